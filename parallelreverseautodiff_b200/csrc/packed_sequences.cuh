// What the kernels over packed sequences share: which rows of the token matrix belong to which sequence, and the scalar
// functions of the layers they run in.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace prad {
namespace seq {

// Sequence s has the rows [end(s - 1), end(s)); offsets == nullptr: `each` rows a sequence.  What is read from the device is
// cut to [0, tokens], so that offsets which do not ascend give wrong rows but never rows outside the matrices.
struct Sequences {
  const int32_t* offsets;
  int count;
  int64_t tokens;
  int64_t each;
  __device__ __forceinline__ int64_t cut(int64_t o) const { return o < 0 ? 0 : o > tokens ? tokens : o; }
  __device__ __forceinline__ int64_t begin() const { return offsets ? cut(offsets[0]) : 0; }
  __device__ __forceinline__ int64_t finish() const { return offsets ? cut(offsets[count]) : tokens; }
  __device__ __forceinline__ int64_t start(int s) const { return offsets ? cut(offsets[s]) : s * each; }
  __device__ __forceinline__ int64_t end(int s) const { return offsets ? cut(offsets[s + 1]) : (s + 1) * each; }
  // the first sequence that ends behind row t (count if there is none)
  __device__ __forceinline__ int at(int64_t t) const {
    if (!offsets) return each > 0 && t < tokens ? (int)(t / each) : count;
    int lo = 0, hi = count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cut(offsets[mid + 1]) > t) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }
};

// 1 / (1 + 2^(-x log2 e)): two steps of the special function unit, each within 2 units of the last place
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float x) { return reciprocal(1.0f + exp2_approx(x * -1.4426950408889634f)); }
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }
template <typename T> __device__ __forceinline__ T swish(T x) { return x * sigmoid(x); }
// d swish / dx
template <typename T> __device__ __forceinline__ T swish_slope(T x) {
  const T s = sigmoid(x);
  return s * ((T)1 + x * ((T)1 - s));
}

}  // namespace seq
}  // namespace prad
