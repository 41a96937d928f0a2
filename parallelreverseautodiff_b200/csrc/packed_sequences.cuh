// What the kernels of state space layers share: which rows of the token matrix belong to which sequence, packs of values, and the
// scalar functions of the layers they run in.
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

// V values side by side, read and written at a time
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }

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

// two values side by side: float works on both with one instruction
template <typename T> struct Two;
template <> struct Two<float> {
  unsigned long long v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
template <> struct Two<double> {
  double a_, b_;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(double a, double b) : a_(a), b_(b) {}
  __device__ __forceinline__ void get(double& a, double& b) const { a = a_, b = b_; }
};
__device__ __forceinline__ Two<float> mul(Two<float> a, Two<float> b) {
  Two<float> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
  Two<float> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two<double> mul(Two<double> a, Two<double> b) { return {a.a_ * b.a_, a.b_ * b.b_}; }
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) {
  return {::fma(a.a_, b.a_, c.a_), ::fma(a.b_, b.b_, c.b_)};
}
// one value, with the same functions
template <typename T> struct One {
  T v;
  __device__ __forceinline__ One() {}
  __device__ __forceinline__ explicit One(T a) : v(a) {}
};
__device__ __forceinline__ One<float> mul(One<float> a, One<float> b) { return One<float>(a.v * b.v); }
__device__ __forceinline__ One<float> fma(One<float> a, One<float> b, One<float> c) { return One<float>(fmaf(a.v, b.v, c.v)); }
__device__ __forceinline__ One<double> mul(One<double> a, One<double> b) { return One<double>(a.v * b.v); }
__device__ __forceinline__ One<double> fma(One<double> a, One<double> b, One<double> c) { return One<double>(::fma(a.v, b.v, c.v)); }
template <typename T> __device__ __forceinline__ Two<T> each(const Two<T>& x, T (*f)(T)) {
  T a, b;
  x.get(a, b);
  return {f(a), f(b)};
}
template <typename T> __device__ __forceinline__ One<T> each(const One<T>& x, T (*f)(T)) { return One<T>(f(x.v)); }
// V = 1 or 2 neighbouring values
template <typename T, int V> struct Few;
template <typename T> struct Few<T, 1> {
  using type = One<T>;
  __device__ static __forceinline__ type from(const T* v) { return One<T>(v[0]); }
  __device__ static __forceinline__ void to(const type& x, T* v) { v[0] = x.v; }
};
template <typename T> struct Few<T, 2> {
  using type = Two<T>;
  __device__ static __forceinline__ type from(const T* v) { return {v[0], v[1]}; }
  __device__ static __forceinline__ void to(const type& x, T* v) { x.get(v[0], v[1]); }
};

}  // namespace seq
}  // namespace prad
