// Dropout whose mask is a function of (seed, offset, element), so that it is never stored: the gradient's way back draws the same
// words again.  Element i keeps x_i / (1 - p) if word i mod 4 of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) with the counter (i / 4, offset) and the key seed is below (1 - p) 2^32, and is 0 otherwise,
// whatever x_i is.  The words depend neither on the launch nor on alignment.
#include "common.cuh"
#include "packed_sequences.cuh"

namespace prad {
namespace drop {

constexpr int THREADS = 256;

__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = (uint32_t)offset, x3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

template <typename T> using Vec = seq::Pack<T, 16 / sizeof(T)>;
template <typename T> struct Four { T v[4]; };
template <typename T, bool VECTOR> __device__ __forceinline__ Four<T> load4(const T* p, int left) {
  Four<T> f;
  if (VECTOR && left >= 4) {
#pragma unroll
    for (int k = 0; k < 4; k += 16 / (int)sizeof(T)) {
      const Vec<T> q = *reinterpret_cast<const Vec<T>*>(p + k);
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(T); ++j) f.v[k + j] = q.v[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) f.v[k] = k < left ? p[k] : (T)0;
  }
  return f;
}
template <typename T, bool VECTOR> __device__ __forceinline__ void store4(T* p, const Four<T>& f, int left) {
  if (VECTOR && left >= 4) {
#pragma unroll
    for (int k = 0; k < 4; k += 16 / (int)sizeof(T)) {
      Vec<T> q;
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(T); ++j) q.v[j] = f.v[k + j];
      *reinterpret_cast<Vec<T>*>(p + k) = q;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = f.v[k];
  }
}

// A thread takes U blocks of four words, THREADS apart.  Bound by memory, and by how the CTAs come and what they compute beside it:
// 65536 x 4096 floats with a residual take 592 us with as many CTAs as the device holds and a loop over the blocks, 463 us (7.0 TB/s
// of the three matrices) with a CTA for every U * THREADS blocks, which the device starts one by one as others end; whole blocks take
// a path without tests, as the generator's integers leave little room under the power limit.
constexpr int U = 4;
template <typename T, bool RESIDUAL>
__device__ __forceinline__ Four<T> drop(const Four<T>& in, const Four<T>& residual, int64_t block, uint64_t keep, T scale, uint64_t seed,
                                        uint64_t offset) {
  const uint4 w = philox((uint64_t)block, offset, seed);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
  Four<T> out;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const T kept = (uint64_t)word[k] < keep ? in.v[k] * scale : (T)0;
    out.v[k] = RESIDUAL ? kept + residual.v[k] : kept;
  }
  return out;
}
template <typename T, bool VECTOR, bool RESIDUAL>
__global__ void __launch_bounds__(THREADS)
dropout_kernel(const T* x, const T* residual, T* y, int64_t n, uint64_t keep, T scale, uint64_t seed, uint64_t offset,
               const uint64_t* step) {
  chain_begin();
  if (step) offset += *step;
  const int64_t blocks = (n + 3) / 4, b0 = (int64_t)blockIdx.x * THREADS * U + threadIdx.x;
  if (VECTOR && (b0 + (U - 1) * THREADS + 1) * 4 <= n) {
    Four<T> in[U], out[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      in[i] = load4<T, true>(x + (b0 + i * THREADS) * 4, 4);
      if (RESIDUAL) out[i] = load4<T, true>(residual + (b0 + i * THREADS) * 4, 4);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      store4<T, true>(y + (b0 + i * THREADS) * 4, drop<T, RESIDUAL>(in[i], out[i], b0 + i * THREADS, keep, scale, seed, offset), 4);
  } else {
    for (int64_t b = b0; b < blocks && b < b0 + U * THREADS; b += THREADS) {
      const int left = n - b * 4 < 4 ? (int)(n - b * 4) : 4;
      Four<T> in = load4<T, VECTOR>(x + b * 4, left), out;
      if (RESIDUAL) out = load4<T, VECTOR>(residual + b * 4, left);
      store4<T, VECTOR>(y + b * 4, drop<T, RESIDUAL>(in, out, b, keep, scale, seed, offset), left);
    }
  }
}

template <typename T>
static prad_status run(prad_ctx* ctx, const void* x, const void* residual, void* y, int64_t n, uint64_t keep, double scale,
                       uint64_t seed, uint64_t offset, const uint64_t* step) {
  const bool vector = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & 15) == 0;
  const unsigned grid = (unsigned)ceil_div((n + 3) / 4, THREADS * U);
  auto kernel = vector ? (residual ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                       : (residual ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
  launch_chained(kernel, grid, THREADS, 0, ctx->stream, (const T*)x, (const T*)residual, (T*)y, n, keep, (T)scale, seed, offset, step);
  PRAD_LAUNCHED(ctx);
  return PRAD_OK;
}

}  // namespace drop
}  // namespace prad

using namespace prad;

extern "C" prad_status prad_dropout(prad_ctx* ctx, prad_dtype dt, const void* x, const void* residual, void* y, int64_t n, double p,
                                    uint64_t seed, uint64_t offset, const uint64_t* step) {
  PRAD_REQUIRE(dtype_ok(dt), PRAD_ERR_INVALID, "prad_dropout: unknown dtype %d", (int)dt);
  PRAD_REQUIRE(n >= 0, PRAD_ERR_SHAPE, "prad_dropout: negative size");
  PRAD_REQUIRE(p >= 0.0 && p <= 1.0, PRAD_ERR_INVALID, "prad_dropout: p must be in [0, 1], got %g", p);
  PRAD_REQUIRE(n <= (int64_t)0x7fffffff * 4 * drop::THREADS * drop::U, PRAD_ERR_UNSUPPORTED, "prad_dropout: too many values");
  PRAD_REQUIRE(n == 0 || (x && y), PRAD_ERR_INVALID, "prad_dropout: null pointer");
  PRAD_REQUIRE(natural(dt, x, residual, y) && ((uintptr_t)step & 7) == 0, PRAD_ERR_INVALID, "prad_dropout: unaligned pointer");
  PRAD_CHECK_CTX(ctx);
  if (n == 0) return PRAD_OK;
  // the nearest whole number of words; p so close to 1 that none is left keeps nothing, as p == 1 does
  const uint64_t keep = (uint64_t)((1.0 - p) * 4294967296.0 + 0.5);
  const double scale = keep ? 1.0 / (1.0 - p) : 0.0;
  return dt == PRAD_F32 ? drop::run<float>(ctx, x, residual, y, n, keep, scale, seed, offset, step)
                        : drop::run<double>(ctx, x, residual, y, n, keep, scale, seed, offset, step);
}
