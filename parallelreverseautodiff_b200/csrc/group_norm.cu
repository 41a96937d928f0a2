// Group normalisation of channels-last data, x[sample][position][channel]: a group is channels / groups neighbouring channels of
// all positions of a sample,  xhat = (x - mean) rstd,  v = gamma xhat + beta,  y = v or swish(v).  Backward, with dv = dy swish'(v):
//   dbeta = sum dv,  dgamma = sum dv xhat,  dx = rstd (gamma dv - mean(gamma dv) - xhat mean(gamma dv xhat)).
//
// Bound by memory; three shapes of work.  One position per sample (a norm per token): a group's values lie side by side and stay in
// the registers of a few lanes, one pass over the memory each way.  Several positions: a cluster of CTAs takes a sample (or some of
// its groups), each CTA a block of its positions; they sum, exchange the sums through each other's shared memory and read their
// blocks again, now out of the L2.  Too few samples for that, or groups wider than a CTA: sums and results in launches of their own.
// Floats, forward and backward: 16384 rows of 2048 in groups of 128, 49 and 66 us (5.5 and 6.1 TB/s); 64 samples of 3136 positions and
// 96 channels in groups of 12 with swish, 39 and 70 us (3.9 and 3.3 TB/s: the clusters of the whole input run at once, so that
// backward its second reading misses the L2; clusters of 16, or blocks of half the channels, took 14 and 17 us longer, and blocks that
// stay in shared memory, so that fewer of them run at a time, 54 and 113 us).
//
// Over several positions a thread sums the deviations of a few values at a time from one of them, the median of three, and joins them
// with the others in double, around a pivot out of the data: neither a mean far from zero nor single values far from the others take
// anything from the variance. With one position per sample the variance is of deviations from the mean that is already there. The
// backward sums of floats go into doubles too, every few values or samples.
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed_sequences.cuh"

namespace prad {
namespace gn {

using seq::load;
using seq::Pack;
using seq::swish;
using seq::swish_slope;

constexpr int THREADS = 256;

template <typename T> struct Args {
  const T *x, *gamma, *beta, *mean, *rstd, *dy;
  T *y, *mean_out, *rstd_out, *dx, *dgamma, *dbeta;
  int64_t samples, positions;
  int channels, groups, per;     // per: channels of a group
  double eps;
  int act, wide;                 // wide: gamma and beta can be read as many values at a time as x
};


// V values of gamma or beta from channel c on; `none` without any
template <typename T, int V> __device__ __forceinline__ Pack<T, V> parameters(const Args<T>& a, const T* p, int c, T none) {
  Pack<T, V> r;
  if (p && a.wide) return load<T, V>(p + c);
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = p ? p[c + j] : none;
  return r;
}

__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }

// ---------------------------------------------------------------- one position per sample
// LW lanes share the values of a (sample, group), E packs of V values each; a lane keeps its channels for all its samples, so the
// sums for dgamma and dbeta stay in registers as well.  Slot k of the grid takes group k mod groups: neighbouring slots read
// neighbouring memory; its samples are `step` apart.
template <int LW, typename A> __device__ __forceinline__ A lanes_sum(A v) {
#pragma unroll
  for (int o = LW / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// the first sample of a slot, and its group
struct Slot {
  int64_t row;
  int group;
  __device__ __forceinline__ Slot(int64_t slot, int groups) {
    if (slot >> 32 == 0) {         // (a division of 64 bits takes as long as a row's arithmetic)
      const uint32_t q = (uint32_t)slot / (uint32_t)groups;
      row = q;
      group = (int)((uint32_t)slot - q * (uint32_t)groups);
    } else {
      row = slot / groups;
      group = (int)(slot - row * groups);
    }
  }
};

// samples of a slot in the forward pass, whose values are on their way at the same time
template <int E> constexpr int rows_at_once() { return E == 1 ? 4 : E == 2 ? 2 : 1; }
template <typename T, int V, int LW, int E>
__global__ void __launch_bounds__(THREADS)
rows_forward_kernel(const Args<T> a, int64_t step) {
  chain_begin();
  constexpr int R = rows_at_once<E>();
  const Slot slot(((int64_t)blockIdx.x * THREADS + threadIdx.x) / LW, a.groups);
  const int l = threadIdx.x % LW, g = slot.group;
  int c[E];
  bool on[E];
  Pack<T, V> gamma[E], beta[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    c[e] = (l + e * LW) * V;
    on[e] = c[e] < a.per;
    if (on[e]) {
      gamma[e] = parameters<T, V>(a, a.gamma, g * a.per + c[e], (T)1);
      beta[e] = parameters<T, V>(a, a.beta, g * a.per + c[e], (T)0);
    }
  }
  // all lanes of a warp take part in its sums: those beyond the last sample with nothing to add
  const int64_t first = slot.row < step ? slot.row : a.samples;
  const T inv = (T)1 / (T)a.per, eps = (T)a.eps;
  Pack<T, V> x[R][E];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t s = first + r * step;
#pragma unroll
      for (int j = 0; j < V; ++j) x[r][e].v[j] = 0;
      if (s < a.samples && on[e]) x[r][e] = load<T, V>(a.x + s * a.channels + (int64_t)g * a.per + c[e]);
    }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t s = first + r * step;
    T sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) sum += x[r][e].v[j];
    const T mean = lanes_sum<LW>(sum) * inv;
    T sq = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const T d = x[r][e].v[j] - mean;
        if (on[e]) sq += d * d;
      }
    const T rstd = inverse_root(lanes_sum<LW>(sq) * inv + eps);
    if (s < a.samples) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (on[e]) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const T v = (x[r][e].v[j] - mean) * rstd * gamma[e].v[j] + beta[e].v[j];
            x[r][e].v[j] = a.act ? swish(v) : v;
          }
          *reinterpret_cast<Pack<T, V>*>(a.y + s * a.channels + g * a.per + c[e]) = x[r][e];
        }
      if (l == 0) {
        a.mean_out[s * a.groups + g] = mean;
        a.rstd_out[s * a.groups + g] = rstd;
      }
    }
  }
}

// partial[row block][2][channels]: this slot's sums of dv xhat and of dv
template <typename T, int V, int LW, int E>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 && E == 1 ? 4 : 0)
rows_backward_kernel(const Args<T> a, int64_t step, T* __restrict__ partial) {
  chain_begin();
  const Slot slot(((int64_t)blockIdx.x * THREADS + threadIdx.x) / LW, a.groups);
  const int l = threadIdx.x % LW, g = slot.group;
  int c[E];
  bool on[E];
  Pack<T, V> gamma[E], beta[E], dg[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    c[e] = (l + e * LW) * V;
    on[e] = c[e] < a.per;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int ch = g * a.per + c[e] + j;
      gamma[e].v[j] = on[e] && a.gamma ? a.gamma[ch] : (T)1;
      beta[e].v[j] = on[e] && a.beta ? a.beta[ch] : (T)0;
      dg[e].v[j] = db[e].v[j] = 0;
    }
  }
  const int64_t first = slot.row < step ? slot.row : a.samples;
  const int64_t rounds = (a.samples + step - 1) / step;
  const T inv = (T)1 / (T)a.per;
  // One pack of floats a lane: the next sample's is on its way while this one's sums go round (16384 rows of 2048 in groups of 128: 72 us,
  // 78 without, and nothing gained if its registers take a CTA of an SM's four); more have no registers for it.
  constexpr bool AHEAD = sizeof(T) == 4 && E == 1;
  Pack<T, V> next_x, next_d;
  T next_mean = 0, next_rstd = 0;
  const auto fetch = [&](int64_t s) {
    if (s >= a.samples) return;
    const int64_t at = s * a.channels + (int64_t)g * a.per;
    next_mean = a.mean[s * a.groups + g];
    next_rstd = a.rstd[s * a.groups + g];
    if (on[0]) {
      next_x = load<T, V>(a.x + at + c[0]);
      next_d = load<T, V>(a.dy + at + c[0]);
    }
  };
  if constexpr (AHEAD) fetch(first);
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t s = first + k * step;
    const bool live = s < a.samples;
    const int64_t at = s * a.channels + (int64_t)g * a.per;
    T mean, rstd;
    Pack<T, V> x[E], d[E];
    T s1 = 0, s2 = 0;
    if constexpr (AHEAD) {
      mean = next_mean, rstd = next_rstd;
      x[0] = next_x, d[0] = next_d;
      fetch(s + step);
    } else {
      mean = live ? a.mean[s * a.groups + g] : (T)0;
      rstd = live ? a.rstd[s * a.groups + g] : (T)0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (live && on[e]) {
          x[e] = load<T, V>(a.x + at + c[e]);
          d[e] = load<T, V>(a.dy + at + c[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (live && on[e]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const T xh = (x[e].v[j] - mean) * rstd;
          T dv = d[e].v[j];
          if (a.act) dv *= swish_slope(xh * gamma[e].v[j] + beta[e].v[j]);
          dg[e].v[j] += dv * xh;
          db[e].v[j] += dv;
          dv *= gamma[e].v[j];
          s1 += dv;
          s2 += dv * xh;
          x[e].v[j] = xh;
          d[e].v[j] = dv;
        }
      }
    s1 = lanes_sum<LW>(s1) * inv;
    s2 = lanes_sum<LW>(s2) * inv;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (live && on[e]) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[e].v[j] = rstd * (d[e].v[j] - s1 - x[e].v[j] * s2);
        *reinterpret_cast<Pack<T, V>*>(a.dx + at + c[e]) = d[e];
      }
  }
  if (slot.row < step)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (on[e])
#pragma unroll
        for (int j = 0; j < V; ++j) {
          T* to = partial + (slot.row * 2) * a.channels + g * a.per + c[e] + j;
          to[0] = dg[e].v[j];
          to[a.channels] = db[e].v[j];
        }
}

// out[0][c], out[1][c] = sums over the blocks of partial[block][2][channels], in the order of the blocks within a warp's share
constexpr int TOTALS = 1024;
template <typename P, typename T>
__global__ void __launch_bounds__(TOTALS)
column_totals_kernel(const P* __restrict__ partial, int64_t blocks, int channels, T* dgamma, T* dbeta) {
  chain_begin();
  __shared__ double part[TOTALS / 32][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  T* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  double sum = 0.0;
  if (c < channels) {
    const P* p = partial + (int64_t)blockIdx.y * channels + c;
#pragma unroll 8
    for (int64_t b = w; b < blocks; b += TOTALS / 32) sum += (double)p[b * 2 * channels];
  }
  part[w][lane] = sum;
  __syncthreads();
  if (w == 0 && c < channels) {
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < TOTALS / 32; ++k) sum += part[k][lane];
    out[c] = (T)sum;
  }
}

// ---------------------------------------------------------------- several positions per sample
// A CTA takes a block of positions of one sample and a part of the channels: as many whole groups as THREADS packs of V channels
// hold (so at most THREADS), the threads in rows of one position each; or one wide group, whose packs the threads walk.
struct Parts {
  int64_t blocks, rows;        // blocks of `rows` positions per sample
  int parts, groups_each;      // of the channels
};
template <typename T> struct Place {
  int64_t s, block, p0, p1;
  int g0, g1, c0, packs, tx, ty, rows;
  __device__ __forceinline__ Place(const Args<T>& a, const Parts& k, int V) {
    s = blockIdx.x / k.blocks;
    block = blockIdx.x % k.blocks;
    p0 = block * k.rows;
    p1 = p0 + k.rows < a.positions ? p0 + k.rows : a.positions;
    g0 = blockIdx.y * k.groups_each;
    g1 = g0 + k.groups_each < a.groups ? g0 + k.groups_each : a.groups;
    c0 = g0 * a.per;
    packs = (g1 - g0) * a.per / V;
    const int width = packs < THREADS ? packs : THREADS;
    tx = threadIdx.x % width;
    ty = threadIdx.x / width;
    rows = THREADS / width;
  }
};

// The second reading of a block goes from its end to its start, as what was read last is what the caches still have (64 images of 3136
// positions and 96 channels, forward and backward: 117.5 us, 119.3 from start to end): N rows of a thread at a time, from these on.
template <int N, typename T> __device__ __forceinline__ int64_t last_rows(const Place<T>& w) {
  const int64_t mine = w.p1 - w.p0 - w.ty - 1;       // (negative: none)
  return mine < 0 ? w.p0 - 1 : w.p0 + w.ty + mine / ((int64_t)N * w.rows) * N * w.rows;
}

// the average of the middle two of four values of a group: what the joined sums are relative to
template <typename T> __device__ __forceinline__ double pivot(const Args<T>& a, int64_t s, int g) {
  const T* x = a.x + s * a.positions * a.channels + (int64_t)g * a.per;
  double v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = (double)x[(a.positions - 1) * k / 3 * a.channels + (a.per - 1) * k / 3];
  const double lower = fmax(fmin(v[0], v[1]), fmin(v[2], v[3])), upper = fmin(fmax(v[0], v[1]), fmax(v[2], v[3]));
  return (double)(T)(0.5 * lower + 0.5 * upper);
}

template <typename T> __device__ __forceinline__ T median(T a, T b, T c) { return max(min(a, b), min(max(a, b), c)); }
constexpr int RUN = 8;     // positions whose deviations are summed in T before they go into a double

// sums of x - pivot and of its square over the CTA's block, for each of its groups, to `out(group, s1, s2)`
template <typename T, int V> struct SumsShared {
  double part[THREADS][2];
  T piv[THREADS];
};
template <typename T, int V, typename Out>
__device__ __forceinline__ void block_sums(const Args<T>& a, const Place<T>& w, SumsShared<T, V>& m, const Out& out) {
  for (int g = threadIdx.x; g < w.g1 - w.g0; g += THREADS) m.piv[g] = (T)pivot(a, w.s, w.g0 + g);
  __syncthreads();
  double s1 = 0.0, s2 = 0.0;
  if (w.ty < w.rows)
    for (int q = w.tx; q < w.packs; q += THREADS) {
      const double k = (double)m.piv[q * V / a.per];
      const T* x = a.x + (w.s * a.positions) * a.channels + w.c0 + (int64_t)q * V;
      for (int64_t p = w.p0 + w.ty; p < w.p1; p += (int64_t)RUN * w.rows) {
        Pack<T, V> v[RUN];
        int rows = 0;
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          const bool live = i == 0 || p + (int64_t)i * w.rows < w.p1;
#pragma unroll
          for (int j = 0; j < V; ++j) v[i].v[j] = 0;
          if (live) v[i] = load<T, V>(x + (p + (int64_t)i * w.rows) * a.channels);
          rows += live;
        }
        const T at = median(v[0].v[0], rows > 1 ? v[1].v[V / 2] : v[0].v[0], rows > 2 ? v[2].v[V - 1] : v[0].v[V - 1]);
        T r1 = 0, r2 = 0;
#pragma unroll
        for (int i = 0; i < RUN; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const T d = i < rows ? v[i].v[j] - at : (T)0;
            r1 += d;
            r2 += d * d;
          }
        const double e = (double)at - k, all = (double)(rows * V) * e, rest = (double)r1;
        s1 += all + rest;
        s2 += (double)r2 + e * (all + 2.0 * rest);
      }
    }
  m.part[threadIdx.x][0] = s1;
  m.part[threadIdx.x][1] = s2;
  __syncthreads();
  // a warp adds up one group: its packs of every row of threads, lanes in a fixed order
  const int lane = threadIdx.x & 31, width = w.packs < THREADS ? w.packs : THREADS;
  const int each = w.g1 - w.g0 == 1 ? width : a.per / V;       // threads of a group in one row of threads
  for (int g = threadIdx.x >> 5; g < w.g1 - w.g0; g += THREADS / 32) {
    s1 = s2 = 0.0;
    for (int i = lane; i < each * w.rows; i += 32) {
      const int t = i / each * width + g * each + i % each;
      s1 += m.part[t][0];
      s2 += m.part[t][1];
    }
    s1 = lanes_sum<32>(s1);
    s2 = lanes_sum<32>(s2);
    if (lane == 0) out(g, s1, s2);
  }
}
template <typename T>
__device__ __forceinline__ void statistics(const Args<T>& a, double pivot, double s1, double s2, T& mean, T& rstd) {
  const double n = (double)a.positions * a.per, m = s1 / n;
  double var = s2 / n - m * m;
  if (var < 0.0) var = 0.0;        // (a NaN stays)
  mean = (T)(pivot + m);
  rstd = (T)(1.0 / sqrt(var + a.eps));
}

// sums[sample][block][group][2]
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
block_sums_kernel(const Args<T> a, const Parts k, double* __restrict__ sums) {
  chain_begin();
  __shared__ SumsShared<T, V> m;
  const Place<T> w(a, k, V);
  block_sums(a, w, m, [&](int g, double s1, double s2) {
    double* to = sums + ((w.s * k.blocks + w.block) * a.groups + w.g0 + g) * 2;
    to[0] = s1;
    to[1] = s2;
  });
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
statistics_kernel(const Args<T> a, int64_t blocks, const double* __restrict__ sums) {
  chain_begin();
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (i >= a.samples * a.groups) return;
  const int64_t s = i / a.groups;
  const int g = (int)(i % a.groups);
  double s1 = 0.0, s2 = 0.0;
#pragma unroll 8
  for (int64_t b = 0; b < blocks; ++b) {
    const double* p = sums + ((s * blocks + b) * a.groups + g) * 2;
    s1 += p[0];
    s2 += p[1];
  }
  statistics(a, pivot(a, s, g), s1, s2, a.mean_out[i], a.rstd_out[i]);
}

// y of the CTA's block; stats(group of the CTA, mean, rstd)
template <typename T, int V, typename Stats>
__device__ __forceinline__ void apply(const Args<T>& a, const Place<T>& w, const Stats& stats) {
  if (w.ty >= w.rows) return;
  for (int q = w.tx; q < w.packs; q += THREADS) {
    const int c = w.c0 + q * V;
    const int64_t at = w.s * a.positions * a.channels + c;
    T mean, rstd;
    stats(q * V / a.per, mean, rstd);
    const Pack<T, V> gammas = parameters<T, V>(a, a.gamma, c, (T)1), betas = parameters<T, V>(a, a.beta, c, (T)0);
    const T(&gamma)[V] = gammas.v;
    const T(&beta)[V] = betas.v;
    for (int64_t p = last_rows<4>(w); p >= w.p0; p -= (int64_t)4 * w.rows) {
      Pack<T, V> v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (p + (int64_t)r * w.rows < w.p1) v[r] = load<T, V>(a.x + at + (p + (int64_t)r * w.rows) * a.channels);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (p + (int64_t)r * w.rows < w.p1) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const T t = (v[r].v[j] - mean) * rstd * gamma[j] + beta[j];
            v[r].v[j] = a.act ? swish(t) : t;
          }
          *reinterpret_cast<Pack<T, V>*>(a.y + at + (p + (int64_t)r * w.rows) * a.channels) = v[r];
        }
    }
  }
}
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
apply_kernel(const Args<T> a, const Parts k) {
  chain_begin();
  const Place<T> w(a, k, V);
  apply<T, V>(a, w, [&](int g, T& mean, T& rstd) {
    mean = a.mean[w.s * a.groups + w.g0 + g];
    rstd = a.rstd[w.s * a.groups + w.g0 + g];
  });
}

// both by one cluster per sample and part: the CTAs' sums through each other's shared memory
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
cluster_forward_kernel(const Args<T> a, const Parts k) {
  chain_begin();
  __shared__ union { SumsShared<T, V> sums; T stats[THREADS][2]; } m;
  __shared__ double own[THREADS][2];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const Place<T> w(a, k, V);
  block_sums(a, w, m.sums, [&](int g, double s1, double s2) {
    own[g][0] = s1;
    own[g][1] = s2;
  });
  cluster.sync();
  for (int g = threadIdx.x; g < w.g1 - w.g0; g += THREADS) {
    double s1 = 0.0, s2 = 0.0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
      const double* p = cluster.map_shared_rank(&own[g][0], r);
      s1 += p[0];
      s2 += p[1];
    }
    T mean, rstd;
    statistics(a, pivot(a, w.s, w.g0 + g), s1, s2, mean, rstd);
    m.stats[g][0] = mean;
    m.stats[g][1] = rstd;
    if (w.block == 0) {
      a.mean_out[w.s * a.groups + w.g0 + g] = mean;
      a.rstd_out[w.s * a.groups + w.g0 + g] = rstd;
    }
  }
  cluster.sync();                  // (no CTA may end while another reads its sums)
  apply<T, V>(a, w, [&](int g, T& mean, T& rstd) {
    mean = m.stats[g][0];
    rstd = m.stats[g][1];
  });
}

// Sums of dv xhat and of dv over the CTA's block, per channel of packs q0 .. q0 + THREADS - 1, by the thread of each pack and row.
template <typename T, int V>
__device__ __forceinline__ void thread_gradients(const Args<T>& a, const Place<T>& w, int q, double (&sg)[V], double (&sb)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) sg[j] = sb[j] = 0.0;
  if (w.ty >= w.rows || q >= w.packs) return;
  const int c = w.c0 + q * V;
  const int64_t i = w.s * a.groups + c / a.per, at = w.s * a.positions * a.channels + c;
  const T mean = a.mean[i], rstd = a.rstd[i];
  const Pack<T, V> gammas = parameters<T, V>(a, a.gamma, c, (T)1), betas = parameters<T, V>(a, a.beta, c, (T)0);
  const T(&gamma)[V] = gammas.v;
  const T(&beta)[V] = betas.v;
  for (int64_t p = w.p0 + w.ty; p < w.p1; p += (int64_t)2 * w.rows) {
    Pack<T, V> x[2], d[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (p + (int64_t)r * w.rows < w.p1) {
        x[r] = load<T, V>(a.x + at + (p + (int64_t)r * w.rows) * a.channels);
        d[r] = load<T, V>(a.dy + at + (p + (int64_t)r * w.rows) * a.channels);
      }
    T rg[V], rb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) rg[j] = rb[j] = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (p + (int64_t)r * w.rows < w.p1) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const T xh = (x[r].v[j] - mean) * rstd;
          T dv = d[r].v[j];
          if (a.act) dv *= swish_slope(xh * gamma[j] + beta[j]);
          rg[j] += dv * xh;
          rb[j] += dv;
        }
      }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sg[j] += (double)rg[j];
      sb[j] += (double)rb[j];
    }
  }
}
// Of packs q0 .. q0 + THREADS - 1: the rows of threads added up, part[0 / 1][channel] and sums[sample][block][2][channels].
template <typename T, int V>
__device__ __forceinline__ void block_gradients(const Args<T>& a, const Parts& k, const Place<T>& w, int q0, double (*part)[THREADS * V],
                                                double* __restrict__ sums) {
  const int width = w.packs < THREADS ? w.packs : THREADS;
  double sg[V], sb[V];
  thread_gradients<T, V>(a, w, q0 + w.tx, sg, sb);
  __syncthreads();
  if (w.ty < w.rows)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      part[0][(w.ty * width + w.tx) * V + j] = sg[j];
      part[1][(w.ty * width + w.tx) * V + j] = sb[j];
    }
  __syncthreads();
  const int here = (w.packs - q0 < THREADS ? w.packs - q0 : THREADS) * V;
  for (int e = threadIdx.x; e < 2 * here; e += THREADS) {
    const int c = e % here;
    double sum = 0.0;
    for (int r = 0; r < w.rows; ++r) sum += part[e / here][r * width * V + c];
    sums[((w.s * k.blocks + w.block) * 2 + e / here) * a.channels + w.c0 + q0 * V + c] = sum;
    part[e / here][c] = sum;       // (this thread alone reads and writes row 0 of channel c)
  }
  __syncthreads();
}
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
block_gradients_kernel(const Args<T> a, const Parts k, double* __restrict__ sums) {
  chain_begin();
  __shared__ double part[2][THREADS * V];
  const Place<T> w(a, k, V);
  for (int q0 = 0; q0 < w.packs; q0 += THREADS) block_gradients<T, V>(a, k, w, q0, part, sums);
}

// Per sample and group: mean(gamma dv) and mean(gamma dv xhat) of the whole sample; a warp each.
template <typename T>
__global__ void __launch_bounds__(THREADS)
group_gradients_kernel(const Args<T> a, int64_t blocks, const double* __restrict__ sums, double* __restrict__ means) {
  chain_begin();
  const int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= a.samples * a.groups) return;
  const int64_t s = i / a.groups;
  const int c0 = (int)(i % a.groups) * a.per;
  double s1 = 0.0, s2 = 0.0;
  for (int64_t e = lane; e < blocks * a.per; e += 32) {
    const int c = c0 + (int)(e % a.per);
    const double* p = sums + (s * blocks + e / a.per) * 2 * a.channels + c;
    const double gamma = a.gamma ? (double)a.gamma[c] : 1.0;
    s2 += gamma * p[0];
    s1 += gamma * p[a.channels];
  }
  s1 = lanes_sum<32>(s1);
  s2 = lanes_sum<32>(s2);
  const double n = (double)a.positions * a.per;
  if (lane == 0) {
    means[i * 2] = s1 / n;
    means[i * 2 + 1] = s2 / n;
  }
}

// dx of the CTA's block; means(group of the CTA, mean(gamma dv), mean(gamma dv xhat))
template <typename T, int V, typename Means>
__device__ __forceinline__ void input_gradients(const Args<T>& a, const Place<T>& w, const Means& means) {
  if (w.ty >= w.rows) return;
  for (int q = w.tx; q < w.packs; q += THREADS) {
    const int c = w.c0 + q * V;
    const int64_t i = w.s * a.groups + c / a.per, at = w.s * a.positions * a.channels + c;
    const T mean = a.mean[i], rstd = a.rstd[i];
    T s1, s2;
    means(q * V / a.per, s1, s2);
    const Pack<T, V> gammas = parameters<T, V>(a, a.gamma, c, (T)1), betas = parameters<T, V>(a, a.beta, c, (T)0);
    const T(&gamma)[V] = gammas.v;
    const T(&beta)[V] = betas.v;
    for (int64_t p = last_rows<2>(w); p >= w.p0; p -= (int64_t)2 * w.rows) {
      Pack<T, V> x[2], d[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (p + (int64_t)r * w.rows < w.p1) {
          x[r] = load<T, V>(a.x + at + (p + (int64_t)r * w.rows) * a.channels);
          d[r] = load<T, V>(a.dy + at + (p + (int64_t)r * w.rows) * a.channels);
        }
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (p + (int64_t)r * w.rows < w.p1) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const T xh = (x[r].v[j] - mean) * rstd;
            T dv = d[r].v[j];
            if (a.act) dv *= swish_slope(xh * gamma[j] + beta[j]);
            d[r].v[j] = rstd * (dv * gamma[j] - s1 - xh * s2);
          }
          *reinterpret_cast<Pack<T, V>*>(a.dx + at + (p + (int64_t)r * w.rows) * a.channels) = d[r];
        }
    }
  }
}
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
input_gradients_kernel(const Args<T> a, const Parts k, const double* __restrict__ means) {
  chain_begin();
  const Place<T> w(a, k, V);
  input_gradients<T, V>(a, w, [&](int g, T& s1, T& s2) {
    const double* p = means + (w.s * a.groups + w.g0 + g) * 2;
    s1 = (T)p[0];
    s2 = (T)p[1];
  });
}

// both by one cluster per sample and part; sums as above, for dgamma and dbeta
template <typename T, int V>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 4 : 2)
cluster_backward_kernel(const Args<T> a, const Parts k, double* __restrict__ sums) {
  chain_begin();
  __shared__ double part[2][THREADS * V];
  __shared__ double own[THREADS][2];
  __shared__ T mine[THREADS][2];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const Place<T> w(a, k, V);
  block_gradients<T, V>(a, k, w, 0, part, sums);
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < w.g1 - w.g0; g += THREADS / 32) {
    double s1 = 0.0, s2 = 0.0;
    for (int c = lane; c < a.per; c += 32) {
      const double gamma = a.gamma ? (double)a.gamma[w.c0 + g * a.per + c] : 1.0;
      s2 += gamma * part[0][g * a.per + c];
      s1 += gamma * part[1][g * a.per + c];
    }
    s1 = lanes_sum<32>(s1);
    s2 = lanes_sum<32>(s2);
    if (lane == 0) {
      own[g][0] = s1;
      own[g][1] = s2;
    }
  }
  cluster.sync();
  const double n = (double)a.positions * a.per;
  for (int g = threadIdx.x; g < w.g1 - w.g0; g += THREADS) {
    double s1 = 0.0, s2 = 0.0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
      const double* p = cluster.map_shared_rank(&own[g][0], r);
      s1 += p[0];
      s2 += p[1];
    }
    mine[g][0] = (T)(s1 / n);
    mine[g][1] = (T)(s2 / n);
  }
  cluster.sync();                  // (no CTA may end while another reads its sums)
  input_gradients<T, V>(a, w, [&](int g, T& s1, T& s2) {
    s1 = mine[g][0];
    s2 = mine[g][1];
  });
}

// ---------------------------------------------------------------- launches
// Samples of a slot at most whose dgamma and dbeta are summed in one float; the slots' sums are joined in double. Slots come in whole
// multiples of what the device holds (131072 rows of 2048 in groups of 128, backward: 516 us with what it holds and 443 samples a
// slot, 529 us with 4 times as many, 554 us with 3.5 times).
constexpr int SUMMED = 512;
template <typename T, int V> constexpr int most_in_registers() { return 32 * 8 * V; }

template <typename T, int V, int LW, int E> static prad_status rows(prad_ctx* ctx, const Args<T>& a, bool backward) {
  // Forward a slot for every R samples of a group.  Backward as many slots as the device holds, or a multiple: each leaves sums of its own.
  int64_t per_group = ceil_div(a.samples, rows_at_once<E>());
  if (backward) {
    const int64_t fill = resident<rows_backward_kernel<T, V, LW, E>>(ctx, THREADS, 0) * THREADS / LW;
    per_group = fill / a.groups;
    if (per_group < 1) per_group = 1;
    if (sizeof(T) == 4) per_group *= ceil_div(a.samples, per_group * SUMMED);
    if (per_group > a.samples) per_group = a.samples;
  }
  const int64_t slots = per_group * a.groups;
  const int64_t grid = ceil_div(slots * LW, THREADS);
  PRAD_REQUIRE(grid <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "group norm: too many groups");
  if (!backward) {
    launch_chained(rows_forward_kernel<T, V, LW, E>, (unsigned)grid, THREADS, 0, ctx->stream, a, per_group);
    PRAD_LAUNCHED(ctx);
    return PRAD_OK;
  }
  prad_status st = ensure_workspace(ctx, (size_t)per_group * 2 * a.channels * sizeof(T));
  if (st) return st;
  launch_chained(rows_backward_kernel<T, V, LW, E>, (unsigned)grid, THREADS, 0, ctx->stream, a, per_group, (T*)ctx->ws);
  PRAD_LAUNCHED(ctx);
  if (a.dgamma || a.dbeta) {
    launch_chained(column_totals_kernel<T, T>, dim3((unsigned)ceil_div(a.channels, 32), 2), TOTALS, 0, ctx->stream, (const T*)ctx->ws, per_group,
                                                                                                      a.channels, a.dgamma, a.dbeta);
    PRAD_LAUNCHED(ctx);
  }
  return PRAD_OK;
}
template <typename T, int V> static prad_status pick_rows(prad_ctx* ctx, const Args<T>& a, bool backward) {
  const int packs = a.per / V;
  if (packs <= 4) return rows<T, V, 4, 1>(ctx, a, backward);
  if (packs <= 8) return rows<T, V, 8, 1>(ctx, a, backward);
  if (packs <= 16) return rows<T, V, 16, 1>(ctx, a, backward);
  if (packs <= 32) return rows<T, V, 32, 1>(ctx, a, backward);
  if (packs <= 64) return rows<T, V, 32, 2>(ctx, a, backward);
  if (packs <= 128) return rows<T, V, 32, 4>(ctx, a, backward);
  return rows<T, V, 32, 8>(ctx, a, backward);
}

// launch_chained with clusters of `ctas` CTAs (grid.x: a multiple of them).
template <typename... P, typename... A>
static void launch_clusters(void (*kernel)(P...), dim3 grid, unsigned ctas, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = THREADS;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);     // (PRAD_LAUNCHED looks at the error)
}

// By clusters: up to eight CTAs a sample and part, each with at least 16 values a thread; parts of fewer groups where the CTAs would
// not fill the device and a row of the part stays 128 bytes or more.  Returns the CTAs of a cluster, or 0 where launches of their own
// are better: groups wider than a CTA, or so few samples that the clusters leave most of a large input to few SMs.
template <typename T> static int by_clusters(prad_ctx* ctx, const Args<T>& a, int V, Parts& k) {
  if (a.per / V > THREADS) return 0;
  int groups = THREADS * V / a.per < a.groups ? THREADS * V / a.per : a.groups, ctas = 8;
  while (ctas > 1 && a.positions * groups * a.per < (int64_t)ctas * THREADS * 16) ctas /= 2;
  while (groups > 1 && a.samples * ctas * ceil_div(a.groups, groups) < 2 * ctx->sm_count &&
         (int64_t)groups * a.per * (int64_t)sizeof(T) >= 256)
    groups = (groups + 1) / 2;
  k.groups_each = groups;
  k.parts = (int)ceil_div(a.groups, groups);
  const int64_t total = a.samples * ctas * k.parts;
  if (total < ctx->sm_count && a.samples * a.positions * a.channels > 1 << 20) return 0;
  k.rows = ceil_div(a.positions, ctas);
  k.blocks = ctas;
  return ctas;
}

template <typename T, int V> static prad_status blocks(prad_ctx* ctx, Args<T> a, bool backward) {
  Parts k;
  const int ctas = by_clusters(ctx, a, V, k);
  if (ctas) {
    PRAD_REQUIRE(a.samples * ctas <= 0x7fffffff && k.parts <= 65535, PRAD_ERR_UNSUPPORTED, "group norm: too many samples or channels");
    const dim3 grid((unsigned)(a.samples * ctas), (unsigned)k.parts);
    if (!backward) {
      launch_clusters(cluster_forward_kernel<T, V>, grid, ctas, ctx->stream, a, k);
      PRAD_LAUNCHED(ctx);
      return PRAD_OK;
    }
    prad_status st = ensure_workspace(ctx, (size_t)(a.samples * ctas) * 2 * a.channels * sizeof(double));
    if (st) return st;
    launch_clusters(cluster_backward_kernel<T, V>, grid, ctas, ctx->stream, a, k, (double*)ctx->ws);
    PRAD_LAUNCHED(ctx);
    if (a.dgamma || a.dbeta) {
      launch_chained(column_totals_kernel<double, T>, dim3((unsigned)ceil_div(a.channels, 32), 2), TOTALS, 0, ctx->stream,
          (const double*)ctx->ws, a.samples * ctas, a.channels, a.dgamma, a.dbeta);
      PRAD_LAUNCHED(ctx);
    }
    return PRAD_OK;
  }
  k.groups_each = THREADS * V / a.per;
  if (k.groups_each < 1) k.groups_each = 1;
  if (k.groups_each > a.groups) k.groups_each = a.groups;
  k.parts = (int)ceil_div(a.groups, k.groups_each);
  // eight CTAs an SM; a block has at least 16 values a thread
  const int64_t want = ceil_div((int64_t)ctx->sm_count * 8, a.samples * k.parts);
  const int64_t row_values = (int64_t)k.groups_each * a.per;
  const int64_t least = ceil_div((int64_t)THREADS * 16, row_values);
  k.rows = ceil_div(a.positions, want);
  if (k.rows < least) k.rows = least;
  if (k.rows > a.positions) k.rows = a.positions;
  k.blocks = ceil_div(a.positions, k.rows);
  PRAD_REQUIRE(a.samples * k.blocks <= 0x7fffffff && k.parts <= 65535, PRAD_ERR_UNSUPPORTED, "group norm: too many samples or channels");
  const dim3 grid((unsigned)(a.samples * k.blocks), (unsigned)k.parts);
  const int64_t each = a.samples * a.groups;
  PRAD_REQUIRE(ceil_div(each * 32, THREADS) <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "group norm: too many groups");
  if (!backward) {
    prad_status st = ensure_workspace(ctx, (size_t)(a.samples * k.blocks * a.groups) * 2 * sizeof(double));
    if (st) return st;
    launch_chained(block_sums_kernel<T, V>, grid, THREADS, 0, ctx->stream, a, k, (double*)ctx->ws);
    PRAD_LAUNCHED(ctx);
    launch_chained(statistics_kernel<T>, (unsigned)ceil_div(each, THREADS), THREADS, 0, ctx->stream, a, k.blocks, (const double*)ctx->ws);
    PRAD_LAUNCHED(ctx);
    a.mean = a.mean_out;
    a.rstd = a.rstd_out;
    launch_chained(apply_kernel<T, V>, grid, THREADS, 0, ctx->stream, a, k);
    PRAD_LAUNCHED(ctx);
    return PRAD_OK;
  }
  const size_t columns = (size_t)(a.samples * k.blocks) * 2 * a.channels;
  prad_status st = ensure_workspace(ctx, (columns + (size_t)each * 2) * sizeof(double));
  if (st) return st;
  double *sums = (double*)ctx->ws, *means = sums + columns;
  launch_chained(block_gradients_kernel<T, V>, grid, THREADS, 0, ctx->stream, a, k, sums);
  PRAD_LAUNCHED(ctx);
  launch_chained(group_gradients_kernel<T>, (unsigned)ceil_div(each * 32, THREADS), THREADS, 0, ctx->stream, a, k.blocks, sums, means);
  PRAD_LAUNCHED(ctx);
  launch_chained(input_gradients_kernel<T, V>, grid, THREADS, 0, ctx->stream, a, k, means);
  PRAD_LAUNCHED(ctx);
  if (a.dgamma || a.dbeta) {
    launch_chained(column_totals_kernel<double, T>, dim3((unsigned)ceil_div(a.channels, 32), 2), TOTALS, 0, ctx->stream,
        sums, a.samples * k.blocks, a.channels, a.dgamma, a.dbeta);
    PRAD_LAUNCHED(ctx);
  }
  return PRAD_OK;
}

template <typename T> static prad_status run(prad_ctx* ctx, Args<T> a, bool backward) {
  constexpr int V = 16 / sizeof(T);
  a.wide = (((uintptr_t)a.gamma | (uintptr_t)a.beta) & 15) == 0;
  const uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.y | (uintptr_t)a.dx;
  const bool vector = a.per % V == 0 && (all & 15) == 0;
  if (a.positions == 1 && a.per <= (vector ? most_in_registers<T, V>() : most_in_registers<T, 1>()))
    return vector ? pick_rows<T, V>(ctx, a, backward) : pick_rows<T, 1>(ctx, a, backward);
  return vector ? blocks<T, V>(ctx, a, backward) : blocks<T, 1>(ctx, a, backward);
}

static prad_status check(const char* who, prad_dtype dt, int64_t samples, int64_t positions, int channels, int groups) {
  PRAD_REQUIRE(dtype_ok(dt), PRAD_ERR_INVALID, "%s: unknown dtype %d", who, (int)dt);
  PRAD_REQUIRE(samples >= 0 && positions >= 0 && channels > 0 && groups > 0, PRAD_ERR_SHAPE, "%s: bad shape", who);
  PRAD_REQUIRE(channels % groups == 0, PRAD_ERR_SHAPE, "%s: %d channels do not divide into %d groups", who, channels, groups);
  return PRAD_OK;
}

}  // namespace gn
}  // namespace prad

using namespace prad;

template <typename T>
static prad_status forward_t(prad_ctx* ctx, const void* x, const void* gamma, const void* beta, void* y, void* mean, void* rstd,
                             int64_t samples, int64_t positions, int channels, int groups, double eps, int act) {
  gn::Args<T> a = {};
  a.x = (const T*)x, a.gamma = (const T*)gamma, a.beta = (const T*)beta;
  a.y = (T*)y, a.mean_out = (T*)mean, a.rstd_out = (T*)rstd;
  a.samples = samples, a.positions = positions, a.channels = channels, a.groups = groups, a.per = channels / groups;
  a.eps = eps, a.act = act;
  return gn::run(ctx, a, false);
}
template <typename T>
static prad_status backward_t(prad_ctx* ctx, const void* x, const void* gamma, const void* beta, const void* mean, const void* rstd,
                              const void* dy, void* dx, void* dgamma, void* dbeta, int64_t samples, int64_t positions, int channels,
                              int groups, int act) {
  gn::Args<T> a = {};
  a.x = (const T*)x, a.gamma = (const T*)gamma, a.beta = (const T*)beta, a.mean = (const T*)mean, a.rstd = (const T*)rstd;
  a.dy = (const T*)dy, a.dx = (T*)dx, a.dgamma = (T*)dgamma, a.dbeta = (T*)dbeta;
  a.samples = samples, a.positions = positions, a.channels = channels, a.groups = groups, a.per = channels / groups;
  a.act = act;
  return gn::run(ctx, a, true);
}

extern "C" prad_status prad_group_norm_forward(prad_ctx* ctx, prad_dtype dt, const void* x, const void* gamma, const void* beta, void* y,
                                               void* mean, void* rstd, int64_t samples, int64_t positions, int channels, int groups,
                                               double eps, int swish) {
  prad_status st = gn::check("prad_group_norm_forward", dt, samples, positions, channels, groups);
  if (st) return st;
  PRAD_REQUIRE(eps >= 0.0, PRAD_ERR_INVALID, "prad_group_norm_forward: eps must not be negative");
  PRAD_REQUIRE(samples == 0 || positions == 0 || (x && y && mean && rstd), PRAD_ERR_INVALID, "prad_group_norm_forward: null pointer");
  PRAD_REQUIRE(natural(dt, x, gamma, beta, y, mean, rstd), PRAD_ERR_INVALID, "prad_group_norm_forward: unaligned pointer");
  PRAD_CHECK_CTX(ctx);
  if (samples == 0 || positions == 0) return PRAD_OK;
  return dt == PRAD_F32 ? forward_t<float>(ctx, x, gamma, beta, y, mean, rstd, samples, positions, channels, groups, eps, swish)
                        : forward_t<double>(ctx, x, gamma, beta, y, mean, rstd, samples, positions, channels, groups, eps, swish);
}

extern "C" prad_status prad_group_norm_backward(prad_ctx* ctx, prad_dtype dt, const void* x, const void* gamma, const void* beta,
                                                const void* mean, const void* rstd, const void* dy, void* dx, void* dgamma, void* dbeta,
                                                int64_t samples, int64_t positions, int channels, int groups, int swish) {
  prad_status st = gn::check("prad_group_norm_backward", dt, samples, positions, channels, groups);
  if (st) return st;
  PRAD_REQUIRE(samples == 0 || positions == 0 || (x && mean && rstd && dy && dx), PRAD_ERR_INVALID,
               "prad_group_norm_backward: null pointer");
  PRAD_REQUIRE(natural(dt, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta), PRAD_ERR_INVALID,
               "prad_group_norm_backward: unaligned pointer");
  PRAD_CHECK_CTX(ctx);
  if (samples == 0 || positions == 0) {      // nothing was normalised: the parameters' gradients are zero
    if (dgamma) PRAD_CUDA(cudaMemsetAsync(dgamma, 0, channels * dtype_size(dt), ctx->stream));
    if (dbeta) PRAD_CUDA(cudaMemsetAsync(dbeta, 0, channels * dtype_size(dt), ctx->stream));
    return PRAD_OK;
  }
  return dt == PRAD_F32
             ? backward_t<float>(ctx, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, samples, positions, channels, groups, swish)
             : backward_t<double>(ctx, x, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, samples, positions, channels, groups, swish);
}
