// The selective state space scan.  Channel d with the states n of its group's rows B, C; per token of a sequence
//   dt = delta + delta_bias (softplus of it where asked),  a_n = exp(dt A_dn),  h_n <- a_n h_n + dt u B_n,
//   r = sum_n C_n h_n + D u,  y = r or r swish(z);
// the state begins at h0 (zero without one) and is given back in h_last.  Backward, with v = dy swish(z) (dy without z):
//   g_n(t) = C_n v + a_n(t + 1) g_n(t + 1),  du = dt sum g B + D v,  ddt = u sum g B + sum g_n A_n a_n h_n(t - 1),
//   dA_n = sum_t g_n dt a_n h_n(t - 1),  dB_n = sum over the group's channels of g_n dt u,  dC_n likewise of v h_n,
//   dD = sum v u,  dz = dy r swish'(z),  ddelta = ddt sigmoid(delta + delta_bias),  dh0 = a_n g_n of the first token.
//
// L lanes share a channel, S states each; a CTA takes THREADS / L channels of one group over a span of the tokens, TT of them at a
// time in shared memory.  What bounds it is arithmetic, not memory: N exponentials and 4 N multiply-adds for 16 bytes of a float.
//
// The token axis of all sequences is one recurrence in which the state is replaced where a sequence begins.  When the sequences
// alone give too few CTAs, it is cut into spans of equal length: one pass finds what each span makes of a zero state (and of any
// other: exp(A sum dt) times it, as decays multiply), a second strings the spans together, and the main pass starts each span from
// the state it has.  The backward pass runs the same way from the last span up, on checkpoints of the state every TT tokens that
// the forward pass leaves.
#include "common.cuh"
#include "packed_sequences.cuh"

namespace prad {
namespace ssm {

using seq::Sequences;
using seq::swish;
using seq::swish_slope;

constexpr int THREADS = 128;
template <typename T> constexpr int tile() { return sizeof(T) == 8 ? 16 : 32; }     // TT; also tokens per checkpoint
constexpr int MAX_STATE = 128;

template <typename T> struct Args {
  Sequences rows;
  int64_t span;                 // tokens of a span
  int spans, dim, state, groups, per, blocks;   // per: channels of a group, in `blocks` CTAs
  int softplus;
  int64_t ld_u, ld_delta, ld_z, ld_B, ld_C, ld_y, ld_dy, ld_du, ld_ddelta, ld_dz, ld_dB, ld_dC;
  const T *u, *delta, *z, *A, *B, *C, *D, *bias, *h0, *dy;
  T *y, *h_last, *saved;
  T *du, *ddelta, *dz, *dA, *dB, *dC, *dD, *dbias, *dh0;
  // between the passes: of each span the state it ends in (then the one it begins with), the sum of its time steps, and whether
  // a state passes through it
  T *edge, *sum;
  int* passes;
  T *part_A, *part_D, *part_bias, *part_BC;
};

// exp(dt A): in float as 2^(dt A') with A' = A log2 e
__device__ __forceinline__ float decay(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double decay(double x) { return exp(x); }
template <typename T> __device__ __forceinline__ T rate(T a);
template <> __device__ __forceinline__ float rate(float a) { return a * 1.4426950408889634f; }
template <> __device__ __forceinline__ double rate(double a) { return a; }
template <typename T> __device__ __forceinline__ T per_rate();         // A per A'
template <> __device__ __forceinline__ float per_rate<float>() { return 0.6931471805599453f; }
template <> __device__ __forceinline__ double per_rate<double>() { return 1.0; }

__device__ __forceinline__ float log1p_(float x) { return log1pf(x); }
__device__ __forceinline__ double log1p_(double x) { return log1p(x); }
__device__ __forceinline__ float exp_(float x) { return expf(x); }
__device__ __forceinline__ double exp_(double x) { return exp(x); }
template <typename T> __device__ __forceinline__ T softplus(T x) {
  return (x > (T)0 ? x : (T)0) + log1p_(exp_(x > (T)0 ? -x : x));
}

template <typename T, int S> struct alignas(sizeof(T) * S) Pack { T v[S]; };

// A CTA's channels and a thread's place among them.
template <typename T, int L, int S> struct Place {
  static constexpr int CH = THREADS / L;
  int q, c0, channels, ch, lane, n0;
  bool on;                       // this thread's channel exists
  __device__ __forceinline__ Place(const Args<T>& a) {
    q = blockIdx.x / a.blocks;
    const int first = blockIdx.x % a.blocks * CH;
    c0 = q * a.per + first;
    channels = a.per - first < CH ? a.per - first : CH;
    ch = threadIdx.x / L;
    lane = threadIdx.x % L;
    n0 = lane * S;
    on = ch < channels;
  }
  // S states of this thread in a [dim][state] matrix
  __device__ __forceinline__ void load(const Args<T>& a, const T* m, T (&h)[S]) const {
#pragma unroll
    for (int j = 0; j < S; ++j) h[j] = on && n0 + j < a.state ? m[(int64_t)(c0 + ch) * a.state + n0 + j] : (T)0;
  }
  __device__ __forceinline__ void store(const Args<T>& a, T* m, const T (&h)[S]) const {
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (on && n0 + j < a.state) m[(int64_t)(c0 + ch) * a.state + n0 + j] = h[j];
  }
};

// Four values a lane, one for each of four tokens, summed over the L lanes of a channel: afterwards lane l holds the sum of token
// l mod 4 (L >= 4).  Half of the values change hands in each of the first two steps.
template <int L, typename T> __device__ __forceinline__ T sum4(const T (&v)[4], int lane) {
  const bool hi = lane & 2, odd = lane & 1;
  T a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 2);
  b += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 2);
  T c = odd ? b : a;
  c += __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
#pragma unroll
  for (int o = 4; o < L; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  return c;
}

// bits of the tile's tokens that begin a sequence; `s` is the sequence of the tile's first token or a later one's that begins in it
template <int TT> __device__ __forceinline__ uint32_t starts_in(const Sequences& rows, int s, int64_t tile0, int64_t finish) {
  uint32_t mask = 0;
  for (; s < rows.count; ++s) {
    const int64_t e = rows.end(s);
    if (e >= tile0 + TT || e >= finish) break;
    if (e >= tile0) mask |= 1u << (int)(e - tile0);
  }
  return mask;
}

// B and C rows of a tile, by asynchronous copies
template <typename T, int N, int TT>
__device__ __forceinline__ void fetch_rows(T (*to)[N], const T* from, int64_t ld, int first, int state, int64_t tile0, int64_t begin,
                                           int64_t finish) {
#pragma unroll
  for (int i = 0; i < (TT * N + THREADS - 1) / THREADS; ++i) {
    const int e = threadIdx.x + i * THREADS, t = e / N, n = e % N;
    if (TT * N % THREADS != 0 && e >= TT * N) break;
    const bool live = tile0 + t >= begin && tile0 + t < finish && n < state;
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(&to[t][n]);
    const T* src = live ? from + (tile0 + t) * ld + first + n : from;
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"((int)sizeof(T)), "r"(live ? (int)sizeof(T) : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void landed() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// the tokens of a span that lie in sequences
template <typename T> struct Span {
  int64_t begin, finish, first;
  __device__ __forceinline__ Span(const Args<T>& a, int p) {
    const int64_t lo = a.rows.begin(), hi = a.rows.finish();
    first = p * a.span;
    begin = first > lo ? first : lo;
    finish = first + a.span < hi ? first + a.span : hi;
  }
};

// ---------------------------------------------------------------- forward
template <typename T, int L, int S> struct Forward {
  static constexpr int CH = THREADS / L, TT = tile<T>(), N = L * S;
  alignas(16) T B[2][TT][N], C[2][TT][N];
  T dt[TT][CH], x[TT][CH], y[TT][CH];
};
// EDGES: only the state that the span ends in when it begins with zero, and the sum of its time steps.
template <typename T, int L, int S, bool EDGES>
__global__ void __launch_bounds__(THREADS)
forward_kernel(const Args<T> a) {
  constexpr int CH = THREADS / L, TT = tile<T>(), N = L * S, CELLS = TT * CH, E = (CELLS + THREADS - 1) / THREADS;
  extern __shared__ __align__(16) unsigned char raw[];
  Forward<T, L, S>& m = *reinterpret_cast<Forward<T, L, S>*>(raw);
  const Place<T, L, S> me(a);
  const int p = blockIdx.y;
  const Span<T> span(a, p);
  int64_t begin = span.begin;
  const int64_t finish = span.finish;
  T A[S], h[S];
  me.load(a, a.A, A);
#pragma unroll
  for (int j = 0; j < S; ++j) {
    A[j] = rate(A[j]);
    h[j] = 0;
  }
  const auto from_h0 = [&](int s, T(&h)[S]) {
#pragma unroll
    for (int j = 0; j < S; ++j) h[j] = 0;
    if (a.h0) me.load(a, a.h0 + (int64_t)s * a.dim * a.state, h);
  };
  // sequences without a token in front of all others
  const int64_t lo = a.rows.begin();
  if (!EDGES && a.h_last && ((span.first <= lo && lo < span.first + a.span) || (p == a.spans - 1 && lo >= span.first + a.span)))
    for (int s = 0; s < a.rows.count && a.rows.end(s) <= lo; ++s) {
      T k[S];
      from_h0(s, k);
      me.store(a, a.h_last + (int64_t)s * a.dim * a.state, k);
    }
  if (EDGES) {
    // what comes before the last sequence that begins in the span does not reach its end
    const int64_t start = begin < finish ? a.rows.start(a.rows.at(finish - 1)) : begin;
    const bool all = start < begin;
    if (!all && start < finish) begin = start;
    if (threadIdx.x == 0 && blockIdx.x == 0) a.passes[p] = all;
  }
  T total = 0;
  if (begin < finish) {
    int s = a.rows.at(begin);
    if (a.rows.start(s) >= begin) from_h0(s, h);
    else if (!EDGES && p > 0) me.load(a, a.edge + (int64_t)p * a.dim * a.state, h);
    const int64_t tiles0 = begin / TT * TT;
    T u[E], d[E], z[E];
    const T bias = a.bias && threadIdx.x % CH < me.channels ? a.bias[me.c0 + threadIdx.x % CH] : (T)0;
    const T D = !EDGES && a.D && threadIdx.x % CH < me.channels ? a.D[me.c0 + threadIdx.x % CH] : (T)0;
    // element e of a tile: token e / CH, channel e % CH
    const auto fetch = [&](int64_t tile0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = threadIdx.x + i * THREADS, c = e % CH;
        const int64_t t = tile0 + e / CH;
        const bool live = t >= begin && t < finish && c < me.channels && (CELLS % THREADS == 0 || e < CELLS);
        u[i] = live ? a.u[t * a.ld_u + me.c0 + c] : (T)0;
        d[i] = live ? a.delta[t * a.ld_delta + me.c0 + c] : (T)0;
        if (!EDGES) z[i] = live && a.z ? a.z[t * a.ld_z + me.c0 + c] : (T)0;
      }
    };
    fetch(tiles0);
    fetch_rows<T, N, TT>(m.B[0], a.B, a.ld_B, me.q * a.state, a.state, tiles0, begin, finish);
    if constexpr (!EDGES) fetch_rows<T, N, TT>(m.C[0], a.C, a.ld_C, me.q * a.state, a.state, tiles0, begin, finish);
    commit();
    int buf = 0;
    for (int64_t tile0 = tiles0; tile0 < finish; tile0 += TT, buf ^= 1) {
      T kept_u[E], kept_z[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = threadIdx.x + i * THREADS, c = e % CH;
        const int64_t t = tile0 + e / CH;
        T dt = d[i] + bias;
        if (a.softplus) dt = softplus(dt);
        if (!(t >= begin && t < finish && c < me.channels)) dt = 0;
        if (CELLS % THREADS == 0 || e < CELLS) {
          m.dt[e / CH][c] = dt;
          m.x[e / CH][c] = dt * u[i];
        }
        kept_u[i] = u[i];
        if (!EDGES) kept_z[i] = z[i];
      }
      if (tile0 + TT < finish) {
        fetch(tile0 + TT);
        fetch_rows<T, N, TT>(m.B[buf ^ 1], a.B, a.ld_B, me.q * a.state, a.state, tile0 + TT, begin, finish);
        if constexpr (!EDGES) fetch_rows<T, N, TT>(m.C[buf ^ 1], a.C, a.ld_C, me.q * a.state, a.state, tile0 + TT, begin, finish);
      }
      commit();
      landed<1>();
      __syncthreads();
      if (!EDGES && a.saved && tile0 >= begin) me.store(a, a.saved + tile0 / TT * a.dim * a.state, h);
      uint32_t starts = starts_in<TT>(a.rows, s, tile0, finish);
      if (tile0 <= begin) starts &= ~(1u << (int)(begin - tile0));       // (the state there is set)
#pragma unroll 2
      for (int t0 = 0; t0 < TT; t0 += 4) {
        T part[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = t0 + k;
          if (starts >> t & 1) {
            // the sequences that end here, and the ones without a token behind them
            const int64_t here = tile0 + t;
            for (; s + 1 < a.rows.count && a.rows.end(s) <= here; ++s) {
              if (!EDGES && a.h_last) {
                T k0[S];
                if (a.rows.start(s) >= here) from_h0(s, h);
#pragma unroll
                for (int j = 0; j < S; ++j) k0[j] = h[j];
                me.store(a, a.h_last + (int64_t)s * a.dim * a.state, k0);
              }
            }
            from_h0(s, h);
            total = 0;
          }
          const T dt = m.dt[t][me.ch], x = m.x[t][me.ch];
          const Pack<T, S> B = *reinterpret_cast<const Pack<T, S>*>(&m.B[buf][t][me.n0]);
          if (EDGES) {
            total += dt;
#pragma unroll
            for (int j = 0; j < S; ++j) h[j] = decay(dt * A[j]) * h[j] + x * B.v[j];
          } else {
            const Pack<T, S> C = *reinterpret_cast<const Pack<T, S>*>(&m.C[buf][t][me.n0]);
            T sum = 0;
#pragma unroll
            for (int j = 0; j < S; ++j) {
              h[j] = decay(dt * A[j]) * h[j] + x * B.v[j];
              sum += C.v[j] * h[j];
            }
            part[k] = sum;
          }
        }
        if (!EDGES) {
          const T r = sum4<L>(part, me.lane);
          if (me.lane < 4) m.y[t0 + me.lane][me.ch] = r;
        }
      }
      __syncthreads();
      if (!EDGES)
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int e = threadIdx.x + i * THREADS, c = e % CH;
          const int64_t t = tile0 + e / CH;
          if (t >= begin && t < finish && c < me.channels && (CELLS % THREADS == 0 || e < CELLS)) {
            T r = m.y[e / CH][c] + D * kept_u[i];
            if (a.z) r *= swish(kept_z[i]);
            a.y[t * a.ld_y + me.c0 + c] = r;
          }
        }
    }
    landed<0>();
    if (!EDGES && a.h_last)
      for (; s < a.rows.count && a.rows.end(s) <= finish; ++s) {
        if (a.rows.start(s) >= finish) from_h0(s, h);
        me.store(a, a.h_last + (int64_t)s * a.dim * a.state, h);
      }
  }
  if (EDGES) {
    me.store(a, a.edge + (int64_t)(p + 1) * a.dim * a.state, h);
    if (me.on && me.lane == 0) a.sum[(int64_t)p * a.dim + me.c0 + me.ch] = total;
  }
}

// Strings the spans together: edge[p] becomes the state that span p begins with.  FORWARD: edge[p + 1] holds what span p ends in
// from zero; otherwise edge[p] holds what span p hands up from zero, and becomes what it is handed from below.
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(THREADS)
join_kernel(const Args<T> a) {
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x, each = (int64_t)a.dim * a.state;
  if (i >= each) return;
  const T A = rate(a.A[i]);
  const int c = (int)(i / a.state);
  T carry = 0;
  if (FORWARD) {
#pragma unroll 4
    for (int p = 0; p + 1 < a.spans; ++p) {
      const T own = a.edge[(p + 1) * each + i];
      const T through = decay(A * a.sum[(int64_t)p * a.dim + c]) * carry;
      carry = own + (a.passes[p] ? through : (T)0);
      a.edge[(p + 1) * each + i] = carry;
    }
  } else {
#pragma unroll 4
    for (int p = a.spans - 1; p >= 0; --p) {
      const T own = a.edge[p * each + i];
      const T through = decay(A * a.sum[(int64_t)p * a.dim + c]) * carry;
      a.edge[p * each + i] = carry;
      carry = own + (a.passes[p] ? through : (T)0);
    }
  }
}

// ---------------------------------------------------------------- backward
// What a span hands to the one above it when it is handed zero: a_n g_n of its first token.
template <typename T, int L, int S>
__global__ void __launch_bounds__(THREADS)
backward_edges_kernel(const Args<T> a) {
  constexpr int CH = THREADS / L, TT = tile<T>(), N = L * S, CELLS = TT * CH, E = (CELLS + THREADS - 1) / THREADS;
  __shared__ T s_dt[TT][CH], s_v[TT][CH];
  __shared__ __align__(16) T s_C[2][TT][N];
  const Place<T, L, S> me(a);
  const int p = blockIdx.y;
  const Span<T> span(a, p);
  const int64_t begin = span.begin;
  int64_t finish = span.finish;
  T A[S], e[S], total = 0;
  me.load(a, a.A, A);
#pragma unroll
  for (int j = 0; j < S; ++j) {
    A[j] = rate(A[j]);
    e[j] = 0;
  }
  int passes = 0;
  if (begin < finish) {
    const int64_t end = a.rows.end(a.rows.at(begin));       // what comes behind the first sequence does not reach the span's start
    passes = end > finish;
    if (end < finish) finish = end;
    T d[E], v[E];
    const T bias = a.bias && threadIdx.x % CH < me.channels ? a.bias[me.c0 + threadIdx.x % CH] : (T)0;
    const auto fetch = [&](int64_t tile0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int x = threadIdx.x + i * THREADS, c = x % CH;
        const int64_t t = tile0 + x / CH;
        const bool live = t >= begin && t < finish && c < me.channels && (CELLS % THREADS == 0 || x < CELLS);
        d[i] = live ? a.delta[t * a.ld_delta + me.c0 + c] : (T)0;
        v[i] = live ? a.dy[t * a.ld_dy + me.c0 + c] : (T)0;
        if (a.z) v[i] *= live ? swish(a.z[t * a.ld_z + me.c0 + c]) : (T)0;
      }
    };
    const int64_t top = (finish - 1) / TT * TT, bottom = begin / TT * TT;
    fetch(top);
    fetch_rows<T, N, TT>(s_C[0], a.C, a.ld_C, me.q * a.state, a.state, top, begin, finish);
    commit();
    int buf = 0;
    for (int64_t tile0 = top; tile0 >= bottom; tile0 -= TT, buf ^= 1) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int x = threadIdx.x + i * THREADS, c = x % CH;
        const int64_t t = tile0 + x / CH;
        T dt = d[i] + bias;
        if (a.softplus) dt = softplus(dt);
        if (!(t >= begin && t < finish && c < me.channels)) dt = 0;
        if (CELLS % THREADS == 0 || x < CELLS) {
          s_dt[x / CH][c] = dt;
          s_v[x / CH][c] = v[i];
        }
      }
      if (tile0 > bottom) {
        fetch(tile0 - TT);
        fetch_rows<T, N, TT>(s_C[buf ^ 1], a.C, a.ld_C, me.q * a.state, a.state, tile0 - TT, begin, finish);
      }
      commit();
      landed<1>();
      __syncthreads();
#pragma unroll 4
      for (int t = TT - 1; t >= 0; --t) {
        const T dt = s_dt[t][me.ch], vt = s_v[t][me.ch];
        const Pack<T, S> C = *reinterpret_cast<const Pack<T, S>*>(&s_C[buf][t][me.n0]);
        total += dt;
#pragma unroll
        for (int j = 0; j < S; ++j) e[j] = decay(dt * A[j]) * (C.v[j] * vt + e[j]);
      }
      __syncthreads();
    }
    landed<0>();
  }
  me.store(a, a.edge + (int64_t)p * a.dim * a.state, e);
  if (me.on && me.lane == 0) a.sum[(int64_t)p * a.dim + me.c0 + me.ch] = total;
  if (threadIdx.x == 0 && blockIdx.x == 0) a.passes[p] = passes;
}

// Values of 2 S sums a lane (dB, then dC of its states) over the warp's 32 / L channels: lanes L apart hold the same states.  As in
// sum4, half of the values change hands in each step until one is left; returns how many are left and which they are.
template <int L, int S, typename T> __device__ __forceinline__ void channel_sums(T (&v)[2 * S], int warp_lane, int& first, int& count) {
  first = 0;
  count = 2 * S;
#pragma unroll
  for (int o = 16; o >= L; o >>= 1) {
    const bool upper = warp_lane & o;
    if (count > 1) {
      count >>= 1;
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (j < count) {
          const T give = upper ? v[j] : v[j + count], keep = upper ? v[j + count] : v[j];
          v[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      if (upper) first += count;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}

// The main pass: a tile's states again from its checkpoint, forwards, into shared memory, then the tile backwards.
template <typename T, int L, int S> struct Backward {
  static constexpr int CH = THREADS / L, TT = tile<T>(), N = L * S, CELLS = TT * CH, E = (CELLS + THREADS - 1) / THREADS;
  static constexpr int WARPS = THREADS / 32;
  static constexpr int FT = TT * 16 / N < TT ? (TT * 16 / N) : TT;      // tokens whose dB and dC are gathered at a time
  struct Shared {
    Pack<T, S> h[TT][THREADS];
    alignas(16) T B[TT][N], C[TT][N];
    T red[WARPS][FT][2 * N];
    T dt[TT][CH], u[TT][CH], v[TT][CH], r[TT][CH], gB[TT][CH], gA[TT][CH];
  };
};

template <typename T, int L, int S>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const Args<T> a) {
  using K = Backward<T, L, S>;
  constexpr int CH = K::CH, TT = K::TT, N = K::N, CELLS = K::CELLS, E = K::E, FT = K::FT;
  extern __shared__ __align__(16) unsigned char raw[];
  typename K::Shared& m = *reinterpret_cast<typename K::Shared*>(raw);
  const Place<T, L, S> me(a);
  const int p = blockIdx.y, wl = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Span<T> span(a, p);
  const int64_t begin = span.begin, finish = span.finish;
  T A[S], e[S], dA[S];
  me.load(a, a.A, A);
#pragma unroll
  for (int j = 0; j < S; ++j) {
    A[j] = rate(A[j]);
    e[j] = dA[j] = 0;
  }
  const int cc = threadIdx.x % CH;
  const bool here = cc < me.channels;
  const T bias = a.bias && here ? a.bias[me.c0 + cc] : (T)0, D = a.D && here ? a.D[me.c0 + cc] : (T)0;
  T dD = 0, dbias = 0;
  if (begin < finish) {
    int s = a.rows.at(finish - 1);                     // the sequence of the token that is looked at
    if (a.rows.end(s) > finish && p + 1 < a.spans) me.load(a, a.edge + (int64_t)p * a.dim * a.state, e);
    const int64_t top = (finish - 1) / TT * TT, bottom = begin / TT * TT;
    for (int64_t tile0 = top; tile0 >= bottom; tile0 -= TT) {
      const int64_t from = tile0 > begin ? tile0 : begin, to = tile0 + TT < finish ? tile0 + TT : finish;
      fetch_rows<T, N, TT>(m.B, a.B, a.ld_B, me.q * a.state, a.state, tile0, begin, finish);
      fetch_rows<T, N, TT>(m.C, a.C, a.ld_C, me.q * a.state, a.state, tile0, begin, finish);
      commit();
      T x_d[E], x_z[E], x_dy[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int x = threadIdx.x + i * THREADS;
        const int64_t t = tile0 + x / CH;
        const bool in = CELLS % THREADS == 0 || x < CELLS, live = t >= from && t < to && here && in;
        const T u = live ? a.u[t * a.ld_u + me.c0 + cc] : (T)0;
        x_d[i] = live ? a.delta[t * a.ld_delta + me.c0 + cc] + bias : (T)0;
        x_z[i] = live && a.z ? a.z[t * a.ld_z + me.c0 + cc] : (T)0;
        x_dy[i] = live ? a.dy[t * a.ld_dy + me.c0 + cc] : (T)0;
        const T dt = a.softplus ? softplus(x_d[i]) : x_d[i];
        if (in) {
          m.dt[x / CH][cc] = live ? dt : (T)0;
          m.u[x / CH][cc] = u;
          m.v[x / CH][cc] = a.z ? x_dy[i] * swish(x_z[i]) : x_dy[i];
        }
      }
      // the state in front of the tile, and the tokens at which it is replaced
      int s0 = a.rows.at(from);
      T h[S], first[S];
#pragma unroll
      for (int j = 0; j < S; ++j) h[j] = 0;
      if (a.rows.start(s0) < from) me.load(a, a.saved + tile0 / TT * a.dim * a.state, h);
      uint32_t starts = starts_in<TT>(a.rows, s0, tile0, to);
      if (a.rows.start(s0) >= from) starts |= 1u << (int)(from - tile0);
#pragma unroll
      for (int j = 0; j < S; ++j) first[j] = h[j];
      landed<0>();
      __syncthreads();
#pragma unroll 2
      for (int t0 = 0; t0 < TT; t0 += 4) {
        T part[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = t0 + k;
          if (starts >> t & 1) {
            const int q = a.rows.at(tile0 + t);
#pragma unroll
            for (int j = 0; j < S; ++j) h[j] = 0;
            if (a.h0) me.load(a, a.h0 + (int64_t)q * a.dim * a.state, h);
          }
          const T dt = m.dt[t][me.ch], x = dt * m.u[t][me.ch];
          const Pack<T, S> B = *reinterpret_cast<const Pack<T, S>*>(&m.B[t][me.n0]);
          const Pack<T, S> C = *reinterpret_cast<const Pack<T, S>*>(&m.C[t][me.n0]);
          Pack<T, S> now;
          T sum = 0;
#pragma unroll
          for (int j = 0; j < S; ++j) {
            h[j] = decay(dt * A[j]) * h[j] + x * B.v[j];
            now.v[j] = h[j];
            sum += C.v[j] * h[j];
          }
          m.h[t][threadIdx.x] = now;
          part[k] = sum;
        }
        const T r = sum4<L>(part, me.lane);
        if (me.lane < 4) m.r[t0 + me.lane][me.ch] = r;
      }
      // backwards
      T tile_dA[S];
#pragma unroll
      for (int j = 0; j < S; ++j) tile_dA[j] = 0;
      for (int f = TT - FT; f >= 0; f -= FT) {
#pragma unroll 1
        for (int t0 = f + FT - 2; t0 >= f; t0 -= 2) {
          T two[4];
#pragma unroll
          for (int k = 1; k >= 0; --k) {
            const int t = t0 + k;
            const bool start = starts >> t & 1;
            T before[S];
            if (start) {
#pragma unroll
              for (int j = 0; j < S; ++j) before[j] = 0;
              if (a.h0) me.load(a, a.h0 + (int64_t)a.rows.at(tile0 + t) * a.dim * a.state, before);
            } else if (t > 0) {
              const Pack<T, S> b = m.h[t - 1][threadIdx.x];
#pragma unroll
              for (int j = 0; j < S; ++j) before[j] = b.v[j];
            } else {
#pragma unroll
              for (int j = 0; j < S; ++j) before[j] = first[j];
            }
            const Pack<T, S> now = m.h[t][threadIdx.x];
            const T dt = m.dt[t][me.ch], x = dt * m.u[t][me.ch], v = m.v[t][me.ch];
            const Pack<T, S> B = *reinterpret_cast<const Pack<T, S>*>(&m.B[t][me.n0]);
            const Pack<T, S> C = *reinterpret_cast<const Pack<T, S>*>(&m.C[t][me.n0]);
            T gB = 0, gA = 0, rows[2 * S];
#pragma unroll
            for (int j = 0; j < S; ++j) {
              const T g = C.v[j] * v + e[j], ag = decay(dt * A[j]) * g;
              const T w = ag * before[j];
              gB += g * B.v[j];
              gA += w * A[j];
              tile_dA[j] += w * dt;
              rows[j] = g * x;
              rows[S + j] = now.v[j] * v;
              e[j] = ag;
            }
            two[2 * k] = gB;
            two[2 * k + 1] = gA;
            int at, left;
            channel_sums<L, S>(rows, wl, at, left);
            // value i of the 2 S: dB (i < S) or dC of state n0 + i mod S
#pragma unroll
            for (int j = 0; j < 2 * S; ++j)
              if (j < left) {      // (lanes that hold the same sum write the same value)
                const int i = at + j;
                m.red[warp][t - f][(i < S ? 0 : N) + me.n0 + i % S] = rows[j];
              }
            if (start) {
              if (a.dh0) me.store(a, a.dh0 + (int64_t)a.rows.at(tile0 + t) * a.dim * a.state, e);
#pragma unroll
              for (int j = 0; j < S; ++j) e[j] = 0;
            }
          }
          const T r = sum4<L>(two, me.lane);
          if (me.lane < 4) (me.lane & 1 ? m.gA : m.gB)[t0 + (me.lane >> 1)][me.ch] = r;
        }
        __syncthreads();
        // the warps' sums, in the order of the warps
        for (int i = threadIdx.x; i < FT * 2 * N; i += THREADS) {
          const int t = i / (2 * N), n = i % (2 * N), state = n < N ? n : n - N;
          const int64_t row = tile0 + f + t;
          if (row >= from && row < to && state < a.state) {
            T sum = 0;
#pragma unroll
            for (int w = 0; w < K::WARPS; ++w) sum += m.red[w][t][n];
            if (a.blocks > 1)
              a.part_BC[((((int64_t)(blockIdx.x % a.blocks) * a.rows.tokens + row) * a.groups + me.q) * 2 + (n >= N)) * a.state + state] = sum;
            else if (n < N) a.dB[row * a.ld_dB + me.q * a.state + state] = sum;
            else a.dC[row * a.ld_dC + me.q * a.state + state] = sum;
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < S; ++j) dA[j] += tile_dA[j];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int x = threadIdx.x + i * THREADS, tt = x / CH;
        const int64_t t = tile0 + tt;
        if (t >= from && t < to && here && (CELLS % THREADS == 0 || x < CELLS)) {
          const T dt = m.dt[tt][cc], u = m.u[tt][cc], v = m.v[tt][cc], gB = m.gB[tt][cc];
          T dd = u * gB + per_rate<T>() * m.gA[tt][cc];
          if (a.softplus) dd *= seq::sigmoid(x_d[i]);
          a.du[t * a.ld_du + me.c0 + cc] = dt * gB + D * v;
          a.ddelta[t * a.ld_ddelta + me.c0 + cc] = dd;
          if (a.z) a.dz[t * a.ld_dz + me.c0 + cc] = x_dy[i] * (m.r[tt][cc] + D * u) * swish_slope(x_z[i]);
          dD += v * u;
          dbias += dd;
        }
      }
      __syncthreads();
    }
  }
  me.store(a, a.part_A + (int64_t)p * a.dim * a.state, dA);
  // the threads of a channel, in their order
  __syncthreads();
  T* const sums = reinterpret_cast<T*>(m.h);
  sums[threadIdx.x] = dD;
  sums[THREADS + threadIdx.x] = dbias;
  __syncthreads();
  if (threadIdx.x < me.channels) {
    dD = dbias = 0;
#pragma unroll
    for (int k = 0; k < L; ++k) {
      dD += sums[k * CH + threadIdx.x];
      dbias += sums[THREADS + k * CH + threadIdx.x];
    }
    a.part_D[(int64_t)p * a.dim + me.c0 + threadIdx.x] = dD;
    a.part_bias[(int64_t)p * a.dim + me.c0 + threadIdx.x] = dbias;
  }
}

// sums of the spans, in double: dA, then dD and dbias
template <typename T>
__global__ void __launch_bounds__(THREADS)
span_totals_kernel(const Args<T> a) {
  int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int64_t states = (int64_t)a.dim * a.state;
  const T* from = a.part_A;
  T* to = a.dA;
  int64_t each = states;
  if (i >= states) {
    i -= states;
    const bool second = i >= a.dim;
    if (second) i -= a.dim;
    if (i >= a.dim) return;
    from = second ? a.part_bias : a.part_D;
    to = second ? a.dbias : a.dD;
    each = a.dim;
  }
  if (!to) return;
  double sum = 0.0;
#pragma unroll 8
  for (int p = 0; p < a.spans; ++p) sum += (double)from[p * each + i];
  to[i] = (T)sum;
}

// dB and dC: sums of the CTAs of a group
template <typename T>
__global__ void __launch_bounds__(256)
row_totals_kernel(const Args<T> a) {
  const int64_t lo = a.rows.begin(), hi = a.rows.finish(), each = (int64_t)a.groups * 2 * a.state;
  const int64_t i = lo * each + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= hi * each) return;
  const int64_t row = i / each, stride = a.rows.tokens * each;
  const int q = (int)(i % each / (2 * a.state)), n = (int)(i % (2 * a.state));
  T sum = 0;
#pragma unroll 8
  for (int b = 0; b < a.blocks; ++b) sum += a.part_BC[b * stride + i];
  if (n < a.state) a.dB[row * a.ld_dB + q * a.state + n] = sum;
  else a.dC[row * a.ld_dC + q * a.state + n - a.state] = sum;
}

// ---------------------------------------------------------------- one token
// one new token for each row of a batch; h_last may be h0
template <typename T, int L, int S>
__global__ void __launch_bounds__(THREADS)
step_kernel(const Args<T> a) {
  const Place<T, L, S> me(a);
  const int64_t row = blockIdx.y;
  const int c = me.c0 + me.ch;
  T A[S], h[S], sum = 0;
  me.load(a, a.A, A);
  me.load(a, a.h0 + row * a.dim * a.state, h);
  const T u = me.on ? a.u[row * a.ld_u + c] : (T)0;
  T dt = me.on ? a.delta[row * a.ld_delta + c] : (T)0;
  if (a.bias && me.on) dt += a.bias[c];
  if (a.softplus) dt = softplus(dt);
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const bool live = me.on && me.n0 + j < a.state;
    const T B = live ? a.B[row * a.ld_B + me.q * a.state + me.n0 + j] : (T)0;
    const T C = live ? a.C[row * a.ld_C + me.q * a.state + me.n0 + j] : (T)0;
    h[j] = decay(dt * rate(A[j])) * h[j] + dt * u * B;
    sum += C * h[j];
  }
  me.store(a, a.h_last + row * a.dim * a.state, h);
#pragma unroll
  for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (me.on && me.lane == 0) {
    if (a.D) sum += a.D[c] * u;
    if (a.z) sum *= swish(a.z[row * a.ld_z + c]);
    a.y[row * a.ld_y + c] = sum;
  }
}

// ---------------------------------------------------------------- launches
enum class Pass { Forward, Backward, Step };

// How the token axis is cut: by sequences where they are of equal length and give CTAs enough for the device, else into spans of
// whole tiles.
template <typename T> static void cut(prad_ctx* ctx, Args<T>& a, int64_t ctas_across) {
  const int64_t full = (int64_t)ctx->sm_count * 4;
  if (!a.rows.offsets && a.rows.count > 0 && (a.rows.count * ctas_across >= full / 2 || a.rows.each <= 2 * tile<T>()) &&
      a.rows.count <= 65535) {
    a.span = a.rows.each > 0 ? a.rows.each : 1;
    a.spans = a.rows.count;
    return;
  }
  int64_t spans = ceil_div(full, ctas_across);
  int64_t span = ceil_div(ceil_div(a.rows.tokens, spans), tile<T>()) * tile<T>();
  if (span < 2 * tile<T>()) span = 2 * tile<T>();
  if (ceil_div(a.rows.tokens, span) > 65535) span = ceil_div(ceil_div(a.rows.tokens, 65535), tile<T>()) * tile<T>();
  a.span = span;
  a.spans = (int)ceil_div(a.rows.tokens, span);
  if (a.spans < 1) a.spans = 1;
}
// whether a span may begin inside a sequence
template <typename T> static bool joined(const Args<T>& a) { return a.spans > 1 && (a.rows.offsets || a.span != a.rows.each); }

template <typename T> struct Carve {
  char* at;
  size_t used = 0;
  template <typename U> U* take(int64_t n) {
    U* p = at ? (U*)(at + used) : nullptr;
    used += ((size_t)n * sizeof(U) + 255) & ~(size_t)255;
    return p;
  }
};
template <typename T> static size_t carve(Args<T>& a, bool backward, void* ws) {
  Carve<T> c{(char*)ws};
  const int64_t states = (int64_t)a.dim * a.state;
  if (joined(a)) {
    a.edge = c.template take<T>((a.spans + 1) * states);
    a.sum = c.template take<T>((int64_t)a.spans * a.dim);
    a.passes = c.template take<int>(a.spans);
  }
  if (backward) {
    a.part_A = c.template take<T>(a.spans * states);
    a.part_D = c.template take<T>((int64_t)a.spans * a.dim);
    a.part_bias = c.template take<T>((int64_t)a.spans * a.dim);
    if (a.blocks > 1) a.part_BC = c.template take<T>((int64_t)a.blocks * a.rows.tokens * a.groups * 2 * a.state);
  }
  return c.used;
}

template <typename T, int L, int S> static prad_status launch(prad_ctx* ctx, Args<T> a, Pass pass) {
  constexpr int CH = THREADS / L;
  a.blocks = (int)ceil_div(a.per, CH);
  const int64_t across = (int64_t)a.groups * a.blocks;
  PRAD_REQUIRE(across <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "selective scan: too many channels");
  if (pass == Pass::Step) {
    for (int64_t r0 = 0; r0 < a.rows.tokens; r0 += 65535) {      // (the grid's second dimension)
      Args<T> b = a;
      const int64_t n = a.rows.tokens - r0 < 65535 ? a.rows.tokens - r0 : 65535, states = (int64_t)a.dim * a.state;
      b.u += r0 * a.ld_u, b.delta += r0 * a.ld_delta, b.B += r0 * a.ld_B, b.C += r0 * a.ld_C, b.y += r0 * a.ld_y;
      if (b.z) b.z += r0 * a.ld_z;
      b.h0 += r0 * states, b.h_last += r0 * states;
      step_kernel<T, L, S><<<dim3((unsigned)across, (unsigned)n), THREADS, 0, ctx->stream>>>(b);
      PRAD_LAUNCHED(ctx);
    }
    return PRAD_OK;
  }
  cut(ctx, a, across);
  const bool backward = pass == Pass::Backward;
  prad_status st = ensure_workspace(ctx, carve(a, backward, nullptr));
  if (st) return st;
  carve(a, backward, ctx->ws);
  const int64_t states = (int64_t)a.dim * a.state;
  const unsigned x = (unsigned)across;
  if (!backward) {
    constexpr int bytes = (int)sizeof(Forward<T, L, S>);
    if (joined(a)) {
      st = allow_smem<forward_kernel<T, L, S, true>>(ctx, bytes);
      if (st) return st;
      forward_kernel<T, L, S, true><<<dim3(x, (unsigned)a.spans - 1), THREADS, bytes, ctx->stream>>>(a);
      PRAD_LAUNCHED(ctx);
      join_kernel<T, true><<<(unsigned)ceil_div(states, THREADS), THREADS, 0, ctx->stream>>>(a);
      PRAD_LAUNCHED(ctx);
    }
    st = allow_smem<forward_kernel<T, L, S, false>>(ctx, bytes);
    if (st) return st;
    forward_kernel<T, L, S, false><<<dim3(x, (unsigned)a.spans), THREADS, bytes, ctx->stream>>>(a);
    PRAD_LAUNCHED(ctx);
    return PRAD_OK;
  }
  using Shared = typename Backward<T, L, S>::Shared;
  st = allow_smem<backward_kernel<T, L, S>>(ctx, (int)sizeof(Shared));
  if (st) return st;
  if (a.dh0) PRAD_CUDA(cudaMemsetAsync(a.dh0, 0, (size_t)a.rows.count * states * sizeof(T), ctx->stream));
  if (joined(a)) {
    backward_edges_kernel<T, L, S><<<dim3(x, (unsigned)a.spans), THREADS, 0, ctx->stream>>>(a);
    PRAD_LAUNCHED(ctx);
    join_kernel<T, false><<<(unsigned)ceil_div(states, THREADS), THREADS, 0, ctx->stream>>>(a);
    PRAD_LAUNCHED(ctx);
  }
  backward_kernel<T, L, S><<<dim3(x, (unsigned)a.spans), THREADS, sizeof(Shared), ctx->stream>>>(a);
  PRAD_LAUNCHED(ctx);
  span_totals_kernel<T><<<(unsigned)ceil_div(states + 2 * (int64_t)a.dim, THREADS), THREADS, 0, ctx->stream>>>(a);
  PRAD_LAUNCHED(ctx);
  if (a.blocks > 1 && a.rows.tokens) {
    const int64_t n = a.rows.tokens * a.groups * 2 * a.state;
    row_totals_kernel<T><<<(unsigned)ceil_div(n, 256), 256, 0, ctx->stream>>>(a);
    PRAD_LAUNCHED(ctx);
  }
  return PRAD_OK;
}
template <typename T> static prad_status pick(prad_ctx* ctx, const Args<T>& a, Pass pass) {
  if (a.state <= 4) return launch<T, 4, 1>(ctx, a, pass);
  if (a.state <= 8) return launch<T, 4, 2>(ctx, a, pass);
  if (a.state <= 16) return launch<T, 4, 4>(ctx, a, pass);
  if (a.state <= 32) return launch<T, 8, 4>(ctx, a, pass);
  if (a.state <= 64) return launch<T, 16, 4>(ctx, a, pass);
  return launch<T, 32, 4>(ctx, a, pass);
}

static prad_status check(const char* who, prad_dtype dt, const prad_scan_t* s) {
  PRAD_REQUIRE(dtype_ok(dt), PRAD_ERR_INVALID, "%s: unknown dtype %d", who, (int)dt);
  PRAD_REQUIRE(s, PRAD_ERR_INVALID, "%s: null scan", who);
  PRAD_REQUIRE(s->tokens >= 0 && s->sequences >= 0 && s->dim > 0 && s->state > 0 && s->groups > 0, PRAD_ERR_SHAPE, "%s: bad shape", who);
  PRAD_REQUIRE(s->dim % s->groups == 0, PRAD_ERR_SHAPE, "%s: %d channels do not divide into %d groups", who, s->dim, s->groups);
  PRAD_REQUIRE(s->state <= MAX_STATE, PRAD_ERR_UNSUPPORTED, "%s: at most %d states, got %d", who, MAX_STATE, s->state);
  PRAD_REQUIRE(s->tokens <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", who);
  PRAD_REQUIRE(s->dim <= 1 << 20, PRAD_ERR_UNSUPPORTED, "%s: more than 2^20 channels", who);
  const int64_t rows = (int64_t)s->groups * s->state;
  PRAD_REQUIRE((!s->ld_u || s->ld_u >= s->dim) && (!s->ld_delta || s->ld_delta >= s->dim) && (!s->ld_z || s->ld_z >= s->dim) &&
                   (!s->ld_B || s->ld_B >= rows) && (!s->ld_C || s->ld_C >= rows),
               PRAD_ERR_SHAPE, "%s: a pitch below the row", who);
  PRAD_REQUIRE(s->tokens == 0 || (s->u && s->delta && s->A && s->B && s->C), PRAD_ERR_INVALID, "%s: null pointer", who);
  return PRAD_OK;
}
static prad_status check_sequences(const char* who, const prad_scan_t* s) {
  PRAD_REQUIRE(s->offsets || (s->sequences > 0 ? s->tokens % s->sequences == 0 : s->tokens == 0), PRAD_ERR_SHAPE,
               "%s: %lld tokens do not divide into %d sequences", who, (long long)s->tokens, s->sequences);
  PRAD_REQUIRE(((uintptr_t)s->offsets & 3) == 0, PRAD_ERR_INVALID, "%s: unaligned offsets", who);
  return PRAD_OK;
}

template <typename T> static Args<T> args_of(const prad_scan_t* s) {
  Args<T> a = {};
  const int64_t rows = (int64_t)s->groups * s->state;
  a.rows = Sequences{s->offsets, s->sequences, s->tokens, s->offsets || s->sequences == 0 ? 0 : s->tokens / s->sequences};
  a.dim = s->dim, a.state = s->state, a.groups = s->groups, a.per = s->dim / s->groups;
  a.softplus = s->delta_softplus;
  a.ld_u = s->ld_u ? s->ld_u : s->dim, a.ld_delta = s->ld_delta ? s->ld_delta : s->dim, a.ld_z = s->ld_z ? s->ld_z : s->dim;
  a.ld_B = s->ld_B ? s->ld_B : rows, a.ld_C = s->ld_C ? s->ld_C : rows;
  a.u = (const T*)s->u, a.delta = (const T*)s->delta, a.z = (const T*)s->z, a.A = (const T*)s->A, a.B = (const T*)s->B;
  a.C = (const T*)s->C, a.D = (const T*)s->D, a.bias = (const T*)s->delta_bias, a.h0 = (const T*)s->h0;
  return a;
}

}  // namespace ssm
}  // namespace prad

using namespace prad;

template <typename T>
static prad_status forward_t(prad_ctx* ctx, const prad_scan_t* scan, void* y, int64_t ld_y, void* h_last, void* saved, ssm::Pass pass) {
  ssm::Args<T> a = ssm::args_of<T>(scan);
  a.y = (T*)y, a.ld_y = ld_y ? ld_y : scan->dim, a.h_last = (T*)h_last, a.saved = (T*)saved;
  return ssm::pick<T>(ctx, a, pass);
}
template <typename T>
static prad_status backward_t(prad_ctx* ctx, const prad_scan_t* scan, const void* saved, const void* dy, int64_t ld_dy,
                              const prad_scan_gradients_t* g) {
  ssm::Args<T> a = ssm::args_of<T>(scan);
  const int64_t rows = (int64_t)scan->groups * scan->state;
  a.saved = (T*)const_cast<void*>(saved), a.dy = (const T*)dy, a.ld_dy = ld_dy ? ld_dy : scan->dim;
  a.du = (T*)g->du, a.ddelta = (T*)g->ddelta, a.dz = (T*)g->dz, a.dA = (T*)g->dA, a.dB = (T*)g->dB, a.dC = (T*)g->dC;
  a.dD = (T*)g->dD, a.dbias = (T*)g->ddelta_bias, a.dh0 = (T*)g->dh0;
  a.ld_du = g->ld_du ? g->ld_du : scan->dim, a.ld_ddelta = g->ld_ddelta ? g->ld_ddelta : scan->dim;
  a.ld_dz = g->ld_dz ? g->ld_dz : scan->dim, a.ld_dB = g->ld_dB ? g->ld_dB : rows, a.ld_dC = g->ld_dC ? g->ld_dC : rows;
  return ssm::pick<T>(ctx, a, ssm::Pass::Backward);
}

extern "C" prad_status prad_selective_scan_saved_bytes(prad_dtype dt, const prad_scan_t* scan, size_t* out_bytes) {
  prad_status st = ssm::check("prad_selective_scan_saved_bytes", dt, scan);
  if (st) return st;
  PRAD_REQUIRE(out_bytes, PRAD_ERR_INVALID, "prad_selective_scan_saved_bytes: null output");
  const int64_t tile = dt == PRAD_F64 ? ssm::tile<double>() : ssm::tile<float>();
  *out_bytes = (size_t)ceil_div(scan->tokens, tile) * scan->dim * scan->state * dtype_size(dt);
  return PRAD_OK;
}

extern "C" prad_status prad_selective_scan_forward(prad_ctx* ctx, prad_dtype dt, const prad_scan_t* scan, void* y, int64_t ld_y,
                                                   void* h_last, void* saved) {
  const char* who = "prad_selective_scan_forward";
  prad_status st = ssm::check(who, dt, scan);
  if (!st) st = ssm::check_sequences(who, scan);
  if (st) return st;
  PRAD_REQUIRE(!ld_y || ld_y >= scan->dim, PRAD_ERR_SHAPE, "%s: a pitch below dim", who);
  PRAD_REQUIRE(scan->tokens == 0 || y, PRAD_ERR_INVALID, "%s: null pointer", who);
  PRAD_REQUIRE(scan->tokens == 0 || (y != scan->u && y != scan->delta && y != scan->z), PRAD_ERR_INVALID, "%s: y may not be an input", who);
  PRAD_REQUIRE(!h_last || h_last != scan->h0, PRAD_ERR_INVALID, "%s: h_last may not be h0", who);
  PRAD_CHECK_CTX(ctx);
  if (scan->tokens == 0) {       // every final state is the initial one
    const size_t bytes = (size_t)scan->sequences * scan->dim * scan->state * dtype_size(dt);
    if (h_last && bytes && scan->h0) PRAD_CUDA(cudaMemcpyAsync(h_last, scan->h0, bytes, cudaMemcpyDeviceToDevice, ctx->stream));
    else if (h_last && bytes) PRAD_CUDA(cudaMemsetAsync(h_last, 0, bytes, ctx->stream));
    return PRAD_OK;
  }
  return dt == PRAD_F32 ? forward_t<float>(ctx, scan, y, ld_y, h_last, saved, ssm::Pass::Forward)
                        : forward_t<double>(ctx, scan, y, ld_y, h_last, saved, ssm::Pass::Forward);
}

extern "C" prad_status prad_selective_scan_backward(prad_ctx* ctx, prad_dtype dt, const prad_scan_t* scan, const void* saved, const void* dy,
                                                    int64_t ld_dy, const prad_scan_gradients_t* g) {
  const char* who = "prad_selective_scan_backward";
  prad_status st = ssm::check(who, dt, scan);
  if (!st) st = ssm::check_sequences(who, scan);
  if (st) return st;
  PRAD_REQUIRE(g, PRAD_ERR_INVALID, "%s: null gradients", who);
  const int64_t rows = (int64_t)scan->groups * scan->state;
  PRAD_REQUIRE((!ld_dy || ld_dy >= scan->dim) && (!g->ld_du || g->ld_du >= scan->dim) && (!g->ld_ddelta || g->ld_ddelta >= scan->dim) &&
                   (!g->ld_dz || g->ld_dz >= scan->dim) && (!g->ld_dB || g->ld_dB >= rows) && (!g->ld_dC || g->ld_dC >= rows),
               PRAD_ERR_SHAPE, "%s: a pitch below the row", who);
  PRAD_REQUIRE(!g->dh0 || scan->h0, PRAD_ERR_INVALID, "%s: dh0 without an h0", who);
  PRAD_REQUIRE(scan->tokens == 0 || (saved && dy && g->du && g->ddelta && g->dB && g->dC && (!scan->z || g->dz)), PRAD_ERR_INVALID,
               "%s: null pointer", who);
  PRAD_CHECK_CTX(ctx);
  if (scan->tokens == 0) {
    const size_t s = dtype_size(dt), states = (size_t)scan->dim * scan->state;
    if (g->dA) PRAD_CUDA(cudaMemsetAsync(g->dA, 0, states * s, ctx->stream));
    if (g->dD) PRAD_CUDA(cudaMemsetAsync(g->dD, 0, scan->dim * s, ctx->stream));
    if (g->ddelta_bias) PRAD_CUDA(cudaMemsetAsync(g->ddelta_bias, 0, scan->dim * s, ctx->stream));
    if (g->dh0 && scan->sequences) PRAD_CUDA(cudaMemsetAsync(g->dh0, 0, scan->sequences * states * s, ctx->stream));
    return PRAD_OK;
  }
  return dt == PRAD_F32 ? backward_t<float>(ctx, scan, saved, dy, ld_dy, g) : backward_t<double>(ctx, scan, saved, dy, ld_dy, g);
}

extern "C" prad_status prad_selective_scan_step(prad_ctx* ctx, prad_dtype dt, const prad_scan_t* scan, void* y, int64_t ld_y, void* h_out) {
  const char* who = "prad_selective_scan_step";
  prad_status st = ssm::check(who, dt, scan);
  if (st) return st;
  PRAD_REQUIRE(!ld_y || ld_y >= scan->dim, PRAD_ERR_SHAPE, "%s: a pitch below dim", who);
  PRAD_REQUIRE(!scan->offsets && scan->sequences == scan->tokens, PRAD_ERR_SHAPE, "%s: one token for each sequence", who);
  PRAD_REQUIRE(scan->tokens == 0 || (scan->h0 && h_out && y), PRAD_ERR_INVALID, "%s: null pointer", who);
  PRAD_CHECK_CTX(ctx);
  if (scan->tokens == 0) return PRAD_OK;
  return dt == PRAD_F32 ? forward_t<float>(ctx, scan, y, ld_y, h_out, nullptr, ssm::Pass::Step)
                        : forward_t<double>(ctx, scan, y, ld_y, h_out, nullptr, ssm::Pass::Step);
}
