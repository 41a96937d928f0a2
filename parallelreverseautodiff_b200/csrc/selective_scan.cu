// The selective state space scan.  Channel d with the states n of its group's rows B, C; per token of a sequence
//   dt = delta + delta_bias (softplus of it where asked),  a_n = exp(dt A_dn),  h_n <- a_n h_n + dt u B_n,
//   r = sum_n C_n h_n + D u,  y = r or r swish(z);
// the state begins at h0 (zero without one) and is given back in h_last.  Backward, with v = dy swish(z) (dy without z):
//   g_n(t) = C_n v + a_n(t + 1) g_n(t + 1),  du = dt sum g B + D v,  ddt = u sum g B + sum g_n A_n a_n h_n(t - 1),
//   dA_n = sum_t g_n dt a_n h_n(t - 1),  dB_n = sum over the group's channels of g_n dt u,  dC_n likewise of v h_n,
//   dD = sum v u,  dz = dy r swish'(z),  ddelta = ddt sigmoid(delta + delta_bias),  dh0 = a_n g_n of the first token.
//
// L lanes share a channel, S states each; a CTA takes THREADS / L channels of one group over a span of the tokens, a tile of TT at a
// time in shared memory.  What bounds it is arithmetic, not memory: N exponentials and 4 N multiply-adds for 16 bytes of a float.
//
// The token axis of all sequences is one recurrence in which the state is replaced where a sequence begins.  When the sequences
// alone give too few CTAs, it is cut into spans of equal length: one pass finds what each span makes of a zero state (and of any
// other: exp(A sum dt) times it, as decays multiply), a second strings the spans together, and the main pass starts each span from
// the state it has.  The backward pass runs the same way from the last span up, on checkpoints of the state every POINT tokens that
// the forward pass leaves.
//
// 16384 tokens of 1024 float channels with 16 states: edges 93 us, main pass 132 us (a prompt; the exponentials alone would take 60 us
// each time, the memory 42 us); backward edges 78 us, main pass 431 to 446 us on two devices.  The edges' passes use the special
// function unit at 70 %.  In both main passes no unit is used much above half of its cycles, and several are at the same time: chains
// of dependent instructions on the twelve (backward) and sixteen warps that registers leave to an SM are what is left.  Tried and taken
// back: more CTAs with fewer registers each (spills; 162 us for 155 forward), one channel a thread backward (614 us for 446, four CTAs
// an SM), and exponentials by polynomials (every fourth pair in the edges' passes: 95 us for 93, backward 83 for 78), which take more
// issue slots than they free.
#include "common.cuh"
#include "packed_sequences.cuh"

namespace prad {
namespace ssm {

using seq::Pack;
using seq::Sequences;
using seq::swish;
using seq::swish_slope;
using seq::Two;
using seq::fma;
using seq::mul;

constexpr int THREADS = 128;
// TT of the passes without a history: 16 where a CTA has 64 channels (or doubles), so that what it fetches stays in registers
template <typename T, int L> constexpr int tile() { return sizeof(T) == 8 || L == 2 ? 16 : 32; }
// spans are multiples of this many tokens, and two of them at least
template <typename T> constexpr int span_unit() { return sizeof(T) == 8 ? 16 : 32; }
// Tokens per checkpoint, and TT of the main backward pass: with 8 shared memory leaves room for three CTAs, with 16 there are half of
// the checkpoints and two CTAs (the pass took 518 us for 470 when this was chosen, with later steps 446).
constexpr int POINT = 8;
constexpr int MAX_STATE = 128;

template <typename T> struct Args {
  Sequences rows;
  int64_t span;                 // tokens of a span
  int spans, dim, state, groups, per, blocks;   // per: channels of a group, in `blocks` CTAs
  int softplus;
  int wide, wide_B, wide_C, wide_h;     // the token matrices, B, C and the matrices of states: 16 bytes at a time
  int block0;                   // backward: the first of a group's CTAs in this launch
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

// exp(dt A): in float as 2^(dt A' + LIFT) with A' = A log2 e.  The special function unit's 2^x is too small by 0.1 to 0.4 of 2^-24 on
// the average over [-b, 0), b = 0.001 to 1 (measured on 2^24 values each), and with 3 2^-27 added to x off by less than 0.17 of it: an
// error that does not average out builds up over the tokens that a state remembers (dA of 16384 tokens: off by 1.7e-6 without, 0.9e-6
// with it), and the sum comes with the product.  2^LIFT is exactly 1, for rows without a token and states that do not exist.
constexpr float LIFT = 2.2351741790771484e-8f;
__device__ __forceinline__ float decay(float dt, float rate) { return seq::exp2_approx(fmaf(dt, rate, LIFT)); }
__device__ __forceinline__ double decay(double dt, double rate) { return exp(dt * rate); }
// A' no lower than the type's lowest value: a state of A = -inf, which forgets everything, keeps its value over rows without a token,
// where dt is zero, and takes no NaN into the gradient of dt.
__device__ __forceinline__ float rate(float a) {
  a *= 1.4426950408889634f;
  return a < -3.402823466e38f ? -3.402823466e38f : a;        // (a NaN stays)
}
__device__ __forceinline__ double rate(double a) { return a < -1.7976931348623157e308 ? -1.7976931348623157e308 : a; }
template <typename T> __device__ __forceinline__ T per_rate();         // A per A'
template <> __device__ __forceinline__ float per_rate<float>() { return 0.6931471805599453f; }
template <> __device__ __forceinline__ double per_rate<double>() { return 1.0; }

// log(1 + e^x) = max(x, 0) + log(1 + w) with w = e^-|x|.  In float log(1 + w) = 2 atanh(r), r = w / (2 + w) <= 1/3, by a polynomial
// in r^2: the Chebyshev interpolation of atanh(r) / r over r^2 <= 1/9, off by 4e-9 of the value; this keeps the small time steps
// of very negative x to their last bits, at a third of the instructions of log1p and exp.
__device__ __forceinline__ float softplus(float x) {
  const float w = seq::exp2_approx(fabsf(x) * -1.4426950408889634f), r = w * seq::reciprocal(w + 2.0f), q = r * r;
  float p = 0.140788892f;
  p = fmaf(p, q, 0.139825789f);
  p = fmaf(p, q, 0.200122976f);
  p = fmaf(p, q, 0.333331608f);
  p = fmaf(p, q, 1.0f);
  return fmaf(r + r, p, fmaxf(x, 0.0f));
}
// of two values
__device__ __forceinline__ Two<float> softplus(Two<float> x) {
  float a, b, c, d;
  x.get(a, b);
  const Two<float> w(seq::exp2_approx(fabsf(a) * -1.4426950408889634f), seq::exp2_approx(fabsf(b) * -1.4426950408889634f));
  fma(w, Two<float>(1.0f, 1.0f), Two<float>(2.0f, 2.0f)).get(c, d);
  const Two<float> r = mul(w, Two<float>(seq::reciprocal(c), seq::reciprocal(d))), q = mul(r, r);
  Two<float> p(2.0f * 0.140788892f, 2.0f * 0.140788892f);
  p = fma(p, q, Two<float>(2.0f * 0.139825789f, 2.0f * 0.139825789f));
  p = fma(p, q, Two<float>(2.0f * 0.200122976f, 2.0f * 0.200122976f));
  p = fma(p, q, Two<float>(2.0f * 0.333331608f, 2.0f * 0.333331608f));
  p = fma(p, q, Two<float>(2.0f, 2.0f));
  return fma(r, p, Two<float>(fmaxf(a, 0.0f), fmaxf(b, 0.0f)));
}
// the same and its derivative, the sigmoid
__device__ __forceinline__ float softplus(float x, float& slope) {
  const float w = seq::exp2_approx(fabsf(x) * -1.4426950408889634f), i = seq::reciprocal(1.0f + w);
  slope = x > 0.0f ? i : w * i;
  return softplus(x);
}
__device__ __forceinline__ double softplus(double x, double& slope) {
  slope = seq::sigmoid(x);
  return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }
__device__ __forceinline__ Two<double> softplus(Two<double> x) { return {softplus(x.a_), softplus(x.b_)}; }
// Time steps of V channels from their rows' delta and the bias; zero for a row that is no token
template <int V, typename T> __device__ __forceinline__ void time_steps(const T (&delta)[V], const T (&bias)[V], bool soft, bool live, T (&dt)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    Two<T> x = fma(Two<T>(delta[j], delta[j + 1]), Two<T>((T)1, (T)1), Two<T>(bias[j], bias[j + 1]));
    if (soft) x = softplus(x);
    x.get(dt[j], dt[j + 1]);
    if (!live) dt[j] = dt[j + 1] = 0;
  }
}

__device__ __forceinline__ Two<float> decay(Two<float> dt, Two<float> rate) {
  float a, b;
  fma(dt, rate, Two<float>(LIFT, LIFT)).get(a, b);
  return {seq::exp2_approx(a), seq::exp2_approx(b)};
}
__device__ __forceinline__ Two<double> decay(Two<double> dt, Two<double> rate) { return {decay(dt.a_, rate.a_), decay(dt.b_, rate.b_)}; }
template <typename T> __device__ __forceinline__ T total(Two<T> x) {
  T a, b;
  x.get(a, b);
  return a + b;
}
// S values of shared memory (16-byte aligned for float) as pairs
template <int P> __device__ __forceinline__ void read(const float* m, Two<float> (&v)[P]) {
  if constexpr (P == 1) {
    v[0].v = *reinterpret_cast<const unsigned long long*>(m);
  } else {
#pragma unroll
    for (int j = 0; j < P; j += 2) {
      const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(m + 2 * j);
      v[j].v = q.x;
      v[j + 1].v = q.y;
    }
  }
}
template <int P> __device__ __forceinline__ void read(const double* m, Two<double> (&v)[P]) {
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const double2 q = *reinterpret_cast<const double2*>(m + 2 * j);
    v[j] = {q.x, q.y};
  }
}
// a token's time step and dt u of a channel, each twice in float
struct alignas(16) StepF { float dt, dt_, x, x_; };
struct alignas(16) StepD { double dt, x; };
template <typename T> struct StepOf { using type = StepF; };
template <> struct StepOf<double> { using type = StepD; };
__device__ __forceinline__ void write(StepF* m, float dt, float x) { *reinterpret_cast<float4*>(m) = make_float4(dt, dt, x, x); }
__device__ __forceinline__ void write(StepD* m, double dt, double x) { *reinterpret_cast<double2*>(m) = make_double2(dt, x); }
__device__ __forceinline__ void read(const StepF* m, Two<float>& dt, Two<float>& x) {
  const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(m);
  dt.v = q.x;
  x.v = q.y;
}
__device__ __forceinline__ void read(const StepD* m, Two<double>& dt, Two<double>& x) {
  const double2 q = *reinterpret_cast<const double2*>(m);
  dt = {q.x, q.x};
  x = {q.y, q.y};
}

// How a warp's lanes share channels and states: a lane's number among the L of its channel is made of the lane's bits 1, 4, 3, 2, 0 (as
// many as L needs), its channel's number of the others.  A 128-bit read of shared memory takes two cycles if its address does not
// depend on bit 0 or does not depend on bit 1 of the lane, and four otherwise: so the reads by channel and those by state both take two.
template <int L> struct Lanes {
  static constexpr int STATE_BITS = L == 2 ? 1 : L == 4 ? 2 : L == 8 ? 3 : L == 16 ? 4 : 5;
  __host__ __device__ static constexpr int state_bit(int i) { return i == 0 ? 1 : i == 4 ? 0 : 5 - i; }
  __host__ __device__ static constexpr int channel_bit(int i) { return i == 0 ? 0 : i + 1; }      // 0, 2, 3, 4
  __device__ static __forceinline__ int state(int lane) {
    int l = 0;
#pragma unroll
    for (int i = 0; i < STATE_BITS; ++i) l |= (lane >> state_bit(i) & 1) << i;
    return l;
  }
  __device__ static __forceinline__ int channel(int lane) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < 5 - STATE_BITS; ++i) c |= (lane >> channel_bit(i) & 1) << i;
    return c;
  }
};

// States n0 .. n0 + S - 1 of a channel in a [dim][state] matrix; those that do not exist are zero.
template <int S, typename T>
__device__ __forceinline__ void read_states(const T* m, int channel, int n0, bool on, const Args<T>& a, T (&h)[S]) {
  constexpr int V = S * sizeof(T) < 16 ? S : 16 / sizeof(T);
  m += (int64_t)channel * a.state + n0;
  if (a.wide_h) {
#pragma unroll
    for (int j = 0; j < S; j += V) {
      Pack<T, V> w;
#pragma unroll
      for (int i = 0; i < V; ++i) w.v[i] = 0;
      if (on && n0 + j < a.state) w = *reinterpret_cast<const Pack<T, V>*>(m + j);
#pragma unroll
      for (int i = 0; i < V; ++i) h[j + i] = w.v[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j) h[j] = on && n0 + j < a.state ? m[j] : (T)0;
  }
}
template <int S, typename T>
__device__ __forceinline__ void write_states(T* m, int channel, int n0, bool on, const Args<T>& a, const T (&h)[S]) {
  constexpr int V = S * sizeof(T) < 16 ? S : 16 / sizeof(T);
  m += (int64_t)channel * a.state + n0;
  if (a.wide_h) {
#pragma unroll
    for (int j = 0; j < S; j += V) {
      Pack<T, V> w;
#pragma unroll
      for (int i = 0; i < V; ++i) w.v[i] = h[j + i];
      if (on && n0 + j < a.state) *reinterpret_cast<Pack<T, V>*>(m + j) = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (on && n0 + j < a.state) m[j] = h[j];
  }
}

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
    ch = threadIdx.x / 32 * (32 / L) + Lanes<L>::channel(threadIdx.x % 32);
    lane = Lanes<L>::state(threadIdx.x % 32);
    n0 = lane * S;
    on = ch < channels;
  }
  // S states of this thread in a [dim][state] matrix
  __device__ __forceinline__ void load(const Args<T>& a, const T* m, T (&h)[S]) const { read_states<S>(m, c0 + ch, n0, on, a, h); }
  __device__ __forceinline__ void store(const Args<T>& a, T* m, const T (&h)[S]) const { write_states<S>(m, c0 + ch, n0, on, a, h); }
};

// Four values a lane, one for each of four tokens, summed over the L lanes of a channel: afterwards lane l holds the sum of token
// l mod 4 (with two lanes: lane l the sums of tokens 2 l and 2 l + 1).  Half of the values change hands in each of the first steps.
template <int L, typename T> __device__ __forceinline__ void sum4(const T (&v)[4], int lane, T& a, T& b) {
  const bool hi = L == 2 ? lane & 1 : lane & 2;
  constexpr int over = 1 << Lanes<L>::state_bit(L == 2 ? 0 : 1);
  a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], over);
  b += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], over);
  if constexpr (L > 2) {
    const bool odd = lane & 1;
    const T give = odd ? a : b;
    a = odd ? b : a;
    a += __shfl_xor_sync(0xffffffffu, give, 1 << Lanes<L>::state_bit(0));
#pragma unroll
    for (int i = 2; i < Lanes<L>::STATE_BITS; ++i) a += __shfl_xor_sync(0xffffffffu, a, 1 << Lanes<L>::state_bit(i));
  }
}
template <int L, typename T> __device__ __forceinline__ T sum4(const T (&v)[4], int lane) {
  static_assert(L > 2, "one sum a lane");
  T a, b;
  sum4<L>(v, lane, a, b);
  return a;
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

// B or C rows of tiles, by asynchronous copies; rows without a token are zero
template <typename T, int N, int TT> struct Rows {
  static constexpr int V = 16 / sizeof(T), ACROSS = N / V, AT_ONCE = THREADS / ACROSS;
  const T *at, *valid;
  int64_t ld;
  int row, n, state;
  bool wide;
  __device__ __forceinline__ Rows(const T* from, int64_t ld, int first, int state, int wide, int64_t tile0)
      : valid(from), ld(ld), row(threadIdx.x / ACROSS), n(threadIdx.x % ACROSS * V), state(state), wide(wide) {
    at = from + tile0 * ld + first;
  }
  // rows [begin, finish) of the tile that `at` is at
  __device__ __forceinline__ void fetch(T (*to)[N], int begin, int finish) const {
    if (wide) {
      if (ACROSS * AT_ONCE != THREADS && row >= AT_ONCE) return;
#pragma unroll
      for (int t0 = 0; t0 < TT; t0 += AT_ONCE) {
        const int t = t0 + row;
        if (TT % AT_ONCE != 0 && t >= TT) break;
        const bool live = t >= begin && t < finish && n < state;
        const uint32_t d = (uint32_t)__cvta_generic_to_shared(&to[t][n]);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(live ? at + t * ld + n : valid), "r"(live ? 16 : 0)
                     : "memory");
      }
      return;
    }
#pragma unroll 1
    for (int e = threadIdx.x; e < TT * N; e += THREADS) {
      const int t = e / N, k = e % N;
      const bool live = t >= begin && t < finish && k < state;
      const uint32_t d = (uint32_t)__cvta_generic_to_shared(&to[t][k]);
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(live ? at + t * ld + k : valid), "n"((int)sizeof(T)),
                   "r"(live ? (int)sizeof(T) : 0)
                   : "memory");
    }
  }
};
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

// The token matrices' part of a tile: a thread has V neighbouring channels of E rows.
template <typename T, int CH, int TT> struct Cells {
  static constexpr int V = 16 / sizeof(T), ACROSS = CH / V, ROWS = THREADS / ACROSS, E = TT > ROWS ? TT / ROWS : 1;
  static_assert(CH % V == 0 && (TT % ROWS == 0 || ROWS % TT == 0), "whole rows of threads");
  int col, row, mine;            // mine: of the V channels, those that exist
  bool wide;
  __device__ __forceinline__ Cells(int channels, bool aligned) {
    col = threadIdx.x % ACROSS * V;
    row = threadIdx.x / ACROSS;
    mine = channels - col < V ? channels - col : V;
    wide = aligned && mine == V;
  }
  // whether row e of this thread lies in the tile
  __device__ __forceinline__ bool in(int e) const { return ROWS <= TT || row < TT; }
  // this thread's first value of a tile
  __device__ __forceinline__ int64_t first(int64_t ld, int64_t tile0) const { return (tile0 + row) * ld + col; }
  // rows [from, to) of the tile; what lies outside, and channels that do not exist, as zero
  __device__ __forceinline__ void load(const T* at, int64_t ld, int from, int to, T (&v)[E][V]) const {
    if (wide && to - from == TT) {
#pragma unroll
      for (int e = 0; e < E; ++e, at += ROWS * ld) {
        if (!in(e)) break;
        const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(at);
#pragma unroll
        for (int j = 0; j < V; ++j) v[e][j] = w.v[j];
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e, at += ROWS * ld) {
      const bool live = row + e * ROWS >= from && row + e * ROWS < to;
#pragma unroll
      for (int j = 0; j < V; ++j) v[e][j] = live && j < mine ? at[j] : (T)0;
    }
  }
  __device__ __forceinline__ void store(T* at, int64_t ld, int from, int to, const T (&v)[E][V]) const {
    if (wide && to - from == TT) {
#pragma unroll
      for (int e = 0; e < E; ++e, at += ROWS * ld) {
        if (!in(e)) break;
        Pack<T, V> w;
#pragma unroll
        for (int j = 0; j < V; ++j) w.v[j] = v[e][j];
        *reinterpret_cast<Pack<T, V>*>(at) = w;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e, at += ROWS * ld) {
      const bool live = row + e * ROWS >= from && row + e * ROWS < to;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (live && j < mine) at[j] = v[e][j];
    }
  }
  // one value per channel
  __device__ __forceinline__ void per_channel(const T* m, T (&v)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = m && j < mine ? m[col + j] : (T)0;
  }
};
// Where channel c's entry of 16 bytes lies in a row of shared memory: threads that write V channels each, and warps that read eight,
// spread over all banks.
template <typename T> __device__ __forceinline__ int spot(int c) { return c ^ (c >> 3 & (16 / (int)sizeof(T) - 1)); }
// the same of channel col + j, j < V, for a thread's first channel
template <typename T> __device__ __forceinline__ int spot(int col, int j) { return col + (j ^ (col >> 3 & (16 / (int)sizeof(T) - 1))); }
// V values side by side in shared memory
template <int V, typename T> __device__ __forceinline__ void put(T* m, const T (&v)[V]) {
  Pack<T, V> w;
#pragma unroll
  for (int j = 0; j < V; ++j) w.v[j] = v[j];
  *reinterpret_cast<Pack<T, V>*>(m) = w;
}
template <int V, typename T> __device__ __forceinline__ void pick(const T* m, T (&v)[V]) {
  const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(m);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = w.v[j];
}

// ---------------------------------------------------------------- forward
template <typename T, int L, int S> struct Forward {
  static constexpr int CH = THREADS / L, TT = tile<T, L>(), N = L * S;
  alignas(16) T B[2][TT][N], C[2][TT][N];
  typename StepOf<T>::type step[TT][CH];
  alignas(16) T y[TT][CH + 8];  // (four tokens of eight channels at a time: no two in one bank)
};

// EDGES: only the state that the span ends in when it begins with zero, and the sum of its time steps.
template <typename T, int L, int S, bool EDGES>
__global__ void __launch_bounds__(THREADS, 4)
forward_kernel(const Args<T> a) {
  chain_begin();
  constexpr int CH = THREADS / L, TT = tile<T, L>(), N = L * S, P = S / 2;
  extern __shared__ __align__(16) unsigned char raw[];
  Forward<T, L, S>& m = *reinterpret_cast<Forward<T, L, S>*>(raw);
  const Place<T, L, S> me(a);
  const int p = blockIdx.y, at = spot<T>(me.ch);
  const Span<T> span(a, p);
  int64_t begin = span.begin;
  const int64_t finish = span.finish;
  const int64_t states = (int64_t)a.dim * a.state;
  Two<T> A[P], h[P];
  {
    T w[S];
    me.load(a, a.A, w);
#pragma unroll
    for (int j = 0; j < P; ++j) A[j] = {rate(w[2 * j]), rate(w[2 * j + 1])};
  }
  const auto set = [&](const T* from) {        // null: zero
    T w[S];
#pragma unroll
    for (int j = 0; j < S; ++j) w[j] = 0;
    if (from) me.load(a, from, w);
#pragma unroll
    for (int j = 0; j < P; ++j) h[j] = {w[2 * j], w[2 * j + 1]};
  };
  const auto keep = [&](T* to) {
    T w[S];
#pragma unroll
    for (int j = 0; j < P; ++j) h[j].get(w[2 * j], w[2 * j + 1]);
    me.store(a, to, w);
  };
  const auto initial = [&](int s) { return a.h0 ? a.h0 + s * states : nullptr; };
  // sequences without a token in front of all others
  const int64_t lo = a.rows.begin();
  if (!EDGES && a.h_last && ((span.first <= lo && lo < span.first + a.span) || (p == a.spans - 1 && lo >= span.first + a.span)))
    for (int s = 0; s < a.rows.count && a.rows.end(s) <= lo; ++s) {
      set(initial(s));
      keep(a.h_last + s * states);
    }
  set(nullptr);
  if (EDGES) {
    // what comes before the last sequence that begins in the span does not reach its end, and nothing does beyond it if another
    // sequence begins there
    const int64_t start = begin < finish ? a.rows.start(a.rows.at(finish - 1)) : begin;
    const bool all = start < begin;
    if (!all && start < finish) begin = start;
    if (begin < finish && a.rows.end(a.rows.at(finish - 1)) <= finish) begin = finish;
    if (threadIdx.x == 0 && blockIdx.x == 0) a.passes[p] = all;
  }
  T sum = 0;
  if (begin < finish) {
    int s = a.rows.at(begin);
    int64_t end = a.rows.end(s);                // of sequence s, the one that the next token belongs to
    if (a.rows.start(s) >= begin) set(initial(s));
    else if (!EDGES && p > 0) set(a.edge + p * states);
    const int64_t tiles0 = begin / TT * TT;
    const Cells<T, CH, TT> mine(me.channels, a.wide);
    constexpr int E = Cells<T, CH, TT>::E, V = Cells<T, CH, TT>::V, ROWS = Cells<T, CH, TT>::ROWS;
    T u[E][V], d[E][V], z[E][V], bias[V], D[V];
    mine.per_channel(a.bias ? a.bias + me.c0 : nullptr, bias);
    mine.per_channel(!EDGES && a.D ? a.D + me.c0 : nullptr, D);
    const T* pu = a.u + me.c0 + mine.first(a.ld_u, tiles0);
    const T* pd = a.delta + me.c0 + mine.first(a.ld_delta, tiles0);
    const T* pz = a.z ? a.z + me.c0 + mine.first(a.ld_z, tiles0) : nullptr;
    T* py = EDGES ? nullptr : a.y + me.c0 + mine.first(a.ld_y, tiles0);
    Rows<T, N, TT> B_rows(a.B, a.ld_B, me.q * a.state, a.state, a.wide_B, tiles0);
    Rows<T, N, TT> C_rows(a.C, a.ld_C, me.q * a.state, a.state, a.wide_C, tiles0);
    const auto fetch = [&](int64_t tile0) {      // of the tiles in turn
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
      mine.load(pu, a.ld_u, from, to, u);
      mine.load(pd, a.ld_delta, from, to, d);
      pu += TT * a.ld_u;
      pd += TT * a.ld_delta;
      B_rows.fetch(m.B[tile0 / TT & 1], from, to);
      B_rows.at += TT * a.ld_B;
      if (!EDGES) {
        if (a.z) {
          mine.load(pz, a.ld_z, from, to, z);
          pz += TT * a.ld_z;
        }
        C_rows.fetch(m.C[tile0 / TT & 1], from, to);
        C_rows.at += TT * a.ld_C;
      }
    };
    fetch(tiles0);
    commit();
    for (int64_t tile0 = tiles0; tile0 < finish; tile0 += TT) {
      const int buf = (int)(tile0 / TT & 1);
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
      T kept_u[E][V], kept_z[E][V];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int r = mine.row + e * ROWS;
        T dt[V];
        time_steps(d[e], bias, a.softplus, r >= from && r < to, dt);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (mine.in(e)) write(&m.step[r][spot<T>(mine.col, j)], dt[j], dt[j] * u[e][j]);
          kept_u[e][j] = u[e][j];
          if (!EDGES) kept_z[e][j] = z[e][j];
        }
      }
      if (tile0 + TT < finish) fetch(tile0 + TT);
      commit();
      landed<1>();
      __syncthreads();
      const uint32_t starts = end < tile0 + TT && end < finish ? starts_in<TT>(a.rows, s, tile0, finish) : 0;
      const T(*rows_B)[N] = m.B[buf];
      const T(*rows_C)[N] = m.C[buf];
      const auto token = [&](int t) {
        Two<T> dt, x, B[P], r;
        read(&m.step[t][at], dt, x);
        read(&rows_B[t][me.n0], B);
        if (EDGES) {
          T one, two;
          dt.get(one, two);
          sum += one;
        }
#pragma unroll
        for (int j = 0; j < P; ++j) h[j] = fma(decay(dt, A[j]), h[j], mul(x, B[j]));
        if (EDGES) return (T)0;
        Two<T> C[P];
        read(&rows_C[t][me.n0], C);
        r = mul(C[0], h[0]);
#pragma unroll
        for (int j = 1; j < P; ++j) r = fma(C[j], h[j], r);
        return total(r);
      };
#pragma unroll 2
      for (int t0 = 0; t0 < TT; t0 += 4) {
        T part[4] = {0, 0, 0, 0};
        if (!EDGES && t0 % POINT == 0 && a.saved && t0 >= from && t0 < to) keep(a.saved + (tile0 + t0) / POINT * states);
        if ((starts >> t0 & 15) == 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k) part[k] = token(t0 + k);
        } else {
          // (a loop that is not unrolled: what tokens that begin sequences need is little used, and long)
#pragma unroll 1
          for (int k = 0; k < 4; ++k) {
            if (starts >> (t0 + k) & 1) {
              // the sequence that ends here, and the ones without a token behind it
              const int64_t here = tile0 + t0 + k;
              for (; s + 1 < a.rows.count && a.rows.end(s) <= here; ++s) {
                if (a.rows.start(s) >= here) set(initial(s));
                if (!EDGES && a.h_last) keep(a.h_last + s * states);
              }
              set(initial(s));
              end = a.rows.end(s);
              sum = 0;
            }
            const T r = token(t0 + k);
            part[0] = k == 0 ? r : part[0];
            part[1] = k == 1 ? r : part[1];
            part[2] = k == 2 ? r : part[2];
            part[3] = k == 3 ? r : part[3];
          }
        }
        if (!EDGES) {
          T one, two;
          sum4<L>(part, me.lane, one, two);
          if (L == 2) {
            m.y[t0 + 2 * me.lane][me.ch] = one;
            m.y[t0 + 2 * me.lane + 1][me.ch] = two;
          } else if (me.lane < 4) {
            m.y[t0 + me.lane][me.ch] = one;
          }
        }
      }
      __syncthreads();
      if (!EDGES) {
        T y[E][V];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          pick(&m.y[mine.in(e) ? mine.row + e * ROWS : 0][mine.col], y[e]);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[e][j] += D[j] * kept_u[e][j];
            if (a.z) y[e][j] *= swish(kept_z[e][j]);
          }
        }
        mine.store(py, a.ld_y, from, to, y);
        py += TT * a.ld_y;
      }
    }
    landed<0>();
    if (!EDGES && a.h_last)
      for (; s < a.rows.count && a.rows.end(s) <= finish; ++s) {
        if (a.rows.start(s) >= finish) set(initial(s));
        keep(a.h_last + s * states);
      }
  }
  if (EDGES) {
    keep(a.edge + (p + 1) * states);
    if (me.on && me.lane == 0) a.sum[(int64_t)p * a.dim + me.c0 + me.ch] = sum;
  }
}

// Strings the spans together: edge[p] becomes the state that span p begins with.  FORWARD: edge[p + 1] holds what span p ends in
// from zero; otherwise edge[p] holds what span p hands up from zero, and becomes what it is handed from below.
// A span takes what it is given, x, to own + through x.  A CTA has JOINED neighbouring states and 32 spans at a time, a warp each
// state: the lanes' maps are composed in five steps (18 spans of 8040 double states: 4 us; one thread for all spans of a state, 28 us).
constexpr int JOINED = 8;
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(32 * JOINED)
join_kernel(const Args<T> a) {
  chain_begin();
  __shared__ T s_own[JOINED][33], s_through[JOINED][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = threadIdx.x / JOINED;                  // of the reading and writing: span k, state i
  const int64_t i0 = (int64_t)blockIdx.x * JOINED, i = i0 + threadIdx.x % JOINED, each = (int64_t)a.dim * a.state;
  const bool on = i < each;
  const T A = on ? rate(a.A[i]) : (T)0;
  const int c = on ? (int)(i / a.state) : 0;
  const int spans = FORWARD ? a.spans - 1 : a.spans;
  T carry = 0;                                         // of this warp's state
  for (int k0 = 0; k0 < spans; k0 += 32) {
    const int p = FORWARD ? k0 + k : spans - 1 - k0 - k;
    const bool live = on && k0 + k < spans;
    T own = 0, through = 1;
    if (live) {
      own = a.edge[(p + FORWARD) * each + i];
      through = a.passes[p] ? decay(a.sum[(int64_t)p * a.dim + c], A) : (T)-1;       // (a decay is never negative)
    }
    s_own[threadIdx.x % JOINED][k] = own;
    s_through[threadIdx.x % JOINED][k] = through;
    __syncthreads();
    own = s_own[warp][lane];
    through = s_through[warp][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T before = __shfl_up_sync(0xffffffffu, own, o), pass = __shfl_up_sync(0xffffffffu, through, o);
      if (lane >= o && !(through < (T)0)) {            // (what a map that passes nothing is given, NaN or not, leaves no trace)
        own += through * before;
        through = pass < (T)0 ? pass : through * pass;
      }
    }
    // behind span k0 + lane, and in front of it
    const T behind = through < (T)0 ? own : own + through * carry;
    T front = __shfl_up_sync(0xffffffffu, behind, 1);
    if (lane == 0) front = carry;
    carry = __shfl_sync(0xffffffffu, behind, 31);
    __syncthreads();
    s_own[warp][lane] = FORWARD ? behind : front;
    __syncthreads();
    if (live) a.edge[(p + FORWARD) * each + i] = s_own[threadIdx.x % JOINED][k];
    __syncthreads();
  }
}

// ---------------------------------------------------------------- backward
// What a span hands to the one above it when it is handed zero: a_n g_n of its first token.
template <typename T, int L, int S> struct Edges {
  static constexpr int CH = THREADS / L, TT = tile<T, L>(), N = L * S;
  alignas(16) T C[2][TT][N];
  typename StepOf<T>::type step[TT][CH];        // dt and v
};
template <typename T, int L, int S>
__global__ void __launch_bounds__(THREADS, 4)
backward_edges_kernel(const Args<T> a) {
  chain_begin();
  constexpr int CH = THREADS / L, TT = tile<T, L>(), N = L * S, P = S / 2;
  extern __shared__ __align__(16) unsigned char raw[];
  Edges<T, L, S>& m = *reinterpret_cast<Edges<T, L, S>*>(raw);
  const Place<T, L, S> me(a);
  const int p = blockIdx.y, at = spot<T>(me.ch);
  const Span<T> span(a, p);
  const int64_t begin = span.begin;
  int64_t finish = span.finish;
  Two<T> A[P], e[P];
  T sum = 0, w[S];
  me.load(a, a.A, w);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    A[j] = {rate(w[2 * j]), rate(w[2 * j + 1])};
    e[j] = {(T)0, (T)0};
  }
  int passes = 0;
  if (begin < finish && p > 0 && a.rows.start(a.rows.at(begin)) < begin) {
    const int64_t end = a.rows.end(a.rows.at(begin));       // what comes behind this sequence does not reach the span's start
    passes = end > finish;
    if (end < finish) finish = end;
    const Cells<T, CH, TT> mine(me.channels, a.wide);
    constexpr int E = Cells<T, CH, TT>::E, V = Cells<T, CH, TT>::V, ROWS = Cells<T, CH, TT>::ROWS;
    T d[E][V], v[E][V], z[E][V], bias[V];
    mine.per_channel(a.bias ? a.bias + me.c0 : nullptr, bias);
    const int64_t top = (finish - 1) / TT * TT, bottom = begin / TT * TT;
    const T* pd = a.delta + me.c0 + mine.first(a.ld_delta, top);
    const T* pv = a.dy + me.c0 + mine.first(a.ld_dy, top);
    const T* pz = a.z ? a.z + me.c0 + mine.first(a.ld_z, top) : nullptr;
    Rows<T, N, TT> C_rows(a.C, a.ld_C, me.q * a.state, a.state, a.wide_C, top);
    const auto fetch = [&](int64_t tile0) {      // of the tiles in turn, from the last one
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
      mine.load(pd, a.ld_delta, from, to, d);
      mine.load(pv, a.ld_dy, from, to, v);
      pd -= TT * a.ld_delta;
      pv -= TT * a.ld_dy;
      if (a.z) {
        mine.load(pz, a.ld_z, from, to, z);
        pz -= TT * a.ld_z;
      }
      C_rows.fetch(m.C[tile0 / TT & 1], from, to);
      C_rows.at -= TT * a.ld_C;
    };
    fetch(top);
    commit();
    for (int64_t tile0 = top; tile0 >= bottom; tile0 -= TT) {
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
#pragma unroll
      for (int e0 = 0; e0 < E; ++e0) {
        const int r = mine.row + e0 * ROWS;
        T dt[V];
        time_steps(d[e0], bias, a.softplus, r >= from && r < to, dt);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (mine.in(e0)) write(&m.step[r][spot<T>(mine.col, j)], dt[j], a.z ? v[e0][j] * swish(z[e0][j]) : v[e0][j]);
        }
      }
      if (tile0 > bottom) fetch(tile0 - TT);
      commit();
      landed<1>();
      __syncthreads();
      const T(*rows)[N] = m.C[tile0 / TT & 1];
      // (16384 tokens of 1024 channels with 16 states, backward: doubles 2338 us one by one and 2519 four by four, floats 560 and 542)
      constexpr int AT_ONCE = sizeof(T) == 8 ? 1 : 4;
#pragma unroll AT_ONCE
      for (int t = TT - 1; t >= 0; --t) {
        Two<T> dt, v2, C[P];
        read(&m.step[t][at], dt, v2);
        read(&rows[t][me.n0], C);
        T one, two;
        dt.get(one, two);
        sum += one;
#pragma unroll
        for (int j = 0; j < P; ++j) e[j] = mul(decay(dt, A[j]), fma(C[j], v2, e[j]));
      }
      __syncthreads();
    }
    landed<0>();
  }
#pragma unroll
  for (int j = 0; j < P; ++j) e[j].get(w[2 * j], w[2 * j + 1]);
  me.store(a, a.edge + (int64_t)p * a.dim * a.state, w);
  if (me.on && me.lane == 0) a.sum[(int64_t)p * a.dim + me.c0 + me.ch] = sum;
  if (threadIdx.x == 0 && blockIdx.x == 0) a.passes[p] = passes;
}

// Values of 2 S sums a lane (dB, then dC of its states) over the warp's 32 / L lanes that hold the same states of other channels.  As
// in sum4, half of the values change hands in each step until one is left; returns how many are left and which they are.
template <int L, int S, typename T> __device__ __forceinline__ void channel_sums(T (&v)[2 * S], int warp_lane, int& first, int& count) {
  first = 0;
  count = 2 * S;
#pragma unroll
  for (int i = 0; i < 5 - Lanes<L>::STATE_BITS; ++i) {
    const int o = 1 << Lanes<L>::channel_bit(i);
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

// The main pass: a tile's states again from its checkpoint, forwards, into shared memory, then the tile backwards.  A thread has its
// states of CC channels: what is summed over the channels (dB, dC) is added up within the thread first, and the exchange between
// the lanes, a quarter of the instructions, is paid once for both.
template <typename T, int L, int S> struct Backward {
  static constexpr int CC = sizeof(T) == 8 && L < 32 ? 1 : 2, HALF = THREADS / L, CH = CC * HALF, TT = POINT, N = L * S, P = S / 2;
  static constexpr int WARPS = THREADS / 32;
  // In double the decays are kept for the way back beside the states: an exponential takes as long there as all else of a token's
  // state, and shared memory has room for them, as registers leave two CTAs to an SM either way.
  static constexpr bool KEEP = sizeof(T) == 8;
  // tokens whose dB and dC are gathered at a time
  static constexpr int FT = 8 * 16 / N < 2 ? 2 : 8 * 16 / N < 8 ? 8 * 16 / N : 8;
  struct alignas(16) Step { T dt, gB, x, gA; };                       // in float first {dt, dt, x, x}
  struct Shared {
    Pack<T, S> h[CC][TT + 1][THREADS];                                // the state in front of each token, and behind the last
    Pack<T, S> a[KEEP ? CC : 1][KEEP ? TT : 1][KEEP ? THREADS : 1];   // the decays, where they are kept
    alignas(16) T B[2][TT][N], C[2][TT][N];
    Step step[TT][CH];
    alignas(16) T red[WARPS][FT][2 * N];
    alignas(16) T v[TT][CH], u[TT][CH], slope[TT][CH], w[TT][CH];      // slope: d dt / d delta, w: dz / r
    alignas(16) T r[TT][CH + 32 / sizeof(T)];
    int begins[TT];                                                   // the sequence that begins at a token
  };
};
__device__ __forceinline__ void read_step(const float* m, Two<float>& dt, Two<float>& x) {
  const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(m);
  dt.v = q.x;
  x.v = q.y;
}
__device__ __forceinline__ void read_step(const double* m, Two<double>& dt, Two<double>& x) {
  dt = {m[0], m[0]};
  x = {m[2], m[2]};
}

template <typename T, int L, int S>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 3 : 2)
backward_kernel(const Args<T> a) {
  chain_begin();
  using K = Backward<T, L, S>;
  constexpr int CC = K::CC, HALF = K::HALF, CH = K::CH, TT = K::TT, N = K::N, P = K::P, FT = K::FT;
  extern __shared__ __align__(16) unsigned char raw[];
  typename K::Shared& m = *reinterpret_cast<typename K::Shared*>(raw);
  // channels of the CTA: CH of a group; of a thread: ch[0], ch[0] + HALF
  const int q = blockIdx.x / a.blocks, chan0 = (a.block0 + (int)(blockIdx.x % a.blocks)) * CH, c0 = q * a.per + chan0;
  const int channels = a.per - chan0 < CH ? a.per - chan0 : CH;
  const int wl = threadIdx.x & 31, warp = threadIdx.x >> 5, lane = Lanes<L>::state(wl), n0 = lane * S;
  const int ch0 = warp * (32 / L) + Lanes<L>::channel(wl);
  int at0[CC];                                  // of this thread's entries of `step`
#pragma unroll
  for (int k = 0; k < CC; ++k) at0[k] = spot<T>(ch0 + k * HALF);
  const int64_t states = (int64_t)a.dim * a.state;
  const int p = blockIdx.y;
  const Span<T> span(a, p);
  const int64_t begin = span.begin, finish = span.finish;
  const auto load = [&](const T* from, int k, Two<T>(&h)[P]) {       // null: zero
    const int ch = ch0 + k * HALF;
    T w[S];
#pragma unroll
    for (int j = 0; j < S; ++j) w[j] = from && ch < channels && n0 + j < a.state ? from[(int64_t)(c0 + ch) * a.state + n0 + j] : (T)0;
#pragma unroll
    for (int j = 0; j < P; ++j) h[j] = {w[2 * j], w[2 * j + 1]};
  };
  const auto store = [&](T* to, int k, const Two<T>(&h)[P]) {
    const int ch = ch0 + k * HALF;
    T w[S];
#pragma unroll
    for (int j = 0; j < P; ++j) h[j].get(w[2 * j], w[2 * j + 1]);
    write_states<S>(to, c0 + ch, n0, ch < channels, a, w);
  };
  Two<T> A[CC][P], e[CC][P], dA[CC][P];
#pragma unroll
  for (int k = 0; k < CC; ++k) {
    load(a.A, k, A[k]);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      T x, y;
      A[k][j].get(x, y);
      A[k][j] = {rate(x), rate(y)};
      e[k][j] = dA[k][j] = {(T)0, (T)0};
    }
  }
  const Cells<T, CH, TT> mine(channels, a.wide);
  constexpr int E = Cells<T, CH, TT>::E, V = Cells<T, CH, TT>::V, ROWS = Cells<T, CH, TT>::ROWS;
  T bias[V], D[V], dD[V], dbias[V];
  mine.per_channel(a.bias ? a.bias + c0 : nullptr, bias);
  mine.per_channel(a.D ? a.D + c0 : nullptr, D);
#pragma unroll
  for (int j = 0; j < V; ++j) dD[j] = dbias[j] = 0;
  if (begin < finish) {
    if (p + 1 < a.spans && a.rows.end(a.rows.at(finish - 1)) > finish)
#pragma unroll
      for (int k = 0; k < CC; ++k) load(a.edge + p * states, k, e[k]);
    const int64_t top = (finish - 1) / TT * TT, bottom = begin / TT * TT;
    T u[E][V], d[E][V], z[E][V], dy[E][V];
    Two<T> next[CC][P];                         // the checkpoint of the tile that is fetched
    const T* pu = a.u + c0 + mine.first(a.ld_u, top);
    const T* pd = a.delta + c0 + mine.first(a.ld_delta, top);
    const T* pv = a.dy + c0 + mine.first(a.ld_dy, top);
    const T* pz = a.z ? a.z + c0 + mine.first(a.ld_z, top) : nullptr;
    T* to_u = a.du + c0 + mine.first(a.ld_du, top);
    T* to_d = a.ddelta + c0 + mine.first(a.ld_ddelta, top);
    T* to_z = a.z ? a.dz + c0 + mine.first(a.ld_dz, top) : nullptr;
    Rows<T, N, TT> B_rows(a.B, a.ld_B, q * a.state, a.state, a.wide_B, top);
    Rows<T, N, TT> C_rows(a.C, a.ld_C, q * a.state, a.state, a.wide_C, top);
    const T* point = a.saved + top / TT * states + (int64_t)(c0 + ch0) * a.state + n0;      // the checkpoint of the tile to fetch
    const bool even = a.state % S == 0;         // then a thread has S states or none
    const auto fetch = [&](int64_t tile0) {      // of the tiles in turn, from the last one
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
      mine.load(pu, a.ld_u, from, to, u);
      mine.load(pd, a.ld_delta, from, to, d);
      mine.load(pv, a.ld_dy, from, to, dy);
      pu -= TT * a.ld_u;
      pd -= TT * a.ld_delta;
      pv -= TT * a.ld_dy;
      if (a.z) {
        mine.load(pz, a.ld_z, from, to, z);
        pz -= TT * a.ld_z;
      }
      B_rows.fetch(m.B[tile0 / TT & 1], from, to);
      C_rows.fetch(m.C[tile0 / TT & 1], from, to);
      B_rows.at -= TT * a.ld_B;
      C_rows.at -= TT * a.ld_C;
#pragma unroll
      for (int k = 0; k < CC; ++k) {
        if (even && from == 0) {      // (value by value: reads of 16 bytes took 590 us for 540, as their zeros wait for what they load into)
          const bool on = ch0 + k * HALF < channels && n0 < a.state;
          const T* at = point + k * HALF * a.state;
          T w[S];
#pragma unroll
          for (int j = 0; j < S; ++j) w[j] = on ? at[j] : (T)0;
#pragma unroll
          for (int j = 0; j < P; ++j) next[k][j] = {w[2 * j], w[2 * j + 1]};
        } else {
          load(from == 0 ? a.saved + tile0 / TT * states : nullptr, k, next[k]);
        }
      }
      point -= states;
    };
    int s = a.rows.at(finish - 1);              // the sequence of the last token of the tile, and its first token
    int64_t start = a.rows.start(s);
    fetch(top);
    commit();
    for (int64_t tile0 = top; tile0 >= bottom; tile0 -= TT) {
      const int buf = (int)(tile0 / TT & 1);
      const int from = begin > tile0 ? (int)(begin - tile0) : 0, to = finish < tile0 + TT ? (int)(finish - tile0) : TT;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int r = mine.row + i * ROWS;
        const bool live = r >= from && r < to;
        T v[V], slope[V], w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {          // (in pairs, as time_steps has them, the kernel took 450 us for 446)
          const T x = d[i][j] + bias[j];
          T dt = x;
          slope[j] = 1;
          if (a.softplus) dt = softplus(x, slope[j]);
          if (!live) dt = 0;
          v[j] = dy[i][j];
          w[j] = 0;
          if (a.z) {
            const T g = seq::sigmoid(z[i][j]);
            w[j] = v[j] * (g * ((T)1 + z[i][j] * ((T)1 - g)));
            v[j] *= z[i][j] * g;
          }
          const typename K::Step st = {dt, dt, dt * u[i][j], dt * u[i][j]};
          if (mine.in(i)) m.step[r][spot<T>(mine.col, j)] = st;
        }
        if (mine.in(i)) {
          put(&m.v[r][mine.col], v);
          put(&m.u[r][mine.col], u[i]);
          put(&m.slope[r][mine.col], slope);
          put(&m.w[r][mine.col], w);
        }
      }
      Two<T> h[CC][P];
#pragma unroll
      for (int k = 0; k < CC; ++k) {
        Pack<T, S> w;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          h[k][j] = next[k][j];
          h[k][j].get(w.v[2 * j], w.v[2 * j + 1]);
        }
        m.h[k][0][threadIdx.x] = w;
      }
      if (tile0 > bottom) fetch(tile0 - TT);
      commit();
      // the tokens that begin sequences
      uint32_t starts = 0;
      while (start >= tile0 + from) {
        if (start < tile0 + to) {
          const uint32_t bit = 1u << (int)(start - tile0);
          if (threadIdx.x == 0 && !(starts & bit)) m.begins[start - tile0] = s;      // (those before it there have no token)
          starts |= bit;
        }
        if (s == 0) {
          start = -1;
          break;
        }
        start = a.rows.start(--s);
      }
      landed<1>();
      __syncthreads();
      const T(*rows_B)[N] = m.B[buf];
      const T(*rows_C)[N] = m.C[buf];
      const auto initial = [&](int t) { return a.h0 ? a.h0 + m.begins[t] * states : nullptr; };
#pragma unroll 1
      for (int t0 = 0; t0 < TT; t0 += 4) {
        T part[CC][4];
        const auto token = [&](int t, T(&sums)[CC]) {
          Two<T> B[P], C[P];
          read(&rows_B[t][n0], B);
          read(&rows_C[t][n0], C);
#pragma unroll
          for (int k = 0; k < CC; ++k) {
            Two<T> dt, x, r;
            read_step(&m.step[t][at0[k]].dt, dt, x);
            Pack<T, S> now, decays;
#pragma unroll
            for (int j = 0; j < P; ++j) {
              const Two<T> d = decay(dt, A[k][j]);
              if constexpr (K::KEEP) d.get(decays.v[2 * j], decays.v[2 * j + 1]);
              h[k][j] = fma(d, h[k][j], mul(x, B[j]));
              h[k][j].get(now.v[2 * j], now.v[2 * j + 1]);
              r = j ? fma(C[j], h[k][j], r) : mul(C[j], h[k][j]);
            }
            m.h[k][t + 1][threadIdx.x] = now;
            if constexpr (K::KEEP) m.a[k][t][threadIdx.x] = decays;
            sums[k] = total(r);
          }
        };
        if ((starts >> t0 & 15) == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            T sums[CC];
            token(t0 + i, sums);
#pragma unroll
            for (int k = 0; k < CC; ++k) part[k][i] = sums[k];
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            if (starts >> (t0 + i) & 1)
#pragma unroll
              for (int k = 0; k < CC; ++k) load(initial(t0 + i), k, h[k]);
            T sums[CC];
            token(t0 + i, sums);
#pragma unroll
            for (int k = 0; k < CC; ++k)
#pragma unroll
              for (int j = 0; j < 4; ++j) part[k][j] = i == j ? sums[k] : part[k][j];
          }
        }
#pragma unroll
        for (int k = 0; k < CC; ++k) {
          const T r = sum4<L>(part[k], lane);
          if (lane < 4) m.r[t0 + lane][ch0 + k * HALF] = r;
        }
      }
      // backwards
      Two<T> tile_dA[CC][P], now[CC][P];        // now: the state behind the token that is looked at
#pragma unroll
      for (int k = 0; k < CC; ++k)
#pragma unroll
        for (int j = 0; j < P; ++j) {
          tile_dA[k][j] = {(T)0, (T)0};
          now[k][j] = h[k][j];
        }
      for (int f = TT - FT; f >= 0; f -= FT) {
#pragma unroll 2
        for (int t0 = f + FT - 2; t0 >= f; t0 -= 2) {
          T two[CC][4];
          // one token: its gradients from the state in front of it
          const auto token = [&](int t, const Two<T>(&behind)[CC][P], const Two<T>(&before)[CC][P], T(&sums)[CC][2]) {
            Two<T> B[P], C[P], dB[P], dC[P];
            read(&rows_B[t][n0], B);
            read(&rows_C[t][n0], C);
#pragma unroll
            for (int k = 0; k < CC; ++k) {
              Two<T> dt, x, gB, gA;
              read_step(&m.step[t][at0[k]].dt, dt, x);
              const T v1 = m.v[t][ch0 + k * HALF];
              const Two<T> v = {v1, v1};
              Two<T> decays[P];
              if constexpr (K::KEEP) read(m.a[k][t][threadIdx.x].v, decays);
#pragma unroll
              for (int j = 0; j < P; ++j) {
                const Two<T> g = fma(C[j], v, e[k][j]);
                if constexpr (K::KEEP) e[k][j] = mul(decays[j], g);
                else e[k][j] = mul(decay(dt, A[k][j]), g);
                const Two<T> w = mul(e[k][j], before[k][j]);
                gB = j ? fma(g, B[j], gB) : mul(g, B[j]);
                gA = j ? fma(w, A[k][j], gA) : mul(w, A[k][j]);
                tile_dA[k][j] = fma(w, dt, tile_dA[k][j]);
                dB[j] = k ? fma(g, x, dB[j]) : mul(g, x);
                dC[j] = k ? fma(behind[k][j], v, dC[j]) : mul(behind[k][j], v);
              }
              sums[k][0] = total(gB);
              sums[k][1] = total(gA);
            }
            T rows[2 * S];
#pragma unroll
            for (int j = 0; j < P; ++j) {
              dB[j].get(rows[2 * j], rows[2 * j + 1]);
              dC[j].get(rows[S + 2 * j], rows[S + 2 * j + 1]);
            }
            int at, left;
            channel_sums<L, S>(rows, wl, at, left);
            // value x of the 2 S: dB (x < S) or dC of state n0 + x mod S
            T* const to = &m.red[warp][t - f][n0 + (at < S ? at : N + at - S)];
#pragma unroll
            for (int j = 0; j < 2 * S; ++j)
              if (j < left) to[left > S && j >= S ? N + j - S : j] = rows[j];      // (lanes with the same sum write the same value)
          };
          const auto in_front = [&](int t, Two<T>(&to)[CC][P]) {
#pragma unroll
            for (int k = 0; k < CC; ++k) read(m.h[k][t][threadIdx.x].v, to[k]);
          };
          Two<T> one[CC][P], zero[CC][P];
          in_front(t0 + 1, one);
          in_front(t0, zero);
          if ((starts >> t0 & 3) == 0) {
            T sums[2][CC][2];
            token(t0 + 1, now, one, sums[1]);
            token(t0, one, zero, sums[0]);
#pragma unroll
            for (int k = 0; k < CC; ++k)
#pragma unroll
              for (int j = 0; j < 4; ++j) two[k][j] = sums[j / 2][k][j % 2];
          } else {
#pragma unroll
            for (int k = 0; k < CC; ++k)
#pragma unroll
              for (int j = 0; j < 4; ++j) two[k][j] = 0;
#pragma unroll 1
            for (int i = 1; i >= 0; --i) {
              const bool begins = starts >> (t0 + i) & 1;
              Two<T> before[CC][P];
              T sums[CC][2];
#pragma unroll
              for (int k = 0; k < CC; ++k) {
#pragma unroll
                for (int j = 0; j < P; ++j) before[k][j] = i ? one[k][j] : zero[k][j];
                if (begins) load(initial(t0 + i), k, before[k]);
              }
              token(t0 + i, now, before, sums);
#pragma unroll
              for (int k = 0; k < CC; ++k) {
#pragma unroll
                for (int j = 0; j < 4; ++j) two[k][j] = j / 2 == i ? sums[k][j % 2] : two[k][j];
                if (begins && a.dh0) store(a.dh0 + m.begins[t0 + i] * states, k, e[k]);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                  if (begins) e[k][j] = {(T)0, (T)0};
                  now[k][j] = one[k][j];
                }
              }
            }
          }
#pragma unroll
          for (int k = 0; k < CC; ++k)
#pragma unroll
            for (int j = 0; j < P; ++j) now[k][j] = zero[k][j];
          // over the second dt and dt u, which the channel's lanes have read
          __syncwarp();
#pragma unroll
          for (int k = 0; k < CC; ++k) {
            const T r = sum4<L>(two[k], lane);
            if (lane < 4) {
              typename K::Step& st = m.step[t0 + (lane >> 1)][at0[k]];
              (lane & 1 ? st.gA : st.gB) = r;
            }
          }
        }
        __syncthreads();
        // the warps' sums, in the order of the warps
        constexpr int WIDE = 16 / sizeof(T), FOURS = 2 * N / WIDE;
        if (a.part_BC && a.state == N) {     // whole rows of the partial sums, 16 bytes at a time
          T* to0 = a.part_BC + ((blockIdx.x % a.blocks * a.rows.tokens + tile0 + f) * a.groups + q) * 2 * N;
          for (int i = threadIdx.x; i < FT * FOURS; i += THREADS) {
            const int t = i / FOURS, n = i % FOURS * WIDE;
            if (f + t >= from && f + t < to) {
              T sum[WIDE], next_sum[WIDE];
              pick(&m.red[0][t][n], sum);
#pragma unroll
              for (int w = 1; w < K::WARPS; ++w) {
                pick(&m.red[w][t][n], next_sum);
#pragma unroll
                for (int j = 0; j < WIDE; ++j) sum[j] += next_sum[j];
              }
              put(to0 + (int64_t)t * a.groups * 2 * N + n, sum);
            }
          }
        } else {
          constexpr int ACROSS = 2 * N < THREADS ? 2 * N : THREADS;
          for (int n = threadIdx.x % ACROSS; n < 2 * N; n += ACROSS) {
            const int state = n < N ? n : n - N;
            if (state >= a.state) continue;
            T* to0 = n < N ? a.dB + q * a.state + state : a.dC + q * a.state + state;
            int64_t ld = n < N ? a.ld_dB : a.ld_dC;
            if (a.part_BC) {
              to0 = a.part_BC + ((int64_t)(blockIdx.x % a.blocks) * a.rows.tokens * a.groups + q) * 2 * a.state + (n < N ? 0 : a.state) + state;
              ld = (int64_t)a.groups * 2 * a.state;
            }
            to0 += (tile0 + f) * ld;
#pragma unroll
            for (int t = threadIdx.x / ACROSS; t < FT; t += THREADS / ACROSS)
              if (f + t >= from && f + t < to) {
                T sum = 0;
#pragma unroll
                for (int w = 0; w < K::WARPS; ++w) sum += m.red[w][t][n];
                to0[t * ld] = sum;
              }
          }
        }
        if (f > 0) __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < CC; ++k)
#pragma unroll
        for (int j = 0; j < P; ++j) dA[k][j] = fma(tile_dA[k][j], Two<T>((T)1, (T)1), dA[k][j]);
      T du[E][V], dd[E][V], dz[E][V];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!mine.in(i)) break;
        const int r = mine.row + i * ROWS;
        const bool live = r >= from && r < to;
        T ut[V], v[V], slope[V], w[V], rt[V];
        pick(&m.u[r][mine.col], ut);
        pick(&m.v[r][mine.col], v);
        pick(&m.slope[r][mine.col], slope);
        pick(&m.w[r][mine.col], w);
        pick(&m.r[r][mine.col], rt);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const typename K::Step st = m.step[r][spot<T>(mine.col, j)];
          du[i][j] = st.dt * st.gB + D[j] * v[j];
          dd[i][j] = (ut[j] * st.gB + per_rate<T>() * st.gA) * slope[j];
          dz[i][j] = w[j] * (rt[j] + D[j] * ut[j]);
          if (live) {
            dD[j] += v[j] * ut[j];
            dbias[j] += dd[i][j];
          }
        }
      }
      mine.store(to_u, a.ld_du, from, to, du);
      mine.store(to_d, a.ld_ddelta, from, to, dd);
      to_u -= TT * a.ld_du;
      to_d -= TT * a.ld_ddelta;
      if (a.z) {
        mine.store(to_z, a.ld_dz, from, to, dz);
        to_z -= TT * a.ld_dz;
      }
      // (no barrier: a thread alone reads and writes its cells of the tile, here and where the next tile's go in)
    }
    landed<0>();
  }
#pragma unroll
  for (int k = 0; k < CC; ++k) store(a.part_A + p * states, k, dA[k]);
  // the threads of a channel, in their order
  __syncthreads();
  T(*const sums)[2][CH] = reinterpret_cast<T(*)[2][CH]>(m.h);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    sums[mine.row][0][mine.col + j] = dD[j];
    sums[mine.row][1][mine.col + j] = dbias[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * CH; i += THREADS) {
    const int c = i % CH;
    T sum = 0;
#pragma unroll
    for (int k = 0; k < (ROWS < TT ? ROWS : TT); ++k) sum += sums[k][i / CH][c];
    if (c < channels) (i < CH ? a.part_D : a.part_bias)[(int64_t)p * a.dim + c0 + c] = sum;
  }
}

// Value i of dA, then of dD and of dbias: the sum of the spans, in double.
template <typename T> __device__ __forceinline__ void span_total(const Args<T>& a, int64_t i) {
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
// Pack i of V values of dB and dC: the sum of the CTAs of a group, added to that of the launches before this one.
template <typename T, int V> __device__ __forceinline__ void row_total(const Args<T>& a, int64_t i) {
  const int64_t lo = a.rows.begin(), hi = a.rows.finish(), each = (int64_t)a.groups * 2 * a.state;
  i = lo * each + i * V;
  if (i >= hi * each) return;
  const int64_t row = i / each, stride = a.rows.tokens * each;
  const int at = (int)(i % each), q = at / (2 * a.state), n = at % (2 * a.state);
  T sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0;
#pragma unroll 8
  for (int b = 0; b < a.blocks; ++b) {
    const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(a.part_BC + b * stride + i);
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] += w.v[j];
  }
  T* to = n < a.state ? a.dB + row * a.ld_dB + q * a.state + n : a.dC + row * a.ld_dC + q * a.state + n - a.state;
#pragma unroll
  for (int j = 0; j < V; ++j) to[j] = a.block0 ? to[j] + sum[j] : sum[j];
}
// the CTAs below `span_blocks` take the spans' sums, the others the rows', 16 bytes at a time where states come in such packs
template <typename T>
__global__ void __launch_bounds__(THREADS)
totals_kernel(const Args<T> a, int span_blocks) {
  chain_begin();
  constexpr int V = 16 / sizeof(T);
  if ((int)blockIdx.x < span_blocks) span_total(a, (int64_t)blockIdx.x * THREADS + threadIdx.x);
  else if (a.state % V == 0) row_total<T, V>(a, (int64_t)(blockIdx.x - span_blocks) * THREADS + threadIdx.x);
  else row_total<T, 1>(a, (int64_t)(blockIdx.x - span_blocks) * THREADS + threadIdx.x);
}

// ---------------------------------------------------------------- one token
// One new token for each row of a batch; h_last may be h0.  A thread takes R rows, whose states are all on their way at a time.
template <typename T, int L, int S, int R>
__global__ void __launch_bounds__(THREADS)
step_kernel(const Args<T> a) {
  chain_begin();
  const Place<T, L, S> me(a);
  const int c = me.c0 + me.ch;
  const int64_t row0 = (int64_t)blockIdx.y * R, states = (int64_t)a.dim * a.state;
  T A[S], h[R][S], B[R][S], C[R][S], u[R], dt[R], z[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int64_t row = row0 + k;
    const bool on = me.on && row < a.rows.tokens;
    read_states<S>(a.h0 + row * states, c, me.n0, on, a, h[k]);
    u[k] = on ? a.u[row * a.ld_u + c] : (T)0;
    dt[k] = on ? a.delta[row * a.ld_delta + c] : (T)0;
    z[k] = on && a.z ? a.z[row * a.ld_z + c] : (T)0;
    const T *b = a.B + row * a.ld_B + me.q * a.state + me.n0, *g = a.C + row * a.ld_C + me.q * a.state + me.n0;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const bool live = on && me.n0 + j < a.state;
      B[k][j] = live ? b[j] : (T)0;
      C[k][j] = live ? g[j] : (T)0;
    }
  }
  me.load(a, a.A, A);
  const T bias = a.bias && me.on ? a.bias[c] : (T)0, D = a.D && me.on ? a.D[c] : (T)0;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int64_t row = row0 + k;
    const bool on = me.on && row < a.rows.tokens;
    dt[k] += bias;
    if (a.softplus) dt[k] = softplus(dt[k]);
    const T x = dt[k] * u[k];
    T sum = 0;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      h[k][j] = decay(dt[k], rate(A[j])) * h[k][j] + x * B[k][j];
      sum += C[k][j] * h[k][j];
    }
    write_states<S>(a.h_last + row * states, c, me.n0, on, a, h[k]);
#pragma unroll
    for (int i = 0; i < Lanes<L>::STATE_BITS; ++i) sum += __shfl_xor_sync(0xffffffffu, sum, 1 << Lanes<L>::state_bit(i));
    if (on && me.lane == 0) {
      sum += D * u[k];
      if (a.z) sum *= swish(z[k]);
      a.y[row * a.ld_y + c] = sum;
    }
  }
}

// ---------------------------------------------------------------- launches
enum class Pass { Forward, Backward, Step };

// How the token axis is cut: by sequences where they are of equal length and fill at least half of the device (the edges' pass is
// about half of the work again), else into spans of whole tiles, as many as the device holds at a time: one CTA more takes as long
// as twice as many.  Each span costs a CTA's beginning and end and leaves sums of its own, dim x state values, which is more than
// short sequences bring: where there are many of those, a span has as many as give every place of the device two CTAs (backward,
// 1024 floats with 16 states: 16384 sequences of one token 772 us, 791 with one CTA a place, 813 with eight and 6190 with a span
// each; 1024 of 16 tokens 471, 472, 492 and 596 us).
template <typename T> static void cut(Args<T>& a, int64_t across, int64_t full) {
  constexpr int unit = span_unit<T>();
  const int64_t count = a.rows.count, each = a.rows.each;
  const auto at_most = [&](int64_t spans) { return spans < 1 ? 1 : spans > 65535 ? 65535 : spans; };
  const bool brief = each <= 2 * unit;
  if (!a.rows.offsets && each > 0 && (brief || (count <= 65535 && count * across >= full / 2))) {
    const int64_t together = brief && count * across > 8 * full ? ceil_div(count, at_most(2 * full / across)) : 1;
    a.span = together * each;
    a.spans = (int)ceil_div(count, together);
    return;
  }
  int64_t span = ceil_div(ceil_div(a.rows.tokens, at_most(full / across)), unit) * unit;
  if (span < 2 * unit) span = 2 * unit;
  a.span = span;
  a.spans = (int)ceil_div(a.rows.tokens, span);
  if (a.spans < 1) a.spans = 1;
}
// whether a span may begin inside a sequence
template <typename T> static bool joined(const Args<T>& a) { return a.spans > 1 && (a.rows.offsets || a.span % a.rows.each != 0); }

struct Carve {
  char* at;
  size_t used = 0;
  template <typename U> U* take(int64_t n) {
    U* p = at ? (U*)(at + used) : nullptr;
    used += ((size_t)n * sizeof(U) + 255) & ~(size_t)255;
    return p;
  }
};
// `rows`: CTAs whose sums of dB and dC there is room for
template <typename T> static size_t carve(Args<T>& a, bool backward, int rows, void* ws) {
  Carve c{(char*)ws};
  const int64_t states = (int64_t)a.dim * a.state;
  if (joined(a)) {
    a.edge = c.take<T>((a.spans + 1) * states);
    a.sum = c.take<T>((int64_t)a.spans * a.dim);
    a.passes = c.take<int>(a.spans);
  }
  if (backward) {
    a.part_A = c.take<T>(a.spans * states);
    a.part_D = c.take<T>((int64_t)a.spans * a.dim);
    a.part_bias = c.take<T>((int64_t)a.spans * a.dim);
    if (rows) a.part_BC = c.take<T>((int64_t)rows * a.rows.tokens * a.groups * 2 * a.state);
  }
  return c.used;
}

constexpr int64_t ROWS_ROOM = 256 << 20;
// FL lanes of FS states a channel in the forward passes, L of S backward and for single tokens
template <typename T, int L, int S, int FL, int FS> static prad_status launch(prad_ctx* ctx, Args<T> a, Pass pass) {
  using Main = Backward<T, L, S>;
  const bool backward = pass == Pass::Backward;
  // the edges' pass has THREADS / L channels a CTA, the main backward pass CC times as many
  const int edge_blocks = (int)ceil_div(a.per, THREADS / L);
  a.blocks = backward ? (int)ceil_div(a.per, Main::CH) : pass == Pass::Forward ? (int)ceil_div(a.per, THREADS / FL) : edge_blocks;
  // Backward each of a group's CTAs leaves sums of dB and dC over its channels, Main::CH, for the last launch to add up: 2 state / CH
  // token matrices in all, half a one with 16 float states and 32 with 128, where CH is 8.  Beyond 256 MB and beyond one token matrix
  // the group's CTAs come in several launches, whose sums go to the same place, on spans that fill the device again (16384 tokens with
  // 128 states: 2048 floats 15.5 ms with 0.4 GB of scratch, 16.6 ms with 5.4 GB in one launch; 1024 doubles 27.8 and 26.5 ms).
  const int all_blocks = a.blocks;
  if (backward) {
    const int64_t each = a.rows.tokens * a.groups * 2 * a.state * (int64_t)sizeof(T), matrix = a.rows.tokens * a.dim * (int64_t)sizeof(T);
    const int64_t most = (matrix > ROWS_ROOM ? matrix : ROWS_ROOM) / each;
    if (most < a.blocks) a.blocks = (int)ceil_div(a.blocks, ceil_div(a.blocks, most < 1 ? 1 : most));
  }
  const int rows = backward && all_blocks > 1 ? a.blocks : 0;
  const int64_t across = (int64_t)a.groups * a.blocks;
  PRAD_REQUIRE(across <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "selective scan: too many channels");
  if (pass == Pass::Step) {
    // four rows a thread where that still gives every SM eight CTAs
    const int R = sizeof(T) == 4 && a.rows.tokens * across >= (int64_t)ctx->sm_count * 32 ? 4 : 1;
    const int64_t most = (int64_t)65535 * R, states = (int64_t)a.dim * a.state;      // (the grid's second dimension)
    for (int64_t r0 = 0; r0 < a.rows.tokens; r0 += most) {
      Args<T> b = a;
      b.rows.tokens = a.rows.tokens - r0 < most ? a.rows.tokens - r0 : most;
      b.u += r0 * a.ld_u, b.delta += r0 * a.ld_delta, b.B += r0 * a.ld_B, b.C += r0 * a.ld_C, b.y += r0 * a.ld_y;
      if (b.z) b.z += r0 * a.ld_z;
      b.h0 += r0 * states, b.h_last += r0 * states;
      const dim3 grid((unsigned)across, (unsigned)ceil_div(b.rows.tokens, R));
      void (*kernel)(const Args<T>) = step_kernel<T, L, S, 1>;
      if constexpr (sizeof(T) == 4)
        if (R == 4) kernel = step_kernel<T, L, S, 4>;
      launch_chained(kernel, grid, THREADS, 0, ctx->stream, b);
      PRAD_LAUNCHED(ctx);
    }
    return PRAD_OK;
  }
  using Shared = typename Main::Shared;
  constexpr int bytes = (int)sizeof(Forward<T, FL, FS>);
  prad_status st = backward ? allow_smem<backward_kernel<T, L, S>>(ctx, (int)sizeof(Shared)) : allow_smem<forward_kernel<T, FL, FS, false>>(ctx, bytes);
  constexpr int edge_bytes = (int)sizeof(Edges<T, L, S>);
  if (!st) st = backward ? allow_smem<backward_edges_kernel<T, L, S>>(ctx, edge_bytes) : allow_smem<forward_kernel<T, FL, FS, true>>(ctx, bytes);
  if (st) return st;
  cut(a, across, backward ? resident<backward_kernel<T, L, S>>(ctx, THREADS, (int)sizeof(Shared)) : resident<forward_kernel<T, FL, FS, false>>(ctx, THREADS, bytes));
  st = ensure_workspace(ctx, carve(a, backward, rows, nullptr));
  if (st) return st;
  carve(a, backward, rows, ctx->ws);
  const int64_t states = (int64_t)a.dim * a.state;
  const unsigned x = (unsigned)across;
  if (!backward) {
    if (joined(a)) {
      launch_chained(forward_kernel<T, FL, FS, true>, dim3(x, (unsigned)a.spans - 1), THREADS, bytes, ctx->stream, a);
      PRAD_LAUNCHED(ctx);
      launch_chained(join_kernel<T, true>, (unsigned)ceil_div(states, JOINED), 32 * JOINED, 0, ctx->stream, a);
      PRAD_LAUNCHED(ctx);
    }
    launch_chained(forward_kernel<T, FL, FS, false>, dim3(x, (unsigned)a.spans), THREADS, bytes, ctx->stream, a);
    PRAD_LAUNCHED(ctx);
    return PRAD_OK;
  }
  // of the last launch: the spans' sums, and the rows of dB and dC in packs
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t span_blocks = ceil_div(states + 2 * (int64_t)a.dim, THREADS);
  const int64_t packs = rows ? a.rows.tokens * a.groups * 2 * a.state / (a.state % V ? 1 : V) : 0;
  PRAD_REQUIRE(span_blocks + ceil_div(packs, THREADS) <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "selective scan: too many rows of B and C");
  if (a.dh0) PRAD_CUDA(cudaMemsetAsync(a.dh0, 0, (size_t)a.rows.count * states * sizeof(T), ctx->stream));
  if (joined(a)) {
    Args<T> b = a;
    b.blocks = edge_blocks;
    launch_chained(backward_edges_kernel<T, L, S>, dim3((unsigned)(a.groups * edge_blocks), (unsigned)a.spans), THREADS, edge_bytes, ctx->stream, b);
    PRAD_LAUNCHED(ctx);
    launch_chained(join_kernel<T, false>, (unsigned)ceil_div(states, JOINED), 32 * JOINED, 0, ctx->stream, a);
    PRAD_LAUNCHED(ctx);
  }
  for (const int most = a.blocks; a.block0 < all_blocks; a.block0 += most) {
    if (a.blocks > all_blocks - a.block0) a.blocks = all_blocks - a.block0;
    const int64_t sums = a.block0 + a.blocks == all_blocks ? span_blocks : 0;
    launch_chained(backward_kernel<T, L, S>, dim3((unsigned)(a.groups * a.blocks), (unsigned)a.spans), THREADS, sizeof(Shared), ctx->stream, a);
    PRAD_LAUNCHED(ctx);
    launch_chained(totals_kernel<T>, (unsigned)(sums + ceil_div(packs, THREADS)), THREADS, 0, ctx->stream, a, (int)sums);
    PRAD_LAUNCHED(ctx);
  }
  return PRAD_OK;
}
template <typename T> static prad_status pick(prad_ctx* ctx, Args<T> a, Pass pass) {
  constexpr int V = 16 / sizeof(T);
  const uintptr_t all = (uintptr_t)a.u | (uintptr_t)a.delta | (uintptr_t)a.z | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.du |
                        (uintptr_t)a.ddelta | (uintptr_t)a.dz;
  const int64_t pitches = a.ld_u | a.ld_delta | a.ld_z | a.ld_y | a.ld_dy | a.ld_du | a.ld_ddelta | a.ld_dz;
  a.wide = (all & 15) == 0 && pitches % V == 0 && (a.groups == 1 || a.per % V == 0);
  const uintptr_t matrices = (uintptr_t)a.A | (uintptr_t)a.h0 | (uintptr_t)a.h_last | (uintptr_t)a.saved | (uintptr_t)a.dh0;
  a.wide_h = (matrices & 15) == 0 && a.state % V == 0;
  // Forward, eight states of a float channel to a lane: half of the sums over lanes and of the reads of dt that four take.
  if constexpr (sizeof(T) == 4) {
    if (a.state <= 8) return launch<T, 4, 2, 2, 4>(ctx, a, pass);
    if (a.state <= 16) return launch<T, 4, 4, 2, 8>(ctx, a, pass);
    if (a.state <= 32) return launch<T, 8, 4, 4, 8>(ctx, a, pass);
    if (a.state <= 64) return launch<T, 16, 4, 8, 8>(ctx, a, pass);
    return launch<T, 32, 4, 16, 8>(ctx, a, pass);
  } else {
    if (a.state <= 8) return launch<T, 4, 2, 4, 2>(ctx, a, pass);
    if (a.state <= 16) return launch<T, 4, 4, 4, 4>(ctx, a, pass);
    if (a.state <= 32) return launch<T, 8, 4, 8, 4>(ctx, a, pass);
    if (a.state <= 64) return launch<T, 16, 4, 16, 4>(ctx, a, pass);
    return launch<T, 32, 4, 32, 4>(ctx, a, pass);
  }
}

static prad_status check_shape(const char* who, prad_dtype dt, const prad_scan_t* s) {
  PRAD_REQUIRE(dtype_ok(dt), PRAD_ERR_INVALID, "%s: unknown dtype %d", who, (int)dt);
  PRAD_REQUIRE(s, PRAD_ERR_INVALID, "%s: null scan", who);
  PRAD_REQUIRE(s->tokens >= 0 && s->sequences >= 0 && s->dim > 0 && s->state > 0 && s->groups > 0, PRAD_ERR_SHAPE, "%s: bad shape", who);
  PRAD_REQUIRE(s->dim % s->groups == 0, PRAD_ERR_SHAPE, "%s: %d channels do not divide into %d groups", who, s->dim, s->groups);
  PRAD_REQUIRE(s->state <= MAX_STATE, PRAD_ERR_UNSUPPORTED, "%s: at most %d states, got %d", who, MAX_STATE, s->state);
  PRAD_REQUIRE(s->tokens <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", who);
  PRAD_REQUIRE(s->dim <= 1 << 20, PRAD_ERR_UNSUPPORTED, "%s: more than 2^20 channels", who);
  return PRAD_OK;
}
static prad_status check(const char* who, prad_dtype dt, const prad_scan_t* s) {
  prad_status st = check_shape(who, dt, s);
  if (st) return st;
  const int64_t rows = (int64_t)s->groups * s->state;
  PRAD_REQUIRE((!s->ld_u || s->ld_u >= s->dim) && (!s->ld_delta || s->ld_delta >= s->dim) && (!s->ld_z || s->ld_z >= s->dim) &&
                   (!s->ld_B || s->ld_B >= rows) && (!s->ld_C || s->ld_C >= rows),
               PRAD_ERR_SHAPE, "%s: a pitch below the row", who);
  PRAD_REQUIRE(s->tokens == 0 || (s->u && s->delta && s->A && s->B && s->C), PRAD_ERR_INVALID, "%s: null pointer", who);
  PRAD_REQUIRE(natural(dt, s->u, s->delta, s->z, s->A, s->B, s->C, s->D, s->delta_bias, s->h0), PRAD_ERR_INVALID, "%s: unaligned pointer", who);
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
  constexpr int V = 16 / sizeof(T);
  const auto wide = [&](const void* m, int64_t ld) { return ((uintptr_t)m & 15) == 0 && ld % V == 0 && s->state % V == 0; };
  a.ld_u = s->ld_u ? s->ld_u : s->dim, a.ld_delta = s->ld_delta ? s->ld_delta : s->dim, a.ld_z = s->ld_z ? s->ld_z : s->dim;
  a.ld_B = s->ld_B ? s->ld_B : rows, a.ld_C = s->ld_C ? s->ld_C : rows;
  a.wide_B = wide(s->B, a.ld_B), a.wide_C = wide(s->C, a.ld_C);
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
  prad_status st = ssm::check_shape("prad_selective_scan_saved_bytes", dt, scan);
  if (st) return st;
  PRAD_REQUIRE(out_bytes, PRAD_ERR_INVALID, "prad_selective_scan_saved_bytes: null output");
  *out_bytes = (size_t)ceil_div(scan->tokens, ssm::POINT) * scan->dim * scan->state * dtype_size(dt);
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
  PRAD_REQUIRE(natural(dt, y, h_last, saved), PRAD_ERR_INVALID, "%s: unaligned pointer", who);
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
  PRAD_REQUIRE(natural(dt, saved, dy, g->du, g->ddelta, g->dz, g->dA, g->dB, g->dC, g->dD, g->ddelta_bias, g->dh0), PRAD_ERR_INVALID,
               "%s: unaligned pointer", who);
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
  PRAD_REQUIRE(natural(dt, y, h_out), PRAD_ERR_INVALID, "%s: unaligned pointer", who);
  PRAD_CHECK_CTX(ctx);
  if (scan->tokens == 0) return PRAD_OK;
  return dt == PRAD_F32 ? forward_t<float>(ctx, scan, y, ld_y, h_out, nullptr, ssm::Pass::Step)
                        : forward_t<double>(ctx, scan, y, ld_y, h_out, nullptr, ssm::Pass::Step);
}
