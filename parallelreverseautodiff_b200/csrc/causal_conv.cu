// The short convolution of a state space layer: per channel c over the tokens of each sequence,
//   p_t = bias_c + sum_k w[c][k] x_(t - (W - 1) + k),  y_t = p_t or swish(p_t),
// where the W - 1 rows before a sequence's first token come from its state (zero without one).  Backward, with g = dy swish'(p):
//   dx_t = sum_k w[c][k] g_(t + W - 1 - k)  over the tokens of the sequence,  dw[c][k] = sum_t g_t x_(t - (W - 1) + k),  dbias = sum g.
//
// Bound by memory: a thread takes V neighbouring channels and walks down a run of tokens with the last W rows in registers, so that a
// row is read once per run and W - 1 rows twice.  The next rows are on their way into a ring of its own in shared memory: in
// registers, four rows ahead took the room of the warps that are to keep the memory busy (16384 tokens of 2048 floats, width 4:
// forward 62 us, and 45 us = 5.9 TB/s with the ring; backward 80 us = 5.0 TB/s, two thirds of the issue slots used).
#include <type_traits>

#include "common.cuh"
#include "packed_sequences.cuh"

namespace prad {
namespace conv {

using seq::load;
using seq::Pack;
using seq::Sequences;
using seq::swish;
using seq::swish_slope;

constexpr int LANES = 32, WARPS = 8, THREADS = LANES * WARPS;
constexpr int AHEAD = 8;         // rows on their way

template <typename T> struct Args {
  Sequences rows;
  const T *x, *w, *bias, *state, *dy;
  T *y, *dx, *state_out, *dw, *dbias, *dstate;
  int64_t ld_x, ld_y, ld_dy, ld_dx;
  int dim, swish, wide_w;        // wide_w: w can be read V values at a time
  int run;                       // tokens of a thread's run
  unsigned blocks;               // CTAs along the tokens; those behind them see to the states
};


// A thread's ring of rows: rows go in by asynchronous copies, one group of copies a row, and come out in their order.
template <typename T, int V> struct Ring {
  Pack<T, V>* at;                // of this thread's first slot; slots are THREADS packs apart
  __device__ __forceinline__ Ring(void* shared, int which) : at((Pack<T, V>*)shared + which * AHEAD * THREADS + threadIdx.x) {}
  __device__ __forceinline__ void put(int slot, const T* from) const {
    constexpr int bytes = sizeof(T) * V;
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(at + slot * THREADS);
    if constexpr (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(from), "n"(bytes) : "memory");
  }
  __device__ __forceinline__ Pack<T, V> get(int slot) const { return at[slot * THREADS]; }
};
__device__ __forceinline__ void end_of_row() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void oldest_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory"); }

// the row at place `p` of sequence s, which begins at row `start`: a token, or below zero a row of its state
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> row_at(const Args<T>& a, int s, int64_t start, int64_t p, int c) {
  Pack<T, V> r;
  if (p >= 0) return load<T, V>(a.x + (start + p) * a.ld_x + c);
  if (a.state) return load<T, V>(a.state + ((int64_t)s * (W - 1) + (W - 1) + p) * a.dim + c);
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = 0;
  return r;
}

template <typename T, int V, int W> struct Weights {
  T w[W][V], bias[V];
  __device__ __forceinline__ Weights(const Args<T>& a, int c) {
    T all[W * V];                // V rows of w, which lie one behind the other
    if (a.wide_w) {
#pragma unroll
      for (int i = 0; i < W * V; i += V) {
        const Pack<T, V> r = load<T, V>(a.w + (int64_t)c * W + i);
#pragma unroll
        for (int j = 0; j < V; ++j) all[i + j] = r.v[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < W * V; ++i) all[i] = a.w[(int64_t)c * W + i];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[k][j] = all[j * W + k];
      bias[j] = a.bias ? a.bias[c + j] : (T)0;
    }
  }
};

// state_out[s] = the last W - 1 rows of state[s] followed by the sequence's tokens
template <typename T, int V, int W>
__device__ __forceinline__ void final_states(const Args<T>& a, int64_t block) {
  const int c = (blockIdx.y * LANES + (threadIdx.x & 31)) * V;
  const int64_t i = block * WARPS + (threadIdx.x >> 5);
  if (c >= a.dim || i >= (int64_t)a.rows.count * (W - 1)) return;
  const int s = (int)(i / (W - 1)), k = (int)(i % (W - 1));
  const int64_t start = a.rows.start(s);
  int64_t len = a.rows.end(s) - start;
  if (len < 0) len = 0;
  *reinterpret_cast<Pack<T, V>*>(a.state_out + i * a.dim + c) = row_at<T, V, W>(a, s, start, len - (W - 1) + k, c);
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS)
forward_kernel(const Args<T> a) {
  chain_begin();
  if (blockIdx.x >= a.blocks) {
    if constexpr (W > 1) final_states<T, V, W>(a, blockIdx.x - a.blocks);
    return;
  }
  const int c = (blockIdx.y * LANES + (threadIdx.x & 31)) * V;
  if (c >= a.dim) return;
  const int64_t run = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int64_t lo = a.rows.begin(), hi = a.rows.finish();
  int64_t t = run * a.run, last = t + a.run;
  if (t < lo) t = lo;
  if (last > hi) last = hi;
  if (t >= last) return;
  const Weights<T, V, W> wt(a, c);
  int s = a.rows.at(t);
  int64_t start = a.rows.start(s), end = a.rows.end(s);
  if (start > t) start = t;     // (offsets that do not ascend)
  Pack<T, V> x[W];              // x[W - 1]: the newest row
#pragma unroll
  for (int k = 1; k < W; ++k) x[k] = row_at<T, V, W>(a, s, start, t - start - (W - k), c);
  extern __shared__ __align__(16) unsigned char raw[];
  const Ring<T, V> ring(raw, 0);
  const T* px = a.x + t * a.ld_x + c;
  T* py = a.y + t * a.ld_y + c;
  const int rows = (int)(last - t);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (i < rows) ring.put(i, px + i * a.ld_x);
    end_of_row();
  }
  px += AHEAD * a.ld_x;
  for (int i0 = 0;; i0 += AHEAD)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (i0 + i >= rows) return;
      if (t == end) {
        do ++s; while (s < a.rows.count && a.rows.end(s) <= t);
        if (s >= a.rows.count) return;
        start = t;
        end = a.rows.end(s);
#pragma unroll
        for (int k = 1; k < W; ++k) x[k] = row_at<T, V, W>(a, s, start, -(W - k), c);
      }
#pragma unroll
      for (int k = 0; k + 1 < W; ++k) x[k] = x[k + 1];
      oldest_landed();
      x[W - 1] = ring.get(i);
      if (i0 + i + AHEAD < rows) ring.put(i, px);
      end_of_row();
      px += a.ld_x;
      Pack<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        T p = wt.bias[j];
#pragma unroll
        for (int k = 0; k < W; ++k) p += wt.w[k][j] * x[k].v[j];
        y.v[j] = a.swish ? swish(p) : p;
      }
      *reinterpret_cast<Pack<T, V>*>(py) = y;
      py += a.ld_y;
      ++t;
    }
}

// g at place q of a sequence
template <typename T, int V, int W>
__device__ __forceinline__ void slope(const Weights<T, V, W>& wt, const Pack<T, V> (&x)[W], const Pack<T, V>& dy, int act, T (&g)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    g[j] = dy.v[j];
    if (act) {
      T p = wt.bias[j];
#pragma unroll
      for (int k = 0; k < W; ++k) p += wt.w[k][j] * x[k].v[j];
      g[j] *= swish_slope(p);
    }
  }
}

// dstate[s][i], the row at place i - (W - 1): sum over the places q <= i of the sequence of w[i - q] g_q
template <typename T, int V, int W>
__device__ __forceinline__ void state_gradients(const Args<T>& a, int64_t block) {
  const int c = (blockIdx.y * LANES + (threadIdx.x & 31)) * V;
  const int64_t s64 = block * WARPS + (threadIdx.x >> 5);
  if (c >= a.dim || s64 >= a.rows.count) return;
  const int s = (int)s64;
  const int64_t start = a.rows.start(s), len = a.rows.end(s) - start;
  const Weights<T, V, W> wt(a, c);
  T sum[W][V];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sum[i][j] = 0;
#pragma unroll
  for (int q = 0; q < W - 1; ++q)
    if (q < len) {
      Pack<T, V> x[W];
#pragma unroll
      for (int k = 0; k < W; ++k) x[k] = row_at<T, V, W>(a, s, start, q - (W - 1) + k, c);
      T g[V];
      slope<T, V, W>(wt, x, load<T, V>(a.dy + (start + q) * a.ld_dy + c), a.swish, g);
#pragma unroll
      for (int i = q; i < W - 1; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[i][j] += wt.w[i - q][j] * g[j];
    }
#pragma unroll
  for (int i = 0; i < W - 1; ++i) {
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = sum[i][j];
    *reinterpret_cast<Pack<T, V>*>(a.dstate + ((int64_t)s * (W - 1) + i) * a.dim + c) = o;
  }
}

// A thread computes g over its run and the W - 1 tokens behind it, and dx of its run from the last W of them.
// partial[block][W + 1][dim]: sums for dw (k = 0 .. W - 1) and dbias over the block's runs.
template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const Args<T> a, T* __restrict__ partial) {
  chain_begin();
  if (blockIdx.x >= a.blocks) {
    if constexpr (W > 1) state_gradients<T, V, W>(a, blockIdx.x - a.blocks);
    return;
  }
  using F = seq::Few<T, V>;
  using Unit = typename F::type;
  __shared__ T part[WARPS][LANES * V];
  extern __shared__ __align__(16) unsigned char raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.y * LANES + lane) * V;
  const bool on = c < a.dim;
  const int64_t lo = a.rows.begin(), hi = a.rows.finish();
  int64_t t = ((int64_t)blockIdx.x * WARPS + warp) * a.run, last = t + a.run;
  if (t < lo) t = lo;
  if (last > hi) last = hi;
  T zeros[V], ones[V], minuses[V];
#pragma unroll
  for (int j = 0; j < V; ++j) zeros[j] = 0, ones[j] = 1, minuses[j] = -1;
  const Unit zero = F::from(zeros), one = F::from(ones), minus = F::from(minuses);
  Unit dw[W], db = zero;
#pragma unroll
  for (int k = 0; k < W; ++k) dw[k] = zero;
  if (on && t < last) {
    Unit w[W], bias;
    {
      const Weights<T, V, W> wt(a, c);
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = F::from(wt.w[k]);
      bias = F::from(wt.bias);
    }
    const Ring<T, V> ring_x(raw, 0), ring_d(raw, 1);
    int s = a.rows.at(t);
    while (t < last && s < a.rows.count) {
      int64_t start = a.rows.start(s);
      const int64_t end = a.rows.end(s);
      if (start > t) start = t;                                // (offsets that do not ascend)
      const int64_t stop = end < last ? end : last;            // of the tokens whose dx is this thread's
      int64_t ahead = stop + W - 1;                            // of the tokens whose g they take
      if (ahead > end) ahead = end;
      Unit x[W], g[W];                                         // x[W - 1], g[W - 1]: the newest token's
#pragma unroll
      for (int k = 1; k < W; ++k) {
        const Pack<T, V> r = row_at<T, V, W>(a, s, start, t - start - (W - k), c);
        x[k] = F::from(r.v);
      }
#pragma unroll
      for (int k = 0; k < W; ++k) g[k] = zero;
      const T *px = a.x + t * a.ld_x + c, *pd = a.dy + t * a.ld_dy + c;
      T* po = a.dx + t * a.ld_dx + c;
      const int all = (int)(stop - t) + W - 1, taken = (int)(ahead - t), own = (int)(stop - t);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (i < taken) {
          ring_x.put(i, px + i * a.ld_x);
          ring_d.put(i, pd + i * a.ld_dy);
        }
        end_of_row();
      }
      px += AHEAD * a.ld_x;
      pd += AHEAD * a.ld_dy;
      // one row; INNER: its dx and the row AHEAD behind it are this run's
      const auto row = [&](auto inner, int q, int i) {
        constexpr bool INNER = decltype(inner)::value;
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) {
          x[k] = x[k + 1];
          g[k] = g[k + 1];
        }
        oldest_landed();
        g[W - 1] = zero;
        if (INNER || q < taken) {
          const Pack<T, V> rx = ring_x.get(i), rd = ring_d.get(i);
          x[W - 1] = F::from(rx.v);
          g[W - 1] = F::from(rd.v);
          if (a.swish) {
            Unit p = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) p = seq::fma(w[k], x[k], p);
            // s (1 + p (1 - s)) = s + s p - s (s p)
            const Unit sig = seq::each<T>(p, seq::sigmoid), sp = seq::mul(sig, p);
            const Unit rest = seq::fma(seq::mul(sig, minus), sp, sp);
            g[W - 1] = seq::mul(g[W - 1], seq::fma(sig, one, rest));
          }
          if (INNER || q < own) {
            db = seq::fma(g[W - 1], one, db);
#pragma unroll
            for (int k = 0; k < W; ++k) dw[k] = seq::fma(g[W - 1], x[k], dw[k]);
          }
        }
        if (INNER || q + AHEAD < taken) {
          ring_x.put(i, px);
          ring_d.put(i, pd);
        }
        end_of_row();
        px += a.ld_x;
        pd += a.ld_dy;
        if (INNER || q >= W - 1) {                             // g[k] belongs to the token W - 1 - k before q
          Unit dx = seq::mul(w[W - 1], g[0]);
#pragma unroll
          for (int k = 1; k < W; ++k) dx = seq::fma(w[W - 1 - k], g[k], dx);
          Pack<T, V> out;
          F::to(dx, out.v);
          *reinterpret_cast<Pack<T, V>*>(po) = out;
          po += a.ld_dx;
        }
      };
      for (int q0 = 0; q0 < all; q0 += AHEAD) {
        if (q0 >= W - 1 && q0 + 2 * AHEAD <= own) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) row(std::true_type(), q0 + i, i);
        } else {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            if (q0 + i >= all) break;
            row(std::false_type(), q0 + i, i);
          }
        }
      }
      t = stop;
      do ++s; while (s < a.rows.count && a.rows.end(s) <= t);
    }
  }
  // the warps' sums in the order of the warps
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
    T sums[V];
    F::to(k < W ? dw[k < W ? k : 0] : db, sums);
#pragma unroll
    for (int j = 0; j < V; ++j) part[warp][lane * V + j] = sums[j];
    __syncthreads();
    for (int e = threadIdx.x; e < LANES * V; e += THREADS) {
      const int ch = blockIdx.y * LANES * V + e;
      T sum = 0;
#pragma unroll
      for (int r = 0; r < WARPS; ++r) sum += part[r][e];
      if (ch < a.dim) partial[((int64_t)blockIdx.x * (W + 1) + k) * a.dim + ch] = sum;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
totals_kernel(const T* __restrict__ partial, int64_t blocks, int dim, int width, T* dw, T* dbias) {
  chain_begin();
  __shared__ double part[WARPS][LANES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * LANES + lane, k = blockIdx.y;
  double sum = 0.0;
  if (c < dim)
#pragma unroll 4
    for (int64_t b = warp; b < blocks; b += WARPS) sum += (double)partial[(b * (width + 1) + k) * dim + c];
  part[warp][lane] = sum;
  __syncthreads();
  if (warp || c >= dim) return;
  sum = 0.0;
#pragma unroll
  for (int r = 0; r < WARPS; ++r) sum += part[r][lane];
  if (k < width) {
    if (dw) dw[(int64_t)c * width + k] = (T)sum;
  } else if (dbias) {
    dbias[c] = (T)sum;
  }
}

// one new row of each sequence; state_out may be the state itself
template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS)
step_kernel(const Args<T> a, int64_t batch) {
  chain_begin();
  const int c = (blockIdx.y * LANES + (threadIdx.x & 31)) * V;
  const int64_t s = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (c >= a.dim || s >= batch) return;
  const Weights<T, V, W> wt(a, c);
  Pack<T, V> x[W];
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) x[k] = load<T, V>(a.state + (s * (W - 1) + k) * a.dim + c);
  x[W - 1] = load<T, V>(a.x + s * a.ld_x + c);
  Pack<T, V> y;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    T p = wt.bias[j];
#pragma unroll
    for (int k = 0; k < W; ++k) p += wt.w[k][j] * x[k].v[j];
    y.v[j] = a.swish ? swish(p) : p;
  }
  *reinterpret_cast<Pack<T, V>*>(a.y + s * a.ld_y + c) = y;
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) *reinterpret_cast<Pack<T, V>*>(a.state_out + (s * (W - 1) + k) * a.dim + c) = x[k + 1];
}

// ---------------------------------------------------------------- launches
enum class Pass { Forward, Backward, Step };

template <typename T, int V, int W, bool BACKWARD> static prad_status launch(prad_ctx* ctx, Args<T> a, Pass pass) {
  const unsigned across = (unsigned)ceil_div(a.dim, LANES * V);
  if constexpr (!BACKWARD)
    if (pass == Pass::Step) {
      launch_chained(step_kernel<T, V, W>, dim3((unsigned)ceil_div(a.rows.tokens, WARPS), across), THREADS, 0, ctx->stream, a, a.rows.tokens);
      PRAD_LAUNCHED(ctx);
      return PRAD_OK;
    }
  // Runs of 32 tokens, of 64 backward (16384 tokens of 2048 floats: forward 45 us, 51 with 64; backward 93 us, 85 with 64), or shorter
  // ones where those give less than two CTAs an SM (2047 tokens of 333 doubles, backward: 26 us with runs of 32, 13 with runs of 8).
  a.run = BACKWARD ? 64 : 32;
  while (a.run > 8 && ceil_div(a.rows.tokens, WARPS * a.run) * across < 2 * ctx->sm_count) a.run /= 2;
  a.blocks = (unsigned)ceil_div(a.rows.tokens, WARPS * a.run);
  if constexpr (!BACKWARD) {
    const int64_t rows = W > 1 && a.state_out ? (int64_t)a.rows.count * (W - 1) : 0;
    const unsigned grid = a.blocks + (unsigned)ceil_div(rows, WARPS);
    if (grid) {
      constexpr int bytes = AHEAD * THREADS * V * (int)sizeof(T);
      prad_status st = allow_smem<forward_kernel<T, V, W>>(ctx, bytes);
      if (st) return st;
      launch_chained(forward_kernel<T, V, W>, dim3(grid, across), THREADS, bytes, ctx->stream, a);
      PRAD_LAUNCHED(ctx);
    }
    return PRAD_OK;
  } else {
    prad_status st = ensure_workspace(ctx, (size_t)(a.blocks ? a.blocks : 1) * (W + 1) * a.dim * sizeof(T));
    if (st) return st;
    const bool states = W > 1 && a.dstate && a.rows.count;
    if (a.blocks) {
      const unsigned grid = a.blocks + (states ? (unsigned)ceil_div(a.rows.count, WARPS) : 0);
      constexpr int bytes = 2 * AHEAD * THREADS * V * (int)sizeof(T);
      st = allow_smem<backward_kernel<T, V, W>>(ctx, bytes);
      if (st) return st;
      launch_chained(backward_kernel<T, V, W>, dim3(grid, across), THREADS, bytes, ctx->stream, a, (T*)ctx->ws);
      PRAD_LAUNCHED(ctx);
    } else if (states) {
      PRAD_CUDA(cudaMemsetAsync(a.dstate, 0, (size_t)a.rows.count * (W - 1) * a.dim * sizeof(T), ctx->stream));
    }
    if (a.dw || a.dbias) {
      launch_chained(totals_kernel<T>, dim3((unsigned)ceil_div(a.dim, LANES), W + 1), THREADS, 0, ctx->stream, (const T*)ctx->ws, a.blocks, a.dim, W,
                                                                                                a.dw, a.dbias);
      PRAD_LAUNCHED(ctx);
    }
    return PRAD_OK;
  }
}
template <typename T, int V, bool BACKWARD> static prad_status pick(prad_ctx* ctx, const Args<T>& a, Pass pass, int width) {
  switch (width) {
    case 1: return launch<T, V, 1, BACKWARD>(ctx, a, pass);
    case 2: return launch<T, V, 2, BACKWARD>(ctx, a, pass);
    case 3: return launch<T, V, 3, BACKWARD>(ctx, a, pass);
    case 4: return launch<T, V, 4, BACKWARD>(ctx, a, pass);
    case 5: return launch<T, V, 5, BACKWARD>(ctx, a, pass);
    case 6: return launch<T, V, 6, BACKWARD>(ctx, a, pass);
    case 7: return launch<T, V, 7, BACKWARD>(ctx, a, pass);
    default: return launch<T, V, 8, BACKWARD>(ctx, a, pass);
  }
}
template <typename T> static prad_status run(prad_ctx* ctx, const Args<T>& a, Pass pass, int width) {
  // Eight bytes a thread in the backward pass: with sixteen its windows, sums and weights leave room for half of the threads.
  const int bytes = pass == Pass::Backward ? 8 : 16;
  const uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx | (uintptr_t)a.state |
                        (uintptr_t)a.state_out | (uintptr_t)a.dstate;
  const int64_t pitches = a.dim | a.ld_x | a.ld_y | a.ld_dy | a.ld_dx;
  const bool vector = all % bytes == 0 && pitches * (int64_t)sizeof(T) % bytes == 0;
  Args<T> b = a;
  b.wide_w = vector && (uintptr_t)a.w % bytes == 0;
  if (pass == Pass::Backward) return vector ? pick<T, 8 / sizeof(T), true>(ctx, b, pass, width) : pick<T, 1, true>(ctx, b, pass, width);
  return vector ? pick<T, 16 / sizeof(T), false>(ctx, b, pass, width) : pick<T, 1, false>(ctx, b, pass, width);
}

static prad_status check(const char* who, prad_dtype dt, int64_t tokens, int sequences, const void* offsets, int dim, int width) {
  PRAD_REQUIRE(dtype_ok(dt), PRAD_ERR_INVALID, "%s: unknown dtype %d", who, (int)dt);
  PRAD_REQUIRE(tokens >= 0 && sequences >= 0 && dim > 0, PRAD_ERR_SHAPE, "%s: bad shape", who);
  PRAD_REQUIRE(dim <= 1 << 20, PRAD_ERR_UNSUPPORTED, "%s: more than 2^20 channels", who);
  PRAD_REQUIRE(width >= 1 && width <= PRAD_CONV_MAX_WIDTH, PRAD_ERR_UNSUPPORTED, "%s: widths of 1 to %d, got %d", who,
               PRAD_CONV_MAX_WIDTH, width);
  PRAD_REQUIRE(tokens <= 0x7fffffff, PRAD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", who);
  PRAD_REQUIRE(offsets || (sequences > 0 ? tokens % sequences == 0 : tokens == 0), PRAD_ERR_SHAPE,
               "%s: %lld tokens do not divide into %d sequences", who, (long long)tokens, sequences);
  PRAD_REQUIRE(((uintptr_t)offsets & 3) == 0, PRAD_ERR_INVALID, "%s: unaligned offsets", who);
  return PRAD_OK;
}
static Sequences sequences_of(int64_t tokens, int sequences, const int32_t* offsets) {
  return Sequences{offsets, sequences, tokens, offsets || sequences == 0 ? 0 : tokens / sequences};
}
static int64_t pitch(int64_t ld, int dim) { return ld ? ld : dim; }

}  // namespace conv
}  // namespace prad

using namespace prad;

template <typename T>
static prad_status forward_t(prad_ctx* ctx, const void* x, int64_t ld_x, const void* w, const void* bias, const void* state,
                             const int32_t* offsets, void* y, int64_t ld_y, void* state_out, int sequences, int64_t tokens, int dim,
                             int width, int swish, conv::Pass pass) {
  conv::Args<T> a = {};
  a.rows = conv::sequences_of(tokens, sequences, offsets);
  a.x = (const T*)x, a.w = (const T*)w, a.bias = (const T*)bias, a.state = (const T*)state;
  a.y = (T*)y, a.state_out = (T*)state_out;
  a.ld_x = ld_x, a.ld_y = ld_y, a.dim = dim, a.swish = swish;
  return conv::run<T>(ctx, a, pass, width);
}
template <typename T>
static prad_status backward_t(prad_ctx* ctx, const void* x, int64_t ld_x, const void* w, const void* bias, const void* state,
                              const int32_t* offsets, const void* dy, int64_t ld_dy, void* dx, int64_t ld_dx, void* dw, void* dbias,
                              void* dstate, int sequences, int64_t tokens, int dim, int width, int swish) {
  conv::Args<T> a = {};
  a.rows = conv::sequences_of(tokens, sequences, offsets);
  a.x = (const T*)x, a.w = (const T*)w, a.bias = (const T*)bias, a.state = (const T*)state, a.dy = (const T*)dy;
  a.dx = (T*)dx, a.dw = (T*)dw, a.dbias = (T*)dbias, a.dstate = (T*)dstate;
  a.ld_x = ld_x, a.ld_dy = ld_dy, a.ld_dx = ld_dx, a.dim = dim, a.swish = swish;
  return conv::run<T>(ctx, a, conv::Pass::Backward, width);
}

extern "C" prad_status prad_causal_conv_forward(prad_ctx* ctx, prad_dtype dt, const void* x, int64_t ld_x, const void* w, const void* bias,
                                                const void* state, const int32_t* offsets, void* y, int64_t ld_y, void* state_out,
                                                int sequences, int64_t tokens, int dim, int width, int swish) {
  prad_status st = conv::check("prad_causal_conv_forward", dt, tokens, sequences, offsets, dim, width);
  if (st) return st;
  ld_x = conv::pitch(ld_x, dim), ld_y = conv::pitch(ld_y, dim);
  PRAD_REQUIRE(ld_x >= dim && ld_y >= dim, PRAD_ERR_SHAPE, "prad_causal_conv_forward: a pitch below dim");
  PRAD_REQUIRE(tokens == 0 || (x && w && y), PRAD_ERR_INVALID, "prad_causal_conv_forward: null pointer");
  PRAD_REQUIRE(natural(dt, x, w, bias, state, y, state_out), PRAD_ERR_INVALID, "prad_causal_conv_forward: unaligned pointer");
  PRAD_REQUIRE(tokens == 0 || y != x, PRAD_ERR_INVALID, "prad_causal_conv_forward: y may not be x");
  PRAD_REQUIRE(!state_out || state_out != state, PRAD_ERR_INVALID, "prad_causal_conv_forward: state_out may not be the state");
  PRAD_CHECK_CTX(ctx);
  return dt == PRAD_F32 ? forward_t<float>(ctx, x, ld_x, w, bias, state, offsets, y, ld_y, state_out, sequences, tokens, dim, width, swish,
                                           conv::Pass::Forward)
                        : forward_t<double>(ctx, x, ld_x, w, bias, state, offsets, y, ld_y, state_out, sequences, tokens, dim, width, swish,
                                            conv::Pass::Forward);
}

extern "C" prad_status prad_causal_conv_backward(prad_ctx* ctx, prad_dtype dt, const void* x, int64_t ld_x, const void* w, const void* bias,
                                                 const void* state, const int32_t* offsets, const void* dy, int64_t ld_dy, void* dx,
                                                 int64_t ld_dx, void* dw, void* dbias, void* dstate, int sequences, int64_t tokens,
                                                 int dim, int width, int swish) {
  prad_status st = conv::check("prad_causal_conv_backward", dt, tokens, sequences, offsets, dim, width);
  if (st) return st;
  ld_x = conv::pitch(ld_x, dim), ld_dy = conv::pitch(ld_dy, dim), ld_dx = conv::pitch(ld_dx, dim);
  PRAD_REQUIRE(ld_x >= dim && ld_dy >= dim && ld_dx >= dim, PRAD_ERR_SHAPE, "prad_causal_conv_backward: a pitch below dim");
  PRAD_REQUIRE(tokens == 0 || (x && w && dy && dx), PRAD_ERR_INVALID, "prad_causal_conv_backward: null pointer");
  PRAD_REQUIRE(natural(dt, x, w, bias, state, dy, dx, dw, dbias, dstate), PRAD_ERR_INVALID, "prad_causal_conv_backward: unaligned pointer");
  PRAD_REQUIRE(tokens == 0 || (dx != x && dx != dy), PRAD_ERR_INVALID, "prad_causal_conv_backward: dx may not be x or dy");
  PRAD_CHECK_CTX(ctx);
  return dt == PRAD_F32 ? backward_t<float>(ctx, x, ld_x, w, bias, state, offsets, dy, ld_dy, dx, ld_dx, dw, dbias, dstate, sequences,
                                            tokens, dim, width, swish)
                        : backward_t<double>(ctx, x, ld_x, w, bias, state, offsets, dy, ld_dy, dx, ld_dx, dw, dbias, dstate, sequences,
                                             tokens, dim, width, swish);
}

extern "C" prad_status prad_causal_conv_step(prad_ctx* ctx, prad_dtype dt, const void* x, int64_t ld_x, const void* w, const void* bias,
                                             const void* state, void* y, int64_t ld_y, void* state_out, int64_t batch, int dim, int width,
                                             int swish) {
  prad_status st = conv::check("prad_causal_conv_step", dt, batch, 1, nullptr, dim, width);
  if (st) return st;
  ld_x = conv::pitch(ld_x, dim), ld_y = conv::pitch(ld_y, dim);
  PRAD_REQUIRE(ld_x >= dim && ld_y >= dim, PRAD_ERR_SHAPE, "prad_causal_conv_step: a pitch below dim");
  PRAD_REQUIRE(batch == 0 || (x && w && y && (width == 1 || (state && state_out))), PRAD_ERR_INVALID,
               "prad_causal_conv_step: null pointer");
  PRAD_REQUIRE(natural(dt, x, w, bias, state, y, state_out), PRAD_ERR_INVALID, "prad_causal_conv_step: unaligned pointer");
  PRAD_CHECK_CTX(ctx);
  if (batch == 0) return PRAD_OK;
  return dt == PRAD_F32 ? forward_t<float>(ctx, x, ld_x, w, bias, state, nullptr, y, ld_y, state_out, 1, batch, dim, width, swish,
                                           conv::Pass::Step)
                        : forward_t<double>(ctx, x, ld_x, w, bias, state, nullptr, y, ld_y, state_out, 1, batch, dim, width, swish,
                                            conv::Pass::Step);
}
