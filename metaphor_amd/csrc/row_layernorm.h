/*
 * Layer normalisation over the last dimension, forward and reverse.
 *
 * The reference has no normalisation kernel; its row-reduce (src/cuda/nvcc_src/reduce_ij_i.cu:3-54)
 * and column-reduce (src/cuda/nvcc_src/reduce_ij_j.cu:3-66) are the nearest patterns. Math:
 *   forward   u_i   = mean_j x_ij,   r_i = (mean_j (x_ij - u_i)^2 + eps)^(-1/2)
 *             y_ij  = (x_ij - u_i) * r_i * g_j + b_j
 *   reverse   h_ij  = (x_ij - u_i) * r_i,   e_ij = dy_ij * g_j
 *             dx_ij = r_i * (e_ij - mean_j e_ij - h_ij * mean_j(e_ij * h_ij)) + alpha * dx_ij
 *             dg_j  = sum_i dy_ij * h_ij + alpha * dg_j
 *             db_j  = sum_i dy_ij        + alpha * db_j
 * Statistics and sums are in precision<T>, the last stage of dg and db in fp64. A gain that is NULL
 * counts as ones, a bias that is NULL as zeros; dg or db that is NULL is not wanted.
 */
#ifndef MP_ROW_LAYERNORM_H
#define MP_ROW_LAYERNORM_H

#include "row_rmsnorm.h"

#if defined(__cplusplus) && defined(__HIPCC__)

namespace mp {

/* The variance from mean((x - c)^2) and mean(x - c): never below zero by rounding, NaN kept. */
template <class P> __device__ __forceinline__ P variance_of(P square, P off) {
  const P v = square - off * off;
  return v < (P)0 ? (P)0 : v;
}

/* ------------------------------------------------------------------ rows read several times */

/* One workgroup a row, which it reads three times: for the mean, for the variance about that mean,
 * and to write. The rounded mean c of a row far from zero is off by more than its values' spread
 * allows (fp32, mean 1000, spread 1: some 1e-4), so the second pass also adds up x - c, which is
 * exact or nearly so, and u = c + mean(x - c) is used as (x - c) - mean(x - c). */
template <class T, int W, bool LOOSE>
__global__ __launch_bounds__(STREAM_THREADS) void layernorm_fwd_stream(
    const T* x, const T* gain, const T* bias, T* y, typename precision<T>::type eps, size_t m, size_t n) {
  using P = typename precision<T>::type;
  constexpr int G = STREAM_THREADS;
  __shared__ P slots[3][G / WAVE];
  const P inv_n = (P)1 / (P)n;
  const int lane = threadIdx.x;
  const RowPacks<T, W, LOOSE> rp(n);
  for (size_t row = blockIdx.x; row < m; row += gridDim.x) {
    const T* xr = x + row * n;
    P s = (P)0;
    for (int p = lane; p < rp.npk; p += G) {
      P v[W];
      rp.template load<false>(xr, p, v);
#pragma unroll
      for (int i = 0; i < W; ++i) s += v[i]; /* past the end of a cut pack: zeros */
    }
    P pivot = group_allreduce<AddOP, G>(s, slots[0], lane) * inv_n;
    settle(pivot); /* the same rounded value in both passes */
    P q = (P)0, t = (P)0;
    for (int p = lane; p < rp.npk; p += G) {
      P v[W];
      rp.template load<false>(xr, p, v);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < rp.valid(p)) {
          q += (v[i] - pivot) * (v[i] - pivot);
          t += v[i] - pivot;
        }
    }
    const P off = group_allreduce<AddOP, G>(t, slots[1], lane) * inv_n;
    const P r = rsqrt_of(variance_of(group_allreduce<AddOP, G>(q, slots[2], lane) * inv_n, off) + eps);
    for (int p = lane; p < rp.npk; p += G) {
      P v[W], g[W], b[W];
      rp.template load<false>(xr, p, v);
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] = (P)1, b[i] = (P)0;
      if (gain) rp.template load<false>(gain, p, g);
      if (bias) rp.template load<false>(bias, p, b);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = (v[i] - pivot - off) * r * g[i] + b[i];
      rp.store(y + row * n, p, v);
    }
  }
}

/* The reverse of the same: the mean, then the variance with both of the gradient's row sums, then the
 * write. A workgroup walks rows and keeps its sums for dg and db in a partial row of 2n values of
 * its own, where a column always belongs to the same thread. */
template <class T, int W, bool BLEND, bool LOOSE>
__global__ __launch_bounds__(STREAM_THREADS) void layernorm_rev_stream(
    const T* x, const T* gain, const T* dy, T* dx, typename precision<T>::type* partials,
    typename precision<T>::type eps, typename precision<T>::type alpha, size_t m, size_t n) {
  using P = typename precision<T>::type;
  constexpr int G = STREAM_THREADS;
  __shared__ P slots[5][G / WAVE];
  const P inv_n = (P)1 / (P)n;
  const int lane = threadIdx.x;
  const RowPacks<T, W, LOOSE> rp(n);
  P* mine = partials + (size_t)blockIdx.x * 2 * n;
  bool first = true;
  for (size_t row = blockIdx.x; row < m; row += gridDim.x, first = false) {
    const T* xr = x + row * n;
    const T* dr = dy + row * n;
    T* out_row = dx + row * n;
    P s = (P)0;
    for (int p = lane; p < rp.npk; p += G) {
      P v[W];
      rp.template load<false>(xr, p, v);
#pragma unroll
      for (int i = 0; i < W; ++i) s += v[i];
    }
    P pivot = group_allreduce<AddOP, G>(s, slots[0], lane) * inv_n;
    settle(pivot); /* the same rounded value in both passes */
    P q = (P)0, sum = (P)0, a = (P)0, c = (P)0;
    for (int p = lane; p < rp.npk; p += G) {
      P v[W], d[W], g[W];
      rp.template load<false>(xr, p, v);
      rp.template load<false>(dr, p, d);
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] = (P)1;
      if (gain) rp.template load<false>(gain, p, g);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < rp.valid(p)) {
          const P t = v[i] - pivot, e = d[i] * g[i];
          q += t * t;
          sum += t;
          a += e;
          c += e * t;
        }
    }
    q = group_allreduce<AddOP, G>(q, slots[1], lane);
    a = group_allreduce<AddOP, G>(a, slots[2], lane);
    c = group_allreduce<AddOP, G>(c, slots[3], lane);
    const P off = group_allreduce<AddOP, G>(sum, slots[4], lane) * inv_n;
    const P r = rsqrt_of(variance_of(q * inv_n, off) + eps);
    const P ma = a * inv_n, mc = (c * inv_n - off * ma) * r;
    for (int p = lane; p < rp.npk; p += G) {
      P v[W], d[W], g[W], out[W];
      rp.template load<false>(xr, p, v);
      rp.template load<false>(dr, p, d);
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] = (P)1;
      if (gain) rp.template load<false>(gain, p, g);
      P old[W];
      if constexpr (BLEND) rp.template load<false>(out_row, p, old);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const P h = (v[i] - pivot - off) * r;
        out[i] = r * (d[i] * g[i] - ma - h * mc);
        if constexpr (BLEND) out[i] += alpha * old[i];
        if (i < rp.valid(p)) {
          P* at = mine + (size_t)p * W + i;
          at[0] = (first ? (P)0 : at[0]) + d[i] * h;
          at[n] = (first ? (P)0 : at[n]) + d[i];
        }
      }
      rp.store(out_row, p, out);
    }
  }
}

/* ------------------------------------------------------------------ a row in registers */

/* How a row's packs lie on the lanes that hold it: pack k * lanes + lane is the k-th of a lane. SUB < 64:
 * a row is held by SUB lanes, 64 / SUB rows a wavefront; SUB = 64: by `gw` wavefronts, any number up
 * to 16 (a kernel argument), so that rows of any length leave fewer than 64 lanes' worth of packs idle.
 * Loads have no conditions: a pack beyond the row reads its first pack and is left out of every
 * sum. */
template <class T, int W, int SUB, int NV, bool LOOSE> struct NormRow {
  using P = typename precision<T>::type;
  using V = typename vec_of<T, W>::type;
  const RowPacks<T, W, LOOSE> rp;
  int lanes, lane; /* lanes a row, and which of them this is */

  __device__ __forceinline__ NormRow(size_t n, int lanes_, int lane_) : rp(n), lanes(lanes_), lane(lane_) {}
  __device__ __forceinline__ int pack(int k) const { return k * lanes + lane; }
  __device__ __forceinline__ bool inside(int k) const { return pack(k) < rp.npk; }
  template <bool NT> __device__ __forceinline__ void fetch(const T* row, V (&out)[NV]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) out[k] = rp.template raw<NT>(row, inside(k) ? pack(k) : 0);
  }
  /* elements the wavefront `w` of the row holds (SUB < 64: the row's own) */
  __device__ __forceinline__ int held(int w, size_t n) const {
    if (SUB < WAVE) return (int)n;
    int packs = 0;
    bool end = false;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int lo = k * lanes + w * WAVE, left = rp.npk - lo;
      packs += left < 0 ? 0 : left > WAVE ? WAVE : left;
      end = end || (left > 0 && left <= WAVE);
    }
    return packs * W - (end ? W - rp.last : 0);
  }
};

/* What the wavefronts of a row hand each other: a pivot near the mean of a wavefront's own elements, the
 * sums of x - pivot and its square, and in the reverse those of e = dy * gain and e * (x - pivot). Every
 * wavefront takes its sums about a pivot of its own, so one exchange does for the mean and the
 * variance, without a difference of squares of values far from zero. */
template <class P> struct NormPart { P pivot, off, square, e, ex; };
template <class P> struct NormStats {
  P pivot, off, r; /* mean = pivot + off: x - mean is (x - pivot) - off, where x - pivot is exact or nearly so */
  P mean_e, mean_eh;
};

/* The row's statistics from the parts of its wavefronts, which lie in LDS behind a barrier; lane i of every
 * 16 takes part i, `held` of whose elements exist (0 from the gw-th on), and all lanes get the same bits. */
template <bool REVERSE, class P>
__device__ __forceinline__ NormStats<P> norm_join(const NormPart<P>* parts, int gw, P held, P inv_n, P eps) {
  const int slot = threadIdx.x & 15;
  NormPart<P> part = parts[slot < gw ? slot : 0];
  NormStats<P> s;
  s.pivot = parts[0].pivot;
  const bool real = slot < gw;
  const P apart = part.pivot - s.pivot;
  s.off = fold_partials<AddOP, 16>(real ? part.off + held * apart : (P)0) * inv_n;
  const P by = apart - s.off; /* pivot - mean */
  const P square = fold_partials<AddOP, 16>(real ? part.square + by * ((P)2 * part.off + held * by) : (P)0) * inv_n;
  s.r = rsqrt_of((square < (P)0 ? (P)0 : square) + eps);
  if constexpr (REVERSE) {
    s.mean_e = fold_partials<AddOP, 16>(real ? part.e : (P)0) * inv_n;
    s.mean_eh = fold_partials<AddOP, 16>(real ? part.ex + by * part.e : (P)0) * inv_n * s.r;
  }
  return s;
}
template <bool REVERSE, class P>
__device__ __forceinline__ NormStats<P> norm_alone(const NormPart<P>& part, P inv_n, P eps) {
  NormStats<P> s;
  s.pivot = part.pivot;
  s.off = part.off * inv_n;
  s.r = rsqrt_of(variance_of(part.square * inv_n, s.off) + eps);
  if constexpr (REVERSE) {
    s.mean_e = part.e * inv_n;
    s.mean_eh = (part.ex - s.off * part.e) * inv_n * s.r;
  }
  return s;
}

constexpr int NORM_WAVES = NORM_BLOCK / WAVE;

/* Half-precision rows are bound by arithmetic as much as by memory (13 instructions an element in the
 * forward when every operand is widened first), so products take their operands as stored:
 * a * b + c with a (and b) in half is one v_fma_mix_f32, exact in the product as fp32 is. */
__device__ __forceinline__ float mix_fma(_Float16 a, float b, float c) { return __builtin_fmaf((float)a, b, c); }
__device__ __forceinline__ float mix_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double mix_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }
/* a - c; `one` is a one that the compiler does not know, or the half case would be two instructions again */
__device__ __forceinline__ float mix_less(_Float16 a, float c, float one) { return __builtin_fmaf((float)a, one, -c); }
__device__ __forceinline__ float mix_less(float a, float c, float) { return a - c; }
__device__ __forceinline__ double mix_less(double a, double c, double) { return a - c; }
__device__ __forceinline__ float mix_add(_Float16 a, float c, float one) { return __builtin_fmaf((float)a, one, c); }
__device__ __forceinline__ float mix_add(float a, float c, float) { return a + c; }
__device__ __forceinline__ double mix_add(double a, double c, double) { return a + c; }
template <class T, class P> __device__ __forceinline__ P mix_mul(T a, T b) {
  if constexpr (sizeof(T) == 2) return __builtin_fmaf((float)a, (float)b, 0.0f);
  else return a * b;
}
__device__ __forceinline__ float norm_out(float h, float g, _Float16 b) { return __builtin_fmaf(h, g, (float)b); }
__device__ __forceinline__ float norm_out(float h, float g, float b) { return __builtin_fmaf(h, g, b); }
__device__ __forceinline__ double norm_out(double h, double g, double b) { return __builtin_fma(h, g, b); }
/* the sum of a pack (two halves an instruction) */
template <class T, int W, class P> __device__ __forceinline__ P pack_sum(const typename vec_of<T, W>::type& v) {
  P s = (P)0;
  if constexpr (sizeof(T) == 2) {
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    const half2_t ones = {(_Float16)1, (_Float16)1};
#pragma unroll
    for (int i = 0; i < W; i += 2) s = __builtin_amdgcn_fdot2(half2_t{v[i], v[i + 1]}, ones, s, false);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) s += v[i];
  }
  return s;
}

/* ------------------------------------------------------------------ forward */

template <class T, int W, int SUB, int NV, bool LOOSE, bool PAIR>
__global__ __launch_bounds__(NORM_BLOCK) void layernorm_fwd_rows(
    const T* x, const T* gain, const T* bias, T* y, typename precision<T>::type eps, size_t m, size_t n, int gw) {
  using P = typename precision<T>::type;
  using Row = NormRow<T, W, SUB, NV, LOOSE>;
  using V = typename Row::V;
  __shared__ NormPart<P> parts[2][NORM_WAVES];
  const P inv_n = (P)1 / (P)n;
  const int wave = threadIdx.x / WAVE, G = SUB < WAVE ? SUB : gw * WAVE;
  const int rows_here = (int)blockDim.x / G, sub = threadIdx.x / G;
  const int base_wave = sub * gw, mine = wave - base_wave; /* of the row's wavefronts */
  const Row rw(n, G, threadIdx.x % G);
  const P held = (P)rw.held(SUB < WAVE ? 0 : mine, n), inv_held = held > (P)0 ? (P)1 / held : (P)0;
  const P held_slot = SUB < WAVE || gw == 1 ? held : (P)rw.held(threadIdx.x & 15, n);

  V gv[NV], bv[NV]; /* as stored, widened where they are used */
  if (gain) rw.template fetch<false>(gain, gv);
  else
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) gv[k][i] = (T)1;
  if (bias) rw.template fetch<false>(bias, bv);
  else
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) bv[k][i] = (T)0;

  const size_t last = m - 1, stride = (size_t)gridDim.x * rows_here;
  auto fetch = [&](V (&xs)[NV], size_t base) { /* a row beyond the last reads the last */
    const size_t row = base + sub;
    rw.template fetch<true>(x + (row < last ? row : last) * n, xs);
  };
  P one = (P)1;
  settle(one);
  auto finish = [&](const V (&xs)[NV], size_t base, NormPart<P>* slots) {
    P s = (P)0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const P sk = pack_sum<T, W, P>(xs[k]); /* past the end of a cut pack: zeros */
      s += rw.inside(k) ? sk : (P)0;
    }
    P d[NV][W];
    NormPart<P> part;
    part.pivot = lanes_allreduce<AddOP, SUB>(s) * inv_held;
    settle(part.pivot); /* rounded here: x - s * inv_held in one step is not x minus what is handed on */
    part.off = part.square = (P)0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      P tk = (P)0, qk = (P)0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        d[k][i] = mix_less(xs[k][i], part.pivot, one);
        if constexpr (LOOSE) d[k][i] = i < rw.rp.valid(rw.pack(k)) ? d[k][i] : (P)0;
        tk += d[k][i];
        qk += d[k][i] * d[k][i];
      }
      part.off += rw.inside(k) ? tk : (P)0;
      part.square += rw.inside(k) ? qk : (P)0;
    }
    part.off = lanes_allreduce<AddOP, SUB>(part.off);
    part.square = lanes_allreduce<AddOP, SUB>(part.square);
    NormStats<P> st;
    if (SUB < WAVE || gw == 1) {
      st = norm_alone<false>(part, inv_n, eps);
    } else {
      if (threadIdx.x % WAVE == 0) slots[wave] = part;
      lds_barrier();
      st = norm_join<false>(slots + base_wave, gw, held_slot, inv_n, eps);
    }
    const P back = part.pivot - st.pivot - st.off; /* what x - mean is above d */
    const size_t row = base + sub;
    if (row < m) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (rw.inside(k)) {
          P out[W];
#pragma unroll
          for (int i = 0; i < W; ++i) out[i] = norm_out(d[k][i] + back, mix_fma(gv[k][i], st.r, (P)0), bv[k][i]);
          rw.rp.store(y + row * n, rw.pack(k), out);
        }
      }
    }
  };

  size_t base = (size_t)blockIdx.x * rows_here;
  V ax[NV];
  if constexpr (PAIR) { /* the next rows are on their way while these are reduced and written */
    V bx[NV];
    fetch(ax, base);
    for (; base < m; base += 2 * stride) {
      fetch(bx, base + stride);
      __builtin_amdgcn_sched_barrier(0);
      finish(ax, base, parts[0]);
      fetch(ax, base + 2 * stride);
      __builtin_amdgcn_sched_barrier(0);
      finish(bx, base + stride, parts[1]);
    }
  } else {
    int parity = 0;
    for (; base < m; base += stride, parity ^= 1) {
      fetch(ax, base);
      finish(ax, base, parts[parity]);
    }
  }
}

/* ------------------------------------------------------------------ reverse */

/* Persistent workgroups walk the rows; the next rows' x and dy are on their way while these are reduced
 * behind a barrier that orders LDS traffic only, and the columns' sums for dg and db stay in registers.
 * At the end the rows of a workgroup are folded in order and it leaves ONE partial row of 2n sums. */
template <class T, int W, int SUB, int NV, bool BLEND, bool LOOSE, bool PAIR>
__global__ __launch_bounds__(NORM_BLOCK) void layernorm_rev_rows(
    const T* x, const T* gain, const T* dy, T* dx, typename precision<T>::type* partials,
    typename precision<T>::type eps, typename precision<T>::type alpha, size_t m, size_t n, int gw) {
  using P = typename precision<T>::type;
  using Row = NormRow<T, W, SUB, NV, LOOSE>;
  using V = typename Row::V;
  __shared__ NormPart<P> parts[2][NORM_WAVES];
  __shared__ P comb[NORM_BLOCK * W];
  const P inv_n = (P)1 / (P)n;
  const int wave = threadIdx.x / WAVE, G = SUB < WAVE ? SUB : gw * WAVE;
  const int rows_here = (int)blockDim.x / G, sub = threadIdx.x / G;
  const int base_wave = sub * gw, mine = wave - base_wave;
  const Row rw(n, G, threadIdx.x % G);
  const P held = (P)rw.held(SUB < WAVE ? 0 : mine, n), inv_held = held > (P)0 ? (P)1 / held : (P)0;
  const P held_slot = SUB < WAVE || gw == 1 ? held : (P)rw.held(threadIdx.x & 15, n);

  V gv[NV];
  if (gain) rw.template fetch<false>(gain, gv);
  else
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) gv[k][i] = (T)1;
  P acc_g[NV][W], acc_b[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < W; ++i) acc_g[k][i] = acc_b[k][i] = (P)0;

  const size_t last = m - 1, stride = (size_t)gridDim.x * rows_here;
  auto fetch = [&](V (&xs)[NV], V (&ds)[NV], size_t base) {
    size_t row = base + sub;
    row = row < last ? row : last;
    rw.template fetch<true>(x + row * n, xs);
    rw.template fetch<true>(dy + row * n, ds);
  };
  P one = (P)1;
  settle(one);
  auto finish = [&](const V (&xs)[NV], const V (&ds)[NV], size_t base, NormPart<P>* slots) {
    P s = (P)0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const P sk = pack_sum<T, W, P>(xs[k]); /* past the end of a cut pack: zeros, as dy's */
      s += rw.inside(k) ? sk : (P)0;
    }
    P t[NV][W], e[NV][W];
    NormPart<P> part;
    part.pivot = lanes_allreduce<AddOP, SUB>(s) * inv_held;
    settle(part.pivot); /* rounded here: x - s * inv_held in one step is not x minus what is handed on */
    part.off = part.square = part.e = part.ex = (P)0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      P tk = (P)0, qk = (P)0, ek = (P)0, fk = (P)0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        t[k][i] = mix_less(xs[k][i], part.pivot, one);
        if constexpr (LOOSE) t[k][i] = i < rw.rp.valid(rw.pack(k)) ? t[k][i] : (P)0;
        e[k][i] = mix_mul<T, P>(ds[k][i], gv[k][i]);
        tk += t[k][i];
        qk += t[k][i] * t[k][i];
        ek += e[k][i];
        fk += e[k][i] * t[k][i];
      }
      const bool in = rw.inside(k);
      part.off += in ? tk : (P)0;
      part.square += in ? qk : (P)0;
      part.e += in ? ek : (P)0;
      part.ex += in ? fk : (P)0;
    }
    part.off = lanes_allreduce<AddOP, SUB>(part.off);
    part.square = lanes_allreduce<AddOP, SUB>(part.square);
    part.e = lanes_allreduce<AddOP, SUB>(part.e);
    part.ex = lanes_allreduce<AddOP, SUB>(part.ex);
    NormStats<P> st;
    if (SUB < WAVE || gw == 1) {
      st = norm_alone<true>(part, inv_n, eps);
    } else {
      if (threadIdx.x % WAVE == 0) slots[wave] = part;
      lds_barrier();
      st = norm_join<true>(slots + base_wave, gw, held_slot, inv_n, eps);
    }
    const P back = (part.pivot - st.pivot - st.off) * st.r; /* h = (x - mean) * r = t * r + back */
    const P re = st.r * st.mean_e, rh = st.r * st.mean_eh;
    const size_t row = base + sub;
    if (row < m) {
      T* out_row = dx + row * n;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (rw.inside(k)) {
          P out[W];
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const P h = t[k][i] * st.r + back;
            out[i] = e[k][i] * st.r - re - h * rh;
            acc_g[k][i] = mix_fma(ds[k][i], h, acc_g[k][i]);
            acc_b[k][i] = mix_add(ds[k][i], acc_b[k][i], one);
          }
          if constexpr (BLEND) {
            P old[W];
            rw.rp.template load<false>(out_row, rw.pack(k), old);
#pragma unroll
            for (int i = 0; i < W; ++i) out[i] += alpha * old[i];
          }
          rw.rp.store(out_row, rw.pack(k), out);
        }
      }
    }
  };

  size_t base = (size_t)blockIdx.x * rows_here;
  V ax[NV], ad[NV];
  if constexpr (PAIR) {
    V bx[NV], bd[NV];
    fetch(ax, ad, base);
#pragma unroll
    for (int k = 0; k < NV; ++k) settle(gv[k]); /* the gain is waited for here, not inside the loop */
    for (; base < m; base += 2 * stride) {
      fetch(bx, bd, base + stride);
      __builtin_amdgcn_sched_barrier(0);
      finish(ax, ad, base, parts[0]);
      fetch(ax, ad, base + 2 * stride);
      __builtin_amdgcn_sched_barrier(0);
      finish(bx, bd, base + stride, parts[1]);
    }
  } else {
    int parity = 0;
    for (; base < m; base += stride, parity ^= 1) {
      fetch(ax, ad, base);
      finish(ax, ad, base, parts[parity]);
    }
  }

  /* the rows of a wavefront, then the row groups of the workgroup, a pack of every lane at a time */
  const int groups = SUB < WAVE ? (int)blockDim.x / WAVE : rows_here;
  const int width = SUB < WAVE ? SUB : G; /* lanes a group */
  P* out = partials + (size_t)blockIdx.x * 2 * n;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      P a[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        a[i] = which ? acc_b[k][i] : acc_g[k][i];
        if constexpr (SUB < WAVE)
          for (int step = SUB; step < WAVE; step <<= 1) a[i] += __shfl_xor(a[i], step, WAVE);
      }
      if (groups == 1) {
        if (rw.inside(k)) {
          const int p = rw.pack(k);
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (i < rw.rp.valid(p)) out[which * n + (size_t)p * W + i] = a[i];
        }
        continue;
      }
      const int group = SUB < WAVE ? wave : sub, at = threadIdx.x % width;
      __syncthreads(); /* the sums before have been read */
      if (SUB == WAVE || threadIdx.x % WAVE < (unsigned)SUB)
#pragma unroll
        for (int i = 0; i < W; ++i) comb[(group * width + at) * W + i] = a[i];
      __syncthreads();
      for (int c = threadIdx.x; c < width * W; c += blockDim.x) {
        const size_t col = (size_t)k * width * W + c;
        if (col < n) {
          P t = (P)0;
          for (int g = 0; g < groups; ++g) t += comb[g * width * W + c];
          out[which * n + col] = t;
        }
      }
    }
}

/* ------------------------------------------------------------------ dg and db from the partial rows */

/* The partial rows (2n columns: dg's, then db's) added in a fixed order in fp64. A workgroup owns
 * FINISH_COLS columns, FINISH_SLICES slices of it take the rows in turn with eight loads on their way. */
constexpr int NORM_FINISH_LANES = 8, NORM_FINISH_SLICES = 64;
template <class T, int CW>
__global__ __launch_bounds__(NORM_FINISH_LANES * NORM_FINISH_SLICES) void layernorm_grads_finish(
    const typename precision<T>::type* partials, T* dg, T* db, double alpha, int rows, size_t n) {
  using P = typename precision<T>::type;
  constexpr int COLS = NORM_FINISH_LANES * CW;
  __shared__ double part[NORM_FINISH_SLICES][COLS + 1];
  const int c = threadIdx.x % NORM_FINISH_LANES, slice = threadIdx.x / NORM_FINISH_LANES;
  const size_t col = ((size_t)blockIdx.x * NORM_FINISH_LANES + c) * CW, width = 2 * n;
  double s[CW];
#pragma unroll
  for (int i = 0; i < CW; ++i) s[i] = 0.0;
  if (col < width) { /* 2n is a multiple of CW */
    constexpr int U = 8;
    for (int p = slice; p < rows; p += U * NORM_FINISH_SLICES) {
      P v[U][CW];
#pragma unroll
      for (int u = 0; u < U; ++u) { /* beyond the last row: the last, left out */
        const int q = p + u * NORM_FINISH_SLICES;
        load_pack<P, CW>(partials + (size_t)(q < rows ? q : rows - 1) * width + col, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < CW; ++i) s[i] += p + u * NORM_FINISH_SLICES < rows ? (double)v[u][i] : 0.0;
    }
  }
#pragma unroll
  for (int i = 0; i < CW; ++i) part[slice][c * CW + i] = s[i];
  __syncthreads();
  const size_t at = (size_t)blockIdx.x * COLS + threadIdx.x;
  if (threadIdx.x < COLS && at < width) {
    T* out = at < n ? dg : db;
    if (!out) return;
    out += at < n ? at : at - n;
    double t = 0.0;
#pragma unroll 8
    for (int i = 0; i < NORM_FINISH_SLICES; ++i) t += part[i][threadIdx.x];
    if (alpha != 0.0) t += alpha * (double)*out;
    *out = (T)t;
  }
}

/* ------------------------------------------------------------------ host dispatch */

/* Partial rows the reverse may write: one per workgroup, at most two workgroups per CU. */
inline size_t layernorm_partial_rows(size_t m) {
  const size_t cap = (size_t)compute_units() * 2;
  return m < cap ? m : cap;
}

template <class T> inline size_t layernorm_reverse_scratch_bytes(size_t m, size_t n) {
  return layernorm_partial_rows(m) * 2 * n * sizeof(typename precision<T>::type);
}

/* How a launch holds its rows: `sub` lanes a row below 64, else `gw` wavefronts, `nv` packs a lane, `rows`
 * rows a workgroup at a time, `per_cu` workgroups a compute unit that walk them (0: one workgroup for
 * every `rows` rows), `pair`: the next rows on their way while these are reduced. nv = 0: rows too long
 * for registers. */
struct NormPlan {
  int sub, nv, gw, rows, per_cu;
  bool pair;
};
inline unsigned norm_grid(const NormPlan& p, size_t m) {
  const size_t need = (m + p.rows - 1) / p.rows, cap = (size_t)compute_units() * p.per_cu;
  require(need < 0x7fffffffull || p.per_cu, "layernorm: too many rows for one grid");
  return (unsigned)(p.per_cu && cap < need ? cap : need);
}
inline unsigned norm_block(const NormPlan& p) { return (unsigned)(p.rows * (p.sub < WAVE ? p.sub : p.gw * WAVE)); }

template <class T> inline NormPlan layernorm_forward_plan(size_t packs) {
  constexpr int MAXNV = sizeof(T) == 2 ? 4 : 8;
  if (packs <= 8) return {8, 1, 1, 32, 0, false};
  if (packs <= 16) return {16, 1, 1, 16, 0, false};
  if (packs <= 32) return {32, 1, 1, 8, 0, false};
  for (int nv = 1; nv <= MAXNV; nv *= 2)
    if (packs <= (size_t)nv * NORM_BLOCK) {
      const int gw = (int)((packs + (size_t)nv * WAVE - 1) / ((size_t)nv * WAVE));
      const int rows = NORM_WAVES / gw;
      return {WAVE, nv, gw, rows, 2, false};
    }
  return {WAVE, 0, 0, 0, 0, false};
}
template <class T> inline NormPlan layernorm_reverse_plan(size_t packs) {
  constexpr int MAXNV = sizeof(T) == 2 ? 2 : 4;
  if (packs <= 8) return {8, 1, 1, 128, 1, true};
  if (packs <= 16) return {16, 1, 1, 64, 1, true};
  if (packs <= 32) return {32, 1, 1, 32, 1, true};
  for (int nv = 1; nv <= MAXNV; nv *= 2)
    if (packs <= (size_t)nv * NORM_BLOCK) {
      const int gw = (int)((packs + (size_t)nv * WAVE - 1) / ((size_t)nv * WAVE));
      return {WAVE, nv, gw, NORM_WAVES / gw, 1, nv == 1};
    }
  return {WAVE, 0, 0, 0, 0, false};
}

/* f.template operator()<SUB, NV, PAIR>() for a plan in registers */
template <int MAXNV, class F> inline void for_norm_plan(const NormPlan& p, F&& f) {
  auto at = [&]<int SUB, int NV>() {
    if (p.pair) f.template operator()<SUB, NV, true>();
    else f.template operator()<SUB, NV, false>();
  };
  if (p.sub == 8) at.template operator()<8, 1>();
  else if (p.sub == 16) at.template operator()<16, 1>();
  else if (p.sub == 32) at.template operator()<32, 1>();
  else if (p.nv == 1) at.template operator()<WAVE, 1>();
  else if (p.nv == 2) at.template operator()<WAVE, 2>();
  else if (p.nv == 4) { if constexpr (MAXNV >= 4) at.template operator()<WAVE, 4>(); }
  else { if constexpr (MAXNV >= 8) at.template operator()<WAVE, 8>(); }
}

template <class T>
inline void layernorm_forward_as(const NormPlan& plan, const T* x, const T* gain, const T* bias, T* y, double eps, size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  const bool loose = !(aligned16(x) && aligned16(y) && (!gain || aligned16(gain)) && (!bias || aligned16(bias)) && n % W == 0);
  if (plan.nv == 0) {
    const size_t cap = (size_t)compute_units() * 2;
    const dim3 grid((unsigned)(m < cap ? m : cap)), block(STREAM_THREADS);
    if (loose) layernorm_fwd_stream<T, W, true><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
    else layernorm_fwd_stream<T, W, false><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
  } else {
    const dim3 grid(norm_grid(plan, m)), block(norm_block(plan));
    for_norm_plan<sizeof(T) == 2 ? 4 : 8>(plan, [&]<int SUB, int NV, bool PAIR>() {
      if (loose) layernorm_fwd_rows<T, W, SUB, NV, true, PAIR><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n, plan.gw);
      else layernorm_fwd_rows<T, W, SUB, NV, false, PAIR><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n, plan.gw);
    });
  }
  MP_CHECK_LAUNCH();
}

template <class T>
inline void layernorm_forward(const T* x, const T* gain, const T* bias, T* y, double eps, size_t m, size_t n, hipStream_t stream) {
  if (m == 0 || n == 0) return;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  require(n <= 0x40000000ull, "layernorm: row length must not exceed 2^30");
  layernorm_forward_as<T>(layernorm_forward_plan<T>((n + W - 1) / W), x, gain, bias, y, eps, m, n, stream);
}

template <class T>
inline void layernorm_reverse_as(const NormPlan& plan, const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, void* scratch, double eps, double alpha,
                                 size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  P* partials = static_cast<P*>(scratch);
  size_t rows = 0;
  if (m > 0) {
    const bool loose = !(aligned16(x) && aligned16(dy) && aligned16(dx) && (!gain || aligned16(gain)) && n % W == 0);
    if (plan.nv == 0) {
      rows = layernorm_partial_rows(m);
      const dim3 grid((unsigned)rows), block(STREAM_THREADS);
      auto go = [&]<bool BLEND, bool LOOSE>() {
        layernorm_rev_stream<T, W, BLEND, LOOSE><<<grid, block, 0, stream>>>(x, gain, dy, dx, partials, (P)eps, (P)alpha, m, n);
      };
      if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
      else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
    } else {
      rows = norm_grid(plan, m);
      require(rows <= layernorm_partial_rows(m), "layernorm reverse: more partial rows than the workspace holds");
      const dim3 grid((unsigned)rows), block(norm_block(plan));
      for_norm_plan<sizeof(T) == 2 ? 2 : 4>(plan, [&]<int SUB, int NV, bool PAIR>() {
        auto go = [&]<bool BLEND, bool LOOSE>() {
          layernorm_rev_rows<T, W, SUB, NV, BLEND, LOOSE, PAIR><<<grid, block, 0, stream>>>(x, gain, dy, dx, partials, (P)eps, (P)alpha, m, n, plan.gw);
        };
        if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
        else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
      });
    }
    MP_CHECK_LAUNCH();
  }
  if (!dg && !db) return;
  /* wide loads need 16-byte aligned partial rows: fp32 sums, 2n % 4 == 0, an aligned workspace */
  const bool wide = sizeof(P) == 4 && n % 2 == 0 && aligned16(partials);
  const size_t cols = wide ? NORM_FINISH_LANES * 4 : NORM_FINISH_LANES;
  const dim3 grid((unsigned)((2 * n + cols - 1) / cols)), block(NORM_FINISH_LANES * NORM_FINISH_SLICES);
  if (wide) { if constexpr (sizeof(P) == 4) layernorm_grads_finish<T, 4><<<grid, block, 0, stream>>>(partials, dg, db, alpha, (int)rows, n); }
  else layernorm_grads_finish<T, 1><<<grid, block, 0, stream>>>(partials, dg, db, alpha, (int)rows, n);
  MP_CHECK_LAUNCH();
}

template <class T>
inline void layernorm_reverse(const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, void* scratch, double eps, double alpha,
                              size_t m, size_t n, hipStream_t stream) {
  if (n == 0) return;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  require(n <= 0x40000000ull, "layernorm reverse: row length must not exceed 2^30");
  require(m == 0 || scratch != nullptr, "layernorm reverse: scratch must hold mpLayernormReverseScratchBytes bytes");
  layernorm_reverse_as<T>(layernorm_reverse_plan<T>((n + W - 1) / W), x, gain, dy, dx, dg, db, scratch, eps, alpha, m, n, stream);
}

}  // namespace mp

#endif
#endif
