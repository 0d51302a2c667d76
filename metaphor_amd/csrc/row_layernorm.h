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

/* A partial row holds dg's sums from its start and db's from partial_apart on: n rounded up to whole packs of
 * T, so that packs of sums are stored and added whole and aligned. */
template <class T> __host__ __device__ inline size_t partial_apart(size_t n) {
  constexpr size_t W = PACK_BYTES / sizeof(T);
  return (n + W - 1) / W * W;
}

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
 * write. A workgroup walks rows and keeps its sums for dg and db in a partial row of its own, where a
 * column always belongs to the same thread. */
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
  const size_t apart = partial_apart<T>(n);
  P* mine = partials + (size_t)blockIdx.x * 2 * apart;
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
          at[apart] = (first ? (P)0 : at[apart]) + d[i];
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
 * sum. The pack that the row's end cuts (LOOSE) is read whole too, into the next row, and masked by the
 * one lane that holds it; only where that would pass the tensor's end are its elements read singly. */
template <class T, int W, int SUB, int NV, bool LOOSE> struct NormRow {
  using P = typename precision<T>::type;
  using V = typename vec_of<T, W>::type;
  using VL = typename std::conditional<LOOSE, typename loose_vec_of<T, W>::type, V>::type;
  const RowPacks<T, W, LOOSE> rp;
  int lanes, lane; /* lanes a row, and which of them this is */

  __device__ __forceinline__ NormRow(size_t n, int lanes_, int lane_) : rp(n), lanes(lanes_), lane(lane_) {}
  __device__ __forceinline__ int pack(int k) const { return k * lanes + lane; }
  __device__ __forceinline__ bool inside(int k) const { return pack(k) < rp.npk; }
  __device__ __forceinline__ bool cut(int k) const { return LOOSE && rp.last != W && pack(k) == rp.npk - 1; }
  /* whether the packs of this row reach past m rows of n (short rows: not the last one alone) */
  __device__ __forceinline__ bool ends(size_t row, size_t m, size_t n) const { return row * n + (size_t)rp.npk * W > m * n; }
  /* a row of x or dy; KEEP: through loads that leave it in the memory-side cache (keep_input, row_cluster.h) */
  template <bool KEEP> __device__ __forceinline__ void fetch(const T* row, V (&out)[NV], bool end) const {
    if (LOOSE && end) {
#pragma unroll
      for (int k = 0; k < NV; ++k) out[k] = rp.template raw<!KEEP>(row, inside(k) ? pack(k) : 0);
      return;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const VL* at = reinterpret_cast<const VL*>(row + (size_t)(unsigned)(inside(k) ? pack(k) : 0) * W);
      out[k] = KEEP ? *at : __builtin_nontemporal_load(at);
    }
  }
  /* a vector that every row uses; NULL: `fill` throughout */
  __device__ __forceinline__ void fetch_vector(const T* vec, V (&out)[NV], T fill) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (vec) {
        out[k] = rp.template raw<false>(vec, inside(k) ? pack(k) : 0);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) out[k][i] = fill;
      }
    }
  }
  /* what a cut pack read behind the row becomes zero */
  __device__ __forceinline__ void mask(V (&v)[NV]) const {
    if constexpr (LOOSE)
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cut(k))
#pragma unroll
          for (int i = 0; i < W; ++i) v[k][i] = i < rp.last ? v[k][i] : (T)0;
  }
  /* elements the wavefront `w` of the row holds in the first `packs` packs of its lanes (SUB < 64: the
   * whole row, whose lanes hold one pack each) */
  __device__ __forceinline__ int held(int w, int depth, size_t n) const {
    if (SUB < WAVE) return (int)n;
    int packs = 0;
    bool end = false;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (k >= depth) break;
      const int lo = k * lanes + w * WAVE, left = rp.npk - lo;
      packs += left < 0 ? 0 : left > WAVE ? WAVE : left;
      end = end || (left > 0 && left <= WAVE);
    }
    return packs * W - (end ? W - rp.last : 0);
  }
};

constexpr int NORM_WAVES = NORM_BLOCK / WAVE;

/* Half-precision rows are bound by arithmetic as much as by memory (23 vector instructions an element in
 * the reverse, 19 us of the 39 a [16384, 2048] pass took, when every operand was widened first), so
 * products take their operands as stored: a * b + c with a (and b) in half is one v_fma_mix_f32, and
 * sums of elements and of products go two at a time through v_dot2_f32_f16, both with fp32 results. */
__device__ __forceinline__ float mix_fma(_Float16 a, float b, float c) { return __builtin_fmaf((float)a, b, c); }
__device__ __forceinline__ float mix_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double mix_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }
/* a - c and a + c; `one` is a one that the compiler does not know, or the half case would be two instructions again */
template <class T, class P> __device__ __forceinline__ P mix_less(T a, P c, P one) {
  if constexpr (sizeof(T) == 2) return __builtin_fmaf((float)a, one, -c);
  else return a - c;
}
template <class T, class P> __device__ __forceinline__ P mix_add(T a, P c, P one) {
  if constexpr (sizeof(T) == 2) return __builtin_fmaf((float)a, one, c);
  else return a + c;
}
template <class T, class P> __device__ __forceinline__ P mix_mul(T a, T b) {
  if constexpr (sizeof(T) == 2) return __builtin_fmaf((float)a, (float)b, 0.0f);
  else return a * b;
}
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
/* s + the sum of a pack's products with another's, or of its elements */
template <int W, class V> __device__ __forceinline__ float half_dot(const V& a, const V& b, float s) {
#pragma unroll
  for (int i = 0; i < W; i += 2) s = __builtin_amdgcn_fdot2(half2_t{a[i], a[i + 1]}, half2_t{b[i], b[i + 1]}, s, false);
  return s;
}
template <class T, int W, class P, class V> __device__ __forceinline__ P pack_sum(const V& v) {
  P s = (P)0;
  if constexpr (sizeof(T) == 2) {
    V ones;
#pragma unroll
    for (int i = 0; i < W; ++i) ones[i] = (T)1;
    s = half_dot<W>(v, ones, s);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) s += v[i];
  }
  return s;
}

/* Several sums over the S lanes of a row at once. Two (four) values a lane become one after a step (two)
 * of the butterfly, the even lanes going on with the first and the odd ones with the second (every
 * fourth lane with one of four), which takes 19 instructions for four values instead of 48. Steps
 * between lanes that agree in their lowest bits follow: rotations by 8 and 4 within 16 lanes, then the
 * swaps of half wavefronts. Lane l ends with the sum of value l % 2 (l % 4). */
constexpr int DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;
template <int S, class P> __device__ __forceinline__ P fold_apart(P v) {
  static_assert(S == 16 || S == 32 || S == 64, "16, 32 or 64 lanes");
  v += dpp_move<DPP_ROR8>(v);
  v += dpp_move<DPP_ROR4>(v);
  if constexpr (S >= 32) v = fold_swap16<AddOP>(v);
  if constexpr (S >= 64) v = fold_swap32<AddOP>(v);
  return v;
}
template <int S, class P> __device__ __forceinline__ P lanes_sum2(P a, P b) {
  const bool odd = threadIdx.x & 1;
  a += dpp_move<DPP_XOR1>(a);
  b += dpp_move<DPP_XOR1>(b);
  P v = odd ? b : a;
  v += dpp_move<DPP_XOR2>(v);
  return fold_apart<S>(v);
}
template <int S, class P> __device__ __forceinline__ P lanes_sum4(P a, P b, P c, P d) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  a += dpp_move<DPP_XOR1>(a);
  b += dpp_move<DPP_XOR1>(b);
  c += dpp_move<DPP_XOR1>(c);
  d += dpp_move<DPP_XOR1>(d);
  P lo = odd ? b : a, hi = odd ? d : c;
  lo += dpp_move<DPP_XOR2>(lo);
  hi += dpp_move<DPP_XOR2>(hi);
  return fold_apart<S>(high ? hi : lo);
}
/* value q of a lanes_sum2 or lanes_sum4 on all lanes: the q-th lane of every four */
template <int Q, class P> __device__ __forceinline__ P quad_lane(P v) { return dpp_move<Q * 0x55>(v); }

/* What the wavefronts of a row hand each other: a pivot near the mean of a wavefront's own elements, the
 * sums of x - pivot (`off`) and its square, and in the reverse those of e = dy * gain and e * (x - pivot).
 * Every wavefront takes its sums about a pivot of its own, so one exchange does for the mean and the
 * variance, without a difference of squares of values far from zero. */
enum { PART_OFF = 0, PART_SQUARE = 1, PART_E = 2, PART_EX = 3, PART_PIVOT = 4, PART_WORDS = 8 };
template <class P> struct alignas(32) NormPart { P v[PART_WORDS]; };
template <class P> struct NormStats {
  P back; /* x - mean is (x - pivot) + back */
  P r, mean_e, mean_eh;
};

/* A value of each of a row's wavefronts added up: lane i holds the (i % pow2)-th wavefront's, pow2 the next
 * power of two from gw. */
template <class P> __device__ __forceinline__ P waves_sum(P v, int gw) {
  v += dpp_move<DPP_XOR1>(v);
  if (gw > 2) v += dpp_move<DPP_XOR2>(v);
  if (gw > 4) v += dpp_move<DPP_HALF_MIRROR>(v);
  if (gw > 8) v += dpp_move<DPP_MIRROR>(v);
  return v;
}

/* The row's statistics from the parts of its wavefronts, which lie in LDS behind a barrier. `held`: how many
 * elements the wavefront of this lane's slot has (0 for a slot from gw on). All lanes get the same bits. */
template <bool REVERSE, class P>
__device__ __forceinline__ NormStats<P> norm_join(const NormPart<P>* parts, int slot, int gw, P held, P pivot, P inv_n, P eps) {
  const bool real = slot < gw;
  const NormPart<P>& part = parts[real ? slot : 0];
  const P first = parts[0].v[PART_PIVOT], off = part.v[PART_OFF], apart = part.v[PART_PIVOT] - first;
  NormStats<P> s;
  const P mean = waves_sum(real ? off + held * apart : (P)0, gw) * inv_n; /* above the first wavefront's pivot */
  const P by = apart - mean;                                             /* pivot - mean, for the slot's wavefront */
  const P square = waves_sum(real ? part.v[PART_SQUARE] + by * ((P)2 * off + held * by) : (P)0, gw) * inv_n;
  s.r = rsqrt_of((square < (P)0 ? (P)0 : square) + eps);
  s.back = pivot - first - mean;
  if constexpr (REVERSE) {
    const P e = part.v[PART_E];
    s.mean_e = waves_sum(real ? e : (P)0, gw) * inv_n;
    s.mean_eh = waves_sum(real ? part.v[PART_EX] + by * e : (P)0, gw) * inv_n * s.r;
  }
  return s;
}
template <bool REVERSE, class P>
__device__ __forceinline__ NormStats<P> norm_alone(P off, P square, P e, P ex, P inv_n, P eps) {
  NormStats<P> s;
  s.back = -off * inv_n;
  s.r = rsqrt_of(variance_of(square * inv_n, s.back) + eps);
  if constexpr (REVERSE) {
    s.mean_e = e * inv_n;
    s.mean_eh = (ex * inv_n + s.back * s.mean_e) * s.r;
  }
  return s;
}

/* The statistics of the row a wavefront has (part of) in registers. sum: of the elements `pivot_held` the pivot
 * is the mean of, over the lanes already; measure(pivot) gives a lane's sums about it. Half-precision
 * rows take their pivot from all elements: it is their mean as fp32 has it, and what its rounding leaves
 * over is sum - held * pivot, so no second sum of differences is needed. The other types take it from
 * a first pack a lane and add up the differences. */
template <class T, int SUB, bool REVERSE, class P, class F>
__device__ __forceinline__ NormStats<P> norm_stats(P sum, P inv_pivot_held, P held, P held_slot, int slot, int gw, NormPart<P>* slots, int mine,
                                                   P inv_n, P eps, F&& measure) {
  sum = lanes_allreduce<AddOP, SUB>(sum);
  P pivot = sum * inv_pivot_held;
  settle(pivot); /* rounded here: x - sum * inv in one step is not x minus what is handed on */
  P off = (P)0, square = (P)0, e = (P)0, ex = (P)0;
  measure(pivot, off, square, e, ex);
  constexpr bool WHOLE = sizeof(T) == 2;
  const bool alone = SUB < WAVE || gw == 1;
  if constexpr (SUB == 8) {
    off = WHOLE ? mix_fma((float)pivot, (float)-held, (float)sum) : lanes_allreduce<AddOP, SUB>(off);
    square = lanes_allreduce<AddOP, SUB>(square);
    if constexpr (REVERSE) {
      e = lanes_allreduce<AddOP, SUB>(e);
      ex = lanes_allreduce<AddOP, SUB>(ex);
    }
    return norm_alone<REVERSE>(off, square, e, ex, inv_n, eps);
  } else {
    P v;
    if constexpr (REVERSE) v = lanes_sum4<SUB>(off, square, e, ex);
    else if constexpr (WHOLE) v = lanes_allreduce<AddOP, SUB>(square);
    else v = lanes_sum2<SUB>(off, square);
    if constexpr (WHOLE) off = mix_fma((float)pivot, (float)-held, (float)sum);
    if (alone) {
      if constexpr (!WHOLE) off = quad_lane<PART_OFF>(v);
      return norm_alone<REVERSE>(off, WHOLE && !REVERSE ? v : quad_lane<PART_SQUARE>(v), quad_lane<PART_E>(v), quad_lane<PART_EX>(v), inv_n, eps);
    }
    const int l = threadIdx.x % WAVE;
    if (l <= PART_PIVOT) {
      if (WHOLE && l == PART_OFF) v = off;
      slots[mine].v[l] = l == PART_PIVOT ? pivot : v;
    }
    lds_barrier();
    return norm_join<REVERSE>(slots, slot, gw, held_slot, pivot, inv_n, eps);
  }
}

/* Where a thread of a launch belongs: rows_here rows a workgroup, held by G lanes each. SINGLE: one row a
 * workgroup, held by all of it. */
template <int SUB, bool SINGLE = false> struct NormPlace {
  int G, rows_here, sub, base_wave, mine, slot;
  __device__ __forceinline__ explicit NormPlace(int gw) {
    G = SUB < WAVE ? SUB : SINGLE ? (int)blockDim.x : gw * WAVE;
    rows_here = SINGLE ? 1 : (int)blockDim.x / G;
    sub = SINGLE ? 0 : threadIdx.x / G;
    base_wave = sub * gw;
    mine = (int)threadIdx.x / WAVE - base_wave;
    slot = threadIdx.x & (gw > 8 ? 15 : gw > 4 ? 7 : gw > 2 ? 3 : 1);
  }
};

/* ------------------------------------------------------------------ forward */

/* SUB <= 64: a wavefront or a part of one holds a row; SUB = ROW_A_BLOCK: the workgroup does. Once x - pivot
 * is taken the registers of x are free again: a workgroup that walks several rows has the next row's
 * loads on their way while this one is reduced and written. */
constexpr int ROW_A_BLOCK = 1024;
template <class T, int W, int SUB_, int NV, bool LOOSE, bool KEEP>
__global__ __launch_bounds__(NORM_BLOCK) void layernorm_fwd_rows(
    const T* x, const T* gain, const T* bias, T* y, typename precision<T>::type eps, size_t m, size_t n) {
  constexpr bool SINGLE = SUB_ == ROW_A_BLOCK;
  constexpr int SUB = SINGLE ? WAVE : SUB_;
  using P = typename precision<T>::type;
  using Row = NormRow<T, W, SUB, NV, LOOSE>;
  using V = typename Row::V;
  constexpr int PIVOT_PACKS = sizeof(T) == 2 ? NV : 1;
  __shared__ NormPart<P> parts[2][SINGLE ? NORM_WAVES : 1];
  const int gw = SINGLE ? (int)blockDim.x / WAVE : 1;
  const NormPlace<SUB, SINGLE> at(gw);
  const Row rw(n, at.G, SINGLE ? (int)threadIdx.x : (int)threadIdx.x % SUB);

  const size_t stride = (size_t)gridDim.x * at.rows_here;
  size_t base = (size_t)blockIdx.x * at.rows_here;
  auto fetch = [&](V (&xs)[NV], size_t from) { /* a row beyond the last reads the last */
    const size_t row = from + at.sub, real = row < m ? row : m - 1;
    rw.template fetch<KEEP>(x + real * n, xs, rw.ends(real, m, n));
  };
  V xs[NV], gv[NV], bv[NV]; /* as stored, widened where they are used */
  fetch(xs, base);
  rw.fetch_vector(gain, gv, (T)1);
  rw.fetch_vector(bias, bv, (T)0);
  const P inv_n = (P)1 / (P)n;
  const P held = (P)rw.held(at.mine, NV, n), pivot_held = (P)rw.held(at.mine, PIVOT_PACKS, n);
  const P inv_pivot_held = pivot_held > (P)0 ? (P)1 / pivot_held : (P)0, held_slot = (P)rw.held(at.slot, NV, n);
  P one = (P)1;
  settle(one);

  int parity = 0;
  for (; base < m; base += stride, parity ^= 1) {
    rw.mask(xs);
    P s = (P)0;
#pragma unroll
    for (int k = 0; k < PIVOT_PACKS; ++k) {
      const P sk = pack_sum<T, W, P>(xs[k]);
      s += rw.inside(k) ? sk : (P)0;
    }
    P d[NV][W];
    const NormStats<P> st = norm_stats<T, SUB, false>(s, inv_pivot_held, held, held_slot, at.slot, gw, parts[parity], at.mine, inv_n, eps,
                                                      [&](P pivot, P& off, P& square, P&, P&) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) d[k][i] = mix_less<T, P>(xs[k][i], pivot, one);
        if (rw.cut(k))
#pragma unroll
          for (int i = 0; i < W; ++i) d[k][i] = i < rw.rp.last ? d[k][i] : (P)0;
      }
      if (base + stride < m) fetch(xs, base + stride);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        P tk = (P)0, qk = (P)0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if constexpr (sizeof(T) != 2) tk += d[k][i];
          qk += d[k][i] * d[k][i];
        }
        off += rw.inside(k) ? tk : (P)0;
        square += rw.inside(k) ? qk : (P)0;
      }
    });
    const size_t row = base + at.sub;
    if (row < m) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (rw.inside(k)) {
          P out[W];
#pragma unroll
          for (int i = 0; i < W; ++i) out[i] = (d[k][i] + st.back) * mix_fma(gv[k][i], st.r, (P)0) + (P)bv[k][i];
          rw.rp.store(y + row * n, rw.pack(k), out);
        }
      }
    }
  }
}

/* ------------------------------------------------------------------ reverse */

/* Persistent workgroups walk the rows; with PAIR the next rows' x and dy are on their way (into a second
 * set of registers) while these are reduced, behind a barrier that orders LDS traffic only, and written.
 * The columns' sums for dg and db stay in registers; at the end the rows of a workgroup are folded in
 * order and it leaves ONE partial row, or, where it is the only workgroup, dg and db themselves. BLOCK 512
 * leaves a lane 256 registers. */
template <class T, int W, int SUB, int NV, bool BLEND, bool LOOSE, bool PAIR, int BLOCK>
__global__ __launch_bounds__(BLOCK) void layernorm_rev_rows(
    const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, typename precision<T>::type* partials,
    typename precision<T>::type eps, typename precision<T>::type alpha, size_t m, size_t n, int gw) {
  using P = typename precision<T>::type;
  using Row = NormRow<T, W, SUB, NV, LOOSE>;
  using V = typename Row::V;
  constexpr int PIVOT_PACKS = sizeof(T) == 2 ? NV : 1;
  constexpr int WAVES = BLOCK / WAVE;
  __shared__ NormPart<P> parts[2][SUB < WAVE ? 1 : WAVES];
  __shared__ P comb[BLOCK * W];
  const P inv_n = (P)1 / (P)n;
  const NormPlace<SUB> at(gw);
  const Row rw(n, at.G, threadIdx.x % at.G);
  const P held = (P)rw.held(at.mine, NV, n), pivot_held = (P)rw.held(at.mine, PIVOT_PACKS, n);
  const P inv_pivot_held = pivot_held > (P)0 ? (P)1 / pivot_held : (P)0, held_slot = (P)rw.held(at.slot, NV, n);
  P one = (P)1;
  settle(one);

  V gv[NV];
  rw.fetch_vector(gain, gv, (T)1);
  P acc_g[NV][W], acc_b[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < W; ++i) acc_g[k][i] = acc_b[k][i] = (P)0;

  const size_t stride = (size_t)gridDim.x * at.rows_here;
  auto fetch = [&](V (&xs)[NV], V (&ds)[NV], size_t base) { /* a row beyond the last reads the last */
    const size_t row = base + at.sub, real = row < m ? row : m - 1;
    const bool end = rw.ends(real, m, n);
    rw.template fetch<false>(x + real * n, xs, end);
    rw.template fetch<false>(dy + real * n, ds, end);
  };
  auto finish = [&](V (&xs)[NV], V (&ds)[NV], size_t base, NormPart<P>* slots) {
    rw.mask(xs);
    rw.mask(ds);
    P s = (P)0;
#pragma unroll
    for (int k = 0; k < PIVOT_PACKS; ++k) {
      const P sk = pack_sum<T, W, P>(xs[k]);
      s += rw.inside(k) ? sk : (P)0;
    }
    P t[NV][W];
    const NormStats<P> st = norm_stats<T, SUB, true>(s, inv_pivot_held, held, held_slot, at.slot, gw, slots + (SUB < WAVE ? 0 : at.base_wave), at.mine,
                                                     inv_n, eps, [&](P pivot, P& off, P& square, P& e, P& ex) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) t[k][i] = mix_less<T, P>(xs[k][i], pivot, one);
        if (rw.cut(k))
#pragma unroll
          for (int i = 0; i < W; ++i) t[k][i] = i < rw.rp.last ? t[k][i] : (P)0;
        P tk = (P)0, qk = (P)0, ek = (P)0, fk = (P)0;
        if constexpr (sizeof(T) == 2) ek = half_dot<W>(ds[k], gv[k], ek);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const P p = mix_mul<T, P>(ds[k][i], gv[k][i]);
          if constexpr (sizeof(T) != 2) {
            tk += t[k][i];
            ek += p;
          }
          qk += t[k][i] * t[k][i];
          fk += p * t[k][i];
        }
        const bool in = rw.inside(k);
        off += in ? tk : (P)0;
        square += in ? qk : (P)0;
        e += in ? ek : (P)0;
        ex += in ? fk : (P)0;
      }
    });
    const P back = st.back * st.r, re = st.r * st.mean_e, rh = st.r * st.mean_eh; /* h = (x - mean) * r = t * r + back */
    const size_t row = base + at.sub;
    if (row < m) {
      T* out_row = dx + row * n;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (rw.inside(k)) {
          P out[W];
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const P h = t[k][i] * st.r + back;
            out[i] = mix_mul<T, P>(ds[k][i], gv[k][i]) * st.r - re - h * rh;
            acc_g[k][i] = mix_fma(ds[k][i], h, acc_g[k][i]);
            acc_b[k][i] = mix_add<T, P>(ds[k][i], acc_b[k][i], one);
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

  size_t base = (size_t)blockIdx.x * at.rows_here;
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
      if (base + stride >= m) break;
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
  const int groups = SUB < WAVE ? (int)blockDim.x / WAVE : at.rows_here;
  const int width = at.G; /* lanes a group */
  const size_t apart = partial_apart<T>(n);
  P* out = partials + (size_t)blockIdx.x * 2 * apart;
  /* a pack of sums of column p * W on; `alone`: in the results' type, added to what they hold */
  const bool alone = gridDim.x == 1;
  auto leave = [&](int which, int p, const P (&a)[W]) {
    if (!alone) {
#pragma unroll
      for (int i = 0; i < W; i += PACK_BYTES / (int)sizeof(P)) {
        P some[PACK_BYTES / sizeof(P)];
#pragma unroll
        for (int j = 0; j < PACK_BYTES / (int)sizeof(P); ++j) some[j] = a[i + j];
        store_pack<P, PACK_BYTES / (int)sizeof(P)>(out + which * apart + (size_t)p * W + i, some);
      }
      return;
    }
    T* to = which ? db : dg;
    if (!to) return;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i >= rw.rp.valid(p)) break;
      T* cell = to + (size_t)p * W + i;
      double t = (double)a[i];
      if constexpr (BLEND) t += (double)alpha * (double)*cell;
      *cell = (T)t;
    }
  };
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
        if (rw.inside(k)) leave(which, rw.pack(k), a);
        continue;
      }
      const int group = SUB < WAVE ? (int)threadIdx.x / WAVE : at.sub, l = threadIdx.x % width;
      __syncthreads(); /* the sums before have been read */
      if (SUB == WAVE || threadIdx.x % WAVE < (unsigned)SUB)
#pragma unroll
        for (int i = 0; i < W; ++i) comb[(group * width + l) * W + i] = a[i];
      __syncthreads();
      const int p = k * width + (int)threadIdx.x;
      if ((int)threadIdx.x < width && p < rw.rp.npk) {
#pragma unroll
        for (int i = 0; i < W; ++i) a[i] = (P)0;
        for (int g = 0; g < groups; ++g)
#pragma unroll
          for (int i = 0; i < W; ++i) a[i] += comb[(g * width + threadIdx.x) * W + i];
        leave(which, p, a);
      }
    }
}

/* ------------------------------------------------------------------ dg and db from the partial rows */

/* The partial rows added in a fixed order in fp64. A workgroup owns a 128-byte line of columns; its 32 slices
 * take the rows in turn, a 16-byte load of eight rows on its way at once. Bound by the latency of a launch that
 * waits for the one before it: 4 us behind the row pass (r32 [8192, 4096], 256 partial rows; 64 slices 0.5 us
 * more, 128 1.7 more, 16 0.3; at 100 partial rows of r16 [100, 12288] the whole reverse 14.3 us at 32 slices,
 * 15.7 at 64, 13.8 at 16). */
constexpr int NORM_FINISH_LANES = 8, NORM_FINISH_SLICES = 32;
template <class T>
__global__ __launch_bounds__(NORM_FINISH_LANES * NORM_FINISH_SLICES) void layernorm_grads_finish(
    const typename precision<T>::type* partials, T* dg, T* db, double alpha, int rows, size_t n, unsigned first_block) {
  using P = typename precision<T>::type;
  constexpr int CW = PACK_BYTES / (int)sizeof(P), COLS = NORM_FINISH_LANES * CW;
  __shared__ double part[NORM_FINISH_SLICES][COLS + 1];
  const int c = threadIdx.x % NORM_FINISH_LANES, slice = threadIdx.x / NORM_FINISH_LANES;
  const size_t apart = partial_apart<T>(n), width = 2 * apart;
  const size_t block = first_block + blockIdx.x, col = (block * NORM_FINISH_LANES + c) * CW;
  double s[CW];
#pragma unroll
  for (int i = 0; i < CW; ++i) s[i] = 0.0;
  if (col < width) { /* a whole number of packs */
    constexpr int U = 8;
    for (int p = slice; p < rows; p += U * NORM_FINISH_SLICES) {
      P v[U][CW];
#pragma unroll
      for (int u = 0; u < U; ++u) { /* beyond the last row: this slice's first, left out */
        const int q = p + u * NORM_FINISH_SLICES;
        load_pack<P, CW>(partials + (size_t)(q < rows ? q : p) * width + col, v[u]);
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
  const size_t at = block * COLS + threadIdx.x, j = at < apart ? at : at - apart;
  if (threadIdx.x < COLS && at < width && j < n) {
    T* out = at < apart ? dg : db;
    if (!out) return;
    out += j;
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
  return layernorm_partial_rows(m) * 2 * partial_apart<T>(n) * sizeof(typename precision<T>::type);
}

/* How a launch holds its rows: `sub` lanes a row below 64, else `gw` wavefronts, `nv` packs a lane, `rows`
 * rows a workgroup at a time, `per_cu` workgroups a compute unit that walk them. nv = 0: rows too long for
 * registers. The choices come from sweeps of all of these (interleaved repeats, launches on operands
 * beyond the caches):
 *   two packs a lane rather than one (r16 [4096, 8192] forward 24.3 us against 25.7, [16384, 2048] reverse 42.7
 *   against 45.9) or four (27.2, 42.6), except where the workgroup would pass 16 wavefronts;
 *   as many workgroups a unit as make 12 wavefronts of four-byte rows (r32 [4099, 5120] 29.9 us at ten, 30.6 at
 *   twenty) and 20 of two-byte ones (r16 [8192, 2560] 16.6 at 18, 17.9 at 12, 18.5 at 30), whose lanes hold
 *   half the bytes;
 *   forward rows of more than 64 KiB, r16 rows of more than 32 KiB, read three times: what is left of the registers
 *   spills (r32 [1024, 32768] 78 us against 87, r16 39 against 59).
 * The reverse holds twice the operands and the sums of the columns, and spills in rows of more than 32 KiB (r32 12 registers
 * of a lane, 21 ragged, r64 37 to 55; r16 of more than 32 KiB 149 to 205), but reading a row's operands five times
 * and the sums from memory costs more for as long as a workgroup can hold the row, 64 KiB in every type: r32 [2034,
 * 12288] 71 us against 199, r64 [1525, 8192] 93 against 173, r16 [2500, 20000] 224 against 624. */
struct NormPlan {
  int sub, nv, gw, rows, per_cu;
};
inline unsigned norm_grid(const NormPlan& p, size_t m) {
  const size_t need = (m + p.rows - 1) / p.rows, cap = (size_t)compute_units() * p.per_cu;
  return (unsigned)(cap < need ? cap : need);
}
inline unsigned norm_block(const NormPlan& p) { return (unsigned)(p.rows * (p.sub < WAVE ? p.sub : p.gw * WAVE)); }
inline int norm_waves(size_t packs, int nv) { return (int)((packs + (size_t)nv * WAVE - 1) / ((size_t)nv * WAVE)); }

template <class T> inline NormPlan layernorm_forward_plan(size_t packs) {
  if (packs <= 8) return {8, 1, 1, 64, 4};
  if (packs <= 16) return {16, 1, 1, 32, 4};
  if (packs <= 32) return {32, 1, 1, 16, 4};
  if (packs <= 64) return {WAVE, 1, 1, 8, 4};
  if (packs <= 128) return {WAVE, 2, 1, 8, 3};
  const int nv = packs <= 1024 || sizeof(T) == 2 ? 2 : 4, gw = norm_waves(packs, nv), waves = sizeof(T) == 2 ? 20 : 12;
  if (gw > NORM_WAVES) return {WAVE, 0, 0, 0, 0};
  return {WAVE, nv, gw, 1, waves / gw ? waves / gw : 1};
}
/* plain: nothing is blended, and rows are whole packs on aligned addresses */
template <class T> inline NormPlan layernorm_reverse_plan(size_t packs, bool plain) {
  if (packs <= 8) return {8, 1, 1, 64, 2};
  if (packs <= 16) return {16, 1, 1, 32, 2};
  if (packs <= 32) return {32, 1, 1, 16, 2};
  if (packs <= 64) return {WAVE, 1, 1, 16, 1};
  /* r16 rows of more than 24 KiB: four packs a lane and no more than eight wavefronts, which leaves room for the
   * next row ([3051, 16384] 68.6 us, two packs on sixteen wavefronts 72.0; 300 rows 28.0 and 25.1), but not for what
   * a blend reads too (114 us against 86) or a cut pack takes ([3051, 16383] 96.8 against 87.3) */
  const int nv = packs <= (sizeof(T) == 2 && plain ? 1536 : 2048) ? 2 : 4, gw = norm_waves(packs, nv), rows = gw < 8 ? 8 / gw : 1;
  if (gw > NORM_WAVES) return {WAVE, 0, 0, 0, 0};
  return {WAVE, nv, gw, rows, sizeof(T) == 2 && nv == 2 && gw > 1 && gw <= 8 ? 2 : 1};
}

template <class T>
inline void layernorm_forward_as(const NormPlan& plan, const T* x, const T* gain, const T* bias, T* y, double eps, size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  const bool loose = !(aligned16(x) && aligned16(y) && (!gain || aligned16(gain)) && (!bias || aligned16(bias)) && n % W == 0);
  /* as RMSNorm's forward: the reverse reads x again */
  const bool keep = keep_input(m * n * sizeof(T));
  if (plan.nv == 0) {
    const size_t cap = (size_t)compute_units() * 2;
    const dim3 grid((unsigned)(m < cap ? m : cap)), block(STREAM_THREADS);
    if (loose) layernorm_fwd_stream<T, W, true><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
    else layernorm_fwd_stream<T, W, false><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
  } else {
    const dim3 grid(norm_grid(plan, m)), block(norm_block(plan));
    auto go = [&]<int SUB, int NV>() {
      auto kept = [&]<bool KEEP>() {
        if (loose) layernorm_fwd_rows<T, W, SUB, NV, true, KEEP><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
        else layernorm_fwd_rows<T, W, SUB, NV, false, KEEP><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
      };
      if (keep) kept.template operator()<true>();
      else kept.template operator()<false>();
    };
    if (plan.sub == 8) go.template operator()<8, 1>();
    else if (plan.sub == 16) go.template operator()<16, 1>();
    else if (plan.sub == 32) go.template operator()<32, 1>();
    else if (plan.nv == 1) go.template operator()<WAVE, 1>();
    else if (plan.gw == 1) go.template operator()<WAVE, 2>();
    else if (plan.nv == 2) go.template operator()<ROW_A_BLOCK, 2>();
    else if constexpr (sizeof(T) != 2) go.template operator()<ROW_A_BLOCK, 4>();
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

/* A few rows: one workgroup takes them all in two turns or up to four, and one launch of two is saved, as long as
 * there is little to read: it walks alone what several would take at once. One against two launches, us:
 *   two turns     r32 [2,8192] 6.1, 7.7   r64 [2,4096] 7.8, 8.2   r16 [2,16384] 8.1, 9.4   beyond 64 KiB: r32
 *                 [2,12288] 9.6, 9.7   [2,16384] 12.7, 11.8   r64 [2,8192] 19.6, 16.9
 *   three, four   r16 [3,8192] 6.7, 7.7   r64 [3,2048] 6.7, 7.5   r32 [3,4096] 5.7, 7.6   beyond 48 KiB: r32 [4,4096]
 *                 6.7, 7.5   r16 [16,2048] 9.2, 8.2   r64 [4,2048] 8.1, 7.5   r32 [4,16384] 22.8, 11.9 */
inline bool layernorm_one_workgroup(size_t workgroups, size_t bytes) {
  return workgroups <= 2 ? bytes <= 65536 : workgroups <= 4 && bytes <= 49152;
}

template <class T> inline bool layernorm_reverse_loose(const T* x, const T* gain, const T* dy, const T* dx, size_t n) {
  return !(aligned16(x) && aligned16(dy) && aligned16(dx) && (!gain || aligned16(gain)) && n % (PACK_BYTES / sizeof(T)) == 0);
}

template <class T>
inline void layernorm_reverse_as(const NormPlan& plan, const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, void* scratch, double eps, double alpha,
                                 size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  P* partials = static_cast<P*>(scratch);
  size_t rows = 0;
  if (m > 0) {
    const bool loose = layernorm_reverse_loose(x, gain, dy, dx, n);
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
      if (layernorm_one_workgroup(rows, m * n * sizeof(T))) rows = 1;
      require(rows <= layernorm_partial_rows(m), "layernorm reverse: more partial rows than the workspace holds");
      const dim3 grid((unsigned)rows), block(norm_block(plan));
      auto go = [&]<int SUB, int NV, bool PAIR, int BLOCK>() {
        auto as = [&]<bool BLEND, bool LOOSE>() {
          layernorm_rev_rows<T, W, SUB, NV, BLEND, LOOSE, PAIR, BLOCK><<<grid, block, 0, stream>>>(x, gain, dy, dx, dg, db, partials, (P)eps, (P)alpha, m, n, plan.gw);
        };
        if (alpha != 0.0) { if (loose) as.template operator()<true, true>(); else as.template operator()<true, false>(); }
        else { if (loose) as.template operator()<false, true>(); else as.template operator()<false, false>(); }
      };
      /* the next rows' loads in flight where the registers hold them (r32 [8192, 4096] 70.6 us against 73.4
       * without; r16 at two packs a lane takes 153 registers then, one workgroup a unit instead of two: [16384, 2048]
       * 46.5 against 41.1) */
      if (plan.sub == 8) go.template operator()<8, 1, false, 512>();
      else if (plan.sub == 16) go.template operator()<16, 1, false, 512>();
      else if (plan.sub == 32) go.template operator()<32, 1, false, 512>();
      else if (plan.nv == 1) go.template operator()<WAVE, 1, false, 1024>();
      else if (plan.nv == 2) {
        if constexpr (sizeof(T) != 2) go.template operator()<WAVE, 2, true, 1024>();
        else if (block.x <= 512) go.template operator()<WAVE, 2, false, 512>();
        else go.template operator()<WAVE, 2, false, 1024>();
      } else {
        if constexpr (sizeof(T) == 2) {
          if (block.x <= 512) { /* the plan's plain rows */
            require(alpha == 0.0 && !loose, "layernorm reverse: a plan for plain rows");
            layernorm_rev_rows<T, W, WAVE, 4, false, false, true, 512><<<grid, block, 0, stream>>>(x, gain, dy, dx, dg, db, partials, (P)eps, (P)alpha, m, n, plan.gw);
          } else go.template operator()<WAVE, 4, false, 1024>();
        } else go.template operator()<WAVE, 4, false, 1024>();
      }
    }
    MP_CHECK_LAUNCH();
  }
  if ((!dg && !db) || (m > 0 && plan.nv != 0 && rows == 1)) return;
  constexpr size_t cols = NORM_FINISH_LANES * PACK_BYTES / sizeof(P);
  in_launches((2 * partial_apart<T>(n) + cols - 1) / cols, [&](dim3 grid, unsigned first) {
    layernorm_grads_finish<T><<<grid, dim3(NORM_FINISH_LANES * NORM_FINISH_SLICES), 0, stream>>>(partials, dg, db, alpha, (int)rows, n, first);
    MP_CHECK_LAUNCH();
  });
}

template <class T>
inline void layernorm_reverse(const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, void* scratch, double eps, double alpha,
                              size_t m, size_t n, hipStream_t stream) {
  if (n == 0) return;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  require(n <= 0x40000000ull, "layernorm reverse: row length must not exceed 2^30");
  require(dg != db || dg == nullptr, "layernorm reverse: gain_grads and bias_grads must be different vectors");
  require(m == 0 || scratch != nullptr, "layernorm reverse: scratch must hold mpLayernormReverseScratchBytes bytes");
  require(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "layernorm reverse: scratch must be aligned to its sums in packs (16-byte aligned)");
  const bool plain = alpha == 0.0 && !layernorm_reverse_loose(x, gain, dy, dx, n);
  layernorm_reverse_as<T>(layernorm_reverse_plan<T>((n + W - 1) / W, plain), x, gain, dy, dx, dg, db, scratch, eps, alpha, m, n, stream);
}

}  // namespace mp

#endif
#endif
