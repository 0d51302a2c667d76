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
    const P pivot = group_allreduce<AddOP, G>(s, slots[0], lane) * inv_n;
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
    const P pivot = group_allreduce<AddOP, G>(s, slots[0], lane) * inv_n;
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

/* ------------------------------------------------------------------ dg and db from the partial rows */

/* Column j of the partial rows (2n of them: dg's, then db's), added in a fixed order in fp64. */
template <class T>
__global__ __launch_bounds__(256) void layernorm_grads_finish(
    const typename precision<T>::type* partials, T* dg, T* db, double alpha, int rows, size_t n) {
  const size_t col = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= 2 * n) return;
  T* out = col < n ? dg : db;
  if (!out) return;
  out += col < n ? col : col - n;
  double t = 0.0;
  for (int p = 0; p < rows; ++p) t += (double)partials[(size_t)p * 2 * n + col];
  if (alpha != 0.0) t += alpha * (double)*out;
  *out = (T)t;
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

template <class T>
inline void layernorm_forward(const T* x, const T* gain, const T* bias, T* y, double eps, size_t m, size_t n, hipStream_t stream) {
  if (m == 0 || n == 0) return;
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  require(n <= 0x40000000ull, "layernorm: row length must not exceed 2^30");
  const bool loose = !(aligned16(x) && aligned16(y) && (!gain || aligned16(gain)) && (!bias || aligned16(bias)) && n % W == 0);
  const size_t cap = (size_t)compute_units() * 2;
  const dim3 grid((unsigned)(m < cap ? m : cap)), block(STREAM_THREADS);
  if (loose) layernorm_fwd_stream<T, W, true><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
  else layernorm_fwd_stream<T, W, false><<<grid, block, 0, stream>>>(x, gain, bias, y, (P)eps, m, n);
  MP_CHECK_LAUNCH();
}

template <class T>
inline void layernorm_reverse(const T* x, const T* gain, const T* dy, T* dx, T* dg, T* db, void* scratch, double eps, double alpha,
                              size_t m, size_t n, hipStream_t stream) {
  if (n == 0) return;
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  require(n <= 0x40000000ull, "layernorm reverse: row length must not exceed 2^30");
  require(m == 0 || scratch != nullptr, "layernorm reverse: scratch must hold mpLayernormReverseScratchBytes bytes");
  P* partials = static_cast<P*>(scratch);
  const size_t rows = layernorm_partial_rows(m);
  if (m > 0) {
    const bool loose = !(aligned16(x) && aligned16(dy) && aligned16(dx) && (!gain || aligned16(gain)) && n % W == 0);
    const dim3 grid((unsigned)rows), block(STREAM_THREADS);
    auto go = [&]<bool BLEND, bool LOOSE>() {
      layernorm_rev_stream<T, W, BLEND, LOOSE><<<grid, block, 0, stream>>>(x, gain, dy, dx, partials, (P)eps, (P)alpha, m, n);
    };
    if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
    else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
    MP_CHECK_LAUNCH();
  }
  if (!dg && !db) return;
  layernorm_grads_finish<T><<<dim3((unsigned)((2 * n + 255) / 256)), dim3(256), 0, stream>>>(partials, dg, db, alpha, (int)rows, n);
  MP_CHECK_LAUNCH();
}

}  // namespace mp

#endif
#endif
