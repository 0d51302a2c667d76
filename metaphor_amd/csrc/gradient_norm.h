/*
 * The norm of many tensors taken as one vector, and scaling them down to a largest norm. The reference
 * has neither; its optimisers walk the leaves of the graph (src/optm/optimizer.zig:56-64). Math:
 *   norm = sqrt(sum over all tensors and elements of g^2 + alpha * norm^2)
 *   out  = g * min(1, max_norm / norm)
 * Squares are added in fp64 whatever the storage type, so neither large nor tiny r16 / r32 gradients
 * overflow or vanish, and in a fixed order, so the norm does not change from run to run. The norm is a
 * double on the device; nothing waits for the host.
 *
 * The tensors' addresses and sizes travel as kernel arguments, NORM_TENSORS of them a launch: nothing
 * is copied to the device and a captured launch keeps its own table. A table's work is cut into pieces of
 * NORM_PIECE bytes that the workgroups take in turn; each leaves one partial sum in the workspace.
 */
#ifndef MP_GRADIENT_NORM_H
#define MP_GRADIENT_NORM_H

#include "row_dispatch.h"

#if defined(__cplusplus) && defined(__HIPCC__)

namespace mp {

constexpr int NORM_TENSORS = 96, NORM_THREADS = 256;
constexpr size_t NORM_PIECE = 16384, NORM_PARTIALS = 2048;

template <class T> struct NormTable {
  const T* src[NORM_TENSORS];
  T* dst[NORM_TENSORS];
  unsigned long long size[NORM_TENSORS];
  unsigned first[NORM_TENSORS + 1]; /* the number of the tensor's first piece; [count] is the end */
  int count;
};

/* The tensor that piece `q` belongs to: the last one whose first piece is not behind it. Tensors of no
 * elements have no piece. */
template <class T> __device__ __forceinline__ int norm_tensor_of(const NormTable<T>& t, unsigned q) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= q) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

/* Sum over the workgroup's threads; every thread gets it. */
__device__ __forceinline__ double norm_block_sum(double s, double* slots) {
  s = wave_allreduce<AddOP>(s);
  if (threadIdx.x % WAVE == 0) slots[threadIdx.x / WAVE] = s;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < NORM_THREADS / WAVE; ++w) t += slots[w];
  return t;
}

template <class T> __global__ __launch_bounds__(NORM_THREADS) void gradient_squares(NormTable<T> t, double* partials) {
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  constexpr size_t PIECE = NORM_PIECE / sizeof(T);
  __shared__ double slots[NORM_THREADS / WAVE];
  double s = 0.0;
  for (unsigned q = blockIdx.x; q < t.first[t.count]; q += gridDim.x) {
    const int k = norm_tensor_of(t, q);
    const size_t lo = (size_t)(q - t.first[k]) * PIECE, size = t.size[k], hi = lo + PIECE < size ? lo + PIECE : size;
    const T* src = t.src[k];
    for (size_t i = lo + (size_t)threadIdx.x * W; i < hi; i += NORM_THREADS * W) {
      if (i + W <= hi) {
        double v[W];
        load_pack_loose<T, W>(src + i, v);
#pragma unroll
        for (int j = 0; j < W; ++j) s += v[j] * v[j];
      } else {
        for (size_t j = i; j < hi; ++j) s += (double)src[j] * (double)src[j];
      }
    }
  }
  s = norm_block_sum(s, slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

/* The partial sums, added by one workgroup in a fixed order. */
__device__ __forceinline__ double norm_of(const double* partials, unsigned count, double* slots) {
  double s = 0.0;
  for (unsigned i = threadIdx.x; i < count; i += NORM_THREADS) s += partials[i];
  return norm_block_sum(s, slots);
}

static __global__ __launch_bounds__(NORM_THREADS) void gradient_norm_finish(const double* partials, unsigned count, double alpha, double* norm) {
  __shared__ double slots[NORM_THREADS / WAVE];
  double s = norm_of(partials, count, slots);
  if (threadIdx.x == 0) {
    if (alpha != 0.0) s += alpha * norm[0] * norm[0];
    norm[0] = ::sqrt(s);
  }
}

template <class T> __global__ __launch_bounds__(NORM_THREADS) void gradient_scaled(NormTable<T> t, const double* norm, double max_norm) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  constexpr size_t PIECE = NORM_PIECE / sizeof(T);
  const double total = norm[0];
  const P factor = total <= max_norm ? (P)1 : (P)(max_norm / total);
  for (unsigned q = blockIdx.x; q < t.first[t.count]; q += gridDim.x) {
    const int k = norm_tensor_of(t, q);
    const size_t lo = (size_t)(q - t.first[k]) * PIECE, size = t.size[k], hi = lo + PIECE < size ? lo + PIECE : size;
    const T* src = t.src[k];
    T* dst = t.dst[k];
    if (src == dst && total <= max_norm) continue; /* nothing to do in place */
    for (size_t i = lo + (size_t)threadIdx.x * W; i < hi; i += NORM_THREADS * W) {
      if (i + W <= hi) {
        P v[W];
        load_pack_loose<T, W>(src + i, v);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] *= factor;
        store_pack_nt_loose<T, W>(dst + i, v);
      } else {
        for (size_t j = i; j < hi; ++j) dst[j] = (T)((P)src[j] * factor);
      }
    }
  }
}

/* ------------------------------------------------------------------ host dispatch */

/* f(table, pieces) for the tensors in groups of NORM_TENSORS. */
template <class T, class F>
inline void for_norm_tables(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count, F&& f) {
  constexpr size_t PIECE = NORM_PIECE / sizeof(T);
  for (size_t base = 0; base < count; base += NORM_TENSORS) {
    NormTable<T> t;
    t.count = (int)(count - base < (size_t)NORM_TENSORS ? count - base : (size_t)NORM_TENSORS);
    size_t pieces = 0;
    for (int k = 0; k < t.count; ++k) {
      t.src[k] = static_cast<const T*>(grads[base + k]);
      t.dst[k] = outs ? const_cast<T*>(static_cast<const T*>(outs[base + k])) : nullptr;
      t.size[k] = sizes[base + k];
      t.first[k] = (unsigned)pieces;
      pieces += (t.size[k] + PIECE - 1) / PIECE;
    }
    t.first[t.count] = (unsigned)pieces;
    f(t, (unsigned)pieces);
  }
}

inline size_t norm_tables(size_t count) { return (count + NORM_TENSORS - 1) / NORM_TENSORS; }

/* Partial sums a table may leave: all of them are added by one workgroup. */
inline size_t norm_partials(size_t count) {
  const size_t each = NORM_PARTIALS / (norm_tables(count) ? norm_tables(count) : 1);
  return each < 64 ? 64 : each;
}
inline size_t gradient_norm_scratch_bytes(size_t count) { return norm_tables(count) * norm_partials(count) * sizeof(double); }

/* Every argument, before the first launch. outs NULL where none are written. */
template <class T>
inline void gradient_check(const void* grads, const void* outs, const void* sizes, const void* norm, size_t count) {
  require(count == 0 || (grads != nullptr && sizes != nullptr), "gradient norm: addresses and sizes must not be NULL");
  require(norm != nullptr && reinterpret_cast<uintptr_t>(norm) % sizeof(double) == 0, "gradient norm: the norm is one aligned double on the device");
  size_t pieces = 0;
  for (size_t k = 0; k < count; ++k) {
    const len_t size = static_cast<const len_t*>(sizes)[k];
    if (size == 0) continue;
    require(static_cast<const void* const*>(grads)[k] != nullptr, "gradient norm: a tensor's address is NULL");
    require(!outs || static_cast<const void* const*>(outs)[k] != nullptr, "gradient clip: a result's address is NULL");
    require(size < 0x1000000000000ull, "gradient norm: a tensor's size is out of range");
    pieces += (size * sizeof(T) + NORM_PIECE - 1) / NORM_PIECE;
    require(pieces < 0x7fffffffull, "gradient norm: too many elements");
  }
}

inline void gradient_check_scratch(const void* scratch, size_t count) {
  require(count == 0 || scratch != nullptr, "gradient norm: scratch must hold mpGradientNormScratchBytes bytes");
  require(reinterpret_cast<uintptr_t>(scratch) % sizeof(double) == 0, "gradient norm: scratch must be 8-byte aligned");
}

inline void gradient_check_limit(const void* outs, double max_norm, size_t count) {
  require(count == 0 || outs != nullptr, "gradient clip: the results' addresses must not be NULL");
  require(max_norm >= 0.0, "gradient clip: the largest norm must not be negative or NaN");
}

/* returns how many partial sums there are */
template <class T>
inline unsigned gradient_squares_all(const void* grads, const void* sizes, void* scratch, size_t count, hipStream_t stream) {
  double* partials = static_cast<double*>(scratch);
  unsigned used = 0;
  for_norm_tables<T>(static_cast<const void* const*>(grads), nullptr, static_cast<const len_t*>(sizes), count, [&](const NormTable<T>& t, unsigned pieces) {
    if (pieces == 0) return;
    const unsigned cap = (unsigned)norm_partials(count), blocks = pieces < cap ? pieces : cap;
    gradient_squares<T><<<dim3(blocks), dim3(NORM_THREADS), 0, stream>>>(t, partials + used);
    MP_CHECK_LAUNCH();
    used += blocks;
  });
  return used;
}

template <class T>
inline void gradient_norm_enqueue(const void* grads, const void* sizes, void* norm, void* scratch, double alpha, size_t count, hipStream_t stream) {
  const unsigned used = gradient_squares_all<T>(grads, sizes, scratch, count, stream);
  gradient_norm_finish<<<dim3(1), dim3(NORM_THREADS), 0, stream>>>(static_cast<const double*>(scratch), used, alpha, static_cast<double*>(norm));
  MP_CHECK_LAUNCH();
}

template <class T>
inline void gradient_scale_enqueue(const void* grads, const void* outs, const void* sizes, const void* norm, double max_norm, size_t count,
                                   hipStream_t stream) {
  for_norm_tables<T>(static_cast<const void* const*>(grads), static_cast<const void* const*>(outs), static_cast<const len_t*>(sizes), count,
                     [&](const NormTable<T>& t, unsigned pieces) {
    if (pieces == 0) return;
    gradient_scaled<T><<<dim3(pieces), dim3(NORM_THREADS), 0, stream>>>(t, static_cast<const double*>(norm), max_norm);
    MP_CHECK_LAUNCH();
  });
}

template <class T>
inline void gradient_norm(const void* grads, const void* sizes, void* norm, void* scratch, double alpha, size_t count, hipStream_t stream) {
  gradient_check<T>(grads, nullptr, sizes, norm, count);
  gradient_check_scratch(scratch, count);
  gradient_norm_enqueue<T>(grads, sizes, norm, scratch, alpha, count, stream);
}

template <class T>
inline void gradient_scale(const void* grads, const void* outs, const void* sizes, const void* norm, double max_norm, size_t count, hipStream_t stream) {
  gradient_check_limit(outs, max_norm, count);
  gradient_check<T>(grads, outs, sizes, norm, count);
  gradient_scale_enqueue<T>(grads, outs, sizes, norm, max_norm, count, stream);
}

template <class T>
inline void gradient_clip(const void* grads, const void* outs, const void* sizes, void* norm, void* scratch, double max_norm, size_t count,
                          hipStream_t stream) {
  gradient_check_limit(outs, max_norm, count);
  gradient_check<T>(grads, outs, sizes, norm, count);
  gradient_check_scratch(scratch, count);
  gradient_norm_enqueue<T>(grads, sizes, norm, scratch, 0.0, count, stream);
  gradient_scale_enqueue<T>(grads, outs, sizes, norm, max_norm, count, stream);
}

}  // namespace mp

#endif
#endif
