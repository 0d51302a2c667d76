/*
 * The norm of many tensors taken as one vector, and scaling them down to a largest norm. The reference
 * has neither; its optimisers walk the leaves of the graph (src/optm/optimizer.zig:56-64). Math:
 *   norm = sqrt(sum over all tensors and elements of g^2 + alpha * norm^2)
 *   out  = g * min(1, max_norm / norm)
 * Squares are added in fp64 whatever the storage type, so neither large nor tiny r16 / r32 gradients
 * overflow or vanish, and in a fixed order, so the norm does not change from run to run. The norm is a
 * double on the device; nothing waits for the host.
 *
 * Tensors that lie one behind the other (a bucket of gradients) are walked as one run. The runs' addresses
 * and sizes travel as kernel arguments, up to 196 of them a launch: nothing is copied to the device and a
 * captured launch keeps its own table. A table's work is cut into pieces of NORM_PIECE bytes, four 16-byte
 * packs a thread; workgroups take them in turn for the squares, each leaving one partial sum in the
 * workspace, and one each for the scaling (1024 workgroups for the squares: 100 tensors of 1000 elements the
 * norm 6.4 us, by 2048 7.0, and 203 M elements in 400 tensors 148 and 154; 196 runs a launch rather than 120
 * make the 148 137).
 *
 * The squares are bound by reading the tensors once, the scaling by reading and writing them once. r32,
 * 203 M elements: squares 124 us (6.6 TB/s), both together 367 us, of which the scaling on its own would
 * take 262: the squares read the last NORM_KEPT_BYTES through loads that leave them in the 256 MiB
 * memory-side cache, where the scaling finds them (all of it through such loads: squares 136 us,
 * together 375; none: 122 and 387; the scaling from the end backwards: 375).
 */
#ifndef MP_GRADIENT_NORM_H
#define MP_GRADIENT_NORM_H

#include "row_dispatch.h"

#include <stdlib.h>
#include <algorithm>

#if defined(__cplusplus) && defined(__HIPCC__)

namespace mp {

constexpr int NORM_THREADS = 256, NORM_PACKS = 4;
constexpr size_t NORM_PIECE = (size_t)NORM_THREADS * NORM_PACKS * PACK_BYTES, NORM_PARTIALS = 1024; /* a table */
/* up to so many pieces the scaling adds up the partial sums itself, in every workgroup, and one launch is
 * saved; beyond, a workgroup would spend as long on that as on its piece */
constexpr size_t NORM_FUSED_PIECES = 2048;

constexpr size_t NORM_KEPT_BYTES = (size_t)224 << 20, NORM_KEPT_PIECES = NORM_KEPT_BYTES / NORM_PIECE;

/* Runs of a launch: as many as 4 KiB of arguments hold. APART: the results lie elsewhere. */
constexpr int norm_runs(bool apart) { return apart ? 140 : 196; }
template <class T, bool APART> struct NormTable {
  static constexpr int RUNS = norm_runs(APART);
  const T* src[RUNS];
  T* dst[APART ? RUNS : 1];
  unsigned long long size[RUNS];
  unsigned first[RUNS + 1]; /* the number of the run's first piece; [count] is the end */
  int count;
};
static_assert(sizeof(NormTable<r16, true>) <= 4032 && sizeof(NormTable<r16, false>) <= 4032, "room for the other arguments");

/* The run that piece `q` belongs to: the last one whose first piece is not behind it (runs have a piece at
 * least). Scalar loads from the argument block; one vector load a wavefront and a vote cost the scaling
 * of 100 runs 3 %. */
template <class TABLE> __device__ __forceinline__ int norm_run_of(const TABLE& t, unsigned q) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= q) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

/* Where a piece lies: pack u of a thread is at(u) elements behind the piece's first. */
template <class T> struct NormPiece {
  static constexpr int W = PACK_BYTES / (int)sizeof(T);
  static constexpr size_t LEN = NORM_PIECE / sizeof(T);
  int run;
  size_t lo, left; /* the piece's first element in its run, and the run's elements from there on */
  template <class TABLE> __device__ __forceinline__ NormPiece(const TABLE& t, unsigned q) {
    run = norm_run_of(t, q);
    lo = (size_t)(q - t.first[run]) * LEN;
    left = t.size[run] - lo;
  }
  __device__ __forceinline__ size_t at(int u) const { return ((size_t)u * NORM_THREADS + threadIdx.x) * W; }
  __device__ __forceinline__ bool whole() const { return left >= LEN; }
  /* pack u where the run ends in this piece: zeros past its end */
  template <int WIDTH> __device__ __forceinline__ typename vec_of<T, WIDTH>::type cut(const T* src, int u) const {
    typename vec_of<T, WIDTH>::type v;
    const size_t i = at(u);
    if (i + WIDTH <= left) return *reinterpret_cast<const typename loose_vec_of<T, WIDTH>::type*>(src + i);
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) v[j] = i + j < left ? src[i + j] : (T)0;
    return v;
  }
};

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

template <bool KEEP, class T> __device__ __forceinline__ double piece_squares(const NormTable<T, false>& t, unsigned q) {
  constexpr int W = NormPiece<T>::W;
  using VL = typename loose_vec_of<T, W>::type;
  const NormPiece<T> piece(t, q);
  const T* src = t.src[piece.run] + piece.lo;
  double s = 0.0;
  if (piece.whole()) {
    typename vec_of<T, W>::type v[NORM_PACKS];
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u) {
      const VL* at = reinterpret_cast<const VL*>(src + piece.at(u));
      v[u] = KEEP ? *at : __builtin_nontemporal_load(at);
    }
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) s += (double)v[u][j] * (double)v[u][j];
  } else { /* the run's last piece: the packs that exist, and the elements behind the last one */
    typename vec_of<T, W>::type v[NORM_PACKS];
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u) v[u] = piece.template cut<W>(src, u);
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u)
#pragma unroll
      for (int j = 0; j < W; ++j) s += (double)v[u][j] * (double)v[u][j];
  }
  return s;
}

/* Pieces from `keep` on through loads that leave them in the memory-side cache. */
template <class T> __global__ __launch_bounds__(NORM_THREADS) void gradient_squares(NormTable<T, false> t, unsigned keep, double* partials) {
  __shared__ double slots[NORM_THREADS / WAVE];
  const unsigned end = t.first[t.count];
  double s = 0.0;
  unsigned q = blockIdx.x;
  for (; q < keep && q < end; q += gridDim.x) s += piece_squares<false>(t, q);
  for (; q < end; q += gridDim.x) s += piece_squares<true>(t, q);
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

/* The smallest normal number of P. A factor below it has lost bits, or all of them, where g * max_norm / norm
 * still is a number of P (r32 gradients of 1e38 and a largest norm of 1e-6): such a product is taken as
 * (g / norm) * max_norm in fp64, whose first factor is at most one and whose second is given. */
template <class P> __device__ constexpr double norm_least_factor() { return sizeof(P) == 4 ? 0x1p-126 : 0x1p-1022; }

/* FUSED: norm_in is what the squares left, `partials` sums; the first workgroup writes the norm. */
template <class T, bool FUSED, bool APART>
__global__ __launch_bounds__(NORM_THREADS) void gradient_scaled(NormTable<T, APART> t, const double* norm_in, unsigned partials, double* norm_out, double max_norm) {
  using P = typename precision<T>::type;
  constexpr int W = NormPiece<T>::W;
  using VL = typename loose_vec_of<T, W>::type;
  const NormPiece<T> piece(t, blockIdx.x);
  const T* src = t.src[piece.run] + piece.lo;
  T* dst = APART ? t.dst[piece.run] + piece.lo : const_cast<T*>(src);
  double inverse = 0.0; /* 1 / norm where the factor has left P's normal range, else zero */
  /* what to scale by; false: nothing to do in place */
  auto factor_of = [&](P& factor) {
    double total;
    if constexpr (FUSED) {
      __shared__ double slots[NORM_THREADS / WAVE];
      total = ::sqrt(norm_of(norm_in, partials, slots));
      if (blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = total;
    } else {
      total = norm_in[0];
    }
    const bool within = total <= max_norm;
    const double ratio = within ? 1.0 : max_norm / total;
    factor = (P)ratio;
    if constexpr (sizeof(T) != 2) /* an r16 result is zero there either way */
      if (ratio < norm_least_factor<P>()) inverse = 1.0 / total;
    return !(within && src == dst);
  };
  typename vec_of<T, W>::type v[NORM_PACKS];
  P factor;
  auto scaled = [&](int u, P (&out)[W]) {
#pragma unroll
    for (int j = 0; j < W; ++j) out[j] = (P)v[u][j] * factor;
    if (sizeof(T) == 2 || inverse == 0.0) return;
#pragma unroll
    for (int j = 0; j < W; ++j) out[j] = (P)((double)v[u][j] * inverse * max_norm);
  };
  if (piece.whole()) { /* on its own from load to store: 203 M elements 262 us, 267 where both share the loops */
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u) v[u] = __builtin_nontemporal_load(reinterpret_cast<const VL*>(src + piece.at(u)));
    asm volatile("" ::: "memory"); /* on their way while the norm is read, not behind it (261 us, 266 without) */
    if (!factor_of(factor)) return;
#pragma unroll
    for (int u = 0; u < NORM_PACKS; ++u) {
      P out[W];
      scaled(u, out);
      store_pack_nt_loose<T, W>(dst + piece.at(u), out);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < NORM_PACKS; ++u) v[u] = piece.template cut<W>(src, u);
  if (!factor_of(factor)) return;
#pragma unroll
  for (int u = 0; u < NORM_PACKS; ++u) {
    const size_t i = piece.at(u);
    P out[W];
    scaled(u, out);
    if (i + W <= piece.left) {
      store_pack_nt_loose<T, W>(dst + i, out);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (i + j < piece.left) dst[i + j] = (T)out[j];
    }
  }
}

/* ------------------------------------------------------------------ host dispatch */

/* The tensors as runs of neighbours: f(first tensor, elements) for each; a run goes on while the next
 * tensor begins where the last one ended, in grads and, where there are any, in outs. */
template <class T, class F> inline void for_norm_runs(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count, F&& f) {
  size_t k = 0;
  while (k < count) {
    if (sizes[k] == 0) {
      ++k;
      continue;
    }
    const size_t begin = k;
    size_t size = 0;
    auto follows = [&](const void* const* a) { return static_cast<const char*>(a[k]) == static_cast<const char*>(a[begin]) + size * sizeof(T); };
    do {
      size += sizes[k++];
      while (k < count && sizes[k] == 0) ++k;
    } while (k < count && follows(grads) && (!outs || follows(outs)));
    f(begin, size);
  }
}

/* whether any result lies elsewhere than its gradient */
inline bool gradients_apart(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count) {
  for (size_t k = 0; k < count; ++k)
    if (sizes[k] && grads[k] != outs[k]) return true;
  return false;
}

struct NormWork { size_t runs, pieces; };
template <class T> inline NormWork norm_work(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count) {
  NormWork w{0, 0};
  for_norm_runs<T>(grads, outs, sizes, count, [&](size_t, size_t size) {
    ++w.runs;
    w.pieces += (size * sizeof(T) + NORM_PIECE - 1) / NORM_PIECE;
  });
  return w;
}

/* f(table) for the runs in groups of a table's */
template <class T, bool APART, class F>
inline void for_norm_tables(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count, F&& f) {
  NormTable<T, APART> t;
  t.count = 0;
  t.first[0] = 0;
  for_norm_runs<T>(grads, APART ? outs : nullptr, sizes, count, [&](size_t k, size_t size) {
    t.src[t.count] = static_cast<const T*>(grads[k]);
    if constexpr (APART) t.dst[t.count] = const_cast<T*>(static_cast<const T*>(outs[k]));
    t.size[t.count] = size;
    const size_t pieces = (size * sizeof(T) + NORM_PIECE - 1) / NORM_PIECE;
    t.first[t.count + 1] = t.first[t.count] + (unsigned)pieces;
    if (++t.count == norm_runs(APART)) {
      f(t);
      t.count = 0;
    }
  });
  if (t.count) f(t);
}

/* Every table leaves at most NORM_PARTIALS sums. Tensors that form runs make fewer tables than they might,
 * never more. */
inline size_t gradient_norm_scratch_bytes(size_t count) { return (count + norm_runs(false) - 1) / norm_runs(false) * NORM_PARTIALS * sizeof(double); }

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
    /* the scaling's workgroups take a piece each, and a launch has fewer than 2^32 threads: 256 GiB of tensors */
    require(pieces < (outs ? ((size_t)1 << 32) / NORM_THREADS : 0x7fffffffull), "gradient norm: too many elements");
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

/* A tensor listed twice, or a result that reaches into another tensor, would be scaled once or twice as the
 * workgroups happen to run: refused. A result is its own gradient or clear of all of them. Results in rising
 * order (a bucket's) are checked in one walk, others are ordered first. */
template <class T> inline void gradient_check_apart(const void* const* grads, const void* const* outs, const len_t* sizes, size_t count) {
  struct Span { uintptr_t begin, end; };
  auto span = [&](const void* const* a, size_t k) { const uintptr_t at = reinterpret_cast<uintptr_t>(a[k]); return Span{at, at + sizes[k] * sizeof(T)}; };
  const char* twice = "gradient clip: a result overlaps another result or another gradient";
  bool rising = true, in_place = true;
  uintptr_t end = 0;
  for (size_t k = 0; k < count; ++k) {
    if (sizes[k] == 0) continue;
    const Span s = span(outs, k);
    rising = rising && s.begin >= end;
    in_place = in_place && grads[k] == outs[k];
    end = s.end;
  }
  if (rising && in_place) return;
  Span* spans = static_cast<Span*>(::malloc(count * sizeof(Span)));
  require(spans != nullptr, "gradient clip: out of host memory");
  size_t used = 0;
  for (size_t k = 0; k < count; ++k)
    if (sizes[k]) spans[used++] = span(outs, k);
  const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  if (!rising) std::sort(spans, spans + used, before);
  for (size_t k = 1; k < used; ++k) require(spans[k - 1].end <= spans[k].begin, twice);
  for (size_t k = 0; k < count && !in_place; ++k) {
    if (sizes[k] == 0 || grads[k] == outs[k]) continue;
    const Span s = span(grads, k);
    const Span* behind = std::lower_bound(spans, spans + used, Span{s.end, 0}, before); /* the first that begins at its end or later */
    require(behind == spans || behind[-1].end <= s.begin, twice);
  }
  ::free(spans);
}

/* returns how many partial sums there are */
template <class T>
inline unsigned gradient_squares_all(const void* const* grads, const len_t* sizes, double* partials, size_t count, hipStream_t stream) {
  unsigned used = 0;
  for_norm_tables<T, false>(grads, nullptr, sizes, count, [&](const NormTable<T, false>& t) {
    const unsigned pieces = t.first[t.count], blocks = pieces < NORM_PARTIALS ? pieces : (unsigned)NORM_PARTIALS;
    const unsigned keep = pieces > NORM_KEPT_PIECES ? pieces - (unsigned)NORM_KEPT_PIECES : 0;
    gradient_squares<T><<<dim3(blocks), dim3(NORM_THREADS), 0, stream>>>(t, keep, partials + used);
    MP_CHECK_LAUNCH();
    used += blocks;
  });
  return used;
}

template <class T>
inline void gradient_scale_all(const void* const* grads, const void* const* outs, const len_t* sizes, const double* norm_in, unsigned partials, double* norm_out,
                               double max_norm, size_t count, hipStream_t stream) {
  auto as = [&]<bool APART>() {
    for_norm_tables<T, APART>(grads, outs, sizes, count, [&](const NormTable<T, APART>& t) {
      const dim3 grid(t.first[t.count]), block(NORM_THREADS);
      if (norm_out) gradient_scaled<T, true, APART><<<grid, block, 0, stream>>>(t, norm_in, partials, norm_out, max_norm);
      else gradient_scaled<T, false, APART><<<grid, block, 0, stream>>>(t, norm_in, 0, nullptr, max_norm);
      MP_CHECK_LAUNCH();
    });
  };
  if (gradients_apart(grads, outs, sizes, count)) as.template operator()<true>();
  else as.template operator()<false>();
}

template <class T>
inline void gradient_norm(const void* grads, const void* sizes, void* norm, void* scratch, double alpha, size_t count, hipStream_t stream) {
  gradient_check<T>(grads, nullptr, sizes, norm, count);
  gradient_check_scratch(scratch, count);
  double* partials = static_cast<double*>(scratch);
  const unsigned used = gradient_squares_all<T>(static_cast<const void* const*>(grads), static_cast<const len_t*>(sizes), partials, count, stream);
  gradient_norm_finish<<<dim3(1), dim3(NORM_THREADS), 0, stream>>>(partials, used, alpha, static_cast<double*>(norm));
  MP_CHECK_LAUNCH();
}

template <class T>
inline void gradient_scale(const void* grads, const void* outs, const void* sizes, const void* norm, double max_norm, size_t count, hipStream_t stream) {
  gradient_check_limit(outs, max_norm, count);
  gradient_check<T>(grads, outs, sizes, norm, count);
  gradient_check_apart<T>(static_cast<const void* const*>(grads), static_cast<const void* const*>(outs), static_cast<const len_t*>(sizes), count);
  gradient_scale_all<T>(static_cast<const void* const*>(grads), static_cast<const void* const*>(outs), static_cast<const len_t*>(sizes),
                        static_cast<const double*>(norm), 0, nullptr, max_norm, count, stream);
}

template <class T>
inline void gradient_clip(const void* grads, const void* outs, const void* sizes, void* norm, void* scratch, double max_norm, size_t count,
                          hipStream_t stream) {
  gradient_check_limit(outs, max_norm, count);
  gradient_check<T>(grads, outs, sizes, norm, count);
  gradient_check_scratch(scratch, count);
  const void* const* src = static_cast<const void* const*>(grads);
  const void* const* dst = static_cast<const void* const*>(outs);
  gradient_check_apart<T>(src, dst, static_cast<const len_t*>(sizes), count);
  const len_t* lengths = static_cast<const len_t*>(sizes);
  double *partials = static_cast<double*>(scratch), *out = static_cast<double*>(norm);
  const unsigned used = gradient_squares_all<T>(src, lengths, partials, count, stream);
  const NormWork work = norm_work<T>(src, dst, lengths, count);
  const bool fused = used > 0 && work.runs <= (size_t)norm_runs(gradients_apart(src, dst, lengths, count)) && work.pieces <= NORM_FUSED_PIECES;
  if (!fused) {
    gradient_norm_finish<<<dim3(1), dim3(NORM_THREADS), 0, stream>>>(partials, used, 0.0, out);
    MP_CHECK_LAUNCH();
  }
  gradient_scale_all<T>(src, dst, lengths, fused ? partials : out, used, fused ? out : nullptr, max_norm, count, stream);
}

}  // namespace mp

#endif
#endif
