/*
 * Rows of a table picked by token ids, and the table's gradient. The reference has neither; its
 * broadcasts (src/cuda/nvcc_src/broadcast_j_ij.cu:9-57) and column sums (reduce_ij_j.cu:3-66) are the
 * nearest patterns. With t_i the id at place i of m, a table of v rows of n and a factor s:
 *   forward   y_ij  = s * table[t_i, j]
 *   reverse   dT_kj = s * sum_{i: t_i = k} dy_ij + alpha * dT_kj
 * An id outside [0, v) (a padded place) gives a row of zeros and takes part in no sum.
 *
 * The reverse adds no floating numbers by atomics, so its results do not change from run to run:
 * the places are sorted by their ids first (a stable radix sort: places of one id stay in order),
 * then chunks of the sorted places are summed in registers, in precision<T>. An id whose places lie
 * within one chunk is written at once; one that crosses chunks leaves a partial row in each, and a
 * last kernel adds those in order. Rows of the table that no id names are cleared (or scaled, by
 * alpha) by workgroups of the same launch as the sums; with alpha = 1 they are not touched.
 */
#ifndef MP_EMBEDDING_H
#define MP_EMBEDDING_H

#include "row_dispatch.h"

#if defined(__cplusplus) && defined(__HIPCC__)

namespace mp {

/* The id at place i as a sort key: ids outside [0, v) become v, which sorts behind every row. */
__device__ __forceinline__ unsigned token_key(const void* tokens, bool wide, size_t i, unsigned v) {
  const long long t = wide ? static_cast<const long long*>(tokens)[i] : (long long)static_cast<const int*>(tokens)[i];
  return t >= 0 && t < (long long)v ? (unsigned)t : v;
}

/* ------------------------------------------------------------------ forward */

/* G lanes hold a strip of G packs of one row, 256 / G rows a workgroup. */
template <class T, int W, int G, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_rows(
    const T* table, const void* tokens, T* y, typename precision<T>::type scale, unsigned wide, unsigned v, size_t m,
    size_t n, unsigned strips) {
  using P = typename precision<T>::type;
  const int sub = threadIdx.x / G, lane = threadIdx.x % G;
  const RowPacks<T, W, LOOSE> rp(n);
  const size_t row = (size_t)(blockIdx.x / strips) * (256 / G) + sub;
  const int p = (int)(blockIdx.x % strips) * G + lane;
  if (row >= m || p >= rp.npk) return;
  const unsigned k = token_key(tokens, wide != 0, row, v);
  P out[W];
#pragma unroll
  for (int i = 0; i < W; ++i) out[i] = (P)0;
  if (k < v) {
    rp.template load<false>(table + (size_t)k * n, p, out);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] *= scale;
  }
  rp.store(y + row * n, p, out);
}

/* ------------------------------------------------------------------ sorting the places by id */

/* A radix sort of 9 bits a pass, lowest first. A tile of the places belongs to one workgroup of 16
 * wavefronts, each of which takes an equal, contiguous part of it, so that counts alone say where
 * every place goes: the places of a digit in earlier tiles, in earlier wavefronts of the tile, and
 * earlier in the wavefront. Two launches a pass: count, then place (each workgroup of the second
 * adds up the counts of all tiles for itself). */
constexpr int SORT_BITS = 9, SORT_DIGITS = 1 << SORT_BITS, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / WAVE;
constexpr size_t SORT_TILES = 256; /* tiles a pass, at most */

inline size_t sort_tile(size_t m) {
  const size_t each = (m + SORT_TILES - 1) / SORT_TILES;
  return (each + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
}

__device__ __forceinline__ unsigned sort_key(const void* tokens, unsigned wide, const unsigned* keys, size_t i, unsigned v) {
  return keys ? keys[i] : token_key(tokens, wide != 0, i, v);
}

static __global__ __launch_bounds__(SORT_THREADS) void embedding_sort_count(
    const void* tokens, unsigned wide, const unsigned* keys, unsigned* counts, unsigned v, size_t m, size_t tile, int shift) {
  __shared__ unsigned hist[SORT_DIGITS];
  for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) hist[d] = 0;
  __syncthreads();
  const size_t lo = (size_t)blockIdx.x * tile, hi = lo + tile < m ? lo + tile : m;
  for (size_t i = lo + threadIdx.x; i < hi; i += SORT_THREADS)
    atomicAdd(&hist[(sort_key(tokens, wide, keys, i, v) >> shift) & (SORT_DIGITS - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) counts[(size_t)blockIdx.x * SORT_DIGITS + d] = hist[d];
}

/* keys NULL: the first pass, from the tokens; the place of an entry is then its index */
static __global__ __launch_bounds__(SORT_THREADS) void embedding_sort_place(
    const void* tokens, unsigned wide, const unsigned* keys, const unsigned* places, const unsigned* counts,
    unsigned* keys_out, unsigned* places_out, unsigned v, size_t m, size_t tile, unsigned tiles, int shift) {
  __shared__ unsigned next[SORT_WAVES][SORT_DIGITS]; /* counts of a wavefront's part, then where its next entry goes */
  __shared__ unsigned total[2][SORT_DIGITS], before[2][SORT_DIGITS], wave_total[SORT_DIGITS / WAVE];
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const size_t part = tile / SORT_WAVES, lo = (size_t)blockIdx.x * tile + wave * part;
  const size_t hi = lo + part < m ? lo + part : m;

  for (int d = lane; d < SORT_DIGITS; d += WAVE) next[wave][d] = 0;
  __syncthreads();
  for (size_t i = lo + lane; i < hi; i += WAVE)
    atomicAdd(&next[wave][(sort_key(tokens, wide, keys, i, v) >> shift) & (SORT_DIGITS - 1)], 1u);

  { /* two threads a digit add up the tiles */
    const int d = tid & (SORT_DIGITS - 1), half = tid / SORT_DIGITS;
    unsigned all = 0, mine = 0;
    for (unsigned t = half; t < tiles; t += 2) {
      const unsigned c = counts[(size_t)t * SORT_DIGITS + d];
      all += c;
      mine += t < blockIdx.x ? c : 0;
    }
    total[half][d] = all;
    before[half][d] = mine;
  }
  __syncthreads();
  unsigned sum = 0, inclusive = 0;
  if (tid < SORT_DIGITS) { /* the digits' exclusive sums: within a wavefront, then over the eight */
    sum = total[0][tid] + total[1][tid];
    inclusive = sum;
#pragma unroll
    for (int step = 1; step < WAVE; step <<= 1) {
      const unsigned up = __shfl_up(inclusive, step, WAVE);
      if (lane >= step) inclusive += up;
    }
    if (lane == WAVE - 1) wave_total[wave] = inclusive;
  }
  __syncthreads();
  if (tid < SORT_DIGITS) {
    unsigned at = inclusive - sum + before[0][tid] + before[1][tid];
    for (int w = 0; w < wave; ++w) at += wave_total[w];
    for (int w = 0; w < SORT_WAVES; ++w) {
      const unsigned c = next[w][tid];
      next[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  for (size_t i0 = lo; i0 < hi; i0 += WAVE) { /* in order: 64 entries at a time */
    const size_t i = i0 + lane;
    const bool live = i < hi;
    const unsigned key = live ? sort_key(tokens, wide, keys, i, v) : 0u;
    const unsigned place = live ? (places ? places[i] : (unsigned)i) : 0u;
    const unsigned digit = (key >> shift) & (SORT_DIGITS - 1);
    unsigned long long same = __ballot(live); /* the lanes that hold my digit */
#pragma unroll
    for (int b = 0; b < SORT_BITS; ++b) {
      const bool set = (digit >> b) & 1u;
      const unsigned long long with = __ballot(set);
      same &= set ? with : ~with;
    }
    const unsigned earlier = (unsigned)__popcll(same & ((1ull << lane) - 1ull));
    const unsigned base = live ? next[wave][digit] : 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* every lane has read before the last of a digit moves it on */
    if (live && (same >> lane) == 1ull) next[wave][digit] = base + earlier + 1u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (live) {
      keys_out[base + earlier] = key;
      places_out[base + earlier] = place;
    }
  }
}

/* ------------------------------------------------------------------ sums over the sorted places */

/* The first of the sorted keys that is at least `key`, m if there is none. */
__device__ __forceinline__ size_t lower_bound(const unsigned* keys, size_t m, unsigned key) {
  size_t lo = 0, hi = m;
  while (lo < hi) {
    const size_t mid = (lo + hi) / 2;
    if (keys[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

constexpr int FILL_ROWS = 64; /* rows of the table a clearing workgroup looks after */

/* Workgroups below sum_blocks: G lanes hold a strip of G packs of the columns and walk one chunk of
 * the sorted places, 256 / G chunks a workgroup. The others clear (BLEND: scale) the rows of the table
 * that no id names. partials: two rows of n for every chunk, the first for an id that begins in an
 * earlier chunk, the second for one that goes on in the next. */
template <class T, int W, int G, bool BLEND, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_sum(
    const unsigned* keys, const unsigned* places, const T* dy, T* grads, typename precision<T>::type* partials,
    typename precision<T>::type scale, typename precision<T>::type alpha, unsigned v, size_t m, size_t n, size_t chunk,
    unsigned strips, unsigned sum_blocks) {
  using P = typename precision<T>::type;
  using V = typename vec_of<T, W>::type;
  const RowPacks<T, W, LOOSE> rp(n);

  if (blockIdx.x >= sum_blocks) {
    __shared__ unsigned named[FILL_ROWS];
    const size_t row0 = (size_t)(blockIdx.x - sum_blocks) * FILL_ROWS;
    const unsigned rows = (unsigned)(v - row0 < FILL_ROWS ? v - row0 : FILL_ROWS);
    if (threadIdx.x < FILL_ROWS) {
      const unsigned key = (unsigned)row0 + threadIdx.x;
      unsigned there = 1;
      if (threadIdx.x < rows) {
        const size_t at = lower_bound(keys, m, key);
        there = at < m && keys[at] == key;
      }
      named[threadIdx.x] = there;
    }
    __syncthreads();
    for (unsigned k = 0; k < rows; ++k) {
      if (named[k]) continue;
      T* row = grads + (row0 + k) * n;
      for (int p = threadIdx.x; p < rp.npk; p += 256) {
        P out[W];
#pragma unroll
        for (int i = 0; i < W; ++i) out[i] = (P)0;
        if constexpr (BLEND) {
          rp.template load<true>(row, p, out);
#pragma unroll
          for (int i = 0; i < W; ++i) out[i] *= alpha;
        }
        rp.store(row, p, out);
      }
    }
    return;
  }

  constexpr int U = 8; /* rows on their way at once */
  const int sub = threadIdx.x / G, lane = threadIdx.x % G;
  const size_t c = (size_t)(blockIdx.x / strips) * (256 / G) + sub;
  const int p = (int)(blockIdx.x % strips) * G + lane;
  const size_t lo = c * chunk;
  if (lo >= m || p >= rp.npk) return;
  const size_t hi = lo + chunk < m ? lo + chunk : m;

  P acc[W];
  unsigned current = keys[lo];
  bool begun = lo > 0 && keys[lo - 1] == current; /* the id's first place lies in an earlier chunk */
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = (P)0;
  };
  auto leave = [&](bool goes_on) {
    if (current >= v) return; /* padded places */
    if (begun || goes_on) {
      P* at = partials + (c * 2 + (begun ? 0 : 1)) * n + (size_t)p * W;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < rp.valid(p)) at[i] = acc[i];
      return;
    }
    T* row = grads + (size_t)current * n;
    P out[W];
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = scale * acc[i];
    if constexpr (BLEND) {
      P old[W];
      rp.template load<true>(row, p, old);
#pragma unroll
      for (int i = 0; i < W; ++i) out[i] += alpha * old[i];
    }
    rp.store(row, p, out);
  };
  clear();
  for (size_t i0 = lo; i0 < hi; i0 += U) {
    unsigned key[U];
    V row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t i = i0 + u < hi ? i0 + u : hi - 1;
      key[u] = keys[i];
      row[u] = rp.template raw<true>(dy + (size_t)places[i] * n, p);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= hi) break;
      if (key[u] != current) {
        leave(false);
        current = key[u];
        begun = false;
        clear();
      }
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] += (P)row[u][i];
    }
  }
  leave(hi < m && keys[hi] == current);
}

/* The ids that cross chunks: the chunk where such an id begins adds up its partial rows in order (a
 * workgroup owns 16 columns of it; 16 slices take the rows in turn, then the slices are added). */
template <class T, bool BLEND>
__global__ __launch_bounds__(256) void embedding_join(
    const unsigned* keys, const typename precision<T>::type* partials, T* grads, typename precision<T>::type scale,
    typename precision<T>::type alpha, unsigned v, size_t m, size_t n, size_t chunk, unsigned strips) {
  using P = typename precision<T>::type;
  constexpr int COLS = 64, SLICES = 256 / COLS;
  __shared__ double part[SLICES][COLS];
  const size_t c = blockIdx.x / strips, lo = c * chunk, hi = lo + chunk;
  if (hi >= m) return;
  const unsigned key = keys[hi - 1];
  if (key >= v || keys[hi] != key) return;
  if (keys[lo] == key && lo > 0 && keys[lo - 1] == key) return; /* it began earlier */
  const size_t end = key + 1 == 0 ? m : lower_bound(keys, m, key + 1); /* behind its last place */
  const size_t later = (end - hi + chunk - 1) / chunk;
  const int col = threadIdx.x % COLS, slice = threadIdx.x / COLS;
  const size_t j = (size_t)(blockIdx.x % strips) * COLS + col;
  double s = 0.0;
  if (j < n)
    for (size_t k = slice; k <= later; k += SLICES) s += (double)partials[((c + k) * 2 + (k == 0 ? 1 : 0)) * n + j];
  part[slice][col] = s;
  __syncthreads();
  if (slice == 0 && j < n) {
    for (int k = 1; k < SLICES; ++k) s += part[k][col];
    T* at = grads + (size_t)key * n + j;
    double out = (double)scale * s;
    if constexpr (BLEND) out += (double)alpha * (double)*at;
    *at = (T)out;
  }
}

/* alpha * dT without any id */
template <class T, bool BLEND> __global__ __launch_bounds__(256) void embedding_scale_all(T* grads, typename precision<T>::type alpha, size_t count) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < count) grads[i] = BLEND ? (T)(alpha * (typename precision<T>::type)grads[i]) : (T)0;
}

/* ------------------------------------------------------------------ host dispatch */

/* The sorted places one chunk holds. */
inline size_t embedding_chunk(size_t m) {
  size_t chunk = 8;
  while (chunk < 64 && m / chunk > 2048) chunk *= 2;
  return chunk;
}

/* Workspace of the reverse: two pairs of keys and places that the sort writes in turn, the counts of
 * its tiles, and two partial rows a chunk. Every part starts on a 256-byte boundary. */
struct EmbeddingScratch {
  size_t keys[2], places[2], counts, partials, bytes;
};
template <class T> inline EmbeddingScratch embedding_scratch(size_t m, size_t n) {
  EmbeddingScratch s{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int k = 0; k < 2; ++k) {
    s.keys[k] = take(m * sizeof(unsigned));
    s.places[k] = take(m * sizeof(unsigned));
  }
  s.counts = take(SORT_TILES * SORT_DIGITS * sizeof(unsigned));
  const size_t chunk = embedding_chunk(m);
  s.partials = take((m + chunk - 1) / chunk * 2 * n * sizeof(typename precision<T>::type));
  s.bytes = at;
  return s;
}

/* Lanes for a strip of a row's packs: the next power of two up to 256. */
template <class F> inline void for_strip(size_t packs, F&& f) {
  if (packs <= 8) f.template operator()<8>();
  else if (packs <= 16) f.template operator()<16>();
  else if (packs <= 32) f.template operator()<32>();
  else if (packs <= 64) f.template operator()<64>();
  else if (packs <= 128) f.template operator()<128>();
  else f.template operator()<256>();
}

inline void embedding_check(const void* tokens, size_t id_bytes, size_t v, size_t m, size_t n) {
  require(id_bytes == 4 || id_bytes == 8, "embedding: token ids are 4 or 8 bytes wide");
  require(reinterpret_cast<uintptr_t>(tokens) % id_bytes == 0, "embedding: token ids must be aligned to their width");
  require(v < 0xffffffffull, "embedding: the table must have fewer than 2^32 - 1 rows");
  require(m < 0x80000000ull, "embedding: at most 2^31 - 1 tokens");
  require(n <= 0x40000000ull, "embedding: row length must not exceed 2^30");
}

template <class T>
inline void embedding_forward(const T* table, const void* tokens, T* y, double scale, size_t id_bytes, size_t v, size_t m, size_t n,
                              hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  embedding_check(tokens, id_bytes, v, m, n);
  if (m == 0 || n == 0) return;
  const bool loose = !(aligned16(table) && aligned16(y) && n % W == 0);
  const size_t packs = (n + W - 1) / W;
  for_strip(packs, [&]<int G>() {
    const size_t strips = (packs + G - 1) / G, blocks = (m + 256 / G - 1) / (256 / G) * strips;
    require(blocks < 0x7fffffffull, "embedding: too many rows for one grid");
    const dim3 grid((unsigned)blocks), block(256);
    if (loose) embedding_rows<T, W, G, true><<<grid, block, 0, stream>>>(table, tokens, y, (P)scale, id_bytes == 8, (unsigned)v, m, n, (unsigned)strips);
    else embedding_rows<T, W, G, false><<<grid, block, 0, stream>>>(table, tokens, y, (P)scale, id_bytes == 8, (unsigned)v, m, n, (unsigned)strips);
  });
  MP_CHECK_LAUNCH();
}

template <class T>
inline void embedding_reverse(const void* tokens, const T* dy, T* grads, void* scratch, double scale, double alpha, size_t id_bytes,
                              size_t v, size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  embedding_check(tokens, id_bytes, v, m, n);
  if (v == 0 || n == 0) return;
  if (m == 0) {
    if (alpha == 1.0) return;
    const size_t count = v * n, blocks = (count + 255) / 256;
    require(blocks < 0x7fffffffull, "embedding reverse: table too large for one grid");
    if (alpha == 0.0) embedding_scale_all<T, false><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(grads, (P)alpha, count);
    else embedding_scale_all<T, true><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(grads, (P)alpha, count);
    MP_CHECK_LAUNCH();
    return;
  }
  require(scratch != nullptr, "embedding reverse: scratch must hold mpEmbeddingReverseScratchBytes bytes");
  require(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "embedding reverse: scratch must be 16-byte aligned");
  const EmbeddingScratch at = embedding_scratch<T>(m, n);
  char* base = static_cast<char*>(scratch);
  unsigned* keys[2] = {reinterpret_cast<unsigned*>(base + at.keys[0]), reinterpret_cast<unsigned*>(base + at.keys[1])};
  unsigned* places[2] = {reinterpret_cast<unsigned*>(base + at.places[0]), reinterpret_cast<unsigned*>(base + at.places[1])};
  unsigned* counts = reinterpret_cast<unsigned*>(base + at.counts);
  P* partials = reinterpret_cast<P*>(base + at.partials);

  const size_t tile = sort_tile(m);
  const unsigned tiles = (unsigned)((m + tile - 1) / tile), wide = id_bytes == 8;
  int from = -1; /* the tokens themselves */
  for (int shift = 0; shift == 0 || (v >> shift) != 0; shift += SORT_BITS) { /* keys run up to v */
    const unsigned *k = from < 0 ? nullptr : keys[from], *p = from < 0 ? nullptr : places[from];
    const int to = from == 0 ? 1 : 0;
    embedding_sort_count<<<dim3(tiles), dim3(SORT_THREADS), 0, stream>>>(tokens, wide, k, counts, (unsigned)v, m, tile, shift);
    embedding_sort_place<<<dim3(tiles), dim3(SORT_THREADS), 0, stream>>>(tokens, wide, k, p, counts, keys[to], places[to], (unsigned)v, m,
                                                                         tile, tiles, shift);
    MP_CHECK_LAUNCH();
    from = to;
  }

  const bool loose = !(aligned16(dy) && aligned16(grads) && n % W == 0);
  const size_t packs = (n + W - 1) / W, chunk = embedding_chunk(m), chunks = (m + chunk - 1) / chunk;
  const size_t fill = alpha == 1.0 ? 0 : (v + FILL_ROWS - 1) / FILL_ROWS;
  for_strip(packs, [&]<int G>() {
    const size_t strips = (packs + G - 1) / G, sums = (chunks + 256 / G - 1) / (256 / G) * strips;
    require(sums + fill < 0x7fffffffull, "embedding reverse: too many rows for one grid");
    const dim3 grid((unsigned)(sums + fill)), block(256);
    auto go = [&]<bool BLEND, bool LOOSE>() {
      embedding_sum<T, W, G, BLEND, LOOSE><<<grid, block, 0, stream>>>(keys[from], places[from], dy, grads, partials, (P)scale, (P)alpha,
                                                                       (unsigned)v, m, n, chunk, (unsigned)strips, (unsigned)sums);
    };
    if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
    else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
  });
  MP_CHECK_LAUNCH();
  if (chunks > 1) {
    const size_t strips = (n + 63) / 64;
    require(chunks * strips < 0x7fffffffull, "embedding reverse: too many rows for one grid");
    const dim3 grid((unsigned)(chunks * strips)), block(256);
    if (alpha != 0.0) embedding_join<T, true><<<grid, block, 0, stream>>>(keys[from], partials, grads, (P)scale, (P)alpha, (unsigned)v, m, n, chunk, (unsigned)strips);
    else embedding_join<T, false><<<grid, block, 0, stream>>>(keys[from], partials, grads, (P)scale, (P)alpha, (unsigned)v, m, n, chunk, (unsigned)strips);
    MP_CHECK_LAUNCH();
  }
}

}  // namespace mp

#endif
#endif
