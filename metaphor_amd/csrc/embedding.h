/*
 * Rows of a table picked by token ids, and the table's gradient. The reference has neither; its
 * broadcasts (src/cuda/nvcc_src/broadcast_j_ij.cu:9-57) and column sums (reduce_ij_j.cu:3-66) are the
 * nearest patterns. With t_i the id at place i of m, a table of v rows of n and a factor s:
 *   forward   y_ij  = s * table[t_i, j]
 *   reverse   dT_kj = s * sum_{i: t_i = k} dy_ij + alpha * dT_kj
 * An id outside [0, v) (a padded place) gives a row of zeros and takes part in no sum.
 *
 * The reverse adds no floating numbers by atomics, so its results do not change from run to run. Up to
 * DIRECT_MOST places one launch does it all. Beyond, the places are sorted by their ids first (places of
 * one id stay in order; by counting up to RANK_MOST places, by a stable radix sort beyond), then chunks
 * of the sorted places are summed in registers, in precision<T>. An id whose places lie
 * within one chunk is written at once; one that crosses chunks leaves a partial row in each, and a
 * last kernel adds those in order. Rows of the table that no id names are cleared (or scaled, by
 * alpha) by workgroups of the same launch as the sums; with alpha = 1 they are not touched. With
 * alpha = 0 the sort's launches, which use a fraction of the GPU, clear the table's first rows on the
 * way, named or not. All of it is bound by memory: dy read once, the table written once. r32 8192 places,
 * 50257 rows of 1024: 54 us (4.3 TB/s, of which the ordering is 13 us and the join 5); r16 65536 places,
 * 151936 rows of 2048: 176 us (5.1 TB/s; the sums' launch 135 us). The lookup, r32 16384 places of rows of 2048:
 * 31 us (6.2 TB/s).
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

/* Pack p of row `row` of a matrix of `rows` rows of n. The pack that the row's end cuts is read whole too, into
 * the next row (what is read there is never stored), except where it would pass the matrix's end: a cut pack
 * read element by element makes its wavefront wait for every row in turn (r16 n = 100, 16000 tokens: the sums
 * 25 us). */
template <class T, int W, bool LOOSE, bool NT>
__device__ __forceinline__ typename vec_of<T, W>::type whole_pack(const RowPacks<T, W, LOOSE>& rp, const T* matrix, size_t row, size_t rows, size_t n, int p) {
  using VL = typename std::conditional<LOOSE, typename loose_vec_of<T, W>::type, typename vec_of<T, W>::type>::type;
  const size_t at = row * n + (size_t)(unsigned)p * W;
  if (LOOSE && at + W > rows * n) return rp.template raw<NT>(matrix + row * n, p);
  const VL* v = reinterpret_cast<const VL*>(matrix + at);
  return NT ? __builtin_nontemporal_load(v) : *v;
}

/* ------------------------------------------------------------------ forward */

/* G lanes hold a strip of G packs of one row, 256 / G rows a workgroup. */
template <class T, int W, int G, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_rows(
    const T* table, const void* tokens, T* y, typename precision<T>::type scale, unsigned wide, unsigned v, size_t m,
    size_t n, unsigned strips, unsigned first_block) {
  using P = typename precision<T>::type;
  const int sub = threadIdx.x / G, lane = threadIdx.x % G;
  const RowPacks<T, W, LOOSE> rp(n);
  const unsigned block = first_block + blockIdx.x;
  const size_t row = (size_t)(block / strips) * (256 / G) + sub;
  const int p = (int)(block % strips) * G + lane;
  if (row >= m || p >= rp.npk) return;
  const unsigned k = token_key(tokens, wide != 0, row, v);
  P out[W];
#pragma unroll
  for (int i = 0; i < W; ++i) out[i] = (P)0;
  if (k < v) {
    const typename vec_of<T, W>::type in = whole_pack<T, W, LOOSE, false>(rp, table, k, v, n, p);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = (P)in[i] * scale;
  }
  rp.store(y + row * n, p, out);
}

/* ------------------------------------------------------------------ clearing rows */

/* Rows [0, rows) of a table cleared by the workgroups of a launch from block `first` on, in units of
 * FILL_PACKS packs a thread. */
constexpr size_t FILL_PACKS = 4;
template <class T, int THREADS> __device__ __forceinline__ void clear_part(T* table, size_t count, unsigned block) {
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  using VL = typename loose_vec_of<T, W>::type;
  const size_t lo = (size_t)block * (THREADS * FILL_PACKS * W);
  typename vec_of<T, W>::type zero;
#pragma unroll
  for (int i = 0; i < W; ++i) zero[i] = (T)0;
#pragma unroll
  for (size_t u = 0; u < FILL_PACKS; ++u) {
    const size_t i = lo + (u * THREADS + threadIdx.x) * W;
    if (i + W <= count) __builtin_nontemporal_store(zero, reinterpret_cast<VL*>(table + i));
    else
      for (size_t j = i; j < count; ++j) table[j] = (T)0;
  }
}

/* ------------------------------------------------------------------ sorting the places by id */

/* A radix sort of 9 bits a pass, lowest first. A tile of the places belongs to one workgroup of 16
 * wavefronts, each of which takes an equal, contiguous part of it, so that counts alone say where
 * every place goes: the places of a digit in earlier tiles, in earlier wavefronts of the tile, and
 * earlier in the wavefront. Two launches a pass: count, then place (each workgroup of the second adds up
 * the counts of all tiles for itself; counting the next pass's digits there with atomics saves a launch
 * and loses more, because a common id's places all meet on one counter: 20 us a launch against 10 + 5). */
constexpr int SORT_BITS = 9, SORT_DIGITS = 1 << SORT_BITS, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / WAVE;
constexpr size_t SORT_TILES = 256; /* tiles a pass, at most */

inline size_t sort_tile(size_t m) {
  const size_t each = (m + SORT_TILES - 1) / SORT_TILES;
  return (each + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
}
inline int sort_passes(size_t v) { /* keys run up to v */
  int passes = 1;
  while (v >> (passes * SORT_BITS)) ++passes;
  return passes;
}

__device__ __forceinline__ unsigned sort_key(const void* tokens, unsigned wide, const unsigned* keys, size_t i, unsigned v) {
  return keys ? keys[i] : token_key(tokens, wide != 0, i, v);
}
__device__ __forceinline__ unsigned sort_digit(unsigned key, int shift) { return (key >> shift) & (SORT_DIGITS - 1); }

/* Counts of the 512 digits by wavefront, turned into where each wavefront's first entry of a digit goes:
 * every digit's start (the sums of the digits before it, and `before` of the thread's own digit) and then
 * the wavefronts in turn. total: of the thread's digit, over everything that is sorted. Threads 0 to 511
 * hold a digit each; all threads call it. */
__device__ __forceinline__ void sort_starts(unsigned (*next)[SORT_DIGITS], unsigned* wave_total, unsigned total, unsigned before) {
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  unsigned inclusive = total;
  if (tid < SORT_DIGITS) {
#pragma unroll
    for (int step = 1; step < WAVE; step <<= 1) {
      const unsigned up = __shfl_up(inclusive, step, WAVE);
      if (lane >= step) inclusive += up;
    }
    if (lane == WAVE - 1) wave_total[wave] = inclusive;
  }
  __syncthreads();
  if (tid < SORT_DIGITS) {
    unsigned at = inclusive - total + before;
    for (int w = 0; w < wave; ++w) at += wave_total[w];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const unsigned c = next[w][tid];
      next[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
}

/* Where the 64 entries of a wavefront go, in order: behind those of the same digit in lower lanes, which
 * votes on the digit's bits find. `starts` is the wavefront's row of `next`. */
__device__ __forceinline__ unsigned sort_target(unsigned* starts, unsigned digit, bool live) {
  const int lane = threadIdx.x % WAVE;
  unsigned long long same = __ballot(live); /* the lanes that hold my digit */
#pragma unroll
  for (int b = 0; b < SORT_BITS; ++b) {
    const bool set = (digit >> b) & 1u;
    const unsigned long long with = __ballot(set);
    same &= set ? with : ~with;
  }
  const unsigned earlier = (unsigned)__popcll(same & ((1ull << lane) - 1ull));
  const unsigned at = (live ? starts[digit] : 0u) + earlier;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* every lane has read before the last of a digit moves it on */
  if (live && (same >> lane) == 1ull) starts[digit] = at + 1u;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return at;
}

/* Up to RANK_MOST places without a radix sort: an entry goes behind the entries of smaller keys and the
 * earlier ones of its own, so its place in the order is counted directly. A workgroup counts for 32 entries;
 * the 32 half wavefronts of it take a share of all keys each, out of LDS, four to a broadcast read. Two
 * instructions a pair of entries. The whole gradient of r16 rows of 100: 5000 places 19 us, 28 by the radix
 * sort below; 9000 32 by either; 12000 38 and 33. Workgroups from `groups` on clear the table's first `cleared` elements. */
constexpr size_t RANK_MOST = 8192;
constexpr int RANK_ENTRIES = 32, RANK_SHARES = SORT_THREADS / RANK_ENTRIES;
template <class T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_rank(
    const void* tokens, unsigned wide, unsigned* keys_out, unsigned* places_out, unsigned* crossing, unsigned v, unsigned m, unsigned groups, T* table,
    size_t cleared) {
  if (blockIdx.x >= groups) {
    clear_part<T, SORT_THREADS>(table, cleared, blockIdx.x - groups);
    return;
  }
  typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
  extern __shared__ unsigned rank_keys[]; /* m rounded up to a whole number of groups, the rest greater than any key */
  __shared__ unsigned part[RANK_SHARES][RANK_ENTRIES];
  const int tid = threadIdx.x, share = tid / RANK_ENTRIES, lane = tid % RANK_ENTRIES;
  for (unsigned i = tid; i < groups * RANK_ENTRIES; i += SORT_THREADS) rank_keys[i] = i < m ? token_key(tokens, wide != 0, i, v) : 0xffffffffu;
  if (blockIdx.x == 0 && tid == 0) *crossing = 0;
  __syncthreads();
  const unsigned mine = blockIdx.x, i = mine * RANK_ENTRIES + lane, key = rank_keys[i];
  unsigned rank = 0;
  for (unsigned b = share; b < groups; b += RANK_SHARES) {
    const uint4_t* others = reinterpret_cast<const uint4_t*>(rank_keys + b * RANK_ENTRIES);
    /* keys below `key`, or up to it in earlier groups: below key + 1 (no key is the largest number) */
    const unsigned below = b < mine ? key + 1u : key;
#pragma unroll
    for (int q = 0; q < RANK_ENTRIES / 4; ++q) {
      const uint4_t o = others[q];
      rank += (o[0] < below) + (o[1] < below) + (o[2] < below) + (o[3] < below);
    }
    if (b == mine)
      for (int j = 0; j < RANK_ENTRIES; ++j) rank += rank_keys[b * RANK_ENTRIES + j] == key && j < lane;
  }
  part[share][lane] = rank;
  __syncthreads();
  if (tid < RANK_ENTRIES && i < m) {
    unsigned at = 0;
#pragma unroll
    for (int w = 0; w < RANK_SHARES; ++w) at += part[w][lane];
    keys_out[at] = key;
    places_out[at] = i;
  }
}

/* A pass's counts by tile. Workgroups from `tiles` on clear the table's first `cleared` elements. */
template <class T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_count(
    const void* tokens, unsigned wide, const unsigned* keys, unsigned* counts, unsigned* crossing, unsigned v, size_t m, size_t tile, unsigned tiles,
    int shift, T* table, size_t cleared) {
  if (blockIdx.x >= tiles) {
    clear_part<T, SORT_THREADS>(table, cleared, blockIdx.x - tiles);
    return;
  }
  __shared__ unsigned hist[SORT_DIGITS];
  for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) hist[d] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *crossing = 0;
  __syncthreads();
  const size_t lo = (size_t)blockIdx.x * tile, hi = lo + tile < m ? lo + tile : m;
  for (size_t i = lo + threadIdx.x; i < hi; i += SORT_THREADS) atomicAdd(&hist[sort_digit(sort_key(tokens, wide, keys, i, v), shift)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_DIGITS; d += SORT_THREADS) counts[blockIdx.x * SORT_DIGITS + d] = hist[d];
}

/* keys NULL: the first pass, from the tokens; the place of an entry is then its index. counts: this pass's, by tile. */
template <class T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_place(
    const void* tokens, unsigned wide, const unsigned* keys, const unsigned* places, const unsigned* counts,
    unsigned* keys_out, unsigned* places_out, unsigned v, size_t m, unsigned tile, unsigned tiles, int shift, T* table, size_t cleared) {
  if (blockIdx.x >= tiles) {
    clear_part<T, SORT_THREADS>(table, cleared, blockIdx.x - tiles);
    return;
  }
  __shared__ unsigned next[SORT_WAVES][SORT_DIGITS]; /* counts of a wavefront's part, then where its next entry goes */
  __shared__ unsigned total[SORT_DIGITS], before[SORT_DIGITS], wave_total[SORT_DIGITS / WAVE];
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const unsigned part = tile / SORT_WAVES;
  const size_t lo = (size_t)blockIdx.x * tile + wave * part, hi = lo + part < m ? lo + part : m;

  for (int d = lane; d < SORT_DIGITS; d += WAVE) next[wave][d] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* a wavefront's row is its own */
  for (size_t i = lo + lane; i < hi; i += WAVE) atomicAdd(&next[wave][sort_digit(sort_key(tokens, wide, keys, i, v), shift)], 1u);

  /* two threads a digit add up the tiles, eight loads on their way */
  const int d = tid & (SORT_DIGITS - 1), half = tid / SORT_DIGITS;
  unsigned all = 0, mine = 0;
  for (unsigned t0 = half; t0 < tiles; t0 += 16) {
    unsigned c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const unsigned t = t0 + 2 * u;
      c[u] = counts[(t < tiles ? t : 0) * SORT_DIGITS + d];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const unsigned t = t0 + 2 * u;
      all += t < tiles ? c[u] : 0;
      mine += t < blockIdx.x ? c[u] : 0;
    }
  }
  if (half == 1) {
    total[d] = all;
    before[d] = mine;
  }
  __syncthreads();
  sort_starts(next, wave_total, half == 0 ? all + total[d] : 0, half == 0 ? mine + before[d] : 0);
  for (size_t i0 = lo; i0 < hi; i0 += WAVE) { /* in order: 64 entries at a time */
    const size_t i = i0 + lane;
    const bool live = i < hi;
    const unsigned key = live ? sort_key(tokens, wide, keys, i, v) : 0u;
    const unsigned place = live ? (places ? places[i] : (unsigned)i) : 0u;
    const unsigned at = sort_target(next[wave], sort_digit(key, shift), live);
    if (live) {
      keys_out[at] = key;
      places_out[at] = place;
    }
  }
}

/* ------------------------------------------------------------------ sums over the sorted places */

/* The first of the sorted keys that is at least `key`, m if there is none. (Seven probes a step are fewer steps
 * and more loads: r16 65536 places, 151936 x 2048, 189 us for 183.) */
__device__ __forceinline__ size_t lower_bound(const unsigned* keys, size_t m, unsigned key) {
  size_t lo = 0, hi = m;
  while (lo < hi) {
    const size_t mid = (lo + hi) / 2;
    if (keys[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

/* Rows of the table that a workgroup of the sums' launch clears: about 16 KiB of them (r16 [65536] tokens of
 * 151936 x 2048, the whole gradient: 64 KiB 202 us, 32 KiB 196, 16 KiB 181, 8 KiB 220; these workgroups in
 * front of the sums 195, between them 214). */
constexpr unsigned FILL_MOST = 64;
constexpr size_t FILL_BYTES = 16384;
inline unsigned embedding_fill_rows(size_t row_bytes) {
  const size_t rows = FILL_BYTES / row_bytes;
  return rows < 1 ? 1 : rows < FILL_MOST ? (unsigned)rows : FILL_MOST;
}

/* What happens at a boundary between chunks, entry i: `cut`: an id's places (a run of equal keys) lie on both
 * sides; then `after` of them from i on, and `over`: there are more than a chunk of them. A lane each looks at
 * a chunk's entries before the boundary and a chunk's behind it, so votes say all of it after one load; binary
 * searches are a dozen loads, one behind the other (the whole gradient, r32 3965 places of 114 rows of 1280:
 * 26.4 us, with votes 22.7; 8192 of 50257 x 1024 added to what is there 31.1 and 29.8). All lanes of the wavefront call it with the same i. */
struct ChunkEdge {
  bool cut, over;
  unsigned after;
};
__device__ __forceinline__ unsigned edge_key(const unsigned* keys, size_t m, size_t i, unsigned chunk) {
  const unsigned l = threadIdx.x % WAVE;
  const size_t at = i - chunk + l;
  return i > 0 && i < m && l < 2 * chunk && at < m ? keys[at] : 0xffffffffu; /* no id's key */
}
__device__ __forceinline__ ChunkEdge chunk_edge(unsigned key, size_t m, size_t i, unsigned chunk) {
  const unsigned long long same = __ballot(key == (unsigned)__builtin_amdgcn_readlane((int)key, (int)chunk));
  const unsigned before = (unsigned)__builtin_clzll(~(same << (WAVE - chunk))); /* up to chunk of them: zeros come in below */
  ChunkEdge e;
  e.after = (unsigned)__builtin_ctzll(~(same >> chunk)); /* likewise */
  e.cut = i > 0 && i < m && before > 0;
  e.over = before + e.after > chunk;
  return e;
}

/* Rows [row0, row0 + rows) of the table but those that are named: cleared, or (BLEND) scaled. */
template <class T, int W, bool BLEND, bool LOOSE>
__device__ __forceinline__ void clear_unnamed(const RowPacks<T, W, LOOSE>& rp, T* grads, const unsigned* named, size_t row0, unsigned rows, size_t n,
                                              typename precision<T>::type alpha) {
  using P = typename precision<T>::type;
  auto clear = [&](unsigned k, int p) {
    if (named[k]) return;
    T* row = grads + (row0 + k) * n;
    P out[W];
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = (P)0;
    if constexpr (BLEND) {
      rp.template load<true>(row, p, out);
#pragma unroll
      for (int i = 0; i < W; ++i) out[i] *= alpha;
    }
    rp.store(row, p, out);
  };
  if (rp.npk >= 256) {
    for (unsigned k = 0; k < rows; ++k)
      for (int p = threadIdx.x; p < rp.npk; p += 256) clear(k, p);
  } else { /* several narrow rows at a time */
    for (unsigned q = threadIdx.x; q < rows * (unsigned)rp.npk; q += 256) clear(q / (unsigned)rp.npk, (int)(q % (unsigned)rp.npk));
  }
}

/* Workgroups below sum_blocks: G lanes hold a strip of G packs of the columns and walk one chunk of
 * the sorted places, 256 / G chunks a workgroup. An id of no more places than a chunk belongs to the chunk
 * it begins in, which goes past its end for it; only longer ones are cut where a chunk ends. The other
 * workgroups clear (BLEND: scale) the rows of the table from `row_begin` on that no id names. partials: two rows of n for every chunk, the first for an id that
 * begins in an earlier chunk, the second for one that goes on in the next; the chunks where such an id begins
 * are listed, in any order. */
template <class T, int W, int G, bool BLEND, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_sum(
    const unsigned* keys, const unsigned* places, const T* dy, T* grads, typename precision<T>::type* partials,
    unsigned* crossing, unsigned* list, typename precision<T>::type scale, typename precision<T>::type alpha, unsigned v, size_t m, size_t n,
    size_t chunk, unsigned strips, unsigned sum_blocks, size_t row_begin, unsigned fill_rows, unsigned first_block) {
  using P = typename precision<T>::type;
  using V = typename vec_of<T, W>::type;
  const RowPacks<T, W, LOOSE> rp(n);
  const unsigned block = first_block + blockIdx.x;

  if (block >= sum_blocks) {
    __shared__ unsigned named[FILL_MOST];
    const size_t row0 = row_begin + (size_t)(block - sum_blocks) * fill_rows;
    const unsigned rows = (unsigned)(v - row0 < fill_rows ? v - row0 : fill_rows);
    if (threadIdx.x < rows) {
      const unsigned key = (unsigned)row0 + threadIdx.x;
      const size_t at = lower_bound(keys, m, key);
      named[threadIdx.x] = at < m && keys[at] == key;
    }
    __syncthreads();
    clear_unnamed<T, W, BLEND>(rp, grads, named, row0, rows, n, alpha);
    return;
  }

  constexpr int U = 8; /* rows on their way at once */
  const int sub = threadIdx.x / G, lane = threadIdx.x % G;
  const size_t c = (size_t)(block / strips) * (256 / G) + sub;
  const int p = (int)(block % strips) * G + lane;
  size_t lo = c * chunk, hi = lo + chunk < m ? lo + chunk : m;
  bool begun = false, goes_on = false; /* the first id began in another chunk, the last one goes on in another */
  constexpr int NG = G < WAVE ? WAVE / G : 1; /* chunks a wavefront */
  const size_t first = G < WAVE ? (size_t)(block / strips) * (256 / G) + threadIdx.x / WAVE * NG : c;
  unsigned at_edge[NG + 1];
#pragma unroll
  for (int g = 0; g <= NG; ++g) at_edge[g] = edge_key(keys, m, (first + g) * chunk, (unsigned)chunk);
#pragma unroll
  for (int g = 0; g <= NG; ++g) {
    const size_t i = (first + g) * chunk;
    const ChunkEdge e = chunk_edge(at_edge[g], m, i, (unsigned)chunk);
    if (!e.cut) continue;
    if (first + g == c) {
      begun = e.over;
      if (!e.over) lo = i + e.after;
    } else if (first + g == c + 1) {
      goes_on = e.over;
      if (!e.over) hi = i + e.after;
    }
  }
  if (lo >= hi || p >= rp.npk) return;

  P acc[W];
  unsigned current = keys[lo];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = (P)0;
  };
  auto leave = [&](bool cut) {
    if (current >= v) return; /* padded places */
    if (begun || cut) {
      P* at = partials + (c * 2 + (begun ? 0 : 1)) * n + (size_t)p * W;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < rp.valid(p)) at[i] = acc[i];
      if (!begun && p == 0) list[atomicAdd(crossing, 1u)] = (unsigned)c;
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
      row[u] = whole_pack<T, W, LOOSE, true>(rp, dy, places[i], m, n, p);
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
  leave(goes_on);
}

/* Up to DIRECT_MOST places in one launch and without a workspace: every workgroup has all keys in LDS. A group
 * of lanes takes a place; where no earlier place has its id, it adds up the rows of that place and of the
 * later ones, in order, and writes the id's row. The workgroups from `place_blocks` on clear (BLEND: scale)
 * the rows that no place names. What this saves is two launches, 3.2 us each of the caller's time; what it costs
 * is that the rows of one id wait for each other, 0.15 to 0.2 us a row. r16, table of 2000 rows of 1024, against
 * ordering the places first: 30 places 4.3 us against 10.4; 256 places of different ids 4.4 against 10.5, of ids as
 * common as one over their rank 6.4 against 10.6, half of them one id 19 against 10.6, all of them 37 against
 * 10.6. Which ids there are the host cannot know. */
constexpr unsigned DIRECT_MOST = 256;
constexpr int DIRECT_WORDS = DIRECT_MOST / WAVE;
template <class T, int W, int G, bool BLEND, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_direct(
    const void* tokens, unsigned wide, const T* dy, T* grads, typename precision<T>::type scale, typename precision<T>::type alpha, unsigned v, unsigned m,
    size_t n, unsigned strips, unsigned place_blocks, unsigned fill_rows, unsigned first_block) {
  using P = typename precision<T>::type;
  using V = typename vec_of<T, W>::type;
  const RowPacks<T, W, LOOSE> rp(n);
  __shared__ unsigned keys[DIRECT_MOST];
  const unsigned block = first_block + blockIdx.x;
  const unsigned mine = threadIdx.x < m ? token_key(tokens, wide != 0, threadIdx.x, v) : v;

  if (block >= place_blocks) {
    __shared__ unsigned named[FILL_MOST];
    const size_t row0 = (size_t)(block - place_blocks) * fill_rows;
    const unsigned rows = (unsigned)(v - row0 < fill_rows ? v - row0 : fill_rows);
    if (threadIdx.x < rows) named[threadIdx.x] = 0;
    __syncthreads();
    if (mine >= row0 && mine - row0 < rows) named[mine - row0] = 1; /* v is in no range: row0 + rows <= v */
    __syncthreads();
    clear_unnamed<T, W, BLEND>(rp, grads, named, row0, rows, n, alpha);
    return;
  }
  keys[threadIdx.x] = mine;
  __syncthreads();
  const int sub = threadIdx.x / G, lane = threadIdx.x % G;
  const unsigned i = (block / strips) * (256 / G) + sub;
  const int p = (int)(block % strips) * G + lane;
  const unsigned key = i < m ? keys[i] : v;
  /* the places of this group's id, a bit each, by votes of the whole wavefront for each of its groups */
  unsigned long long places[DIRECT_WORDS];
#pragma unroll
  for (int g = 0; g < (G < WAVE ? WAVE / G : 1); ++g) {
    const unsigned asked = __shfl(key, g * (G < WAVE ? G : 0), WAVE);
#pragma unroll
    for (int w = 0; w < DIRECT_WORDS; ++w) {
      const unsigned long long same = __ballot(keys[w * WAVE + threadIdx.x % WAVE] == asked);
      if (G >= WAVE || (int)(threadIdx.x % WAVE) / G == g) places[w] = same;
    }
  }
  if (i >= m || p >= rp.npk || key >= v) return;
  unsigned long long left = 0;
  bool earlier = false; /* then an earlier place's group adds this one's row */
#pragma unroll
  for (int w = 0; w < DIRECT_WORDS; ++w) {
    const unsigned long long before = i / WAVE > (unsigned)w ? ~0ull : i / WAVE == (unsigned)w ? (1ull << (i % WAVE)) - 1ull : 0ull;
    earlier = earlier || (places[w] & before) != 0;
    left |= places[w];
  }
  if (earlier) return;
  P acc[W];
  double sum[W]; /* of every 32 rows, as many as a chunk of the longer batches has */
#pragma unroll
  for (int e = 0; e < W; ++e) {
    acc[e] = (P)0;
    sum[e] = 0.0;
  }
  constexpr int U = 8;
  for (int turn = 1; left; ++turn) {
    unsigned found[U]; /* the next places of the id, the last one again where there are fewer */
    int count = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unsigned at = u ? found[u - 1] : 0u;
#pragma unroll
      for (int w = DIRECT_WORDS - 1; w >= 0; --w) /* the lowest place that is left */
        if (places[w]) at = w * WAVE + (unsigned)__builtin_ctzll(places[w]);
      found[u] = at;
      count += left ? 1 : 0;
      left = 0;
#pragma unroll
      for (int w = 0; w < DIRECT_WORDS; ++w) {
        if (at / WAVE == (unsigned)w) places[w] &= ~(1ull << (at % WAVE));
        left |= places[w];
      }
    }
    V row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = whole_pack<T, W, LOOSE, true>(rp, dy, found[u], m, n, p);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += u < count ? (P)row[u][e] : (P)0;
    if (turn % (32 / U) == 0) {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        sum[e] += (double)acc[e];
        acc[e] = (P)0;
      }
    }
  }
  T* row = grads + (size_t)key * n;
  P out[W];
#pragma unroll
  for (int e = 0; e < W; ++e) out[e] = scale * (P)(sum[e] + (double)acc[e]);
  if constexpr (BLEND) {
    P old[W];
    rp.template load<true>(row, p, old);
#pragma unroll
    for (int e = 0; e < W; ++e) out[e] += alpha * old[e];
  }
  rp.store(row, p, out);
}

/* The ids that cross chunks: the partial rows of each are added up in order, in fp64. Workgroups take (id,
 * strip of JOIN_LANES * CW columns) in turn; the slices of a workgroup take the partial rows in turn, up
 * to eight on their way, and are then added. One, four and eight of them by how many there are (always four:
 * r16 22002 places of 383 rows of 128 take 35.6 us for 31.1; always eight: 65536 of 151936 x 2048 178 for 176);
 * the chunks an id reaches are looked for among 256 first, then 1024 at a time (always 1024: 183). */
constexpr int JOIN_LANES = 32, JOIN_SLICES = 256 / JOIN_LANES, JOIN_LOOKS = 4;
template <class T, int CW, bool BLEND>
__global__ __launch_bounds__(256) void embedding_join(
    const unsigned* keys, const typename precision<T>::type* partials, const unsigned* crossing, const unsigned* list, T* grads,
    typename precision<T>::type scale, typename precision<T>::type alpha, size_t m, size_t n, size_t chunk, unsigned strips) {
  using P = typename precision<T>::type;
  constexpr int COLS = JOIN_LANES * CW;
  __shared__ double part[JOIN_SLICES][COLS + 1];
  __shared__ unsigned ends[256 / WAVE];
  const unsigned work = *crossing * strips;
  const int l = threadIdx.x % JOIN_LANES, slice = threadIdx.x / JOIN_LANES;
  for (unsigned q = blockIdx.x; q < work; q += gridDim.x) {
    const size_t c = list[q / strips];
    const unsigned key = keys[(c + 1) * chunk - 1]; /* the id that goes on in the chunk behind */
    /* the chunks behind c that begin with the id: sorted, so they are the first ones */
    size_t later = 0;
    for (int looks = 1;; looks = JOIN_LOOKS) {
      unsigned same = 0;
#pragma unroll
      for (int k = 0; k < JOIN_LOOKS; ++k) {
        const size_t at = (c + 1 + later + k * 256 + threadIdx.x) * chunk;
        const bool look = k < looks && at < m;
        same += (unsigned)__builtin_popcountll(__ballot(look && keys[look ? at : 0] == key));
      }
      if (threadIdx.x % WAVE == 0) ends[threadIdx.x / WAVE] = same;
      __syncthreads();
      unsigned found = 0;
#pragma unroll
      for (int w = 0; w < 256 / WAVE; ++w) found += ends[w];
      later += found;
      __syncthreads();
      if (found < (unsigned)looks * 256) break;
    }
    const size_t j = (size_t)(q % strips) * COLS + l * CW;
    double s[CW];
#pragma unroll
    for (int i = 0; i < CW; ++i) s[i] = 0.0;
    if (j < n) { /* CW > 1: n is a multiple of it */
      auto add = [&]<int R>() { /* R partial rows on their way */
        for (size_t k0 = slice; k0 <= later; k0 += R * JOIN_SLICES) {
          P t[R][CW];
#pragma unroll
          for (int u = 0; u < R; ++u) {
            const size_t k = k0 + u * JOIN_SLICES <= later ? k0 + u * JOIN_SLICES : k0;
            load_pack_nt<P, CW>(partials + ((c + k) * 2 + (k == 0 ? 1 : 0)) * n + j, t[u]);
          }
#pragma unroll
          for (int u = 0; u < R; ++u)
#pragma unroll
            for (int i = 0; i < CW; ++i) s[i] += k0 + u * JOIN_SLICES <= later ? (double)t[u][i] : 0.0;
        }
      };
      if (later < JOIN_SLICES) add.template operator()<1>();
      else if (later < 4 * JOIN_SLICES) add.template operator()<4>();
      else add.template operator()<8>();
    }
#pragma unroll
    for (int i = 0; i < CW; ++i) part[slice][l * CW + i] = s[i];
    __syncthreads();
    for (int col = threadIdx.x; col < COLS && (size_t)(q % strips) * COLS + col < n; col += 256) {
      double t = 0.0;
#pragma unroll
      for (int k = 0; k < JOIN_SLICES; ++k) t += part[k][col];
      T* at = grads + (size_t)key * n + (size_t)(q % strips) * COLS + col;
      double out = (double)scale * t;
      if constexpr (BLEND) out += (double)alpha * (double)*at;
      *at = (T)out;
    }
    __syncthreads();
  }
}

/* ------------------------------------------------------------------ host dispatch */

/* The sorted places one chunk holds: as many as leave the GPU 1024 workgroups, or half of that
 * for narrow rows, from 4 to 32. */
inline size_t embedding_chunk(size_t m, size_t row_bytes) {
  const size_t lanes = (row_bytes + PACK_BYTES - 1) / PACK_BYTES, groups = lanes >= 256 ? 1 : 256 / lanes; /* chunks a workgroup */
  size_t chunk = 4;
  while (chunk < 32 && m / chunk > 1024 * (groups < 8 ? groups : 8)) chunk *= 2;
  return chunk;
}

/* Bytes of the table that a launch of the sort clears beside it: what the rest of the GPU writes in the time
 * the sort takes anyway. */
constexpr size_t RANK_CLEARS = (size_t)32 << 20, SORT_COUNT_CLEARS = (size_t)24 << 20, SORT_PLACE_CLEARS = (size_t)48 << 20;

/* Workspace of the reverse: two pairs of keys and places that the sort writes in turn, the counts of its
 * tiles, the ids that cross chunks with their number, and two partial rows a chunk. Every
 * part starts on a 256-byte boundary. */
struct EmbeddingScratch {
  size_t keys[2], places[2], counts, crossing, list, partials, bytes;
};
template <class T> inline EmbeddingScratch embedding_scratch(size_t m, size_t n) {
  EmbeddingScratch s{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t chunk = embedding_chunk(m, n * sizeof(T)), chunks = (m + chunk - 1) / chunk, pairs = m > RANK_MOST ? 2 : 1;
  for (size_t k = 0; k < pairs; ++k) {
    s.keys[k] = take(m * sizeof(unsigned));
    s.places[k] = take(m * sizeof(unsigned));
  }
  const size_t tile = sort_tile(m), tiles = m > RANK_MOST ? (m + tile - 1) / tile : 0;
  s.counts = take(tiles * SORT_DIGITS * sizeof(unsigned));
  s.crossing = take(sizeof(unsigned));
  s.list = take(chunks * sizeof(unsigned));
  s.partials = take(chunks * 2 * n * sizeof(typename precision<T>::type));
  s.bytes = at;
  return s;
}

/* Lanes for a strip of a row's packs: the next power of two, from 8 to 256. */
inline size_t strip_lanes(size_t packs) {
  size_t lanes = 8;
  while (lanes < 256 && lanes < packs) lanes *= 2;
  return lanes;
}
template <class F> inline void for_strip(size_t packs, F&& f) {
  switch (strip_lanes(packs)) {
    case 8: f.template operator()<8>(); break;
    case 16: f.template operator()<16>(); break;
    case 32: f.template operator()<32>(); break;
    case 64: f.template operator()<64>(); break;
    case 128: f.template operator()<128>(); break;
    default: f.template operator()<256>();
  }
}
/* Workgroups of 256 threads that take `rows` rows of `packs` packs: a strip of 256 / lanes rows each. */
struct StripGrid { size_t strips, blocks; };
inline StripGrid strip_grid(size_t rows, size_t packs) {
  const size_t lanes = strip_lanes(packs), strips = (packs + lanes - 1) / lanes, each = 256 / lanes;
  return {strips, (rows + each - 1) / each * strips};
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
  const StripGrid rows = strip_grid(m, packs);
  require(rows.blocks < 0x7fffffffull, "embedding: too many rows for one call");
  for_strip(packs, [&]<int G>() {
    in_launches(rows.blocks, [&](dim3 grid, unsigned first) {
      auto go = [&]<bool LOOSE>() {
        embedding_rows<T, W, G, LOOSE><<<grid, dim3(256), 0, stream>>>(table, tokens, y, (P)scale, id_bytes == 8, (unsigned)v, m, n, (unsigned)rows.strips, first);
      };
      if (loose) go.template operator()<true>();
      else go.template operator()<false>();
      MP_CHECK_LAUNCH();
    });
  });
}

template <class T>
inline void embedding_reverse(const void* tokens, const T* dy, T* grads, void* scratch, double scale, double alpha, size_t id_bytes,
                              size_t v, size_t m, size_t n, hipStream_t stream) {
  using P = typename precision<T>::type;
  constexpr int W = PACK_BYTES / (int)sizeof(T);
  embedding_check(tokens, id_bytes, v, m, n);
  if (v == 0 || n == 0) return;
  require(m == 0 || scratch != nullptr, "embedding reverse: scratch must hold mpEmbeddingReverseScratchBytes bytes");
  require(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "embedding reverse: scratch must be 16-byte aligned");
  const bool loose = !(aligned16(dy) && aligned16(grads) && n % W == 0);
  const size_t packs = (n + W - 1) / W;
  const unsigned wide = id_bytes == 8, fill_rows = embedding_fill_rows(n * sizeof(T));
  const size_t fill_all = alpha == 1.0 ? 0 : (v + fill_rows - 1) / fill_rows; /* workgroups for all rows of the table */
  if (m <= DIRECT_MOST) {
    const StripGrid places = strip_grid(m, packs);
    require(places.blocks + fill_all < 0x7fffffffull, "embedding reverse: too many rows for one call");
    for_strip(packs, [&]<int G>() {
      in_launches(places.blocks + fill_all, [&](dim3 grid, unsigned first) { /* none: no token, and nothing to clear or to scale */
        auto go = [&]<bool BLEND, bool LOOSE>() {
          embedding_direct<T, W, G, BLEND, LOOSE><<<grid, dim3(256), 0, stream>>>(tokens, wide, dy, grads, (P)scale, (P)alpha, (unsigned)v, (unsigned)m, n,
                                                                                  (unsigned)places.strips, (unsigned)places.blocks, fill_rows, first);
        };
        if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
        else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
        MP_CHECK_LAUNCH();
      });
    });
    return;
  }
  /* every grid, before the first launch */
  const size_t chunk = embedding_chunk(m, n * sizeof(T)), chunks = (m + chunk - 1) / chunk;
  const StripGrid sums = strip_grid(chunks, packs);
  require(sums.blocks + fill_all < 0x7fffffffull, "embedding reverse: too many rows for one call");
  constexpr bool FP32 = sizeof(P) == 4;
  const bool four = FP32 && n % 4 == 0; /* columns a thread of the join: four where the partial rows are 16-byte aligned */
  const size_t join_cols = JOIN_LANES * (four ? 4 : 1), join_strips = (n + join_cols - 1) / join_cols, joins = (chunks - 1) * join_strips;
  require(chunks * join_strips < 0x7fffffffull, "embedding reverse: too many rows for one call");

  const EmbeddingScratch at = embedding_scratch<T>(m, n);
  char* base = static_cast<char*>(scratch);
  auto words = [&](size_t offset) { return reinterpret_cast<unsigned*>(base + offset); };
  unsigned *keys[2] = {words(at.keys[0]), words(at.keys[1])}, *places[2] = {words(at.places[0]), words(at.places[1])};
  unsigned *counts = words(at.counts), *crossing = words(at.crossing), *list = words(at.list);
  P* partials = reinterpret_cast<P*>(base + at.partials);

  /* the sort, with a part of the clearing in each of its launches */
  const int passes = sort_passes(v);
  const size_t unit = (size_t)SORT_THREADS * FILL_PACKS * W; /* elements a clearing workgroup of a sort's launch takes */
  const size_t elements = alpha == 0.0 ? v * n : 0;
  size_t cleared = 0; /* elements so far, from the table's start */
  auto share = [&](size_t bytes) { /* of the next launch: elements, a whole number of its workgroups' */
    const size_t want = bytes / sizeof(T) / unit * unit, left = elements - cleared;
    return want < left ? want : left;
  };
  const unsigned *sorted_keys, *sorted_places;
  if (m <= RANK_MOST) {
    const size_t part = share(RANK_CLEARS);
    const unsigned groups = (unsigned)((m + RANK_ENTRIES - 1) / RANK_ENTRIES);
    embedding_rank<T><<<dim3(groups + (unsigned)((part + unit - 1) / unit)), dim3(SORT_THREADS), groups * RANK_ENTRIES * sizeof(unsigned), stream>>>(
        tokens, wide, keys[0], places[0], crossing, (unsigned)v, (unsigned)m, groups, grads, part);
    MP_CHECK_LAUNCH();
    cleared += part;
    sorted_keys = keys[0];
    sorted_places = places[0];
  } else {
    const size_t tile = sort_tile(m);
    const unsigned tiles = (unsigned)((m + tile - 1) / tile);
    for (int pass = 0; pass < passes; ++pass) {
      const int to = pass & 1;
      const unsigned* from_keys = pass ? keys[to ^ 1] : nullptr;
      size_t part = share(SORT_COUNT_CLEARS);
      embedding_sort_count<T><<<dim3(tiles + (unsigned)((part + unit - 1) / unit)), dim3(SORT_THREADS), 0, stream>>>(
          tokens, wide, from_keys, counts, crossing, (unsigned)v, m, tile, tiles, pass * SORT_BITS, grads + cleared, part);
      MP_CHECK_LAUNCH();
      cleared += part;
      part = share(SORT_PLACE_CLEARS);
      embedding_sort_place<T><<<dim3(tiles + (unsigned)((part + unit - 1) / unit)), dim3(SORT_THREADS), 0, stream>>>(
          tokens, wide, from_keys, pass ? places[to ^ 1] : nullptr, counts, keys[to], places[to], (unsigned)v, m, (unsigned)tile, tiles,
          pass * SORT_BITS, grads + cleared, part);
      MP_CHECK_LAUNCH();
      cleared += part;
    }
    sorted_keys = keys[(passes - 1) & 1];
    sorted_places = places[(passes - 1) & 1];
  }

  const size_t row_begin = cleared / n; /* rows from here on are still to be looked at, the first of them perhaps half cleared */
  const size_t fill = alpha == 1.0 ? 0 : (v - row_begin + fill_rows - 1) / fill_rows;
  for_strip(packs, [&]<int G>() {
    in_launches(sums.blocks + fill, [&](dim3 grid, unsigned first) {
      auto go = [&]<bool BLEND, bool LOOSE>() {
        embedding_sum<T, W, G, BLEND, LOOSE><<<grid, dim3(256), 0, stream>>>(sorted_keys, sorted_places, dy, grads, partials, crossing, list, (P)scale, (P)alpha,
                                                                             (unsigned)v, m, n, chunk, (unsigned)sums.strips, (unsigned)sums.blocks, row_begin,
                                                                             fill_rows, first);
      };
      if (alpha != 0.0) { if (loose) go.template operator()<true, true>(); else go.template operator()<true, false>(); }
      else { if (loose) go.template operator()<false, true>(); else go.template operator()<false, false>(); }
      MP_CHECK_LAUNCH();
    });
  });
  if (chunks > 1) {
    const size_t cap = (size_t)compute_units() * 8;
    const dim3 grid((unsigned)(joins < cap ? joins : cap)), block(256);
    auto go = [&]<int CW, bool BLEND>() {
      embedding_join<T, CW, BLEND><<<grid, block, 0, stream>>>(sorted_keys, partials, crossing, list, grads, (P)scale, (P)alpha, m, n, chunk, (unsigned)join_strips);
    };
    if (four) { if constexpr (FP32) { if (alpha != 0.0) go.template operator()<4, true>(); else go.template operator()<4, false>(); } }
    else { if (alpha != 0.0) go.template operator()<1, true>(); else go.template operator()<1, false>(); }
    MP_CHECK_LAUNCH();
  }
}

}  // namespace mp

#endif
#endif
