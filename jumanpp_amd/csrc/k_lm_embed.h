// Language-model operators 1: rows of a table by word (k_lm_embed), and the gradient of a table whose rows were read by
// word: dW_v = sum over the entries j with word v of w_j src_(j / K).  For the lookup w_j is the scale, K = 1 and src the
// gradient of the rows; for the noise-contrastive loss (k_lm_nce.h) w_j is the gradient of the score of candidate j and
// src_(j / K) the state of its token.
//
// The gradient sums by word without atomics on floats, so its bits follow from the inputs:
//   k_lm_sort_one / k_lm_sort_count, _scan, _scatter   entries into ascending (word, entry): least digit first, stable; an
//                                                      entry takes its row of src and its weight along
//   k_lm_seg_sum                                       a workgroup takes a tile of sorted entries, a group of lanes a part of
//                                                      it: a word that lies inside one part is written at once, one that
//                                                      crosses parts is put together in LDS, one that crosses tiles leaves a
//                                                      partial row per tile
//   k_lm_seg_join                                      the partial rows of those words, in tile order
// 507 904 bfloat16 rows of 256 columns, 65 521 words: 44 us to sort, 73 to sum, 9 to join.
// For the loss, 2.2 M entries on 65 536 such rows: 74, 128 and 5.
// Rows of words that do not occur are zeroed by workgroups that ride in the grid of the first sorting kernel: that one uses
// a fraction of the chip.  Zeros and finished rows leave with the non-temporal hint: the gradient is not read here, src is
// (134 us without for the lookup's gradient above, 126 with; small ones are within 1 % either way).
#ifndef JPP_K_LM_EMBED_H
#define JPP_K_LM_EMBED_H

#include "jpp_lm.h"

namespace jpp {

// ---- lookup --------------------------------------------------------------------
// y_t = scale * W[id_t].  A thread moves packs of V elements, a workgroup `rowsPerBlock` rows; nothing but the loads and
// stores counts.  The ids of PER packs are loaded together, then their rows: one wait each, not one a pack.  2 031 616 rows of
// 128 columns, a 32-bit table of 31 200 rows into bfloat16: 101 us, 5.4 TB/s of ids and results (the table stays in the
// caches; filling memory reaches 6.8).
template <class Tin, class Tout, int V, int PER, bool STREAM>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_embed(const typename Tin::store* __restrict__ table, i64 tableStride, u32 vocab, u32 dim, LmIds ids, u64 n, float scale,
               typename Tout::store* __restrict__ out, i64 outStride, u32 rowsPerBlock) {
  const u32 packs = (dim + V - 1) / V;
  const u64 groups = (n + rowsPerBlock - 1) / rowsPerBlock;
  for (u64 g = blockIdx.x; g < groups; g += gridDim.x) {
    const u64 t0 = g * rowsPerBlock;
    const u32 rows = n - t0 < rowsPerBlock ? (u32)(n - t0) : rowsPerBlock;
    const u32 total = rows * packs;
    for (u32 i0 = threadIdx.x; i0 < total; i0 += kLmThreads * PER) {
      u32 r[PER], c[PER], row[PER];
      LmPack<Tin, V> x[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const u32 i = i0 + (u32)k * kLmThreads < total ? i0 + (u32)k * kLmThreads : i0;
        r[k] = i / packs;
        c[k] = lm_col<V>(i - r[k] * packs, dim);
        row[k] = lm_row(ids, t0 + r[k], vocab);
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        x[k].zero();
        // (an id that names no word reads row 0, if there is one, for nothing)
        if (vocab != 0) x[k] = lm_load<Tin, V>(table + (i64)(row[k] < vocab ? row[k] : 0u) * tableStride + c[k]);
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = row[k] < vocab ? x[k].get(e) * scale : 0.f;
        if (i0 + (u32)k * kLmThreads < total) lm_store<Tout, V, STREAM>(out + (i64)(t0 + r[k]) * outStride + c[k], lm_pack<Tout, V>(y));
      }
    }
  }
}

// ---- sorting the entries by word -------------------------------------------------
struct LmZero {      // the matrix that the riding workgroups clear
  float* data;
  i64 stride;
  u64 rows;
  u32 cols, lastCols;   // (a matrix without gaps is cut into long rows, the last one shorter)
};

__device__ __forceinline__ void lm_zero_rows(const LmZero& z, u64 first, u64 step) {
  for (u64 r = first; r < z.rows; r += step) {
    float* row = z.data + (i64)r * z.stride;
    const u32 cols = r + 1 == z.rows ? z.lastCols : z.cols;
    const u32 packs = cols / 4;
    LmPack<LmF32, 4> zero;
    zero.zero();
    for (u32 c = threadIdx.x; c < packs; c += blockDim.x) lm_store<LmF32, 4, true>(row + 4 * (u64)c, zero);
    for (u32 c = packs * 4 + threadIdx.x; c < cols; c += blockDim.x) row[c] = 0.f;
  }
}

__global__ void __launch_bounds__(kLmThreads) k_lm_zero(LmZero z) { lm_zero_rows(z, blockIdx.x, gridDim.x); }

// an entry on its way through the sort
struct LmPair {
  u32 key;           // word, `vocab` for none
  u32 row;           // of src
  static constexpr bool kWeighted = false;
};
struct LmEntry {
  u32 key;
  u32 row;
  float weight;
  static constexpr bool kWeighted = true;
};

// where the first pass finds its entries
template <class E>
struct LmKeysOfIds {
  LmIds ids;
  u32 vocab;
  u32 perToken;      // entries of a token (= of a row of src); the token counts only if its entry 0 names a word
  LmDiv token;       // ... and the division by it
  const float* weights;
  __device__ __forceinline__ u32 key(u32 j) const {
    u32 k = lm_row(ids, j, vocab);
    if (perToken > 1 && k < vocab && lm_row(ids, token(j) * perToken, vocab) == vocab) k = vocab;
    return k;
  }
  __device__ __forceinline__ E entry(u32 j) const {
    if constexpr (E::kWeighted) return E{key(j), token(j), weights[j]};
    else return E{key(j), j};
  }
};
template <class E>
struct LmKeysOfPass {
  const E* entries;
  __device__ __forceinline__ u32 key(u32 j) const { return entries[j].key; }
  __device__ __forceinline__ E entry(u32 j) const { return entries[j]; }
};

constexpr u32 kLmBins = 256;   // (= kLmThreads: a digit a thread)
constexpr int kLmOneThreads = 1024, kLmOneRounds = 4;
constexpr u32 kLmSortOne = kLmOneThreads * kLmOneRounds;           // up to here one workgroup sorts everything in LDS

// inclusive sum over the lanes
__device__ __forceinline__ u32 lm_scan_incl(u32 v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u32 o = wave_shfl_u32(v, lane - d < 0 ? lane : lane - d);
    if (lane >= d) v += o;
  }
  return v;
}

// Rank of a wavefront's keys among equal digits, in the order (round, lane).  cnt: this wavefront's kLmBins counters in
// LDS, zero before the first round.  One ballot per digit bit finds the lanes with the same digit.
__device__ __forceinline__ u32 lm_rank_round(u32 digit, bool act, u32 bits, u32* cnt, int lane) {
  u64 same = wave_ballot(act);
  for (u32 b = 0; b < bits; ++b) {
    const u64 set = wave_ballot(((digit >> b) & 1u) != 0);
    same &= ((digit >> b) & 1u) != 0 ? set : ~set;
  }
  const u64 below = same & ((u64{1} << lane) - 1);
  u32 before = 0;
  if (act) before = cnt[digit];
  wave_sync();
  if (act && below == 0) cnt[digit] = before + (u32)popc64(same);
  wave_sync();
  return before + (u32)popc64(below);
}

// Exclusive sums of the kLmBins values in `v` (LDS), by the first kLmBins threads; `part`: 4 words of LDS.
__device__ __forceinline__ void lm_scan_bins(u32* v, u32* part, int lane, int wv) {
  u32 x = 0, incl = 0;
  if (wv < 4) {
    x = v[threadIdx.x];
    incl = lm_scan_incl(x, lane);
    if (lane == 63) part[wv] = incl;
  }
  __syncthreads();
  if (wv < 4) {
    u32 base = 0;
    for (int w = 0; w < wv; ++w) base += part[w];
    v[threadIdx.x] = base + incl - x;
  }
  __syncthreads();
}

// Few entries: one workgroup, every pass in LDS.  A thread's keys are those of its rounds, wavefront after wavefront, so
// the order (wavefront, round, lane) is the order of the list.
template <class E>
__global__ void __launch_bounds__(kLmOneThreads)
    k_lm_sort_one(LmKeysOfIds<E> keys, u32 n, u32 keyBits, u32 passes, E* __restrict__ out, u32* __restrict__ spanCount, LmZero zero) {
  constexpr int kWaves = kLmOneThreads / 64;
  __shared__ u32 s_key[kLmSortOne];
  __shared__ u32 s_entry[kLmSortOne];
  __shared__ u32 s_cnt[kWaves][kLmBins];
  __shared__ u32 s_bin[kLmBins];
  __shared__ u32 s_part[4];
  if (blockIdx.x != 0) {
    lm_zero_rows(zero, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  if (threadIdx.x < 2) spanCount[threadIdx.x] = 0;
  const u32 rounds = (n + kLmOneThreads - 1) / kLmOneThreads;   // (1 .. kLmOneRounds)
  const u32 pos0 = (u32)wv * 64u * rounds + (u32)lane;
  u32 key[kLmOneRounds], entry[kLmOneRounds];
#pragma unroll
  for (u32 r = 0; r < (u32)kLmOneRounds; ++r) {
    entry[r] = pos0 + 64 * r;
    key[r] = 0;
    if (r < rounds && entry[r] < n) key[r] = keys.key(entry[r]);
  }
  const u32 digitBits = (keyBits + passes - 1) / passes;
  for (u32 pass = 0; pass < passes; ++pass) {
    const u32 shift = pass * digitBits, mask = (1u << digitBits) - 1;
    for (u32 i = threadIdx.x; i < (u32)kWaves * kLmBins; i += kLmOneThreads) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    u32 rank[kLmOneRounds];
#pragma unroll
    for (u32 r = 0; r < (u32)kLmOneRounds; ++r) {
      rank[r] = 0;
      if (r < rounds) rank[r] = lm_rank_round((key[r] >> shift) & mask, pos0 + 64 * r < n, digitBits, s_cnt[wv], lane);
    }
    __syncthreads();
    if (threadIdx.x < kLmBins) {
      u32 run = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const u32 x = s_cnt[w][threadIdx.x];
        s_cnt[w][threadIdx.x] = run;
        run += x;
      }
      s_bin[threadIdx.x] = run;
    }
    __syncthreads();
    lm_scan_bins(s_bin, s_part, lane, wv);
    const bool last = pass + 1 == passes;
#pragma unroll
    for (u32 r = 0; r < (u32)kLmOneRounds; ++r) {
      if (r < rounds && pos0 + 64 * r < n) {
        const u32 d = (key[r] >> shift) & mask;
        const u32 to = s_bin[d] + s_cnt[wv][d] + rank[r];
        if (last) {
          out[to] = keys.entry(entry[r]);
        } else {
          s_key[to] = key[r];
          s_entry[to] = entry[r];
        }
      }
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (u32 r = 0; r < (u32)kLmOneRounds; ++r) {
        if (r < rounds && pos0 + 64 * r < n) {
          key[r] = s_key[pos0 + 64 * r];
          entry[r] = s_entry[pos0 + 64 * r];
        }
      }
      __syncthreads();
    }
  }
}

// Many entries, a pass, a tile of R entries a thread a workgroup: the digits of every tile ...  counts: [tile][bin] where the
// scatter kernel sums them itself, [bin][tile] for k_lm_sort_scan.  What bounds these kernels is not bytes (a few megabytes a
// pass) but the chain of a tile: load, rank, place.
// Tiles up to which the scatter kernel looks back by itself: a launch a pass costs more than 64 rows of 1 KB (the loss of
// 1 021 tokens, 42 tiles: 37 us, 51 with the launches).
constexpr u32 kLmSortOwn = 64;
template <int R, class Keys>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_sort_count(Keys keys, u32 n, u32 shift, u32 mask, u32* __restrict__ counts, u32 tiles, u32* __restrict__ spanCount, LmZero zero) {
  __shared__ u32 s_cnt[kLmBins];
  if (blockIdx.x >= tiles) {
    lm_zero_rows(zero, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x < 2) spanCount[threadIdx.x] = 0;
  s_cnt[threadIdx.x] = 0;
  __syncthreads();
  const u32 j0 = blockIdx.x * (kLmThreads * R) + threadIdx.x;
  u32 key[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const u32 j = j0 + (u32)r * kLmThreads;
    key[r] = keys.key(j < n ? j : n - 1);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (j0 + (u32)r * kLmThreads < n) atomicAdd(&s_cnt[(key[r] >> shift) & mask], 1u);
  __syncthreads();
  counts[tiles <= kLmSortOwn ? blockIdx.x * (u64)kLmBins + threadIdx.x : threadIdx.x * (u64)tiles + blockIdx.x] = s_cnt[threadIdx.x];
}

// ... per digit the exclusive sums over the tiles and the total, a workgroup a digit ...
constexpr int kLmScanPer = 8;
__global__ void __launch_bounds__(kLmThreads) k_lm_sort_scan(u32* __restrict__ counts, u32 tiles, u32* __restrict__ totals) {
  __shared__ u32 s_part[4];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  u32* c = counts + blockIdx.x * (u64)tiles;
  u32 run = 0;
  for (u32 i0 = 0; i0 < tiles; i0 += kLmThreads * kLmScanPer) {
    u32 x[kLmScanPer], sum = 0;
    const u32 i = i0 + threadIdx.x * kLmScanPer;
#pragma unroll
    for (int k = 0; k < kLmScanPer; ++k) x[k] = i + (u32)k < tiles ? c[i + (u32)k] : 0u;
#pragma unroll
    for (int k = 0; k < kLmScanPer; ++k) sum += x[k];
    const u32 incl = lm_scan_incl(sum, lane);
    if (lane == 63) s_part[wv] = incl;
    __syncthreads();
    u32 before = run + incl - sum;
    for (int w = 0; w < 4; ++w) {
      if (w < wv) before += s_part[w];
      run += s_part[w];
    }
#pragma unroll
    for (int k = 0; k < kLmScanPer; ++k) {
      if (i + (u32)k < tiles) c[i + (u32)k] = before;
      before += x[k];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// ... and every entry to its place
template <int R, class E, class Keys>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_sort_scatter(Keys keys, u32 n, u32 shift, u32 bits, const u32* __restrict__ counts, u32 tiles, const u32* __restrict__ totals,
                      E* __restrict__ out) {
  constexpr int kWaves = kLmThreads / 64;
  __shared__ u32 s_cnt[kWaves][kLmBins];
  __shared__ u32 s_bin[kLmBins];
  __shared__ u32 s_part[4];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 mask = (1u << bits) - 1;
  const u32 pos0 = blockIdx.x * (kLmThreads * R) + (u32)wv * (64u * R) + (u32)lane;
  E p[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const u32 j = pos0 + 64u * (u32)r;
    p[r] = keys.entry(j < n ? j : n - 1);
  }
  // of this thread's digit: entries in earlier tiles, in all
  u32 mine = 0, total = 0;
  if (tiles <= kLmSortOwn) {
#pragma unroll 16
    for (u32 t = 0; t < tiles; ++t) {
      const u32 x = counts[t * (u64)kLmBins + threadIdx.x];
      mine += t < blockIdx.x ? x : 0u;
      total += x;
    }
  } else {
    mine = counts[threadIdx.x * (u64)tiles + blockIdx.x];
    total = totals[threadIdx.x];
  }
  s_bin[threadIdx.x] = total;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s_cnt[w][threadIdx.x] = 0;
  __syncthreads();
  lm_scan_bins(s_bin, s_part, lane, wv);
  u32 rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    rank[r] = lm_rank_round((p[r].key >> shift) & mask, pos0 + 64u * (u32)r < n, bits, s_cnt[wv], lane);
  __syncthreads();
  {
    u32 run = s_bin[threadIdx.x] + mine;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const u32 x = s_cnt[w][threadIdx.x];
      s_cnt[w][threadIdx.x] = run;
      run += x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (pos0 + 64u * (u32)r < n) out[s_cnt[wv][(p[r].key >> shift) & mask] + rank[r]] = p[r];
}

// ---- sums by word ----------------------------------------------------------------
template <class E>
struct LmSeg {
  const E* entries;      // sorted
  u32 n;
  u32 part;              // entries of a group, a multiple of 8
  u32 tile;              // entries of a workgroup
  u32 tiles;
  u32 vocab, dim, colBlocks;
  float scale;           // weight of every entry that has none of its own
  u32 srcStride;
  float* grad;
  i64 gradStride;
  float* head;           // [tiles][dim] partial row of the word that began in an earlier tile
  float* tail;           // [tiles][dim] ... of the word that goes on in the next
  u32* span;             // tiles whose last word began there and goes on
  u32* spanCount;
};

// A group of L lanes owns L V columns of `part` entries; a workgroup's groups, in order, own its tile.  The rows of src are
// the bytes that count.  For the lookup's gradient each is read once and a group takes as much of it as it can (L V >= dim).
// For the loss each is read by every candidate of its token, from anywhere in the chip: there a group takes one cache line
// of a row, and as the workgroups of a tile's column blocks go round the XCDs, an XCD sees a part of src's columns only,
// most of which its own L2 then holds (half lines, eight blocks of 256 columns of bf16, were no use: the L2 fetches whole
// ones).  The loss of 65 536 tokens: 1.1 GB of rows through the L2s in 129 us, of which 0.75 GB come from outside them, which
// is what bounds it; with whole rows a group the step takes 39 us longer.  The lookup's gradient reads 260 MB and writes
// 67 MB in 73 us: 4.5 TB/s.
template <class T, int V, int L, class E>
__global__ void __launch_bounds__(kLmThreads) k_lm_seg_sum(LmSeg<E> q, const typename T::store* __restrict__ src) {
  constexpr int kGroups = kLmThreads / L, kCols = L * V;
  __shared__ float s_head[kGroups][kCols];
  __shared__ float s_tail[kGroups][kCols];
  __shared__ u32 s_flags[kGroups];      // 1: head, 2: the head's word goes on, 4: tail
  __shared__ u32 s_headKey[kGroups];
  const u32 gl = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  const u64 blocks = (u64)q.tiles * q.colBlocks;
  for (u64 block = blockIdx.x; block < blocks; block += gridDim.x) {
    const u32 cb = (u32)(block % q.colBlocks), tile = (u32)(block / q.colBlocks);
    const u32 pack = cb * L + gl;
    const bool on = pack * V < q.dim;
    const u32 col = on ? lm_col<V>(pack, q.dim) : 0u;
    const u32 j0 = tile * q.tile + grp * q.part;
    const u32 cnt = j0 < q.n ? (q.n - j0 < q.part ? q.n - j0 : q.part) : 0u;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    u32 flags = 0, headKey = 0;
    if (cnt > 0) {
      const u32 prevKey = j0 > 0 ? q.entries[j0 - 1].key : ~0u;
      const u32 nextKey = j0 + cnt < q.n ? q.entries[j0 + cnt].key : ~0u;
      u32 cur = q.entries[j0].key;
      headKey = cur;
      bool first = cur == prevKey;   // the running word began in an earlier part
      auto load8 = [&](E (&p)[8], u32 i0) {
#pragma unroll
        for (u32 i = 0; i < 8; ++i) p[i] = q.entries[j0 + (i0 + i < cnt ? i0 + i : cnt - 1)];
      };
      E p[8];
      load8(p, 0);
      for (u32 i0 = 0; i0 < cnt && cur < q.vocab; i0 += 8) {
        LmPack<T, V> x[8];
        u32 key[8];
        float w[8];
#pragma unroll
        for (u32 i = 0; i < 8; ++i) {
          x[i] = lm_load<T, V>(src + (u64)p[i].row * q.srcStride + col);   // (an entry that names no word has a row too)
          key[i] = p[i].key;
          if constexpr (E::kWeighted) w[i] = p[i].weight;
          else w[i] = q.scale;
        }
        load8(p, i0 + 8 < cnt ? i0 + 8 : i0);
#pragma unroll
        for (u32 i = 0; i < 8; ++i) {
          if (i0 + i < cnt) {
            if (key[i] != cur) {
              if (cur < q.vocab) {
                if (first) {
#pragma unroll
                  for (int e = 0; e < V; ++e) s_head[grp][gl * V + (u32)e] = acc[e];
                  flags |= 1;
                } else if (on) {
                  lm_store<LmF32, V, true>(q.grad + (i64)cur * q.gradStride + col, lm_pack<LmF32, V>(acc));
                }
              }
              first = false;
              cur = key[i];
#pragma unroll
              for (int e = 0; e < V; ++e) acc[e] = 0.f;
            }
            if (cur < q.vocab) {
#pragma unroll
              for (int e = 0; e < V; ++e) acc[e] = __builtin_fmaf(w[i], x[i].get(e), acc[e]);
            }
          }
        }
      }
      if (cur < q.vocab) {
        const bool on2 = cur == nextKey;   // goes on behind the part
        if (first) {
#pragma unroll
          for (int e = 0; e < V; ++e) s_head[grp][gl * V + (u32)e] = acc[e];
          flags |= on2 ? 3 : 1;
        } else if (on2) {
#pragma unroll
          for (int e = 0; e < V; ++e) s_tail[grp][gl * V + (u32)e] = acc[e];
          flags |= 4;
        } else if (on) {
          lm_store<LmF32, V, true>(q.grad + (i64)cur * q.gradStride + col, lm_pack<LmF32, V>(acc));
        }
      }
    }
    if (gl == 0) {
      s_flags[grp] = flags;
      s_headKey[grp] = headKey;
    }
    __syncthreads();
    // the words that cross parts, a thread a column, the parts in order
    for (u32 c = threadIdx.x; c < (u32)kCols; c += kLmThreads) {
      const u32 pk = cb * L + c / V;
      if (pk * V >= q.dim) continue;
      const u32 cc = lm_col<V>(pk, q.dim) + c % V;
      float run = 0.f;
      bool outside = true, open = false;   // the word began in an earlier tile; it goes on
      for (int g = 0; g < kGroups; ++g) {
        const u32 f = s_flags[g];
        if ((f & 1) != 0) {
          run += s_head[g][c];
          open = (f & 2) != 0;
          if (!open) {
            if (outside) q.head[(u64)tile * q.dim + cc] = run;
            else q.grad[(i64)s_headKey[g] * q.gradStride + cc] = run;
          }
        }
        if ((f & 4) != 0) {
          run = s_tail[g][c];
          outside = false;
          open = true;
        }
      }
      if (open) {
        (outside ? q.head : q.tail)[(u64)tile * q.dim + cc] = run;
        if (!outside && c == 0 && cb == 0) q.span[atomicAdd(q.spanCount, 1u)] = tile;
      }
    }
    __syncthreads();   // (the next tile writes what this one reads)
  }
}

// A word over several tiles: tail of the first, heads of the following ones.  A workgroup takes 64 V columns of a word; its
// wavefronts take consecutive parts of the tiles, and their sums are added in that order.  Latency bounds it: the list, the
// key, the tiles' keys, their rows, one after the other (a word of every fifteenth of 507 904 rows is 264 tiles: 9 us; 13
// with a column a lane).
constexpr int kLmJoinWaves = 4;
template <int V, class E>
__global__ void __launch_bounds__(64 * kLmJoinWaves) k_lm_seg_join(LmSeg<E> q) {
  constexpr u32 R = 8;   // partial rows in flight
  __shared__ float s_sum[kLmJoinWaves][64 * V];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 packs = (q.dim + V - 1) / V, colBlocks = (packs + 63) / 64;
  const u64 tasks = (u64)*q.spanCount * colBlocks;
  for (u64 task = blockIdx.x; task < tasks; task += gridDim.x) {
    const u32 a = q.span[task / colBlocks];
    const u32 pack = (u32)(task % colBlocks) * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    const u32 key = q.entries[(a + 1) * q.tile - 1].key;
    // tiles a + 1 .. b start with the word
    u32 b = a + 1;
    for (;;) {
      const u32 t = b + 1 + (u32)lane;
      const u64 m = wave_ballot(t < q.tiles && q.entries[(u64)t * q.tile].key == key);
      const u32 k = ~m == 0 ? 64u : (u32)__builtin_ctzll(~m);
      b += k;
      if (k < 64) break;
    }
    const u32 heads = b - a;
    const u32 per = (heads + kLmJoinWaves - 1) / kLmJoinWaves;
    const u32 h0 = a + 1 + per * (u32)wv, h1 = h0 + per < b + 1 ? h0 + per : b + 1;
    LmPack<LmF32, V> x;
    x.zero();
    if (wv == 0) x = lm_load<LmF32, V>(q.tail + (u64)a * q.dim + col);
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = x.get(e);
    for (u32 t = h0; t < h1; t += R) {
      LmPack<LmF32, V> y[R];
#pragma unroll
      for (u32 i = 0; i < R; ++i) y[i] = lm_load<LmF32, V>(q.head + (u64)(t + i < h1 ? t + i : t) * q.dim + col);
#pragma unroll
      for (u32 i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += t + i < h1 ? y[i].get(e) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s_sum[wv][lane * V + e] = sum[e];
    __syncthreads();
    if (wv == 0) {
      for (int w = 1; w < kLmJoinWaves; ++w)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += s_sum[w][lane * V + e];
      if (pack < packs) lm_store<LmF32, V>(q.grad + (i64)key * q.gradStride + col, lm_pack<LmF32, V>(sum));
    }
    __syncthreads();
  }
}

}  // namespace jpp

#endif  // JPP_K_LM_EMBED_H
