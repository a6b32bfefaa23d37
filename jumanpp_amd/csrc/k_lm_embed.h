// Language-model operators 1: rows of a table by word (k_lm_embed), and the gradient of a table whose rows were read by
// word: dW_v = sum over the entries j with word v of w_j src_(j / K).  For the lookup w_j is the scale, K = 1 and src the
// gradient of the rows; for the noise-contrastive loss (k_lm_nce.h) w_j is the gradient of the score of candidate j and
// src_(j / K) the state of its token.
//
// The gradient sums by word without atomics on floats, so its bits follow from the inputs:
//   k_lm_sort_one / k_lm_sort_count, _scan, _scatter   entries into ascending (word, entry): least digit first, stable
//   k_lm_seg_sum                                       tiles of M sorted entries, a wavefront each: a word whose entries
//                                                      lie inside one tile is written at once, one that crosses a border
//                                                      leaves a partial row per tile
//   k_lm_seg_join                                      the partial rows of those words, in tile order
// Rows of words that do not occur are zeroed by workgroups that ride in the grid of the first sorting kernel: that one uses
// a fraction of the chip.
#ifndef JPP_K_LM_EMBED_H
#define JPP_K_LM_EMBED_H

#include "jpp_lm.h"

namespace jpp {

// ---- lookup --------------------------------------------------------------------
// y_t = scale * W[id_t].  A thread moves packs of V elements, a workgroup `rowsPerBlock` rows; nothing but the loads and
// stores counts.  The ids of PER packs are loaded together, then their rows: one wait each, not one a pack.
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
    for (u32 c = threadIdx.x; c < packs; c += blockDim.x) lm_store<LmF32, 4>(row + 4 * (u64)c, zero);
    for (u32 c = packs * 4 + threadIdx.x; c < cols; c += blockDim.x) row[c] = 0.f;
  }
}

__global__ void __launch_bounds__(kLmThreads) k_lm_zero(LmZero z) { lm_zero_rows(z, blockIdx.x, gridDim.x); }

struct LmPair {      // an entry on its way through the sort
  u32 key;           // word, `vocab` for none
  u32 entry;
};

// where the first pass finds its keys
struct LmKeysOfIds {
  LmIds ids;
  u32 vocab;
  u32 perToken;      // entries of a token; the token counts only if its entry 0 names a word
  __device__ __forceinline__ LmPair operator()(u32 j) const {
    u32 key = lm_row(ids, j, vocab);
    if (perToken > 1 && key < vocab && lm_row(ids, j / perToken * perToken, vocab) == vocab) key = vocab;
    return LmPair{key, j};
  }
};
struct LmKeysOfPairs {
  const LmPair* pairs;
  __device__ __forceinline__ LmPair operator()(u32 j) const { return pairs[j]; }
};

constexpr u32 kLmBins = 256;
constexpr int kLmSortRounds = 8;                                   // keys of a thread
constexpr u32 kLmSortTile = kLmThreads * kLmSortRounds;            // keys of a workgroup
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
template <class Keys>
__global__ void __launch_bounds__(kLmOneThreads)
    k_lm_sort_one(Keys keys, u32 n, u32 keyBits, u32 passes, LmPair* __restrict__ out, u32* __restrict__ spanCount, LmZero zero) {
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
  if (threadIdx.x == 0) *spanCount = 0;
  const u32 rounds = (n + kLmOneThreads - 1) / kLmOneThreads;   // (1 .. kLmOneRounds)
  const u32 pos0 = (u32)wv * 64u * rounds + (u32)lane;
  LmPair p[kLmOneRounds];
#pragma unroll
  for (u32 r = 0; r < (u32)kLmOneRounds; ++r) {
    p[r] = LmPair{0, 0};
    if (r < rounds && pos0 + 64 * r < n) p[r] = keys(pos0 + 64 * r);
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
      if (r < rounds) rank[r] = lm_rank_round((p[r].key >> shift) & mask, pos0 + 64 * r < n, digitBits, s_cnt[wv], lane);
    }
    __syncthreads();
    if (threadIdx.x < kLmBins) {
      u32 run = 0;
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
        const u32 d = (p[r].key >> shift) & mask;
        const u32 to = s_bin[d] + s_cnt[wv][d] + rank[r];
        if (last) {
          out[to] = p[r];
        } else {
          s_key[to] = p[r].key;
          s_entry[to] = p[r].entry;
        }
      }
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (u32 r = 0; r < (u32)kLmOneRounds; ++r)
        if (r < rounds && pos0 + 64 * r < n) p[r] = LmPair{s_key[pos0 + 64 * r], s_entry[pos0 + 64 * r]};
      __syncthreads();
    }
  }
}

// One pass over many entries: digits per tile ...
template <class Keys>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_sort_count(Keys keys, u32 n, u32 shift, u32 mask, u32* __restrict__ counts, u32 tiles, u32* __restrict__ spanCount, LmZero zero) {
  __shared__ u32 s_cnt[kLmBins];
  if (blockIdx.x >= tiles) {
    lm_zero_rows(zero, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *spanCount = 0;
  s_cnt[threadIdx.x] = 0;
  __syncthreads();
  const u32 j0 = blockIdx.x * kLmSortTile + threadIdx.x;
#pragma unroll
  for (int r = 0; r < kLmSortRounds; ++r) {
    const u32 j = j0 + (u32)r * kLmThreads;
    if (j < n) atomicAdd(&s_cnt[(keys(j).key >> shift) & mask], 1u);
  }
  __syncthreads();
  counts[threadIdx.x * (u64)tiles + blockIdx.x] = s_cnt[threadIdx.x];
}

// ... per digit the exclusive sums over the tiles and the total, a wavefront a digit ...
__global__ void __launch_bounds__(kLmThreads) k_lm_sort_scan(u32* __restrict__ counts, u32 tiles, u32* __restrict__ totals) {
  const int lane = (int)(threadIdx.x & 63);
  const u32 bin = blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6);
  u32* c = counts + bin * (u64)tiles;
  u32 run = 0;
  for (u32 i0 = 0; i0 < tiles; i0 += 64) {
    const u32 i = i0 + (u32)lane;
    const u32 x = i < tiles ? c[i] : 0u;
    const u32 incl = lm_scan_incl(x, lane);
    if (i < tiles) c[i] = run + incl - x;
    run += wave_bcast_u32(incl, 63);
  }
  if (lane == 0) totals[bin] = run;
}

// ... and every key to its place
template <class Keys>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_sort_scatter(Keys keys, u32 n, u32 shift, u32 bits, const u32* __restrict__ counts, u32 tiles, const u32* __restrict__ totals,
                      LmPair* __restrict__ out) {
  constexpr int kWaves = kLmThreads / 64;
  __shared__ u32 s_cnt[kWaves][kLmBins];
  __shared__ u32 s_bin[kLmBins];
  __shared__ u32 s_part[4];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 mask = (1u << bits) - 1;
  const u32 mine = counts[threadIdx.x * (u64)tiles + blockIdx.x];
  s_bin[threadIdx.x] = totals[threadIdx.x];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s_cnt[w][threadIdx.x] = 0;
  const u32 pos0 = blockIdx.x * kLmSortTile + (u32)wv * (64u * kLmSortRounds) + (u32)lane;
  LmPair p[kLmSortRounds];
#pragma unroll
  for (int r = 0; r < kLmSortRounds; ++r) {
    p[r] = LmPair{0, 0};
    if (pos0 + 64u * (u32)r < n) p[r] = keys(pos0 + 64u * (u32)r);
  }
  __syncthreads();
  lm_scan_bins(s_bin, s_part, lane, wv);
  u32 rank[kLmSortRounds];
#pragma unroll
  for (int r = 0; r < kLmSortRounds; ++r)
    rank[r] = lm_rank_round((p[r].key >> shift) & mask, pos0 + 64u * (u32)r < n, bits, s_cnt[wv], lane);
  __syncthreads();
  {
    u32 run = s_bin[threadIdx.x] + mine;
    for (int w = 0; w < kWaves; ++w) {
      const u32 x = s_cnt[w][threadIdx.x];
      s_cnt[w][threadIdx.x] = run;
      run += x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kLmSortRounds; ++r)
    if (pos0 + 64u * (u32)r < n) out[s_cnt[wv][(p[r].key >> shift) & mask] + rank[r]] = p[r];
}

// ---- sums by word ----------------------------------------------------------------
struct LmSeg {
  const LmPair* pairs;   // sorted
  u32 n;
  u32 tile;              // entries of a tile, a multiple of 8, at most 64
  u32 tiles;
  u32 vocab, dim, colBlocks;
  u32 perToken;          // entries of a row of src
  float scale;           // weight of every entry ...
  const float* weights;  // ... or of each
  i64 srcStride;
  float* grad;
  i64 gradStride;
  float* head;           // [tiles][dim] partial row of the word that began in an earlier tile
  float* tail;           // [tiles][dim] ... of the word that goes on in the next
  u32* span;             // tiles whose last word began there and goes on
  u32* spanCount;
};

template <class T, int V>
__global__ void __launch_bounds__(kLmThreads) k_lm_seg_sum(LmSeg q, const typename T::store* __restrict__ src) {
  const int lane = (int)(threadIdx.x & 63);
  const u64 tasks = (u64)q.tiles * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 tile = uni((u32)(task / q.colBlocks));
    const u32 cb = uni((u32)(task - (u64)tile * q.colBlocks));
    const u32 j0 = tile * q.tile;
    const u32 cnt = uni(q.n - j0 < q.tile ? q.n - j0 : q.tile);
    const bool on = (cb * 64u + (u32)lane) * V < q.dim;
    const u32 col = on ? lm_col<V>(cb * 64u + (u32)lane, q.dim) : 0u;
    LmPair p = {q.vocab, 0};
    if ((u32)lane < cnt) p = q.pairs[j0 + (u32)lane];
    const u32 prevKey = tile > 0 ? q.pairs[j0 - 1].key : ~0u;
    const u32 nextKey = j0 + cnt < q.n ? q.pairs[j0 + cnt].key : ~0u;
    float w = q.scale;
    if (q.weights != nullptr) w = p.key < q.vocab ? q.weights[p.entry] : 0.f;
    const u32 srow = q.perToken > 1 ? p.entry / q.perToken : p.entry;
    u32 cur = wave_bcast_u32(p.key, 0);
    bool first = cur == prevKey;   // the running word began in an earlier tile
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    auto put = [&](float* row) {
      if (on) lm_store<LmF32, V>(row + col, lm_pack<LmF32, V>(acc));
    };
    for (u32 i0 = 0; i0 < cnt && cur < q.vocab; i0 += 8) {
      LmPack<T, V> x[8];
      // (entries that name no word are last and read row 0 of src's own rows: their entry is in range)
#pragma unroll
      for (u32 i = 0; i < 8; ++i) {
        const u32 at = i0 + i < cnt ? i0 + i : cnt - 1;
        const u32 r = wave_bcast_u32(srow, (int)at);
        x[i] = lm_load<T, V>(src + (i64)r * q.srcStride + col);
      }
#pragma unroll
      for (u32 i = 0; i < 8; ++i) {
        if (i0 + i < cnt) {
          const u32 key = wave_bcast_u32(p.key, (int)(i0 + i));
          const float wi = wave_bcast_f32(w, (int)(i0 + i));
          if (key != cur) {
            if (cur < q.vocab) put(first ? q.head + (u64)tile * q.dim : q.grad + (i64)cur * q.gradStride);
            first = false;
            cur = key;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = 0.f;
          }
          if (key < q.vocab) {
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = __builtin_fmaf(wi, x[i].get(e), acc[e]);
          }
        }
      }
    }
    if (cur < q.vocab) {
      if (first) {
        put(q.head + (u64)tile * q.dim);
      } else if (cur == nextKey) {
        put(q.tail + (u64)tile * q.dim);
        if (cb == 0 && lane == 0) q.span[atomicAdd(q.spanCount, 1u)] = tile;
      } else {
        put(q.grad + (i64)cur * q.gradStride);
      }
    }
  }
}

// A word over several tiles: tail of the first, heads of the following ones.  A workgroup takes 64 columns of a word; its
// wavefronts take consecutive parts of the tiles, and their sums are added in that order.
constexpr int kLmJoinWaves = 8;
__global__ void __launch_bounds__(64 * kLmJoinWaves) k_lm_seg_join(LmSeg q) {
  __shared__ float s_sum[kLmJoinWaves][64];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 colBlocks = (q.dim + 63) / 64;
  const u64 tasks = (u64)*q.spanCount * colBlocks;
  for (u64 task = blockIdx.x; task < tasks; task += gridDim.x) {
    const u32 a = q.span[task / colBlocks];
    const u32 col = (u32)(task % colBlocks) * 64u + (u32)lane;
    const u32 key = q.pairs[(a + 1) * q.tile - 1].key;
    // tiles a + 1 .. b start with the word
    u32 b = a + 1;
    for (;;) {
      const u32 t = b + 1 + (u32)lane;
      const u64 m = wave_ballot(t < q.tiles && q.pairs[(u64)t * q.tile].key == key);
      const u32 k = ~m == 0 ? 64u : (u32)__builtin_ctzll(~m);
      b += k;
      if (k < 64) break;
    }
    const u32 heads = b - a;
    const u32 per = (heads + kLmJoinWaves - 1) / kLmJoinWaves;
    const u32 h0 = a + 1 + per * (u32)wv, h1 = h0 + per < b + 1 ? h0 + per : b + 1;
    float sum = 0.f;
    if (col < q.dim) {
      if (wv == 0) sum = q.tail[(u64)a * q.dim + col];
#pragma unroll 8
      for (u32 t = h0; t < h1; ++t) sum += q.head[(u64)t * q.dim + col];
    }
    s_sum[wv][lane] = sum;
    __syncthreads();
    if (wv == 0 && col < q.dim) {
      for (int w = 1; w < kLmJoinWaves; ++w) sum += s_sum[w][lane];
      q.grad[(i64)key * q.gradStride + col] = sum;
    }
    __syncthreads();
  }
}

}  // namespace jpp

#endif  // JPP_K_LM_EMBED_H
