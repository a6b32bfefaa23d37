// Language-model operators 2: the gated linear recurrence h_t = a_t h_(t-1) + b_t x_t, a = sigmoid(gate), b = 1 - a, over the
// sentences of a packed batch, and its gradient.
//
// Columns are independent, so a wavefront owns 64 V columns of some rows and walks the rows; the bytes of gate, x and h
// decide.  Two splits:
//   short sentences (k_lm_scan_seq, k_lm_scan_grad_seq)  a wavefront per sentence and column block, one pass over the data;
//   long ones   the packed rows in chunks of C rows, whatever sentences they belong to.  A chunk maps the state in front of
//               it to the state behind it by s -> A s + B, or to B alone where a sentence begins inside (A = -1 says so: 0 s
//               would let a NaN of one sentence into the next):
//                 k_lm_scan_agg, k_lm_scan_grad_agg   A and B of every chunk, put together in groups of four
//                 k_lm_scan_carry                     the states between the groups
//                 k_lm_scan_chunk, k_lm_scan_grad_chunk   the rows themselves, from the states
//               at the price of reading gate and x (in the gradient gate and dh) twice.
// The gradient runs backwards: with e the gradient of the state that reaches a row from behind,
//     delta_t = dh_t + e, dx = delta b, dgate = delta (h_(t-1) - x) a b, e <- a delta.
// Measured: 16 384 sentences of 31 rows of 128 floats, a wavefront each: 174 us with saved states, 291 us backwards, both
// 4.6 TB/s (a copy of sets beyond the caches reaches 4.8).  One sentence of 65 536 rows of 1 024 bfloat16 columns in chunks:
// 55 us for the maps (4.9 TB/s), 6.5 for the states, 68 for the rows (5.9 TB/s).  Walked by one wavefront a column block it
// takes 19.8 ms.
// It needs h_(t-1) in 32 bits.  The forward pass leaves the state in front of every kLmSave-th row (an eighth of h's
// elements); from there the gradient re-makes the states of kLmSave rows in registers, which costs fewer bytes than
// reading h and does not see h's rounding to 16 bits.
#ifndef JPP_K_LM_SCAN_H
#define JPP_K_LM_SCAN_H

#include "jpp_lm.h"

namespace jpp {

constexpr u32 kLmSave = 8;   // rows between saved states, and rows in flight

template <class T>
struct LmScan {
  typedef typename T::store S;
  const S* gate;
  const S* x;
  i64 gateStride, xStride;
  const i32* offsets;
  u32 n, rows, dim, colBlocks;
  const float* state;     // or null: zero
  i64 stateStride;
  S* h;
  i64 hStride;
  float* last;            // or null
  i64 lastStride;
  float* saved;           // [(rows + kLmSave - 1) / kLmSave][dim], or null in the forward pass
  // gradient
  const S* dh;
  i64 dhStride;
  const float* dlast;     // or null: zero
  i64 dlastStride;
  S* dgate;
  S* dx;
  i64 dgateStride, dxStride;
  float* dstate;          // or null
  i64 dstateStride;
  // chunks
  u32 chunk, chunks;      // rows of a chunk (a multiple of kLmSave), chunks
  float *aggA, *aggB;     // [chunks][dim] map of the chunks of its group that lie in front of a chunk
  float *groupA, *groupB; // [groups][dim] map of a group of kLmGroup chunks; k_lm_scan_carry turns B into the state that enters it
};
constexpr u32 kLmGroup = kLmThreads / 64;   // chunks that a workgroup of the aggregating kernels takes, a wavefront each

// the rows of sentence i, inside the batch whatever the offsets hold
__device__ __forceinline__ u32 lm_offset(const i32* offsets, u32 i, u32 rows) {
  const i32 o = as_global(offsets)[i];
  return uni(o < 0 ? 0u : (u32)o < rows ? (u32)o : rows);
}

// The last sentence that begins at or before `row`, or n where the batch begins behind it; 64 offsets a step, all lanes
// taking part.  (Offsets that fall give some sentence, in as many steps.)
__device__ __forceinline__ u32 lm_sentence_of(const i32* offsets, u32 n, u32 row, int lane) {
  u32 lo = 0, hi = n;   // offsets[lo - 1] <= row < offsets[hi]
  while (lo < hi) {
    const u32 step = (hi - lo + 63) / 64;
    const u64 at = (u64)lo + (u64)(lane + 1) * step - 1;
    bool before = false;
    if (at < hi) before = as_global(offsets)[at] <= (i32)row;
    const u32 c = (u32)popc64(wave_ballot(before));
    const u64 end = (u64)lo + (u64)(c + 1) * step - 1;
    lo += c * step;
    if (end < hi) hi = (u32)end;
  }
  return lo == 0 ? n : lo - 1;
}

template <int V>
__device__ __forceinline__ void lm_row_f32(const float* base, i64 stride, u32 row, u32 col, float (&v)[V]) {
  if (base == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    return;
  }
  const LmPack<LmF32, V> p = lm_load<LmF32, V>(base + (i64)row * stride + col);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = p.get(e);
}
template <int V>
__device__ __forceinline__ void lm_put_f32(float* base, i64 stride, u32 row, u32 col, const float (&v)[V]) {
  lm_store<LmF32, V>(base + (i64)row * stride + col, lm_pack<LmF32, V>(v));
}

// Rows [r0, r1) of one sentence, forward, from state v.
template <class T, int V, bool SAVE, bool STREAM>
__device__ __forceinline__ void lm_scan_rows(const LmScan<T>& q, u32 r0, u32 r1, u32 col, float (&v)[V]) {
  for (u32 t = r0; t < r1;) {
    const u32 cut = (t / kLmSave + 1) * kLmSave;
    const u32 cnt = (cut < r1 ? cut : r1) - t;
    LmPack<T, V> f[kLmSave], x[kLmSave];
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
      const u32 r = t + (i < cnt ? i : cnt - 1);
      f[i] = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col);
      x[i] = lm_load<T, V>(q.x + (i64)r * q.xStride + col);
    }
    if (SAVE && t % kLmSave == 0) lm_put_f32<V>(q.saved, q.dim, t / kLmSave, col, v);
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
      if (i < cnt) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float a, b;
          lm_row_gate<T>(f[i].get(e), a, b);
          v[e] = __builtin_fmaf(a, v[e], b * x[i].get(e));
        }
        lm_store<T, V, STREAM>(q.h + (i64)(t + i) * q.hStride + col, lm_pack<T, V>(v));
      }
    }
    t += cnt;
  }
}

// Rows [r0, r1) of a sentence that begins at row `begin`, backward; e: gradient of the state behind row r1 - 1 on entry, of
// the state in front of row r0 on return.
template <class T, int V, bool STREAM>
__device__ __forceinline__ void lm_scan_grad_rows(const LmScan<T>& q, u32 sentence, u32 begin, u32 r0, u32 r1, u32 col, float (&e)[V]) {
  for (u32 end = r1; end > r0;) {
    const u32 cut = (end - 1) / kLmSave * kLmSave;
    const u32 t = cut > r0 ? cut : r0;
    const u32 cnt = end - t;
    LmPack<T, V> f[kLmSave], x[kLmSave], d[kLmSave];
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
      const u32 r = t + (i < cnt ? i : cnt - 1);
      f[i] = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col);
      x[i] = lm_load<T, V>(q.x + (i64)r * q.xStride + col);
      d[i] = lm_load<T, V>(q.dh + (i64)r * q.dhStride + col);
    }
    // the state in front of row t: t is the sentence's first row or a saved one (chunks begin on saved rows)
    float v[V], before[kLmSave][V], a[kLmSave][V], b[kLmSave][V];
    if (t == begin) lm_row_f32<V>(q.state, q.stateStride, sentence, col, v);
    else lm_row_f32<V>(q.saved, q.dim, t / kLmSave, col, v);
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        lm_row_gate<T>(f[i].get(k), a[i][k], b[i][k]);
        before[i][k] = v[k];
        v[k] = __builtin_fmaf(a[i][k], v[k], b[i][k] * x[i].get(k));
      }
    }
#pragma unroll
    for (u32 j = 0; j < kLmSave; ++j) {
      const u32 i = kLmSave - 1 - j;
      if (i < cnt) {
        float df[V], dx[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float delta = d[i].get(k) + e[k];
          dx[k] = delta * b[i][k];
          e[k] = delta * a[i][k];
          df[k] = dx[k] * (before[i][k] - x[i].get(k)) * a[i][k];
        }
        lm_store<T, V, STREAM>(q.dgate + (i64)(t + i) * q.dgateStride + col, lm_pack<T, V>(df));
        lm_store<T, V, STREAM>(q.dx + (i64)(t + i) * q.dxStride + col, lm_pack<T, V>(dx));
      }
    }
    end = t;
  }
}

// ---- a wavefront per sentence and column block -----------------------------------
template <class T, int V, bool SAVE, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_seq(LmScan<T> q) {
  const u64 tasks = (u64)q.n * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 i = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)i * q.colBlocks));
    const u32 pack = cb * 64u + (threadIdx.x & 63u);
    if (pack * V >= q.dim) continue;
    const u32 col = lm_col<V>(pack, q.dim);
    const u32 r0 = lm_offset(q.offsets, i, q.rows), r1 = lm_offset(q.offsets, i + 1, q.rows);
    float v[V];
    lm_row_f32<V>(q.state, q.stateStride, i, col, v);
    if (r0 < r1) lm_scan_rows<T, V, SAVE, STREAM>(q, r0, r1, col, v);
    if (q.last != nullptr) lm_put_f32<V>(q.last, q.lastStride, i, col, v);
  }
}

template <class T, int V, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_seq(LmScan<T> q) {
  const u64 tasks = (u64)q.n * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 i = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)i * q.colBlocks));
    const u32 pack = cb * 64u + (threadIdx.x & 63u);
    if (pack * V >= q.dim) continue;
    const u32 col = lm_col<V>(pack, q.dim);
    const u32 r0 = lm_offset(q.offsets, i, q.rows), r1 = lm_offset(q.offsets, i + 1, q.rows);
    float e[V];
    lm_row_f32<V>(q.dlast, q.dlastStride, i, col, e);
    if (r0 < r1) lm_scan_grad_rows<T, V, STREAM>(q, i, r0, r0, r1, col, e);
    if (q.dstate != nullptr) lm_put_f32<V>(q.dstate, q.dstateStride, i, col, e);
  }
}

// ---- chunks ------------------------------------------------------------------------
template <int V>
struct LmMap {   // s -> A s + B, or B where A < 0
  float A[V], B[V];
  __device__ __forceinline__ void one() {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      A[e] = 1.f;
      B[e] = 0.f;
    }
  }
  // this map, then the map (a, b)
  __device__ __forceinline__ void then(int e, float a, float b) {
    B[e] = a < 0.f ? b : __builtin_fmaf(a, B[e], b);
    A[e] = a < 0.f || A[e] < 0.f ? -1.f : A[e] * a;
  }
};

// The maps of a workgroup's chunks, a wavefront each: what lies in front of a chunk inside the group, and the group's own.
// BACK: in front is behind.
template <int V, bool BACK>
__device__ __forceinline__ void lm_scan_group(LmMap<V>& m, float (&sA)[kLmGroup][64 * V], float (&sB)[kLmGroup][64 * V], float* aggA, float* aggB,
                                              float* groupA, float* groupB, u32 group, u32 chunk, u32 chunks, u32 dim, u32 col, int lane, int wv) {
  // order of the walk
  const int at = BACK ? (int)kLmGroup - 1 - wv : wv;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sA[at][lane * V + e] = m.A[e];
    sB[at][lane * V + e] = m.B[e];
  }
  __syncthreads();
  m.one();
  for (int w = 0; w < at; ++w)
#pragma unroll
    for (int e = 0; e < V; ++e) m.then(e, sA[w][lane * V + e], sB[w][lane * V + e]);
  if (chunk < chunks) {
    lm_put_f32<V>(aggA, dim, chunk, col, m.A);
    lm_put_f32<V>(aggB, dim, chunk, col, m.B);
  }
  if (at == (int)kLmGroup - 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) m.then(e, sA[at][lane * V + e], sB[at][lane * V + e]);
    lm_put_f32<V>(groupA, dim, group, col, m.A);
    lm_put_f32<V>(groupB, dim, group, col, m.B);
  }
  __syncthreads();
}

// state behind the chunk = A * state in front of it + B
template <class T, int V>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_agg(LmScan<T> q) {
  __shared__ float s_A[kLmGroup][64 * V], s_B[kLmGroup][64 * V];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 blocks = (u64)((q.chunks + kLmGroup - 1) / kLmGroup) * q.colBlocks;
  for (u64 block = blockIdx.x; block < blocks; block += gridDim.x) {
    const u32 g = (u32)(block / q.colBlocks), cb = (u32)(block - (u64)g * q.colBlocks), c = g * kLmGroup + (u32)wv;
    // (lanes behind the last column repeat it: the same loads, the same stores)
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    LmMap<V> m;
    m.one();
    if (c < q.chunks) {
      const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
      // only the sentence that holds the chunk's last row reaches past it
      const u32 i = uni(lm_sentence_of(q.offsets, q.n, r1 - 1, lane));
      bool fresh = false;   // nothing passes
      u32 from = r0, to = r0;
      if (i < q.n) {
        const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows);
        from = begin > r0 ? begin : r0;
        to = end < r1 ? end : r1;
        fresh = begin >= r0;
        if (fresh) lm_row_f32<V>(q.state, q.stateStride, i, col, m.B);
      }
      for (u32 t = from; t < to; t += kLmSave) {
        const u32 cnt = to - t;
        LmPack<T, V> f[kLmSave], x[kLmSave];
#pragma unroll
        for (u32 k = 0; k < kLmSave; ++k) {
          const u32 r = t + (k < cnt ? k : cnt - 1);
          f[k] = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col);
          x[k] = lm_load<T, V>(q.x + (i64)r * q.xStride + col);
        }
#pragma unroll
        for (u32 k = 0; k < kLmSave; ++k) {
          if (k < cnt) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float a, b;
              lm_row_gate<T>(f[k].get(e), a, b);
              m.A[e] *= a;
              m.B[e] = __builtin_fmaf(a, m.B[e], b * x[k].get(e));
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) m.A[e] = fresh ? -1.f : m.A[e];
    }
    lm_scan_group<V, false>(m, s_A, s_B, q.aggA, q.aggB, q.groupA, q.groupB, g, c, q.chunks, q.dim, col, lane, wv);
  }
}

// gradient of the state in front of the chunk = A * gradient of the state behind it + B
template <class T, int V>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_agg(LmScan<T> q) {
  __shared__ float s_A[kLmGroup][64 * V], s_B[kLmGroup][64 * V];
  const int lane = (int)(threadIdx.x & 63), wv = (int)(threadIdx.x >> 6);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 blocks = (u64)((q.chunks + kLmGroup - 1) / kLmGroup) * q.colBlocks;
  for (u64 block = blockIdx.x; block < blocks; block += gridDim.x) {
    const u32 g = (u32)(block / q.colBlocks), cb = (u32)(block - (u64)g * q.colBlocks), c = g * kLmGroup + (u32)wv;
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    LmMap<V> m;
    m.one();
    if (c < q.chunks) {
      const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
      // only the sentence that holds the chunk's first row reaches in front of it
      const u32 i = uni(lm_sentence_of(q.offsets, q.n, r0, lane));
      bool fresh = false;   // nothing passes
      u32 to = r0;
      if (i < q.n) {
        const u32 end = lm_offset(q.offsets, i + 1, q.rows);
        to = end < r1 ? end : r1;
        fresh = end <= r1;
        if (fresh) lm_row_f32<V>(q.dlast, q.dlastStride, i, col, m.B);
      }
      for (u32 end = to; end > r0;) {
        const u32 t = end - r0 > kLmSave ? end - kLmSave : r0;
        const u32 cnt = end - t;
        LmPack<T, V> f[kLmSave], d[kLmSave];
#pragma unroll
        for (u32 k = 0; k < kLmSave; ++k) {
          const u32 r = t + (k < cnt ? k : cnt - 1);
          f[k] = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col);
          d[k] = lm_load<T, V>(q.dh + (i64)r * q.dhStride + col);
        }
#pragma unroll
        for (u32 j = 0; j < kLmSave; ++j) {
          const u32 k = kLmSave - 1 - j;
          if (k < cnt) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float a, b;
              lm_row_gate<T>(f[k].get(e), a, b);
              m.A[e] *= a;
              m.B[e] = a * (m.B[e] + d[k].get(e));
            }
          }
        }
        end = t;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) m.A[e] = fresh ? -1.f : m.A[e];
    }
    lm_scan_group<V, true>(m, s_A, s_B, q.aggA, q.aggB, q.groupA, q.groupB, g, c, q.chunks, q.dim, col, lane, wv);
  }
}

// the state (BACK: its gradient) that enters a chunk, from the one that enters its group
template <class T, int V>
__device__ __forceinline__ void lm_scan_enter(const LmScan<T>& q, u32 c, u32 col, float (&v)[V]) {
  float a[V], b[V];
  lm_row_f32<V>(q.groupB, q.dim, c / kLmGroup, col, v);
  lm_row_f32<V>(q.aggA, q.dim, c, col, a);
  lm_row_f32<V>(q.aggB, q.dim, c, col, b);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = a[e] < 0.f ? b[e] : __builtin_fmaf(a[e], v[e], b[e]);
}

// The states between the groups: groupB[c] becomes the state that enters group c (BACK: from behind).  A workgroup owns 16
// columns; 64 threads a column take consecutive runs of groups, first as one map each, then, from the state in front of
// their run, state by state.  What a compute unit can have in flight bounds it, hence the groups: 10 us for the maps of
// 1 024 chunks of 1 024 columns, 17 us with 64 columns a workgroup and 16 threads each.
constexpr u32 kLmCarryCols = 16, kLmCarryRuns = 64;
template <bool BACK>
__global__ void __launch_bounds__(kLmCarryCols * kLmCarryRuns) k_lm_scan_carry(const float* __restrict__ aggA, float* __restrict__ aggB, u32 chunks, u32 dim) {
  __shared__ float s_A[kLmCarryRuns][kLmCarryCols], s_B[kLmCarryRuns][kLmCarryCols];
  const u32 cl = threadIdx.x % kLmCarryCols, run = threadIdx.x / kLmCarryCols;
  const u32 colBlocks = (dim + kLmCarryCols - 1) / kLmCarryCols;
  for (u32 block = blockIdx.x; block < colBlocks; block += gridDim.x) {
    const u32 col = block * kLmCarryCols + cl;
    const bool on = col < dim;
    const u32 per = (chunks + kLmCarryRuns - 1) / kLmCarryRuns;
    const u32 c0 = per * run < chunks ? per * run : chunks, c1 = c0 + per < chunks ? c0 + per : chunks;
    auto at = [&](u32 c) { return (u64)(BACK ? chunks - 1 - c : c) * dim + col; };
    // up to kHold maps of a run stay in registers for the second walk
    constexpr u32 kHold = 16;
    float a[kHold], b[kHold];
    auto load = [&](u32 c) {
#pragma unroll
      for (u32 k = 0; k < kHold; ++k) {
        const u32 ck = c + k < c1 ? c + k : c1 - 1;
        a[k] = aggA[at(ck)];
        b[k] = aggB[at(ck)];
      }
    };
    float A = 1.f, B = 0.f;
    if (on) {
      for (u32 c = c0; c < c1; c += kHold) {
        load(c);
#pragma unroll
        for (u32 k = 0; k < kHold; ++k) {
          if (c + k < c1) {
            B = a[k] < 0.f ? b[k] : __builtin_fmaf(a[k], B, b[k]);
            A = a[k] < 0.f || A < 0.f ? -1.f : A * a[k];
          }
        }
      }
    }
    s_A[run][cl] = A;
    s_B[run][cl] = B;
    __syncthreads();
    float v = 0.f;   // (no state enters the first chunk: its sentences begin inside it)
#pragma unroll 8
    for (u32 w = 0; w < run; ++w) v = s_A[w][cl] < 0.f ? s_B[w][cl] : __builtin_fmaf(s_A[w][cl], v, s_B[w][cl]);
    if (on) {
      for (u32 c = c0; c < c1; c += kHold) {
        if (per > kHold) load(c);
#pragma unroll
        for (u32 k = 0; k < kHold; ++k) {
          if (c + k < c1) {
            aggB[at(c + k)] = v;
            v = a[k] < 0.f ? b[k] : __builtin_fmaf(a[k], v, b[k]);
          }
        }
      }
    }
    __syncthreads();
  }
}

// initial states straight through the sentences without a row (a wavefront per sentence and column block, over the grid)
template <int V>
__device__ __forceinline__ void lm_scan_empty(const i32* offsets, u32 n, u32 rows, u32 dim, u32 colBlocks, const float* in, i64 inStride,
                                              float* out, i64 outStride) {
  if (out == nullptr) return;
  const u64 tasks = (u64)n * colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 i = uni((u32)(task / colBlocks)), cb = uni((u32)(task - (u64)i * colBlocks));
    if (lm_offset(offsets, i, rows) < lm_offset(offsets, i + 1, rows)) continue;
    const u32 pack = cb * 64u + (threadIdx.x & 63u);
    if (pack * V >= dim) continue;
    const u32 col = lm_col<V>(pack, dim);
    float v[V];
    lm_row_f32<V>(in, inStride, i, col, v);
    lm_put_f32<V>(out, outStride, i, col, v);
  }
}

template <class T, int V, bool SAVE, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_chunk(LmScan<T> q) {
  const int lane = (int)(threadIdx.x & 63);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 tasks = (u64)q.chunks * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 c = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)c * q.colBlocks));
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
    u32 i = uni(lm_sentence_of(q.offsets, q.n, r0, lane));
    if (i == q.n) i = 0;   // the batch begins behind r0
    for (u32 t = r0; i < q.n; ++i) {
      const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows);
      if (begin >= r1) break;
      if (end <= t || end <= begin) continue;
      if (begin > t) t = begin;
      float v[V];
      if (begin >= r0) lm_row_f32<V>(q.state, q.stateStride, i, col, v);
      else lm_scan_enter<T, V>(q, c, col, v);
      const u32 to = end < r1 ? end : r1;
      lm_scan_rows<T, V, SAVE, STREAM>(q, t, to, col, v);
      if (to == end && q.last != nullptr) lm_put_f32<V>(q.last, q.lastStride, i, col, v);
      t = to;
      if (t == r1) break;
    }
  }
  lm_scan_empty<V>(q.offsets, q.n, q.rows, q.dim, q.colBlocks, q.state, q.stateStride, q.last, q.lastStride);
}

template <class T, int V, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_chunk(LmScan<T> q) {
  const int lane = (int)(threadIdx.x & 63);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 tasks = (u64)q.chunks * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 c = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)c * q.colBlocks));
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
    // sentences from the one with the last row down to the one with the first
    u32 i = uni(lm_sentence_of(q.offsets, q.n, r1 - 1, lane));
    if (i == q.n) continue;   // the batch begins behind the chunk
    for (u32 t = r1;; --i) {
      const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows);
      if (end <= r0 && begin < end) break;
      const u32 to = end < t ? end : t, from = begin > r0 ? begin : r0;
      if (from < to) {
        float e[V];
        if (end <= r1) lm_row_f32<V>(q.dlast, q.dlastStride, i, col, e);
        else lm_scan_enter<T, V>(q, c, col, e);
        lm_scan_grad_rows<T, V, STREAM>(q, i, begin, from, to, col, e);
        if (from == begin && q.dstate != nullptr) lm_put_f32<V>(q.dstate, q.dstateStride, i, col, e);
        t = from;
      }
      if (i == 0 || t == r0) break;
    }
  }
  lm_scan_empty<V>(q.offsets, q.n, q.rows, q.dim, q.colBlocks, q.dlast, q.dlastStride, q.dstate, q.dstateStride);
}

}  // namespace jpp

#endif  // JPP_K_LM_SCAN_H
