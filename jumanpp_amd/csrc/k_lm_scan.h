// Language-model operators 2: the gated linear recurrence h_t = a_t h_(t-1) + b_t x_t, a = sigmoid(gate), b = 1 - a, over the
// sentences of a packed batch, and its gradient.
//
// Columns are independent, so a wavefront owns 64 V columns of some rows and walks the rows; the bytes of gate, x and h
// decide.  Two splits:
//   short sentences (k_lm_scan_seq, k_lm_scan_grad_seq)  a wavefront per sentence and column block, one pass over the data;
//   long ones   the packed rows in chunks of C rows, whatever sentences they belong to.  A chunk maps the state in front of
//               it to the state behind it by s -> A s + B, or to B alone where a sentence begins inside:
//                 k_lm_scan_agg, k_lm_scan_grad_agg   A and B of every chunk, put together in groups of four
//                 k_lm_scan_carry                     the states between the groups
//                 k_lm_scan_chunk, k_lm_scan_grad_chunk   the rows themselves, from the states
//               at the price of reading gate and x (in the gradient gate and dh) twice.
// A row's step is made from the smaller of its two weights, s (jpp_lm.h): h_t = h_(t-1) + s (x_t - h_(t-1)), or from x_t's side,
// so that the weights sum to one and no rounding of a weight is gathered up over a long memory.  A state that is not a number
// afterwards, every eight rows, has them made again from the two weights, which is what the formula says of infinities.
// The gradient runs backwards: with e the gradient of the state that reaches a row from behind,
//     delta_t = dh_t + e, dx = delta b, dgate = delta (h_(t-1) - x) a b, e <- a delta.
// Measured: 16 384 sentences of 31 rows of 128 floats, a wavefront each: 175 us with saved states, 294 us backwards, both
// 4.6 TB/s (a copy of sets beyond the caches reaches 4.8).  One sentence of 65 536 rows of 1 024 bfloat16 columns in chunks:
// 59 us for the maps (4.6 TB/s, the vector unit at 0.7 of its slots), 8 for the states, 71 for the rows (5.7 TB/s).  Walked by
// one wavefront a column block it takes 21.8 ms.
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
  u32 clear;              // kLmClear*: results whose rows of no sentence are set to zero
  // chunks
  u32 chunk, chunks;      // rows of a chunk (a multiple of kLmSave), chunks
  float *aggW, *aggB;     // [chunks][dim] map of the chunks of its group that lie in front of a chunk
  float *groupW, *groupB; // [groups][dim] map of a group of kLmGroup chunks; k_lm_scan_carry turns B into the state that enters it
};
enum { kLmClearRows = 1, kLmClearDgate = 1, kLmClearDx = 2 };
constexpr u32 kLmGroup = kLmThreads / 64;   // chunks that a workgroup of the aggregating kernels takes, a wavefront each

// the rows of sentence i, inside the batch whatever the offsets hold
__device__ __forceinline__ u32 lm_inside(i32 o, u32 rows) { return uni(o < 0 ? 0u : (u32)o < rows ? (u32)o : rows); }
__device__ __forceinline__ u32 lm_offset(const i32* offsets, u32 i, u32 rows) { return lm_inside(as_global(offsets)[i], rows); }

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

// Rows [r0, r1) of one sentence, forward, from state v, by the two weights: for the elements of a pack that are `odd`, the others
// as ever (two lanes may share a column).  STORE: h too.  Rare, so nothing is held or unrolled for it.
template <class T, int V, bool STORE, bool STREAM>
__device__ __forceinline__ void lm_scan_rows_weights(const LmScan<T>& q, u32 r0, u32 r1, u32 col, const bool (&odd)[V], float (&v)[V]) {
#pragma unroll 1
  for (u32 r = r0; r < r1; ++r) {
    const LmPack<T, V> f = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col), x = lm_load<T, V>(q.x + (i64)r * q.xStride + col);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float w = lm_gate_weight(f.get(e));
      const LmWeights p(w);
      v[e] = odd[e] ? __builtin_fmaf(p.a, v[e], p.b * x.get(e)) : lm_step(w, v[e], x.get(e));
    }
    if constexpr (STORE) lm_store<T, V, STREAM>(q.h + (i64)r * q.hStride + col, lm_pack<T, V>(v));
  }
}
// which elements are not numbers (a state that is none stays so to the end of its sentence)
template <int V>
__device__ __forceinline__ bool lm_odd(const float (&v)[V], bool (&odd)[V]) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    odd[e] = !lm_finite(v[e]);
    any = any || odd[e];
  }
  return any;
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
    float v0[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v0[e] = v[e];
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
      if (i < cnt) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = lm_step(lm_gate_weight(f[i].get(e)), v[e], x[i].get(e));
        lm_store<T, V, STREAM>(q.h + (i64)(t + i) * q.hStride + col, lm_pack<T, V>(v));
      }
    }
    bool odd[V];
    if (__builtin_expect(lm_odd<V>(v, odd), 0)) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v0[e];
      lm_scan_rows_weights<T, V, true, STREAM>(q, t, t + cnt, col, odd, v);
    }
    t += cnt;
  }
}

// Rows [r0, r1), at most kLmSave of them from a sentence's first or a saved one on, backward, by the two weights (see
// lm_scan_rows_weights): the state in front of every row is walked to anew.
template <class T, int V, bool STREAM>
__device__ __forceinline__ void lm_scan_grad_rows_weights(const LmScan<T>& q, u32 sentence, u32 begin, u32 r0, u32 r1, u32 col,
                                                          const bool (&odd)[V], float (&e)[V]) {
#pragma unroll 1
  for (u32 r = r1; r-- > r0;) {
    float v[V], df[V], dx[V];
    if (r0 == begin) lm_row_f32<V>(q.state, q.stateStride, sentence, col, v);
    else lm_row_f32<V>(q.saved, q.dim, r0 / kLmSave, col, v);
    lm_scan_rows_weights<T, V, false, STREAM>(q, r0, r, col, odd, v);
    const LmPack<T, V> f = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col), x = lm_load<T, V>(q.x + (i64)r * q.xStride + col);
    const LmPack<T, V> d = lm_load<T, V>(q.dh + (i64)r * q.dhStride + col);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float w = lm_gate_weight(f.get(k)), delta = d.get(k) + e[k];
      const LmWeights p(w);
      float both;
      lm_parts(w, delta, e[k], dx[k], both);
      if (odd[k]) {
        dx[k] = p.b * delta;
        e[k] = p.a * delta;
        both = p.a * p.b * delta;
      }
      df[k] = both * (v[k] - x.get(k));
    }
    lm_store<T, V, STREAM>(q.dgate + (i64)r * q.dgateStride + col, lm_pack<T, V>(df));
    lm_store<T, V, STREAM>(q.dx + (i64)r * q.dxStride + col, lm_pack<T, V>(dx));
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
    float v[V], before[kLmSave][V], w[kLmSave][V], e1[V];
    if (t == begin) lm_row_f32<V>(q.state, q.stateStride, sentence, col, v);
    else lm_row_f32<V>(q.saved, q.dim, t / kLmSave, col, v);
#pragma unroll
    for (u32 i = 0; i < kLmSave; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        w[i][k] = lm_gate_weight(f[i].get(k));
        before[i][k] = v[k];
        v[k] = lm_step(w[i][k], v[k], x[i].get(k));
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) e1[k] = e[k];
#pragma unroll
    for (u32 j = 0; j < kLmSave; ++j) {
      const u32 i = kLmSave - 1 - j;
      if (i < cnt) {
        float df[V], dx[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float both;
          lm_parts(w[i][k], d[i].get(k) + e[k], e[k], dx[k], both);
          df[k] = both * (before[i][k] - x[i].get(k));
        }
        lm_store<T, V, STREAM>(q.dgate + (i64)(t + i) * q.dgateStride + col, lm_pack<T, V>(df));
        lm_store<T, V, STREAM>(q.dx + (i64)(t + i) * q.dxStride + col, lm_pack<T, V>(dx));
      }
    }
    bool odd[V], oddV[V];
    const bool oddE = lm_odd<V>(e, odd);
    if (__builtin_expect(lm_odd<V>(v, oddV) || oddE, 0)) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        odd[k] = odd[k] || oddV[k];
        e[k] = e1[k];
      }
      lm_scan_grad_rows_weights<T, V, STREAM>(q, sentence, begin, t, end, col, odd, e);
    }
    end = t;
  }
}

// The rows in front of the first sentence and behind the last one, a wavefront per row and column block, over the grid.  The two
// offsets are asked for when the kernel begins and looked at when the rest is done.
struct LmRest {
  i32 first, total;
};
template <class T>
__device__ __forceinline__ LmRest lm_scan_rest(const LmScan<T>& q) {
  LmRest r = {(i32)q.rows, (i32)q.rows};
  if (q.clear != 0 && q.n != 0) {
    r.first = as_global(q.offsets)[0];
    r.total = as_global(q.offsets)[q.n];
  }
  return r;
}
template <class T, int V, bool STREAM>
__device__ __forceinline__ void lm_scan_clear(const LmScan<T>& q, const LmRest& r, u32 which, typename T::store* out, i64 stride) {
  if ((q.clear & which) == 0) return;
  const u32 first = lm_inside(r.first, q.rows), total = lm_inside(r.total, q.rows);
  const u64 tasks = ((u64)first + q.rows - total) * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 i = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)i * q.colBlocks));
    const u32 pack = cb * 64u + (threadIdx.x & 63u);
    if (pack * V >= q.dim) continue;
    LmPack<T, V> zero;
    zero.zero();
    lm_store<T, V, STREAM>(out + (i64)(i < first ? i : total + (i - first)) * stride + lm_col<V>(pack, q.dim), zero);
  }
}

// ---- a wavefront per sentence and column block -----------------------------------
template <class T, int V, bool SAVE, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_seq(LmScan<T> q) {
  const LmRest rest = lm_scan_rest(q);
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
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearRows, q.h, q.hStride);
}

template <class T, int V, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_seq(LmScan<T> q) {
  const LmRest rest = lm_scan_rest(q);
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
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearDgate, q.dgate, q.dgateStride);
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearDx, q.dx, q.dxStride);
}

// ---- chunks ------------------------------------------------------------------------
template <int V>
struct LmMap {   // s -> A s + B
  float A[V], C[V], B[V];   // C = 1 - A as long as all weights are open ones; behind a closed one A is at most a half
  bool fresh;               // s -> B
  __device__ __forceinline__ void one() {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      A[e] = 1.f;
      C[e] = B[e] = 0.f;
    }
    fresh = false;
  }
  // the weight of this map, then of one of weight w
  __device__ __forceinline__ void pass(int e, float w) {
    C[e] = __builtin_fmaf(__builtin_fabsf(w), A[e], C[e]);
    A[e] = lm_kept(w, A[e]);
  }
  // this map, then the map (w, b)
  template <bool EXACT>
  __device__ __forceinline__ void then(int e, float w, float b) {
    pass(e, w);
    B[e] = lm_map<EXACT>(w, B[e], b);
    fresh = fresh || w == kLmFresh;   // (of one element, of all)
  }
  __device__ __forceinline__ float weight(int e) const { return fresh ? kLmFresh : lm_map_weight(A[e], C[e]); }
  __device__ __forceinline__ void put(float* w, float* b, u32 dim, u32 row, u32 col) const {
    float W[V];
#pragma unroll
    for (int e = 0; e < V; ++e) W[e] = weight(e);
    lm_put_f32<V>(w, dim, row, col, W);
    lm_put_f32<V>(b, dim, row, col, B);
  }
};

// The maps of a workgroup's chunks, a wavefront each: what lies in front of a chunk inside the group, and the group's own.
// BACK: in front is behind.
template <int V, bool BACK>
__device__ __forceinline__ void lm_scan_group(const LmMap<V>& own, float (&sW)[kLmGroup][64 * V], float (&sB)[kLmGroup][64 * V], float* aggW, float* aggB,
                                              float* groupW, float* groupB, u32 group, u32 chunk, u32 chunks, u32 dim, u32 col, int lane, int wv) {
  // order of the walk
  const int at = BACK ? (int)kLmGroup - 1 - wv : wv;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sW[at][lane * V + e] = own.weight(e);
    sB[at][lane * V + e] = own.B[e];
  }
  __syncthreads();
  LmMap<V> m;
  auto front = [&](auto exact) {
    bool finite = true;
    m.one();
    for (int w = 0; w < at; ++w)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        m.template then<decltype(exact)::value != 0>(e, sW[w][lane * V + e], sB[w][lane * V + e]);
        finite = finite && lm_finite(m.B[e]);
      }
    return finite;
  };
  if (__builtin_expect(!front(LmConst<0>()), 0)) front(LmConst<1>());
  if (chunk < chunks) m.put(aggW, aggB, dim, chunk, col);
  if (at == (int)kLmGroup - 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) m.template then<true>(e, sW[at][lane * V + e], sB[at][lane * V + e]);
    m.put(groupW, groupB, dim, group, col);
  }
  __syncthreads();
}

// state behind the chunk = A state in front of it + B
template <class T, int V>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_agg(LmScan<T> q) {
  __shared__ float s_W[kLmGroup][64 * V], s_B[kLmGroup][64 * V];
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
      u32 from = r0, to = r0;
      if (i < q.n) {
        const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows);
        from = begin > r0 ? begin : r0;
        to = end < r1 ? end : r1;
        m.fresh = begin >= r0;
        if (m.fresh) lm_row_f32<V>(q.state, q.stateStride, i, col, m.B);
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
        float B0[V];
#pragma unroll
        for (int e = 0; e < V; ++e) B0[e] = m.B[e];
#pragma unroll
        for (u32 k = 0; k < kLmSave; ++k) {
          if (k < cnt) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float w = lm_gate_weight(f[k].get(e));
              m.pass(e, w);
              m.B[e] = lm_step(w, m.B[e], x[k].get(e));
            }
          }
        }
        bool odd[V];
        if (__builtin_expect(lm_odd<V>(m.B, odd), 0)) {
#pragma unroll
          for (int e = 0; e < V; ++e) m.B[e] = B0[e];
          lm_scan_rows_weights<T, V, false, false>(q, t, cnt < kLmSave ? to : t + kLmSave, col, odd, m.B);
        }
      }
    }
    lm_scan_group<V, false>(m, s_W, s_B, q.aggW, q.aggB, q.groupW, q.groupB, g, c, q.chunks, q.dim, col, lane, wv);
  }
}

// gradient of the state in front of the chunk = A gradient of the state behind it + B
template <class T, int V>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_agg(LmScan<T> q) {
  __shared__ float s_W[kLmGroup][64 * V], s_B[kLmGroup][64 * V];
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
      u32 to = r0;
      if (i < q.n) {
        const u32 end = lm_offset(q.offsets, i + 1, q.rows);
        to = end < r1 ? end : r1;
        m.fresh = end <= r1;
        if (m.fresh) lm_row_f32<V>(q.dlast, q.dlastStride, i, col, m.B);
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
        float B0[V];
#pragma unroll
        for (int e = 0; e < V; ++e) B0[e] = m.B[e];
#pragma unroll
        for (u32 j = 0; j < kLmSave; ++j) {
          const u32 k = kLmSave - 1 - j;
          if (k < cnt) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float w = lm_gate_weight(f[k].get(e));
              m.pass(e, w);
              m.B[e] = lm_kept(w, m.B[e] + d[k].get(e));
            }
          }
        }
        bool odd[V];
        if (__builtin_expect(lm_odd<V>(m.B, odd), 0)) {
#pragma unroll 1
          for (u32 r = end; r-- > t;) {
            const LmPack<T, V> g = lm_load<T, V>(q.gate + (i64)r * q.gateStride + col), u = lm_load<T, V>(q.dh + (i64)r * q.dhStride + col);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float w = lm_gate_weight(g.get(e));
              B0[e] += u.get(e);
              B0[e] = odd[e] ? LmWeights(w).a * B0[e] : lm_kept(w, B0[e]);
            }
          }
#pragma unroll
          for (int e = 0; e < V; ++e) m.B[e] = B0[e];
        }
        end = t;
      }
    }
    lm_scan_group<V, true>(m, s_W, s_B, q.aggW, q.aggB, q.groupW, q.groupB, g, c, q.chunks, q.dim, col, lane, wv);
  }
}

// the state (BACK: its gradient) that enters a chunk, from the one that enters its group
template <class T, int V>
__device__ __forceinline__ void lm_scan_enter(const LmScan<T>& q, u32 c, u32 col, float (&v)[V]) {
  float w[V], b[V];
  lm_row_f32<V>(q.groupB, q.dim, c / kLmGroup, col, v);
  lm_row_f32<V>(q.aggW, q.dim, c, col, w);
  lm_row_f32<V>(q.aggB, q.dim, c, col, b);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = lm_map<true>(w[e], v[e], b[e]);
}

// The states between the groups: groupB[c] becomes the state that enters group c (BACK: from behind).  A workgroup owns 16
// columns; 64 threads a column take consecutive runs of groups, first as one map each, then, from the state in front of
// their run, state by state.  What a compute unit can have in flight bounds it, hence the groups: 8 us for 256 groups of
// 1 024 columns (for 1 024 chunks without groups 10, and 17 with 64 columns a workgroup and 16 threads each).
constexpr u32 kLmCarryCols = 16, kLmCarryRuns = 64;
template <bool BACK>
__global__ void __launch_bounds__(kLmCarryCols * kLmCarryRuns) k_lm_scan_carry(const float* __restrict__ aggW, float* __restrict__ aggB, u32 chunks, u32 dim) {
  __shared__ float s_W[kLmCarryRuns][kLmCarryCols], s_B[kLmCarryRuns][kLmCarryCols], s_k[kLmCarryRuns][kLmCarryCols], s_m[kLmCarryRuns][kLmCarryCols];
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
    float w[kHold], b[kHold];
    auto load = [&](u32 c) {
#pragma unroll
      for (u32 k = 0; k < kHold; ++k) {
        const u32 ck = c + k < c1 ? c + k : c1 - 1;
        w[k] = aggW[at(ck)];
        b[k] = aggB[at(ck)];
      }
    };
    // the states behind the maps held in registers, from v on; s[k]: in front of map k.  (Two operations a map: v comes through
    // whole or not at all, and the weight's part of it is taken off; what is not finite stays so, also behind a fresh map.)
    auto states = [&](u32 cnt, float& v, float (&s)[kHold]) {
      const float v0 = v;
#pragma unroll
      for (u32 k = 0; k < kHold; ++k) {
        s[k] = v;
        if (k < cnt) v = __builtin_fmaf(lm_map_whole(w[k]), v, __builtin_fmaf(lm_map_minus(w[k]), v, b[k]));
      }
      if (__builtin_expect(!lm_finite(v), 0)) {
        v = v0;
#pragma unroll
        for (u32 k = 0; k < kHold; ++k) {
          s[k] = v;
          if (k < cnt) v = lm_map<true>(w[k], v, b[k]);
        }
      }
    };
    LmMap<1> m;
    m.one();
    float s[kHold];
    if (on) {
      for (u32 c = c0; c < c1; c += kHold) {
        load(c);
#pragma unroll
        for (u32 k = 0; k < kHold; ++k) {
          if (c + k < c1) {
            m.pass(0, w[k]);
            m.fresh = m.fresh || w[k] == kLmFresh;
          }
        }
        states(c1 - c, m.B[0], s);
      }
    }
    const float W = m.weight(0);
    s_W[run][cl] = W;
    s_k[run][cl] = lm_map_whole(W);
    s_m[run][cl] = lm_map_minus(W);
    s_B[run][cl] = m.B[0];
    __syncthreads();
    float v = 0.f;   // (no state enters the first chunk: its sentences begin inside it)
#pragma unroll 8
    for (u32 r = 0; r < run; ++r) v = __builtin_fmaf(s_k[r][cl], v, __builtin_fmaf(s_m[r][cl], v, s_B[r][cl]));
    if (__builtin_expect(!lm_finite(v), 0)) {
      v = 0.f;
#pragma unroll 1
      for (u32 r = 0; r < run; ++r) v = lm_map<true>(s_W[r][cl], v, s_B[r][cl]);
    }
    if (on) {
      for (u32 c = c0; c < c1; c += kHold) {
        if (per > kHold) load(c);
        states(c1 - c, v, s);
#pragma unroll
        for (u32 k = 0; k < kHold; ++k)
          if (c + k < c1) aggB[at(c + k)] = s[k];
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
  const LmRest rest = lm_scan_rest(q);
  const int lane = (int)(threadIdx.x & 63);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 tasks = (u64)q.chunks * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 c = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)c * q.colBlocks));
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
    u32 t = r0, i = uni(lm_sentence_of(q.offsets, q.n, r0, lane));
    if (i == q.n) {   // the batch begins behind r0
      t = lm_offset(q.offsets, 0, q.rows);
      if (t >= r1) continue;
      i = uni(lm_sentence_of(q.offsets, q.n, t, lane));
    }
    // From sentence to sentence; sentences without a row may be many, so they are passed over by a search.
    while (i < q.n) {
      const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows), to = end < r1 ? end : r1;
      if (begin > t) t = begin;
      if (t >= to) break;   // (behind the last sentence)
      float v[V];
      if (begin >= r0) lm_row_f32<V>(q.state, q.stateStride, i, col, v);
      else lm_scan_enter<T, V>(q, c, col, v);
      lm_scan_rows<T, V, SAVE, STREAM>(q, t, to, col, v);
      if (to == end && q.last != nullptr) lm_put_f32<V>(q.last, q.lastStride, i, col, v);
      t = to;
      if (t == r1 || i + 1 == q.n) break;
      ++i;
      if (lm_offset(q.offsets, i + 1, q.rows) <= t) i = uni(lm_sentence_of(q.offsets, q.n, t, lane));
    }
  }
  lm_scan_empty<V>(q.offsets, q.n, q.rows, q.dim, q.colBlocks, q.state, q.stateStride, q.last, q.lastStride);
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearRows, q.h, q.hStride);
}

template <class T, int V, bool STREAM>
__global__ void __launch_bounds__(kLmThreads) k_lm_scan_grad_chunk(LmScan<T> q) {
  const LmRest rest = lm_scan_rest(q);
  const int lane = (int)(threadIdx.x & 63);
  const u32 packs = (q.dim + V - 1) / V;
  const u64 tasks = (u64)q.chunks * q.colBlocks;
  for (u64 task = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); task < tasks; task += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 c = uni((u32)(task / q.colBlocks)), cb = uni((u32)(task - (u64)c * q.colBlocks));
    const u32 pack = cb * 64u + (u32)lane;
    const u32 col = lm_col<V>(pack < packs ? pack : packs - 1, q.dim);
    const u32 r0 = c * q.chunk, r1 = q.rows - r0 < q.chunk ? q.rows : r0 + q.chunk;
    // sentences from the one with the last row down to the one with the first, those without a row passed over
    u32 t = r1, i = uni(lm_sentence_of(q.offsets, q.n, r1 - 1, lane));
    if (i + 1 == q.n && lm_offset(q.offsets, q.n, q.rows) < r1) {   // the batch ends in front of r1
      t = lm_offset(q.offsets, q.n, q.rows);
      if (t <= r0) continue;
      i = uni(lm_sentence_of(q.offsets, q.n, t - 1, lane));
    }
    while (i < q.n) {
      const u32 begin = lm_offset(q.offsets, i, q.rows), end = lm_offset(q.offsets, i + 1, q.rows);
      const u32 to = end < t ? end : t, from = begin > r0 ? begin : r0;
      if (from >= to) break;   // (in front of the first sentence)
      float e[V];
      if (end <= r1) lm_row_f32<V>(q.dlast, q.dlastStride, i, col, e);
      else lm_scan_enter<T, V>(q, c, col, e);
      lm_scan_grad_rows<T, V, STREAM>(q, i, begin, from, to, col, e);
      if (from == begin && q.dstate != nullptr) lm_put_f32<V>(q.dstate, q.dstateStride, i, col, e);
      t = from;
      if (t == r0 || i == 0) break;
      --i;
      if (lm_offset(q.offsets, i, q.rows) >= t) i = uni(lm_sentence_of(q.offsets, q.n, t - 1, lane));
    }
  }
  lm_scan_empty<V>(q.offsets, q.n, q.rows, q.dim, q.colBlocks, q.dlast, q.dlastStride, q.dstate, q.dstateStride);
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearDgate, q.dgate, q.dgateStride);
  lm_scan_clear<T, V, STREAM>(q, rest, kLmClearDx, q.dx, q.dxStride);
}

}  // namespace jpp

#endif  // JPP_K_LM_SCAN_H
