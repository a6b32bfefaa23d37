// Language-model operators 3: the noise-contrastive score of candidate words and the loss with its gradients.
//
//   score   s = <h_t, W[c]> - C
//   loss    z_k = s_k - ln(K p(c_k)), L_t = w_t (softplus(-z_0) + sum over k > 0 of softplus(z_k))
//           dL/dz_0 = -w sigmoid(-z_0), dL/dz_k = w sigmoid(z_k); dh_t = sum of g_k W[c_k]; dW by word: k_lm_embed.h
//
// The rows of W are gathered: the bytes of K rows a token decide, from L2 and the memory-side cache for a table that fits
// there.  A group of G lanes holds a row in registers, so the loss reads every row once -- the product with h, then
// g_k times the same registers into dh.  G = 16 keeps the product's reduction inside a row of 16 lanes (four DPP steps,
// four candidates side by side); longer rows take the whole wavefront.
#ifndef JPP_K_LM_NCE_H
#define JPP_K_LM_NCE_H

#include "jpp_lm.h"

namespace jpp {

struct LmNce {
  u32 vocab, dim;
  u64 n;                  // tokens
  u32 cands;              // candidates of a token
  i64 hStride, tableStride, dhStride;
  float constant;
  const float* logNoise;
  const float* weight;    // of a token's loss, or null
  float* out;             // scores or losses
  float* g;               // [n * cands] gradients of the scores, for the table's gradient (and for dh, where rows are walked in
                          // blocks); or null
};

// A lane's part of a row: packs l, l + G, ... of V elements (from pack `p0` on, `packs` in the row) and, where V does not
// divide the row, one of its last elements.  Parts that do not exist are zero, so a product over the group counts every
// element once.
struct LmRowShape {
  u32 packs, rest;   // full packs, elements behind them
};
template <class T, int V, int G, int NV>
struct LmRowPart {
  LmPack<T, V> p[NV];
  typename T::store tail;
  __device__ __forceinline__ void load(const typename T::store* row, u32 p0, u32 gl, const LmRowShape& s) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const u32 at = p0 + gl + (u32)(G * i);
      if (at < s.packs) {
        p[i] = lm_load<T, V>(row + at * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) p[i].v[e] = 0;
      }
    }
    tail = 0;
    if (s.rest != 0 && p0 == 0 && gl < s.rest) tail = as_global(row)[s.packs * V + gl];
  }
};
template <int V, int NV>
struct LmRowSum {    // the same part in 32 bits
  float p[NV][V];
  float tail;
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) p[i][e] = 0.f;
    tail = 0.f;
  }
  template <class T, int G>
  __device__ __forceinline__ void add(float w, const LmRowPart<T, V, G, NV>& x) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) p[i][e] = __builtin_fmaf(w, T::get(x.p[i].v[e]), p[i][e]);
    tail = __builtin_fmaf(w, T::get(x.tail), tail);
  }
  template <class T, int G>
  __device__ __forceinline__ float dot(const LmRowPart<T, V, G, NV>& x) const {
    float d = tail * T::get(x.tail);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) d = __builtin_fmaf(p[i][e], T::get(x.p[i].v[e]), d);
    return d;
  }
  template <class T, int G>
  __device__ __forceinline__ void store(typename T::store* row, u32 p0, u32 gl, const LmRowShape& s) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const u32 at = p0 + gl + (u32)(G * i);
      if (at < s.packs) lm_store<T, V>(row + at * V, lm_pack<T, V>(p[i]));
    }
    if (s.rest != 0 && p0 == 0 && gl < s.rest) ((typename T::store JPP_GLOBAL*)row)[s.packs * V + gl] = T::put(tail);
  }
};

// NV packs of V elements a lane cover G NV packs; BLOCKS: the row has more and is walked in such blocks (the loss then reads
// the rows of W twice)
template <class T, int V, int G, int NV, bool BLOCKS>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_nce_score(LmNce q, const typename T::store* __restrict__ h, const typename T::store* __restrict__ table, LmIds ids) {
  const u32 gl = threadIdx.x & (G - 1);
  const LmRowShape shape = {q.dim / V, q.dim % V};
  const u64 pairs = q.n * q.cands;
  const u64 step = (u64)gridDim.x * (kLmThreads / G);
  // (whole wavefronts stay in the loop: the group sums are wavefront operations)
  for (u64 j0 = (u64)blockIdx.x * (kLmThreads / G); j0 < pairs; j0 += step) {
    const u64 j = j0 + threadIdx.x / G;
    const u32 row = j < pairs ? lm_row(ids, j, q.vocab) : q.vocab;
    const u64 t = j < pairs ? (pairs <= 0xffffffffu ? (u64)((u32)j / q.cands) : j / q.cands) : 0u;
    float dot = 0.f;
    if (row < q.vocab) {
      for (u32 p0 = 0; p0 < (BLOCKS ? shape.packs : 1u); p0 += G * NV) {
        LmRowPart<T, V, G, NV> a, b;
        a.load(h + (i64)t * q.hStride, p0, gl, shape);
        b.load(table + (i64)row * q.tableStride, p0, gl, shape);
        LmRowSum<V, NV> x;
        x.zero();
        x.template add<T, G>(1.f, a);
        dot += x.template dot<T, G>(b);
      }
    }
    dot = lm_group_sum<G>(dot);
    if (gl == 0 && j < pairs) q.out[j] = row < q.vocab ? dot - q.constant : -__builtin_inff();
  }
}

template <class T, int V, int G, int NV, bool BLOCKS, bool DH>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_nce_loss(LmNce q, const typename T::store* __restrict__ h, const typename T::store* __restrict__ table, LmIds ids,
                  typename T::store* __restrict__ dh) {
  constexpr u32 kGroups = 64 / G;
  constexpr int U = NV * V >= 32 ? 1 : NV * V >= 16 ? 2 : 4;   // candidates of a group in flight
  const int lane = (int)(threadIdx.x & 63);
  const u32 gl = threadIdx.x & (G - 1), grp = (u32)lane / G;
  const LmRowShape shape = {q.dim / V, q.dim % V};
  for (u64 t = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6); t < q.n; t += (u64)gridDim.x * (kLmThreads / 64)) {
    const u32 target = uni(lm_row(ids, t * q.cands, q.vocab));
    const bool live = target < q.vocab;
    const float w = q.weight != nullptr ? q.weight[t] : 1.f;
    LmRowSum<V, NV> hr, acc;
    hr.zero();
    acc.zero();
    float loss = 0.f;
    if (live && !BLOCKS) {
      LmRowPart<T, V, G, NV> a;
      a.load(h + (i64)t * q.hStride, 0, gl, shape);
      hr.template add<T, G>(1.f, a);
    }
    for (u32 kb = 0; live && kb < q.cands; kb += 64) {
      // the rows of 64 candidates, a lane each, ahead of the gathers that need them
      const u32 kn = q.cands - kb < 64 ? q.cands - kb : 64u;
      u32 rowL = q.vocab;
      if ((u32)lane < kn) rowL = lm_row(ids, t * q.cands + kb + (u32)lane, q.vocab);
      const float biasL = rowL < q.vocab ? q.constant + q.logNoise[rowL] : 0.f;
      float gL = 0.f;
      for (u32 k0 = 0; k0 < kn; k0 += kGroups * U) {
        LmRowPart<T, V, G, NV> b[U];
        u32 row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const u32 k = k0 + (u32)u * kGroups + grp;
          row[u] = wave_shfl_u32(rowL, (int)(k & 63));
          if (k >= kn) row[u] = q.vocab;
          // (a candidate that names no word reads the target's row and leaves with g = 0)
          if (!BLOCKS) b[u].load(table + (i64)(row[u] < q.vocab ? row[u] : target) * q.tableStride, 0, gl, shape);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const u32 k = k0 + (u32)u * kGroups + grp;
          const bool ok = row[u] < q.vocab;
          float dot = 0.f;
          if constexpr (BLOCKS) {
            for (u32 p0 = 0; ok && p0 < shape.packs; p0 += G * NV) {
              LmRowPart<T, V, G, NV> a;
              a.load(h + (i64)t * q.hStride, p0, gl, shape);
              b[u].load(table + (i64)row[u] * q.tableStride, p0, gl, shape);
              LmRowSum<V, NV> x;
              x.zero();
              x.template add<T, G>(1.f, a);
              dot += x.template dot<T, G>(b[u]);
            }
          } else {
            dot = hr.template dot<T, G>(b[u]);
          }
          dot = lm_group_sum<G>(dot);
          const float z = dot - wave_shfl_f32(biasL, (int)(k & 63));
          const float sign = kb + k == 0 ? -1.f : 1.f;
          float sg;
          const float l = lm_softplus(sign * z, sg);
          loss += ok ? l : 0.f;
          const float g = ok ? sign * sg * w : 0.f;
          // lane k keeps candidate k's gradient: group k mod kGroups holds it now
          const float mine = wave_shfl_f32(g, (int)(((u32)lane & (kGroups - 1)) * G));
          const u32 k1 = k0 + (u32)u * kGroups;
          if ((u32)lane >= k1 && (u32)lane < k1 + kGroups) gL = mine;
          if (DH && !BLOCKS && ok) acc.template add<T, G>(g, b[u]);
        }
      }
      if (q.g != nullptr && (u32)lane < kn) q.g[t * q.cands + kb + (u32)lane] = gL;
    }
    if constexpr (BLOCKS) {
      if (DH) {
        // dh block by block of columns; this wavefront's own q.g, written above by other lanes
        wave_fence_global();
        wave_sync();
        for (u32 p0 = 0; p0 < shape.packs; p0 += G * NV) {
          acc.zero();
          for (u32 k = 0; live && k < q.cands; ++k) {
            const u32 r = uni(lm_row(ids, t * q.cands + k, q.vocab));
            if (r == q.vocab) continue;
            LmRowPart<T, V, G, NV> b;
            b.load(table + (i64)r * q.tableStride, p0, gl, shape);
            acc.template add<T, G>(q.g[t * q.cands + k], b);
          }
          acc.template store<T, G>(dh + (i64)t * q.dhStride, p0, gl, shape);
        }
      }
    } else {
      // the groups' parts, in a fixed tree
#pragma unroll
      for (int d = G; d < 64; d *= 2) {
        loss += wave_shfl_f32(loss, lane ^ d);
        if (DH) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) acc.p[i][e] += wave_shfl_f32(acc.p[i][e], lane ^ d);
          acc.tail += wave_shfl_f32(acc.tail, lane ^ d);
        }
      }
      if (DH && grp == 0) acc.template store<T, G>(dh + (i64)t * q.dhStride, 0, gl, shape);
    }
    if (lane == 0) q.out[t] = live ? loss * w : 0.f;
  }
}

}  // namespace jpp

#endif  // JPP_K_LM_NCE_H
