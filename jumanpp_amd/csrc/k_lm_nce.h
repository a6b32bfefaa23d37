// Language-model operators 3: the noise-contrastive score of candidate words and the loss with its gradients.
//
//   score   s = <h_t, W[c]> - C
//   loss    z_k = s_k - ln(K p(c_k)), L_t = w_t (softplus(-z_0) + sum over k > 0 of softplus(z_k))
//           dL/dz_0 = -w sigmoid(-z_0), dL/dz_k = w sigmoid(z_k); dh_t = sum of g_k W[c_k]; dW by word: k_lm_embed.h
//
// The rows of W are gathered: the bytes of K rows a token decide, from L2 and the memory-side cache for a table that fits
// there.  A group of G lanes holds a row in registers, so the loss reads every row once -- the product with h, then
// g_k times the same registers into dh.  G = 16 keeps the product's reduction inside a row of 16 lanes (four DPP steps,
// four candidates side by side); longer rows take the whole wavefront (for 256 columns of 16 bits the loss would take three
// times as long: a reduction over 64 lanes for every candidate, none side by side).
// 507 904 tokens, 6 candidates, 128 bfloat16 columns are scored in 57 us: 0.72 GB asked of the L2s, 0.28 GB of it from outside,
// the vector unit taking 0.6 of its slots.  The loss of 65 536 tokens, 33 candidates, 256 columns takes 110 us with dh, the
// vector unit 0.77 of its slots: that is the bound there.  Hence the products in pairs (lm_dot2), addresses made once and
// handed on, and the exact row length as a kind of its own: 57 us against 70 with the masks of shorter rows; the loss gains
// 35 us.
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
// element once; they are loaded from the row's start and cleared (no branch, so that a wait covers many rows).  FULL: every
// part exists.
struct LmRowShape {
  u32 packs, rest;   // full packs, elements behind them
};
template <class T, int V, int G, int NV, bool FULL>
struct LmRowPart {
  LmPack<T, V> p[NV];
  LmPack<T, 1> tail;
  __device__ __forceinline__ void load(const typename T::store* row, u32 p0, u32 gl, const LmRowShape& s) {
    if constexpr (FULL) {
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i] = lm_load<T, V>(row + (gl + (u32)(G * i)) * V);
      tail.zero();
    } else {
      // (where V > dim there is no full pack: the tail has it all)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        p[i].zero();
        if (s.packs != 0) p[i] = lm_load<T, V>(row + (p0 + gl + (u32)(G * i) < s.packs ? p0 + gl + (u32)(G * i) : 0u) * V);
      }
      tail.zero();
      if (s.rest != 0) tail = lm_load<T, 1>(row + s.packs * V + (gl < s.rest ? gl : 0u));
    }
  }
  // cleared unless `ok`
  __device__ __forceinline__ void keep(bool ok) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < LmPack<T, V>::kWords; ++k) p[i].w[k] = ok ? p[i].w[k] : 0u;
    tail.w[0] = ok ? tail.w[0] : 0u;
  }
  __device__ __forceinline__ void mask(u32 p0, u32 gl, const LmRowShape& s) {
    if constexpr (!FULL) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < LmPack<T, V>::kWords; ++k) p[i].w[k] = p0 + gl + (u32)(G * i) < s.packs ? p[i].w[k] : 0u;
      tail.w[0] = p0 == 0 && gl < s.rest ? tail.w[0] : 0u;
    }
  }
};
// the product of two parts; both cleared where they do not exist
template <class T, int V, int G, int NV, bool FULL>
__device__ __forceinline__ float lm_dot_parts(const LmRowPart<T, V, G, NV, FULL>& x, const LmRowPart<T, V, G, NV, FULL>& y) {
  float d = 0.f;
  if constexpr (!FULL) d = x.tail.get(0) * y.tail.get(0);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (sizeof(typename T::store) == 2) {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) d = lm_dot2<T>(x.p[i].w[k], y.p[i].w[k], d);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d = __builtin_fmaf(x.p[i].get(e), y.p[i].get(e), d);
    }
  }
  return d;
}
template <int V, int NV, bool FULL>
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
  __device__ __forceinline__ void add(float w, const LmRowPart<T, V, G, NV, FULL>& x) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) p[i][e] = __builtin_fmaf(w, x.p[i].get(e), p[i][e]);
    if constexpr (!FULL) tail = __builtin_fmaf(w, x.tail.get(0), tail);
  }
  template <class T, int G>
  __device__ __forceinline__ void store(typename T::store* row, u32 p0, u32 gl, const LmRowShape& s) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const u32 at = p0 + gl + (u32)(G * i);
      if (FULL || at < s.packs) lm_store<T, V>(row + at * V, lm_pack<T, V>(p[i]));
    }
    if (!FULL && s.rest != 0 && p0 == 0 && gl < s.rest) {
      const float x[1] = {tail};
      lm_store<T, 1>(row + s.packs * V + gl, lm_pack<T, 1>(x));
    }
  }
};

// the product of two rows, block of columns by block
template <class T, int V, int G, int NV>
__device__ __forceinline__ float lm_dot_blocks(const typename T::store* x, const typename T::store* y, u32 gl, const LmRowShape& s) {
  float d = 0.f;
  for (u32 p0 = 0; p0 < s.packs; p0 += G * NV) {
    LmRowPart<T, V, G, NV, false> a, b;
    a.load(x, p0, gl, s);
    b.load(y, p0, gl, s);
    a.mask(p0, gl, s);
    b.mask(p0, gl, s);
    d += lm_dot_parts<T, V, G, NV, false>(a, b);
  }
  return d;
}

// NV packs of V elements a lane cover G NV packs: the whole row exactly (kLmFull), the whole row (kLmPart), or a block of it,
// the row being longer (kLmBlocks: the loss then reads the rows of W twice).
enum LmRowKind { kLmFull, kLmPart, kLmBlocks };
// Rows in flight a group: about 32 registers of them.
template <class T, int V, int NV>
constexpr int lm_rows_in_flight() {
  return NV * V * (int)sizeof(typename T::store) >= 64 ? 2 : NV * V * (int)sizeof(typename T::store) >= 32 ? 4 : 8;
}

// where a row is, to hand from lane to lane
template <class S>
__device__ __forceinline__ u64 lm_address(const S* row) {
  return (u64) reinterpret_cast<uintptr_t>(row);
}

// A group takes up to kLmScoreCands candidates of a token: h comes in once for them, their ids with one load (a lane each),
// their rows several at a time.  The vector unit decides: where a row starts is worked out once, by the lane that loaded the
// id (a 64-bit product is a dozen full-rate operations), and handed to the group.
constexpr u32 kLmScoreCands = 16;
template <class T, int V, int G, int NV, LmRowKind KIND>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_nce_score(LmNce q, const typename T::store* __restrict__ h, const typename T::store* __restrict__ table, LmIds ids) {
  typedef typename T::store S;
  constexpr bool BLOCKS = KIND == kLmBlocks, FULL = KIND == kLmFull;
  constexpr int U = BLOCKS ? 1 : lm_rows_in_flight<T, V, NV>();
  const int lane = (int)(threadIdx.x & 63);
  const u32 gl = threadIdx.x & (G - 1);
  const LmRowShape shape = {q.dim / V, q.dim % V};
  const u32 parts = (q.cands + kLmScoreCands - 1) / kLmScoreCands;
  const u64 tasks = q.n * parts;
  const u64 step = (u64)gridDim.x * (kLmThreads / G);
  // (whole wavefronts stay in the loop: the group sums are wavefront operations)
  for (u64 task0 = (u64)blockIdx.x * (kLmThreads / G); task0 < tasks; task0 += step) {
    const u64 task = task0 + threadIdx.x / G;
    const bool some = task < tasks;
    const u64 t = some ? (parts == 1 ? task : task / parts) : 0u;
    const u32 k0 = some ? (u32)(task - t * parts) * kLmScoreCands : 0u;
    const u32 cnt = some ? (q.cands - k0 < kLmScoreCands ? q.cands - k0 : kLmScoreCands) : 0u;
    const u32 rowL = gl < cnt ? lm_row(ids, t * q.cands + k0 + gl, q.vocab) : q.vocab;
    float mine = 0.f;
    if (q.vocab != 0) {
      LmRowPart<T, V, G, NV, FULL> hr;
      if constexpr (!BLOCKS) {
        hr.load(h + (i64)t * q.hStride, 0, gl, shape);
        hr.mask(0, gl, shape);
      }
      // (an id that names no word reads row 0 for nothing)
      const u64 atL = lm_address(table + (rowL < q.vocab ? (u64)rowL * (u64)q.tableStride : 0u));
      const u32 most = uni(wave_max_u32(cnt));
      // candidates k .. k + R - 1 of every group; k + R <= 16 <= G
      auto rows = [&](auto many, u32 k) {
        constexpr u32 R = decltype(many)::value;
        LmRowPart<T, V, G, NV, FULL> b[R];
        const S* row[R];
#pragma unroll
        for (u32 u = 0; u < R; ++u) {
          row[u] = reinterpret_cast<const S*>(wave_shfl_u64(atL, (int)((lane & ~(G - 1)) + k + u)));
          if constexpr (!BLOCKS) b[u].load(row[u], 0, gl, shape);
        }
#pragma unroll
        for (u32 u = 0; u < R; ++u) {
          float dot;
          if constexpr (BLOCKS) {
            dot = lm_dot_blocks<T, V, G, NV>(h + (i64)t * q.hStride, row[u], gl, shape);
          } else {
            b[u].mask(0, gl, shape);
            dot = lm_dot_parts<T, V, G, NV, FULL>(hr, b[u]);
          }
          dot = lm_group_sum<G>(dot);
          mine = gl == k + u ? dot : mine;
        }
      };
      u32 k = 0;
      for (; k + U <= most; k += U) rows(LmConst<U>(), k);
      if (U > 4 && k + 4 <= most) {
        rows(LmConst<4>(), k);
        k += 4;
      }
      if (U > 2 && k + 2 <= most) {
        rows(LmConst<2>(), k);
        k += 2;
      }
      if (k < most) rows(LmConst<1>(), k);
    }
    if (gl < cnt) q.out[t * q.cands + k0 + gl] = rowL < q.vocab ? mine - q.constant : -__builtin_inff();
  }
}

// A wavefront a token, its groups side by side over the candidates.  What the next token needs is requested while this one's
// rows are on their way: its ids first, then, from them, the logarithms of its noise, and its row of h.
template <class T, int V, int G, int NV, LmRowKind KIND, bool DH>
__global__ void __launch_bounds__(kLmThreads)
    k_lm_nce_loss(LmNce q, const typename T::store* __restrict__ h, const typename T::store* __restrict__ table, LmIds ids,
                  typename T::store* __restrict__ dh) {
  typedef typename T::store S;
  constexpr bool BLOCKS = KIND == kLmBlocks, FULL = KIND == kLmFull;
  constexpr u32 kGroups = 64 / G;
  constexpr int U = BLOCKS ? 1 : lm_rows_in_flight<T, V, NV>();
  const int lane = (int)(threadIdx.x & 63);
  const u32 gl = threadIdx.x & (G - 1), grp = (u32)lane / G;
  const LmRowShape shape = {q.dim / V, q.dim % V};
  const u64 step = (u64)gridDim.x * (kLmThreads / 64);
  const u64 t00 = (u64)blockIdx.x * (kLmThreads / 64) + (threadIdx.x >> 6);
  const u32 ahead = q.cands < 64 ? q.cands : 64u;
  u32 rowN = q.vocab;
  float lnN = 0.f;
  LmRowPart<T, V, G, NV, FULL> hN;
  auto fetch_ids = [&](u64 t) {
    rowN = q.vocab;
    if (t < q.n && (u32)lane < ahead) rowN = lm_row(ids, t * q.cands + (u32)lane, q.vocab);
  };
  auto fetch_rest = [&](u64 t) {
    lnN = 0.f;
    if (rowN < q.vocab) lnN = q.logNoise[rowN];
    if constexpr (!BLOCKS) hN.load(h + (i64)(t < q.n ? t : t00) * q.hStride, 0, gl, shape);
  };
  if (t00 >= q.n) return;
  fetch_ids(t00);
  fetch_rest(t00);
  for (u64 t = t00; t < q.n; t += step) {
    u32 rowL = rowN;
    float lnL = lnN;
    const u32 target = wave_bcast_u32(rowL, 0);
    const bool live = target < q.vocab;
    const float w = q.weight != nullptr ? q.weight[t] : 1.f;
    LmRowSum<V, NV, FULL> acc;
    acc.zero();
    float loss = 0.f;
    LmRowPart<T, V, G, NV, FULL> hr = hN;
    if constexpr (!BLOCKS) hr.mask(0, gl, shape);
    fetch_ids(t + step);
    if (!live) fetch_rest(t + step);
    for (u32 kb = 0; live && kb < q.cands; kb += 64) {
      const u32 kn = q.cands - kb < 64 ? q.cands - kb : 64u;
      if (kb > 0) {
        rowL = (u32)lane < kn ? lm_row(ids, t * q.cands + kb + (u32)lane, q.vocab) : q.vocab;
        lnL = rowL < q.vocab ? q.logNoise[rowL] : 0.f;
      }
      const u64 named = wave_ballot(rowL < q.vocab);
      const float biasL = q.constant + lnL;
      // (a candidate that names no word reads the target's row and leaves with a gradient of zero)
      const u64 atL = lm_address(table + (u64)(rowL < q.vocab ? rowL : target) * (u64)q.tableStride);
      // lane k keeps what is candidate k's alone: its logit now, its loss and gradient once for all 64 behind the loop
      float zL = 0.f;
      // candidates k0 .. k0 + R kGroups - 1, those behind kn as ones without a word
      auto rows = [&](auto many, u32 k0) {
        constexpr u32 R = decltype(many)::value;
        static_assert(R * kGroups < 64 && R <= 8, "a step does not pass the 64th candidate");
        LmRowPart<T, V, G, NV, FULL> b[R];
        const S* row[R];
#pragma unroll
        for (u32 u = 0; u < R; ++u) {
          row[u] = reinterpret_cast<const S*>(wave_shfl_u64(atL, (int)(k0 + u * kGroups + grp)));
          if (!BLOCKS) b[u].load(row[u], 0, gl, shape);
        }
        if (kb + k0 == 0) fetch_rest(t + step);
        constexpr u64 kThese = (u64{1} << (R * kGroups)) - 1;
        const bool all = ((named >> k0) & kThese) == kThese;
        float zg = 0.f;   // of the group's candidate gl
#pragma unroll
        for (u32 u = 0; u < R; ++u) {
          const u32 k1 = k0 + u * kGroups, k = k1 + grp;
          float dot;
          if constexpr (BLOCKS) {
            dot = lm_dot_blocks<T, V, G, NV>(h + (i64)t * q.hStride, row[u], gl, shape);
          } else {
            b[u].mask(0, gl, shape);
            dot = lm_dot_parts<T, V, G, NV, FULL>(hr, b[u]);
          }
          const float z = lm_group_sum<G>(dot) - wave_shfl_f32(biasL, (int)k);
          // (lane k of the 64 reads group k mod kGroups)
          const float mine = kGroups == 1 ? z : wave_shfl_f32(z, (int)(((u32)lane & (kGroups - 1)) * G));
          zL = (u32)lane - k1 < kGroups ? mine : zL;
          if constexpr (DH && !BLOCKS) zg = gl == u ? z : zg;
        }
        if constexpr (DH && !BLOCKS) {
          // a lane a candidate makes the gradient once, and hands it to its group
          const u32 kL = k0 + gl * kGroups + grp;
          const float s = kb + kL == 0 ? -1.f : 1.f;
          const float gL = lm_sigmoid(s * zg) * (s * w);
          auto add = [&](auto at) {
            constexpr int I = decltype(at)::value;
            if constexpr (I < (int)R) {
              float gk = lm_group_bcast<G, I>(gL);
              if (!all) {   // (a branch around the sum, on its candidates or on their number, has the compiler copy the sum: 16 moves a row)
                const bool ok = ((named >> (k0 + (u32)I * kGroups + grp)) & 1u) != 0;
                gk = ok ? gk : 0.f;
                b[I].keep(ok);
              }
              acc.template add<T, G>(gk, b[I]);
            }
          };
          add(LmConst<0>()), add(LmConst<1>()), add(LmConst<2>()), add(LmConst<3>());
          add(LmConst<4>()), add(LmConst<5>()), add(LmConst<6>()), add(LmConst<7>());
        }
      };
      u32 k0 = 0;
      for (; k0 + kGroups < kn; k0 += kGroups * U) rows(LmConst<U>(), k0);
      if (k0 < kn) rows(LmConst<1>(), k0);
      const float sign = kb + (u32)lane == 0 ? -1.f : 1.f;
      float sg;
      const float l = lm_softplus(sign * zL, sg);
      const bool okL = rowL < q.vocab;
      loss += okL ? l : 0.f;
      if (q.g != nullptr && (u32)lane < kn) q.g[t * q.cands + kb + (u32)lane] = okL ? sign * sg * w : 0.f;
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
            LmRowPart<T, V, G, NV, FULL> b;
            b.load(table + (i64)r * q.tableStride, p0, gl, shape);
            b.mask(p0, gl, shape);
            acc.template add<T, G>(q.g[t * q.cands + k], b);
          }
          acc.template store<T, G>(dh + (i64)t * q.dhStride, p0, gl, shape);
        }
      }
    } else {
      if constexpr (DH && G == 64) {
        acc.template store<T, G>(dh + (i64)t * q.dhStride, 0, gl, shape);
      } else if constexpr (DH) {
        // the four groups' parts are added and shared out: group r stores a quarter of every lane's elements
        static_assert(G == 16, "a group is a row of lanes");
        constexpr int Q = NV * V / 4;
        float flat[NV * V];
#pragma unroll
        for (int i = 0; i < NV * V; ++i) flat[i] = acc.p[i / V][i % V];
        lm_rows_share(flat);
        float mine[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) mine[i] = flat[i];
        typename T::store* row = dh + (i64)t * q.dhStride;
        constexpr int kStore = Q < V ? Q : V;   // elements of one pack that a group has
#pragma unroll
        for (int i = 0; i < Q; i += kStore) {
          const u32 at = grp * (u32)Q + (u32)i, pack = gl + G * (at / V);
          float part[kStore];
#pragma unroll
          for (int e = 0; e < kStore; ++e) part[e] = mine[i + e];
          if (FULL || pack < shape.packs) lm_store<T, kStore>(row + pack * V + at % V, lm_pack<T, kStore>(part));
        }
        if constexpr (!FULL) {
          if (shape.rest != 0) {
            float tail = acc.tail;
            tail += wave_shfl_f32(tail, lane ^ 32);
            tail += wave_shfl_f32(tail, lane ^ 16);
            const float one[1] = {tail};
            if (grp == 0 && gl < shape.rest) lm_store<T, 1>(row + shape.packs * V + gl, lm_pack<T, 1>(one));
          }
        }
      }
    }
    loss = lm_group_sum<64>(loss);
    if (lane == 0) q.out[t] = live ? loss * w : 0.f;
  }
}

}  // namespace jpp

#endif  // JPP_K_LM_NCE_H
