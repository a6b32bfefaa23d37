// Language-model operators: element types, packs of a row, the arithmetic they share.
#ifndef JPP_LM_H
#define JPP_LM_H

#include <cmath>
#include <type_traits>

#include "jpp_rt.h"

namespace jpp {

// ---- elements ----------------------------------------------------------------
// An element type is its storage and its way to and from 32 bits; nothing is computed in 16.
struct LmF32 {
  typedef float store;
  static __device__ __forceinline__ float get(u32 bits) {
    float r;
    __builtin_memcpy(&r, &bits, 4);
    return r;
  }
  static __device__ __forceinline__ u32 put(float v) {
    u32 w;
    __builtin_memcpy(&w, &v, 4);
    return w;
  }
};

struct LmBf16 {
  typedef u16 store;
  static __device__ __forceinline__ float get(u32 bits) { return LmF32::get(bits << 16); }
  static __device__ __forceinline__ u32 put(float v) {   // to nearest, ties to even
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(u16, (__bf16)v);
#else
    const u32 w = LmF32::put(v);
    if (v != v) return (w >> 16) | 0x40u;
    return (w + 0x7fffu + ((w >> 16) & 1u)) >> 16;
#endif
  }
};

struct LmF16 {
  typedef u16 store;
  static __device__ __forceinline__ float get(u32 bits) {
#if defined(__HIP_DEVICE_COMPILE__)
    return (float)__builtin_bit_cast(_Float16, (u16)bits);
#else
    const int e = (bits >> 10) & 31, m = bits & 1023;
    float r;
    if (e == 31) r = m ? NAN : INFINITY;
    else if (e == 0) r = std::ldexp((float)m, -24);
    else r = std::ldexp((float)(m + 1024), e - 25);
    return (bits & 0x8000u) != 0 ? -r : r;
#endif
  }
  static __device__ __forceinline__ u32 put(float v) {   // to nearest, ties to even
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(u16, (_Float16)v);
#else
    const u32 sign = (LmF32::put(v) >> 16) & 0x8000u;
    const float a = std::fabs(v);
    if (v != v) return sign | 0x7e00u;
    if (a == 0.f) return sign;
    if (a >= 65520.f) return sign | 0x7c00u;
    int e = 0;
    std::frexp(a, &e);                           // a < 2^e
    const int ulp = e - 11 < -24 ? -24 : e - 11; // the last bit of a half of that size
    const int m = (int)std::nearbyint(std::ldexp(a, -ulp));
    const int be = ulp + 24;                     // 0 for subnormals and the lowest normal binade
    return sign | (u32)((be << 10) + m);         // (m >= 1024 carries into the exponent by itself)
#endif
  }
};

// d + the products of two pairs of 16-bit elements, without taking them apart
template <class T>
__device__ __forceinline__ float lm_dot2(u32 a, u32 b, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (std::is_same<T, LmBf16>::value) {
    typedef __bf16 h2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(h2_t, a), __builtin_bit_cast(h2_t, b), d, false);
  } else {
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, a), __builtin_bit_cast(h2_t, b), d, false);
  }
#else
  return __builtin_fmaf(T::get(a >> 16), T::get(b >> 16), __builtin_fmaf(T::get(a & 0xffffu), T::get(b & 0xffffu), d));
#endif
}

// N elements of a row, moved as one access of up to 16 bytes and held as the words that came.  (Held as an array of 16-bit
// elements, a pack that is loaded under a condition is taken apart inside the branch, behind a wait of its own.)  The access
// asks for no more alignment than an element has: the global memory path takes a wide one at any element's address, so rows
// of odd lengths and strides use the same loads (one that crosses a cache line costs a second look-up) and no kernel exists
// once per alignment.
template <class T, int N>
struct LmPack {
  static constexpr int kBytes = N * (int)sizeof(typename T::store), kWords = (kBytes + 3) / 4;
  u32 w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(typename T::store) == 4) return T::get(w[i]);
    else return T::get((i & 1) != 0 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
  }
  __device__ __forceinline__ void set(const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(typename T::store) == 4) w[i] = T::put(x[i]);
      else w[i] = T::put(x[2 * i]) | (2 * i + 1 < N ? T::put(x[2 * i + 1 < N ? 2 * i + 1 : 0]) << 16 : 0u);
    }
  }
};

#if defined(__HIP_DEVICE_COMPILE__)
// the register image of a pack, with the alignment of an element
template <int BYTES, int ALIGN>
struct LmRaw {
  typedef u32 type __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN)));
};
template <>
struct LmRaw<4, 4> {
  typedef u32 type;
};
template <>
struct LmRaw<4, 2> {
  typedef u32 type __attribute__((aligned(2)));
};
template <>
struct LmRaw<2, 2> {
  typedef u16 type;
};
#endif

template <class T, int N>
__device__ __forceinline__ LmPack<T, N> lm_load(const typename T::store* p) {
  LmPack<T, N> x;
#if defined(__HIP_DEVICE_COMPILE__)
  typedef typename LmRaw<LmPack<T, N>::kBytes, sizeof(typename T::store)>::type Raw;
  const Raw r = *(const Raw JPP_GLOBAL*)p;
  if constexpr (LmPack<T, N>::kBytes == 2) x.w[0] = r;
  else __builtin_memcpy(&x, &r, sizeof(x));
#else
  x.w[LmPack<T, N>::kWords - 1] = 0;
  __builtin_memcpy(&x, p, LmPack<T, N>::kBytes);
#endif
  return x;
}
// STREAM: with the non-temporal hint, for results too large to be found in a cache by whoever reads them, so that they do not
// push out what this kernel itself reads again.  (A template argument: two stores under a condition that differ in the hint
// alone are merged into one without it.)
template <class T, int N, bool STREAM = false>
__device__ __forceinline__ void lm_store(typename T::store* p, const LmPack<T, N>& x) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef typename LmRaw<LmPack<T, N>::kBytes, sizeof(typename T::store)>::type Raw;
  Raw r;
  if constexpr (LmPack<T, N>::kBytes == 2) r = (Raw)x.w[0];
  else __builtin_memcpy(&r, &x, sizeof(x));
  if constexpr (STREAM) __builtin_nontemporal_store(r, (Raw JPP_GLOBAL*)p);
  else *(Raw JPP_GLOBAL*)p = r;
#else
  __builtin_memcpy(p, &x, LmPack<T, N>::kBytes);
#endif
}
template <class T, int N>
__device__ __forceinline__ LmPack<T, N> lm_pack(const float (&x)[N]) {
  LmPack<T, N> r;
  r.set(x);
  return r;
}
// A row whose length N does not divide ends in a pack moved back to its last N elements: the lanes that share elements
// compute and store the same values.
// first column of pack `i` of a row of dim >= N columns
template <int N>
__device__ __forceinline__ u32 lm_col(u32 i, u32 dim) {
  const u32 c = i * N;
  return N == 1 || c + N <= dim ? c : dim - N;
}
// ---- arithmetic ----------------------------------------------------------------
__device__ __forceinline__ float lm_exp2(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);   // (results below 2^-126 flush to zero: nothing here tells them from it)
#else
  return std::exp2(x);
#endif
}

// 1 / d for 1 <= d <= 2: the reciprocal instruction and one Newton step (within half a unit and a bit)
__device__ __forceinline__ float lm_rcp(float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
#else
  return 1.f / d;
#endif
}

// exp(-y), y >= 0: 2^(-y log2 e).  The product's rounding and the digits of log2 e behind its 24th are put back to first
// order (without either the relative error grows with y: 1e-6 at y = 20, and at y = 60).  NaN stays NaN, infinity gives 0.
__device__ __forceinline__ float lm_exp_neg(float y) {
  constexpr float kL = 1.44269504088896341f, kLlo = 1.92596303e-8f, kLn2 = 0.693147180559945309f;
  const float t = -y * kL;
  const float lo = __builtin_fmaf(-y, kLlo, __builtin_fmaf(-y, kL, -t));
  const float e = lm_exp2(t);
  return y > 104.f ? 0.f : __builtin_fmaf(e * lo, kLn2, e);
}

// to full relative precision at either end
__device__ __forceinline__ float lm_sigmoid(float z) {
  const float e = lm_exp_neg(__builtin_fabsf(z));
  const float r = lm_rcp(1.f + e);
  return z >= 0.f ? r : e * r;
}

// A gate as the smaller of sigmoid(z) and sigmoid(-z), with the sign of z: a step's weights are it and what it leaves of one, so
// they sum to one however they are rounded.  (Rounded apart, they miss it by up to 2^-24, and a state that is a mean over
// 1 / (1 - a) rows shows that as many times over: 3e-4 of itself behind 40 000 gates of 10.)
// To full precision whatever the rows' type: their states, and the gradients of those, come back in 32 bits.  1 / (1 + 2^t (1 + lo
// ln 2)), t the rounded y log2 e and lo what it misses: the instructions' 2 units of 2^-24 each, the rounding of 1 + lo ln 2 and of
// the sum.  (t ends at 1000, where the weight is zero, so that an infinite y has no infinity taken from itself; a NaN comes
// through lo.)
__device__ __forceinline__ float lm_gate_weight(float z) {
  constexpr float kL = 1.44269504088896341f, kLlo = 1.92596303e-8f, kLn2 = 0.693147180559945309f;
  const float y = __builtin_fabsf(z), t = __builtin_fminf(y * kL, 1000.f);
  const float lo = __builtin_fmaf(y, kLlo, __builtin_fmaf(y, kL, -t));
  const float d = __builtin_fmaf(lm_exp2(t), __builtin_fmaf(lo, kLn2, 1.f), 1.f);
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_copysignf(__builtin_amdgcn_rcpf(d), z);
#else
  return __builtin_copysignf(1.f / d, z);
#endif
}
__device__ __forceinline__ bool lm_open(float w) { return (i32)LmF32::put(w) >= 0; }   // (a weight may be a zero with a sign)
// a v + (1 - a) x, from the larger weight's side
__device__ __forceinline__ float lm_step(float w, float v, float x) { return __builtin_fmaf(w, x - v, lm_open(w) ? v : x); }
// a v
__device__ __forceinline__ float lm_kept(float w, float v) { return __builtin_fmaf(-w, v, lm_open(w) ? v : 0.f); }
// a v, (1 - a) v, a (1 - a) v
__device__ __forceinline__ void lm_parts(float w, float v, float& kept, float& in, float& both) {
  const float s = __builtin_fabsf(w), p = s * v, q = __builtin_fmaf(-s, v, v);
  kept = lm_open(w) ? q : p;
  in = lm_open(w) ? p : q;
  both = __builtin_fmaf(-s, p, p);
}
// The same from the two weights, for states that are not finite, or further than the largest number from what comes in: there
// differences are NaN or infinite where the formula's value is not.
struct LmWeights {
  float a, b;
  __device__ __forceinline__ explicit LmWeights(float w) {
    const float s = __builtin_fabsf(w), l = 1.f - s;
    a = lm_open(w) ? l : s;
    b = lm_open(w) ? s : l;
  }
};
__device__ __forceinline__ bool lm_finite(float v) { return __builtin_fabsf(v) < __builtin_inff(); }

// Many steps are v -> A v + B.  Their A is held like a gate's weights, and for the same reason (the same sentence may have the same
// gates in every chunk, and the same rounding of their product): 1 - A, or - A where that is the smaller.  kLmFresh: nothing of v
// passes, also where v is no number.
constexpr float kLmFresh = -2.f;
__device__ __forceinline__ float lm_map_weight(float A, float C) { return A > 0.5f ? C : -A; }   // C: 1 - A, made for itself
// A v + B = whole v + (minus v + B), for finite v
__device__ __forceinline__ float lm_map_whole(float w) { return lm_open(w) ? 1.f : 0.f; }
__device__ __forceinline__ float lm_map_minus(float w) { return w == kLmFresh ? 0.f : -w; }
// A v + B.  EXACT: also where v is not finite, or the difference v (A - 1) + B is not; a caller takes it where the other form's
// result is not finite.  (A is never zero, though its product may be: an infinity passes.)
template <bool EXACT>
__device__ __forceinline__ float lm_map(float w, float v, float B) {
  float r = __builtin_fmaf(-w, v, B) + (lm_open(w) ? v : 0.f);
  if constexpr (EXACT) {
    const float s = lm_finite(v) ? __builtin_fmaf(lm_open(w) ? 1.f - w : -w, v, B) : v + B;
    r = lm_finite(r) ? r : s;
  }
  return w == kLmFresh ? B : r;
}

// softplus(z) = max(z, 0) + ln(1 + exp(-|z|)), s = sigmoid(z); ln(1 + e) with the rounding of 1 + e put back
__device__ __forceinline__ float lm_softplus(float z, float& s) {
  const float e = lm_exp_neg(__builtin_fabsf(z));
  const float u = 1.f + e;
  const float r = lm_rcp(u);
  s = z >= 0.f ? r : e * r;
#if defined(__HIP_DEVICE_COMPILE__)
  const float ln = __builtin_amdgcn_logf(u) * 0.693147180559945309f;   // (the instruction is a base-2 logarithm)
#else
  const float ln = std::log2(u) * 0.693147180559945309f;
#endif
  const float l = e < 0x1p-12f ? e - 0.5f * e * e : ln + (e - (u - 1.f)) * r;
  return z != z ? z : (z > 0.f ? z : 0.f) + l;
}

template <int V>
struct LmConst {
  static constexpr int value = V;
};

// sum over aligned groups of N lanes (N = 4, 8, 16, 32 or 64), the same value in every lane of the group; the tree is
// fixed, so the bits are
template <int N>
__device__ __forceinline__ float lm_group_sum(float v) {
#if defined(JPP_EMU) || !defined(__HIP_DEVICE_COMPILE__)
  for (int d = 1; d < N; d *= 2) v += wave_shfl_f32(v, lane_id() ^ d);
  return v;
#else
  // inside rows of 16 lanes through DPP: quad permutes, half-row and row mirrors
  auto dpp = [](float x, auto ctrl) {
    int y;
    __builtin_memcpy(&y, &x, 4);
    y = __builtin_amdgcn_update_dpp(0, y, decltype(ctrl)::value, 0xf, 0xf, false);
    __builtin_memcpy(&x, &y, 4);
    return x;
  };
  if constexpr (N >= 2) v += dpp(v, LmConst<0xB1>());    // quad_perm 1,0,3,2
  if constexpr (N >= 4) v += dpp(v, LmConst<0x4E>());    // quad_perm 2,3,0,1
  if constexpr (N >= 8) v += dpp(v, LmConst<0x141>());   // row_half_mirror
  if constexpr (N >= 16) v += dpp(v, LmConst<0x140>());  // row_mirror
  if constexpr (N >= 32) v += wave_shfl_f32(v, lane_id() ^ 16);
  if constexpr (N >= 64) v += wave_shfl_f32(v, lane_id() ^ 32);
  return v;
#endif
}

// Lane I of every aligned group of N lanes (N = 16 or 64), in all lanes of the group.
template <int N, int I>
__device__ __forceinline__ float lm_group_bcast(float v) {
  static_assert((N == 16 || N == 64) && I < 16, "a row of lanes, or all of them");
#if defined(JPP_EMU) || !defined(__HIP_DEVICE_COMPILE__)
  return wave_shfl_f32(v, (lane_id() & ~(N - 1)) + I);
#else
  if constexpr (N == 64) return wave_bcast_f32(v, I);
  const int x = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, 0x150 + I, 0xf, 0xf, false));   // row_newbcast
#endif
}

// Sums over the four rows of 16 lanes, the rows sharing the result: of v[0 .. N - 1] in every row, row r keeps the N / 4
// sums of elements r N / 4 .. in v[0 .. N / 4 - 1].  Lanes 32 apart swap halves of the array, then lanes 16 apart.
template <int N>
__device__ __forceinline__ void lm_rows_share(float (&v)[N]) {
  static_assert(N % 4 == 0, "a quarter each");
  auto exchange = [&](float& a, float& b, auto half) {   // a: the sum over the pair in the lower lanes, b's in the upper
#if defined(__HIP_DEVICE_COMPILE__)
    const u32 x = __builtin_bit_cast(u32, a), y = __builtin_bit_cast(u32, b);
    u32 p, q;   // (words of their own: a bit cast of the result's second element takes the first)
    if constexpr (decltype(half)::value == 32) {
      const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
      p = r[0], q = r[1];
    } else {
      const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
      p = r[0], q = r[1];
    }
    a = __builtin_bit_cast(float, p) + __builtin_bit_cast(float, q);
#else
    constexpr int d = decltype(half)::value;
    const bool up = (lane_id() & d) != 0;
    const float mine = up ? b : a, other = wave_shfl_f32(up ? a : b, lane_id() ^ d);
    a = up ? other + mine : mine + other;
#endif
  };
#pragma unroll
  for (int i = 0; i < N / 2; ++i) exchange(v[i], v[i + N / 2], LmConst<32>());
#pragma unroll
  for (int i = 0; i < N / 4; ++i) exchange(v[i], v[i + N / 4], LmConst<16>());
}

// ---- ids -----------------------------------------------------------------------
struct LmIds {
  const void* data;
  u32 wide;   // int64 ids, not int32
};
// the id as a row of the table, or `vocab` where it names no word
__device__ __forceinline__ u32 lm_row(const LmIds& ids, u64 i, u32 vocab) {
  const i64 v = ids.wide ? as_global(static_cast<const i64*>(ids.data))[i] : (i64)as_global(static_cast<const i32*>(ids.data))[i];
  return v >= 0 && v < (i64)vocab ? (u32)v : vocab;
}

// j / d for 0 <= j < 2^31, 1 <= d < 2^31, by a product: m = ceil(2^(31 + s) / d) with 2^s >= d, so the error of j m / 2^(31 + s)
// stays below 1 / d
struct LmDiv {
  u32 mul, shift;
  static LmDiv by(u32 d) {
    u32 s = 0;
    while ((u64{1} << s) < d) ++s;
    return LmDiv{(u32)(((u64{1} << (31 + s)) + d - 1) / d), 31 + s};
  }
  __device__ __forceinline__ u32 operator()(u32 j) const { return (u32)((u64)j * mul >> shift); }
};

constexpr u32 kLmThreads = 256;        // threads of a workgroup, where a kernel has no reason for another number
constexpr u64 kLmChipBlocks = 256 * 8; // workgroups of kLmThreads threads that the 256 compute units hold, at up to 64 registers a lane
constexpr u32 kLmMaxBlocks = 1u << 21; // largest grid (the sort of 2^31 entries has half of it); kernels that may need more loop

}  // namespace jpp

#endif  // JPP_LM_H
