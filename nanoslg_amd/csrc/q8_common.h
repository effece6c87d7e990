// 8-bit KV caches: the code types, their conversion to MFMA operands, and the write of
// one block of tokens.
//
// A cache layer is codes [P, page_size, Hkv, D] (1 byte) and fp32 scales [P, nb, Hkv],
// nb = ceil(page_size / 16): one scale for each block of 16 slots of a page and KV head,
// for K and for V. A stored value is code * scale; scales are powers of two (or 0), so
// that x / scale is exact, a code is x / scale rounded once, and raising a block's scale
// shifts its codes (exactly for e4m3, but for its subnormals).
#pragma once

#include "nslg_common.h"

namespace nslg {

constexpr int kBlockToks = 16;  // tokens of a block (the last block of a page may be shorter)

// The pool holds the 16-bit elements themselves.
struct Raw16 {
  static constexpr bool kQ8 = false;
  static constexpr bool kNanScale = false;
  static constexpr int kBytes = 2;  // of an element
};

__device__ inline float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }

// Smallest power of two s >= 2^-126 with amax <= kMost * s, as its biased exponent (0: amax
// is 0). kMost = (1 + kMant / 2^23) 2^kExp.
template <typename F>
__device__ inline float scale_for(uint32_t amax_bits) {
  int e = (int)(amax_bits >> 23) - F::kExp + ((amax_bits & 0x7fffffu) > F::kMant ? 1 : 0);
  e = e < 1 ? 1 : e;
  return amax_bits ? pow2_bits(e) : 0.f;
}

// 1 / scale for a power of two (biased exponents 1 .. 253); 0 for scale 0.
__device__ inline float inv_scale(float scale) {
  return scale > 0.f ? pow2_bits(254 - (int)(__float_as_uint(scale) >> 23)) : 0.f;
}

// OCP e4m3 without infinities: codes 0x7f / 0xff are NaN, the largest value is 448.
struct E4M3 {
  static constexpr bool kQ8 = true;
  static constexpr int kBytes = 1;
  static constexpr int kExp = 8;
  static constexpr uint32_t kMant = 0x600000;  // 448 = 1.75 * 2^8
  static constexpr bool kNanScale = false;     // has codes for what is not finite
  // four values (|y| <= 448, or NaN) as codes, rounded to nearest even
  __device__ static inline uint32_t encode4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
  __device__ static inline void decode4(uint32_t w, float (&f)[4]) {
    f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  }
};

// Integers in [-127, 127]; a block that was given a value that is not finite has K scale NaN.
struct Int8 {
  static constexpr bool kQ8 = true;
  static constexpr int kBytes = 1;
  static constexpr int kExp = 6;
  static constexpr uint32_t kMant = 0x7e0000;  // 127 = 1.984375 * 2^6
  static constexpr bool kNanScale = true;
  __device__ static inline uint32_t encode4(float a, float b, float c, float d) {
    const uint32_t i0 = (uint32_t)(int)__builtin_rintf(a), i1 = (uint32_t)(int)__builtin_rintf(b);
    const uint32_t i2 = (uint32_t)(int)__builtin_rintf(c), i3 = (uint32_t)(int)__builtin_rintf(d);
    const uint32_t lo = __builtin_amdgcn_perm(i1, i0, 0x0c0c0400u), hi = __builtin_amdgcn_perm(i3, i2, 0x04000c0cu);
    return lo | hi;
  }
  __device__ static inline void decode4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Four codes as 16-bit elements of type T, exactly.
template <typename T, typename F>
__device__ inline u16x4 codes_as16(uint32_t w) {
  u32x2 r;
  if constexpr (!F::kNanScale && T::kDtype == NSLG_F16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  } else if constexpr (!F::kNanScale) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
  } else if constexpr (T::kDtype == NSLG_F16) {
    // 0x6400 | u is the half 1024 + u: with u = code + 128, minus 1152 gives the code
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    r[0] = __builtin_bit_cast(uint32_t, a - off);
    r[1] = __builtin_bit_cast(uint32_t, b - off);
  } else {  // 8 significant bits hold a code: the upper half of its fp32 value is exact
    float f[4];
    F::decode4(w, f);
    r[0] = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
    r[1] = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
  }
  return __builtin_bit_cast(u16x4, r);
}

template <typename T, typename F>
__device__ inline u16x8 codes_as16(u32x2 w) {
  const u16x4 a = codes_as16<T, F>(w[0]), b = codes_as16<T, F>(w[1]);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Scales that codes_to16 takes as they are for int8 codes in half: a half themselves, and 1152 times them too.
constexpr float kHalfScaleMin = 0x1p-24f, kHalfScaleMax = 32.f;

// Four codes times `scale` (a power of two; NaN gives NaN) as 16-bit elements of type T, exact wherever the
// product is a normal number of T. kWide: int8 codes in half with a scale past the two above.
template <typename T, typename F, bool kWide = false>
__device__ inline u16x4 codes_to16(uint32_t w, float scale) {
  u32x2 r;
  if constexpr (T::kDtype == NSLG_F16 && !F::kNanScale) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
  } else if constexpr (T::kDtype == NSLG_BF16 && !F::kNanScale) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
  } else if constexpr (T::kDtype == NSLG_F16 && !kWide) {
    // as in codes_as16: (1152 + code) * scale - 1152 * scale, every step exact
    const uint32_t u = w ^ 0x80808080u;
    const _Float16 s = (_Float16)scale, n = (_Float16)(-1152.f * scale);
    const f16x2 ss = {s, s}, nn = {n, n};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    r[0] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(a, ss, nn));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, ss, nn));
  } else {
    float f[4];
    F::decode4(w, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= scale;
    if constexpr (T::kDtype == NSLG_BF16) {
      r[0] = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
      r[1] = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
    } else {  // rounded into half's subnormals
      return u16x4{T::from_f32(f[0]), T::from_f32(f[1]), T::from_f32(f[2]), T::from_f32(f[3])};
    }
  }
  return __builtin_bit_cast(u16x4, r);
}

// Eight codes, any power of two as the scale; or, with kWide given, what four take.
template <typename T, typename F>
__device__ inline u16x8 codes_to16(u32x2 w, float scale) {
  u16x4 a, b;
  if (F::kNanScale && T::kDtype == NSLG_F16 && (scale < kHalfScaleMin || scale > kHalfScaleMax)) {
    a = codes_to16<T, F, true>(w[0], scale), b = codes_to16<T, F, true>(w[1], scale);
  } else {
    a = codes_to16<T, F>(w[0], scale), b = codes_to16<T, F>(w[1], scale);
  }
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T, typename F, bool kWide>
__device__ inline u16x8 codes_to16(u32x2 w, float scale) {
  const u16x4 a = codes_to16<T, F, kWide>(w[0], scale), b = codes_to16<T, F, kWide>(w[1], scale);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Byte n of the words r[0 .. 3], for n = 0 .. 3: c[n] = (r[0].n, r[1].n, r[2].n, r[3].n).
__device__ inline void transpose4x4(const uint32_t (&r)[4], uint32_t (&c)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), t1 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const uint32_t t2 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), t3 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  c[0] = __builtin_amdgcn_perm(t2, t0, 0x05040100u);
  c[1] = __builtin_amdgcn_perm(t2, t0, 0x07060302u);
  c[2] = __builtin_amdgcn_perm(t3, t1, 0x05040100u);
  c[3] = __builtin_amdgcn_perm(t3, t1, 0x07060302u);
}

// Largest of the lanes' values (bit patterns of non-negative floats).
__device__ inline uint32_t wave_max_bits(uint32_t x) { return (uint32_t)wave_max_i32((int)x); }

// A wave's new rows of one block of one KV head: each lane holds 8 elements of one row, 512 / D rows a
// step. They stay in registers between the maximum and the rounding, so they are read once.
template <int D>
struct BlockRows {
  static constexpr int kLanes = D / 8;
  static constexpr int kRows = 64 / kLanes;
  static constexpr int kIters = kBlockToks / kRows;
  u16x8 x[kIters];
};

// row(i, e) gives elements e .. e + 7 of the block's row i (a u16x8 of T), for new rows only.
template <int D, typename Row>
__device__ inline void load_block_rows(BlockRows<D>& b, int a, int cnt, Row row) {
  const int lane = threadIdx.x & 63;
  const int i0 = lane / b.kLanes, e = 8 * (lane % b.kLanes);
#pragma unroll
  for (int it = 0; it < b.kIters; ++it) {
    const int i = b.kRows * it + i0;
    b.x[it] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (i >= a && i < a + cnt) b.x[it] = row(i, e);
  }
}

__device__ inline bool finite_bits(uint32_t abs_bits) { return abs_bits < 0x7f800000u; }

template <typename T>
__device__ inline uint32_t abs_bits(uint16_t x) {
  return __float_as_uint(T::to_f32(x)) & 0x7fffffffu;
}

// Bit `it`: the lane's 8 elements of step `it` hold one that is not finite.
template <typename T, int D>
__device__ inline uint32_t not_finite(const BlockRows<D>& rows) {
  uint32_t bad = 0;
#pragma unroll
  for (int it = 0; it < BlockRows<D>::kIters; ++it) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits<T>(rows.x[it][j]));
    bad |= finite_bits(m) ? 0u : 1u << it;
  }
  return bad;
}

// Sets the lane's elements of K to NaN where those of V are not all finite (`bad`: not_finite of V's rows).
template <int D>
__device__ inline void spoil(BlockRows<D>& k, uint32_t bad) {
#pragma unroll
  for (int it = 0; it < BlockRows<D>::kIters; ++it)
    if ((bad >> it) & 1) k.x[it] = u16x8(0x7fff);  // NaN in half and in bfloat16
}

// One wave writes its rows a .. a + cnt - 1 (1 <= cnt, a + cnt <= 16) of K (kIsK) or V of one block of one KV head
// and sets the block's scale. `codes`: the block's row 0 at this head, rows row_bytes apart.
//
// A block written from its first row takes the scale its new rows need. Otherwise the scale is the larger of
// its own and that one, and where it grew the rows 0 .. a - 1 are rounded to it; rows past a + cnt - 1 (of no
// token) are left as they are.
//
// A token's value that is not finite, in K or V, goes into K alone (the caller spoils K's rows with V's): its score
// is then NaN for the queries that see it, and masked for those that do not, while a NaN in V would reach these too
// (0 * NaN). e4m3: NaN codes in the row; int8, which has no such code: K's scale, so the whole block's K, until it is
// written from its first row.
template <typename T, typename F, int D, bool kIsK>
__device__ inline void write_block(const BlockRows<D>& rows, char* codes, int64_t row_bytes, float* scale_ptr, int a,
                                   int cnt) {
  constexpr int kLanes = BlockRows<D>::kLanes, kRows = BlockRows<D>::kRows, kIters = BlockRows<D>::kIters;
  constexpr bool kNanScale = kIsK && F::kNanScale, kNanCode = kIsK && !F::kNanScale;
  const int lane = threadIdx.x & 63;
  const int i0 = lane / kLanes, e = 8 * (lane % kLanes);
  const float old = a > 0 ? *scale_ptr : 0.f;
  uint32_t amax = 0;
#pragma unroll
  for (int it = 0; it < kIters; ++it)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = abs_bits<T>(rows.x[it][j]);
      amax = max(amax, kNanScale || finite_bits(m) ? m : 0u);
    }
  amax = wave_max_bits(amax);
  float scale = fmaxf(old, scale_for<F>(amax));
  if (kNanScale && (!finite_bits(amax) || old != old)) scale = __uint_as_float(0x7fc00000u);
  const float inv = inv_scale(scale);  // 0 for NaN: codes 0
  if (a > 0 && scale > old) {          // the block's earlier rows to the new scale
    const float shift = old * inv;
#pragma unroll
    for (int it = 0; it < kIters; ++it) {
      const int i = kRows * it + i0;
      if (i < a) {
        u32x2* at = reinterpret_cast<u32x2*>(codes + i * row_bytes + e);
        u32x2 w = *at;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[4];
          F::decode4(w[h], f);
          w[h] = F::encode4(f[0] * shift, f[1] * shift, f[2] * shift, f[3] * shift);
        }
        *at = w;
      }
    }
  }
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int i = kRows * it + i0;
    if (i >= a && i < a + cnt) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = finite_bits(abs_bits<T>(rows.x[it][j])) ? T::to_f32(rows.x[it][j]) * inv
                                                       : (kNanCode ? __uint_as_float(0x7fc00000u) : 0.f);
      const u32x2 w = {F::encode4(f[0], f[1], f[2], f[3]), F::encode4(f[4], f[5], f[6], f[7])};
      *reinterpret_cast<u32x2*>(codes + i * row_bytes + e) = w;
    }
  }
  if (lane == 0) *scale_ptr = scale;
}

// Index of the scale of slot `slot` of page pid at head h.
__device__ inline int64_t scale_index(int64_t pid, int slot, int nb, int num_kv_heads, int h) {
  return (pid * nb + slot / kBlockToks) * num_kv_heads + h;
}

}  // namespace nslg
