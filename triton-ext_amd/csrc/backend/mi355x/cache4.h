// e2m1 codes under block scales, as the 4-bit paged cache holds them (tx_cache4.h): values to codes
// and back.
//
// The gfx950 conversions do both: v_cvt_scalef32_pk_{bf16,f16,f32}_fp4 multiply two codes by
// a power of two (the exponent of their fp32 operand: byte << 23 is an e8m0 scale as it
// stands, 0 is 2^-127 and 255 NaN), v_cvt_scalef32_pk_fp4_f32 divides by one, rounds to nearest even and
// saturates at 6.  (Compared on the card with the formats' definitions: all 255 x 16 products in
// the three types, 200000 quotients and the border cases.)  An e4m3 scale has three bits of
// mantissa, so its products are taken after the conversion: 2 + 4 bits, exact in fp16 and bf16.
#pragma once

#include <hip/hip_runtime.h>

#include "tile_common.h"

namespace txk {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

// Two codes (byte SEL of w) times 2^(exponent of scale), as two halves of a dword.
template <bool BF, int SEL> __device__ __forceinline__ uint32_t cvt_e2m1(uint32_t w, float scale) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}

// A block scale as a number (NaN where its byte says so).
template <bool NV> __device__ __forceinline__ float scale4_f32(uint32_t byte) {
  if constexpr (NV)
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
  else
    return byte == 0 ? 0x1p-127f : byte == 255 ? __builtin_nanf("") : __uint_as_float(byte << 23);
}

// ---------------------------------------------------------------------------
// Values to codes
// ---------------------------------------------------------------------------

// The largest magnitude of a block as the bits of its absolute value (NaN above infinity above
// numbers): 8 values a lane, LANES adjacent lanes.
template <int LANES> __device__ __forceinline__ uint32_t block4_max(const float (&y)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(y[i]) & 0x7fffffffu;
    a = b > a ? b : a;
  }
  uint32_t b = __builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, true); // lane ^ 1
  a = b > a ? b : a;
  if constexpr (LANES == 4) {
    b = __builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, true); // lane ^ 2
    a = b > a ? b : a;
  }
  return a;
}

// The scale of a block whose largest magnitude has the bits `a`; lo, hi: the least and the
// largest exponent of MX32.
template <bool NV> __device__ __forceinline__ uint32_t block4_scale(uint32_t a, int lo, int hi) {
  if (a >= 0x7f800000u)
    return NV ? 0x7f : 255;
  if constexpr (NV) {
    float s = __uint_as_float(a) / 6.f;
    s = s < 0x1p-9f ? 0x1p-9f : s > 448.f ? 448.f : s;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s, s, 0, false) & 0xff;
  } else {
    // a = 1.m 2^E: e = E - 2, or E - 1 where 1.m > 1.75, which the sum carries into E
    const int e = (int)((a + 0x1fffffu) >> 23) - 127 - 2;
    return (uint32_t)((e < lo ? lo : e > hi ? hi : e) + 127);
  }
}

// 8 values as codes under that scale.
template <bool NV> __device__ __forceinline__ uint32_t block4_codes(const float (&y)[8], uint32_t scale) {
  if (scale == (NV ? 0x7fu : 255u))
    return 0;
  const float s = scale4_f32<NV>(scale);
  uint32_t w = 0;
  auto two = [&](float a, float b, auto sel) __attribute__((always_inline)) {
    if constexpr (NV)
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a / s, b / s, 1.f, decltype(sel)::value);
    else
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a, b, s, decltype(sel)::value);
  };
  two(y[0], y[1], std::integral_constant<int, 0>());
  two(y[2], y[3], std::integral_constant<int, 1>());
  two(y[4], y[5], std::integral_constant<int, 2>());
  two(y[6], y[7], std::integral_constant<int, 3>());
  return w;
}

// ---------------------------------------------------------------------------
// Codes to values
// ---------------------------------------------------------------------------

// 8 codes in fp32, before any scale but MX32's.
template <bool NV> __device__ __forceinline__ void codes4_f32(uint32_t w, uint32_t scale, float (&y)[8]) {
  const float s = NV ? 1.f : __uint_as_float(scale << 23);
  auto two = [&](auto sel) __attribute__((always_inline)) {
    constexpr int I = decltype(sel)::value;
    const float2_t f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, I);
    y[2 * I] = f[0], y[2 * I + 1] = f[1];
  };
  two(std::integral_constant<int, 0>());
  two(std::integral_constant<int, 1>());
  two(std::integral_constant<int, 2>());
  two(std::integral_constant<int, 3>());
  if constexpr (NV) {
    const float f = scale4_f32<true>(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] *= f;
  }
}

// Codes as operands of the matrix cores in bf16 (BF; MX32 alone) or fp16.
template <bool BF, bool NV> struct Code4 {
  static_assert(!(BF && NV), "e4m3 scales in fp16");
  // Whether values under this scale byte may not be numbers of the type: what tx_cache4.h says
  // makes NaN of a row.
  __device__ __forceinline__ static bool bad(uint32_t byte) {
    return NV ? (byte & 0x7f) == 0x7f : byte > (BF ? 125 + 127 : 13 + 127);
  }
  // The factor of `eight`, as bits; a bad scale makes NaN, or 0 if `zero`.
  __device__ __forceinline__ static uint32_t factor(uint32_t byte, bool zero) {
    if constexpr (NV) {
      const _Float16 f = (_Float16)__builtin_amdgcn_cvt_f32_fp8((int)(zero && bad(byte) ? 0 : byte), 0);
      return __builtin_bit_cast(uint32_t, half2_t{f, f});
    } else {
      return bad(byte) ? zero ? 0 : 255u << 23 : byte << 23;
    }
  }
  // 8 codes times their factor.
  __device__ __forceinline__ static u32x4 eight(uint32_t w, uint32_t factor) {
    u32x4 r;
    const float s = NV ? 1.f : __uint_as_float(factor);
    r[0] = cvt_e2m1<BF, 0>(w, s), r[1] = cvt_e2m1<BF, 1>(w, s);
    r[2] = cvt_e2m1<BF, 2>(w, s), r[3] = cvt_e2m1<BF, 3>(w, s);
    if constexpr (NV) {
      const half2_t f = __builtin_bit_cast(half2_t, factor);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, (uint32_t)r[i]) * f);
    }
    return r;
  }
};

} // namespace txk
