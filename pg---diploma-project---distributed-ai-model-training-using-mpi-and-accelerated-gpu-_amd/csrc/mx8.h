// 8-bit activation checkpoints: e4m3 codes [M][C] and one power-of-two scale for every 32
// channels of a row, held as its biased exponent [M][ceil(C/32)].
//
// Scale: the least e with amax <= 448 * 2^e (448 = e4m3's largest), so no finite value saturates;
// a power of two, so x * 2^-e and code * 2^e are exact, the only rounding is e4m3's own (half a
// step is 2^-4 of a normal value), and a decoded value (4 significant bits) is exact in bf16.
// e stays within [-117, 120]: the smallest code, 2^-9, then decodes to a normal fp32 / bf16 number.
// amax is taken over the finite values; NaN and infinities are kept as NaN (e4m3 has no infinity).
#pragma once
#include "common.h"

#include <cmath>

constexpr int kMxBlock = 32;

PG_DEVICE float tof(bf16_t v) { return bf2f(v); }
PG_DEVICE float tof(_Float16 v) { return (float)v; }
PG_DEVICE float tof(float v) { return v; }
template <class T> PG_DEVICE T fromf(float v);
template <> PG_DEVICE bf16_t fromf<bf16_t>(float v) { return f2bf(v); }
template <> PG_DEVICE _Float16 fromf<_Float16>(float v) { return (_Float16)v; }
template <> PG_DEVICE float fromf<float>(float v) { return v; }

PG_DEVICE bool mx8_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
// |v|, or 0 for NaN and infinities
PG_DEVICE float mx8_mag(float v) { return mx8_finite(v) ? fabsf(v) : 0.f; }

// biased exponent (e + 127) of a block's scale; 448 = 1.75 * 2^8
PG_DEVICE int mx8_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, 10), 247);
}
PG_DEVICE float mx8_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }            // 2^e
PG_DEVICE float mx8_inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // 2^-e

// two values (already times 2^-e: 448 at most, or not finite) -> two codes in the low or high half of
// w; the conversion gives NaN for infinities
template <bool HI> PG_DEVICE int mx8_enc2(float a, float b, int w) { return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, HI); }
PG_DEVICE uint32_t mx8_enc4(float a, float b, float c, float d) {
  return (uint32_t)mx8_enc2<true>(c, d, mx8_enc2<false>(a, b, 0));
}
PG_DEVICE uint8_t mx8_enc1(float a) { return (uint8_t)(mx8_enc2<false>(a, 0.f, 0) & 0xff); }
typedef float f32x2_t __attribute__((ext_vector_type(2)));
// codes of the low or high half of w -> values (code times sc)
template <bool HI> PG_DEVICE void mx8_dec2(uint32_t w, float sc, float &a, float &b) {
  const f32x2_t v = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, HI);
  a = v.x * sc;
  b = v.y * sc;
}
PG_DEVICE void mx8_dec4(uint32_t w, float sc, float &a, float &b, float &c, float &d) {
  mx8_dec2<false>(w, sc, a, b);
  mx8_dec2<true>(w, sc, c, d);
}
PG_DEVICE float mx8_dec1(uint8_t q) { return __builtin_amdgcn_cvt_f32_fp8((int)q, 0); }
