// Vectors of V neighbouring channels: their values and their 8-bit codes (mx8.h).
#pragma once
#include "mx8.h"

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 type; };
template <> struct RawOf<8> { typedef uint2 type; };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<2> { typedef uint16_t type; };
template <> struct RawOf<1> { typedef uint8_t type; };

template <class T, int V> struct Vec {
  typedef typename RawOf<V * (int)sizeof(T)>::type raw;
  struct alignas(sizeof(raw)) arr { T v[V]; };
  // by 32-bit words: taken apart into 16-bit values, rows held over a loop cost twice the registers
  static PG_DEVICE void unpack(const raw &r, float (&f)[V]) {
    if constexpr (sizeof(T) == 2 && V >= 2) {
      struct alignas(sizeof(raw)) Words { uint32_t w[V / 2]; };
      const Words a = __builtin_bit_cast(Words, r);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        if constexpr (__is_same(T, bf16_t)) {
          f[2 * j] = __uint_as_float(a.w[j] << 16);
          f[2 * j + 1] = __uint_as_float(a.w[j] & 0xffff0000u);
        } else {
          f[2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)a.w[j]);
          f[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a.w[j] >> 16));
        }
      }
    } else {
      const arr a = __builtin_bit_cast(arr, r);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = tof(a.v[j]);
    }
  }
  static PG_DEVICE raw pack(const float (&f)[V]) {
    if constexpr (sizeof(T) == 2 && V >= 2 && __is_same(T, bf16_t)) {
      struct alignas(sizeof(raw)) { uint32_t w[V / 2]; } a;
#pragma unroll
      for (int j = 0; j < V / 2; ++j) a.w[j] = pack2(f[2 * j], f[2 * j + 1]);
      return __builtin_bit_cast(raw, a);
    } else {
      arr a;
#pragma unroll
      for (int j = 0; j < V; ++j) a.v[j] = fromf<T>(f[j]);
      return __builtin_bit_cast(raw, a);
    }
  }
};

// V codes
template <int V> struct Codes {
  typedef typename RawOf<V>::type raw;
  static PG_DEVICE raw encode(const float (&f)[V], float inv) {
    if constexpr (V == 8)
      return make_uint2(mx8_enc4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                        mx8_enc4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
    else if constexpr (V == 4) return mx8_enc4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    else if constexpr (V == 2) return (uint16_t)mx8_enc2<false>(f[0] * inv, f[1] * inv, 0);
    else return mx8_enc1(f[0] * inv);
  }
  static PG_DEVICE void decode(const raw &r, float sc, float (&f)[V]) {
    if constexpr (V == 8) {
      mx8_dec4(r.x, sc, f[0], f[1], f[2], f[3]);
      mx8_dec4(r.y, sc, f[4], f[5], f[6], f[7]);
    } else if constexpr (V == 4) mx8_dec4(r, sc, f[0], f[1], f[2], f[3]);
    else if constexpr (V == 2) mx8_dec2<false>(r, sc, f[0], f[1]);
    else f[0] = mx8_dec1(r) * sc;
  }
};

// The largest finite magnitude of a 32-channel block, whose 32 / V neighbouring lanes (aligned) hold V
// channels each; lanes without `on` count as zeros.  Magnitudes are compared as whole numbers, two
// 16-bit ones an instruction; non-finite ones, the largest of all, take the long way.
template <class T, int V> PG_DEVICE float block_amax(const typename Vec<T, V>::raw &raw, bool on) {
  uint32_t m = 0;   // bits of the largest magnitude
  constexpr uint32_t inf = sizeof(T) == 4 || __is_same(T, bf16_t) ? 0x7f800000u : 0x7c000000u;   // 16-bit: in the high half
  if constexpr (sizeof(T) == 2 && V >= 2) {
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    struct alignas(sizeof(raw)) Words { uint32_t w[V / 2]; };
    const Words a = __builtin_bit_cast(Words, raw);
    u16x2_t x = __builtin_bit_cast(u16x2_t, a.w[0] & 0x7fff7fffu);
#pragma unroll
    for (int j = 1; j < V / 2; ++j) x = __builtin_elementwise_max(x, __builtin_bit_cast(u16x2_t, a.w[j] & 0x7fff7fffu));
    m = (uint32_t)(x.x > x.y ? x.x : x.y) << 16;
  } else if constexpr (sizeof(T) == 2) {
    m = ((uint32_t)__builtin_bit_cast(uint16_t, raw) & 0x7fffu) << 16;
  } else {
    struct alignas(sizeof(raw)) Words { uint32_t w[V]; };
    const Words a = __builtin_bit_cast(Words, raw);
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, a.w[j] & 0x7fffffffu);
  }
  if (__ballot(m >= inf)) {   // one branch for the wave
    m = 0;
    float f[V];
    Vec<T, V>::unpack(raw, f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const T t = fromf<T>(mx8_mag(f[j]));
      if constexpr (sizeof(T) == 4) m = max(m, __builtin_bit_cast(uint32_t, t));
      else m = max(m, (uint32_t)__builtin_bit_cast(uint16_t, t) << 16);
    }
  }
  m = on ? m : 0;
  // neighbours 1 and 2 apart within a quad, then further
  if constexpr (kMxBlock / V > 1) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp((int)m, (int)m, 0xB1, 0xf, 0xf, false));
  if constexpr (kMxBlock / V > 2) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp((int)m, (int)m, 0x4E, 0xf, 0xf, false));
#pragma unroll
  for (int o = 4; o < kMxBlock / V; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  if constexpr (sizeof(T) == 4 || __is_same(T, bf16_t)) return __uint_as_float(m);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(m >> 16));
}
