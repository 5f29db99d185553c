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

