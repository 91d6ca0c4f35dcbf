// Rows held in 4 bits: blocks of 32 numbers share a scale 2^e, kept as the byte
// e + 127; a number is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (codes 0..7, the sign in
// bit 3) times the scale, two codes a byte, the first in the low half.
// gfx950 converts both ways (two numbers an instruction, the scale as a float's
// exponent): to 16 bits exactly, subnormals among them, NaN from the scale byte
// 255; from fp32 to the nearest code, ties to the even one, past 6 to 6.
#pragma once

#include "gdn_common.h"

namespace {

// Block scales of a paged cache: (blocks, heads, D / 32, page) bytes.
struct ScaleSource {
  uint8_t* base;
  int64_t sb, sh, sd;  // byte strides: block, head, 32 dims (the slots of a page lie side by side)
};

ScaleSource scale_source(const gdn_tensor* t) {
  return {reinterpret_cast<uint8_t*>(t->data), t->stride[0], t->stride[1], t->stride[2]};
}

GDN_DEVICE float fp4_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// The two numbers of byte SEL of w.
template <typename T> struct Fp4;
template <> struct Fp4<bf16_t> {
  static constexpr int32_t kTop = 125;          // largest exponent: 6 * 2^kTop and 2^-kTop / 2 are normal numbers
  static constexpr uint32_t kInfinite = 0x7F80;  // magnitudes from here on are not finite
  template <int SEL> static GDN_DEVICE uint32_t pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  }
  static GDN_DEVICE float value(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }
};
template <> struct Fp4<f16_t> {
  static constexpr int32_t kTop = 13;
  static constexpr uint32_t kInfinite = 0x7C00;
  template <int SEL> static GDN_DEVICE uint32_t pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
  }
  static GDN_DEVICE float value(uint32_t bits) { return (float)__builtin_bit_cast(f16_t, (uint16_t)bits); }
};

// The eight numbers of a word, in 16 bits.
template <typename T> GDN_DEVICE uint4 fp4_eight(uint32_t w, float scale) {
  typedef Fp4<T> F;
  return uint4{F::template pair<0>(w, scale), F::template pair<1>(w, scale), F::template pair<2>(w, scale),
               F::template pair<3>(w, scale)};
}

// The scale byte of a block whose largest magnitude has the 16-bit pattern
// `top`: the smallest e with max <= 6 * 2^e, held to the exponents that keep
// every value a normal number of T; 255 where it is not finite.  (With max =
// m 2^k, 1 <= m < 2, e is k - 2 up to m = 1.5, else k - 1: the sum below carries
// into the exponent past m = 1.5.)
template <typename T> GDN_DEVICE uint32_t fp4_scale_byte(uint32_t top) {
  typedef Fp4<T> F;
  const uint32_t bits = __builtin_bit_cast(uint32_t, F::value(top));
  int32_t e = (int32_t)((bits + 0x3FFFFFu) >> 23) - 2;
  e = e < 127 - F::kTop ? 127 - F::kTop : e;
  e = e > 127 + F::kTop ? 127 + F::kTop : e;
  return top >= F::kInfinite ? 255u : (uint32_t)e;
}

// Eight numbers as a word of codes (0 in a block that is not finite).
template <typename T, typename V8> GDN_DEVICE uint32_t fp4_codes(V8 x, uint32_t byte) {
  const float s = fp4_scale(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, (float)x[0], (float)x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, (float)x[2], (float)x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, (float)x[4], (float)x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, (float)x[6], (float)x[7], s, 3);
  return byte == 255u ? 0u : w;
}

// Largest magnitude of eight numbers, as its 16-bit pattern (which grows with it).
template <typename V8> GDN_DEVICE uint32_t top_of_eight(V8 x) {
  const uint4 u = __builtin_bit_cast(uint4, x);
  uint32_t m = 0;
  auto up = [&](uint32_t w) __attribute__((always_inline)) {
    const uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
    m = lo > m ? lo : m;
    m = hi > m ? hi : m;
  };
  up(u.x);
  up(u.y);
  up(u.z);
  up(u.w);
  return m;
}

}  // namespace
