// The 8-bit cache: codes with one power-of-two scale for each block of 16 tokens and kv head, K and V apart.
//   value = code * s,  s = 2^k,  -24 <= k <= 10
// The codes are int8 (-127 .. 127) or e4m3. A power of two makes every scaling exact: a value is rounded once, when its code
// is made, a code times its scale is an fp16 number (which a matrix instruction takes as it is), and a block whose scale
// grows divides its int8 codes by a power of two (at most one step of the new scale off in all, however often) and moves its
// e4m3 codes' exponents (exact down to the subnormals). It costs int8 half a bit on average against a scale of amax / 127.
#pragma once
#include "attn_common.hpp"
#include "launch.hpp"

namespace dk {

constexpr float kKv8MaxScale = 1024.f;  // 2^10: 65504 / 127 fits below it

template <int CACHE>
struct Kv8Codes;
template <>
struct Kv8Codes<kCacheInt8> {
  static constexpr float most = 127.f;
  static constexpr int most_exp = 6, most_mant = 0x7E0000;  // 127 = 1.984375 * 2^6
  // from this scale on the largest code is one whose value fits fp16: 63 * 1024
  static constexpr float top_scale = 1024.f, top_code = 63.f;
};
template <>
struct Kv8Codes<kCacheE4m3> {
  static constexpr float most = 448.f;
  static constexpr int most_exp = 8, most_mant = 0x600000;  // 448 = 1.75 * 2^8
  static constexpr float top_scale = 256.f, top_code = 240.f;  // 240 * 256 = 120 * 512 = 60 * 1024
};

// The scale of a block whose largest finite |x| is `top` (a non-negative fp16 value): 2^k with the smallest k >= -24 such
// that top <= most * 2^k.
template <int CACHE>
__device__ __forceinline__ float kv8_scale(float top) {
  const uint32_t b = __float_as_uint(top);
  const int k = (int)(b >> 23) - 127 - Kv8Codes<CACHE>::most_exp + ((int)(b & 0x7FFFFF) > Kv8Codes<CACHE>::most_mant ? 1 : 0);
  return __uint_as_float((uint32_t)(max(k, -24) + 127) << 23);
}

// Codes of four values y = x / s, in the bytes of a word, to nearest with ties to even; `big`: the largest code at this
// scale. NaN stays NaN in e4m3 and becomes 0 in int8, which has none.
template <int CACHE>
__device__ __forceinline__ uint32_t kv8_encode4(const float (&y)[4], float big) {
  float c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = fminf(fmaxf(y[i], -big), big);
    c[i] = y[i] != y[i] ? (CACHE == kCacheInt8 ? 0.f : y[i]) : c[i];
  }
  if constexpr (CACHE == kCacheInt8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)((int)rintf(c[i]) & 0xFF) << (8 * i);
    return w;
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
  }
}

// The values of four codes in fp16. A product that passes fp16 (codes that this library did not write) is infinite.
template <int CACHE>
__device__ __forceinline__ u32x2 kv8_decode4(uint32_t w, float s) {
  if constexpr (CACHE == kCacheInt8) {
    const f16 sh = (f16)s;
    const f16x2 sc = {sh, sh}, bias = {(f16)-1152.f, (f16)-1152.f};
    const uint32_t u = w ^ 0x80808080u;  // code + 128; as the low byte of 0x6400 it is 1024 + code + 128
    return u32x2{as_u32((as_f16x2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias) * sc),
                 as_u32((as_f16x2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias) * sc)};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true))};
  }
}
template <int CACHE>
__device__ __forceinline__ u32x4 kv8_decode8(u32x2 w, float s) {
  const u32x2 lo = kv8_decode4<CACHE>(w[0], s), hi = kv8_decode4<CACHE>(w[1], s);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// The scale of a block that had `had` (0: no rows ahead of the new ones) and whose new rows need `need`: the larger one. (A
// scale that this library did not write is not taken further than its own go.)
__device__ __forceinline__ float kv8_grown(float had, float need) { return had > need && had <= kKv8MaxScale ? had : need; }
template <int CACHE>
__device__ __forceinline__ float kv8_big(float s, float inv) {  // the largest code at scale s (inv = 1 / s)
  return s < Kv8Codes<CACHE>::top_scale ? Kv8Codes<CACHE>::most : Kv8Codes<CACHE>::top_code * Kv8Codes<CACHE>::top_scale * inv;
}
// The larger of `top` and the magnitudes of two fp16 values, as fp16 bits (an infinity counts as the largest fp16 value, as
// which it is stored, NaN for nothing).
__device__ __forceinline__ uint32_t kv8_top(uint32_t w, uint32_t top) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t m = (w >> (16 * e)) & 0x7FFFu;
    m = m == 0x7C00u ? 0x7BFFu : m;
    top = max(top, m < 0x7C00u ? m : 0u);
  }
  return top;
}
// Codes of four fp16 values times `by`.
template <int CACHE>
__device__ __forceinline__ uint32_t kv8_code4(uint32_t lo, uint32_t hi, float by, float big) {
  const f16x2 a = as_f16x2(lo), b = as_f16x2(hi);
  const float y[4] = {(float)a[0] * by, (float)a[1] * by, (float)b[0] * by, (float)b[1] * by};
  return kv8_encode4<CACHE>(y, big);
}
// Codes at another scale, `ratio` the old one over the new.
template <int CACHE>
__device__ __forceinline__ uint32_t kv8_recode4(uint32_t w, float ratio, float big) {
  const u32x2 x = kv8_decode4<CACHE>(w, 1.0f);  // (times 1: the codes themselves)
  return kv8_code4<CACHE>(x[0], x[1], ratio, big);
}

}  // namespace dk
