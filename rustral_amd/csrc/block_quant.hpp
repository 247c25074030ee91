// block_quant.hpp -- the arithmetic of the 8-bit pools with one scale for each
// (block, KV head) tile (RKV_I8_BLOCK, RKV_FP8_BLOCK): the scale a tile needs,
// a value's byte, and an older byte brought to a larger scale.
//
// Bytes are the exactly rounded quotients x / scale and byte * old / scale
// (nearest, ties to even), so they do not depend on how a quotient was
// approximated: an int8 product with the reciprocal is within 2^-15 of the
// quotient (|quotient| <= 127, three roundings of 2^-24), and where it falls
// that near to the middle between two integers the remainder is formed in 64
// bits, exactly (24 and 31 bit factors), and decides.
#pragma once

#include "common.hpp"

namespace rkv {

inline bool block_scaled(int dtype) { return dtype == RKV_I8_BLOCK || dtype == RKV_FP8_BLOCK; }

constexpr float kTinyTile = 0x1p-110f;  // a smaller maximum: scale 0, zeros

// |x| where it is finite, else 0 (an infinity or NaN sets no scale).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

// The scale of a tile whose largest finite magnitude is amax.
template <int DT>
__device__ __forceinline__ float tile_scale(float amax) {
  if (amax < kTinyTile) return 0.0f;
  if constexpr (DT == RKV_I8_BLOCK) {
    return amax * (1.0f / 127.0f);
  } else {
    // amax = m 2^e, 1 <= m < 2, and 448 = 1.75 2^8: 2^(e-8) for m <= 1.75,
    // else 2^(e-7)
    const uint32_t u = __float_as_uint(amax);
    const uint32_t e = (u >> 23) - 8u + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
    return __uint_as_float(e << 23);
  }
}

// r, the rounding of y, corrected to that of the exact num / den (y is within
// 2^-15 of it).
__device__ __forceinline__ float exact_round(float y, double num, double den) {
  float r = fminf(fmaxf(rintf(y), -127.0f), 127.0f);
  if (fabsf(fabsf(y - r) - 0.5f) < 1e-4f) {
    const double e = fma(-(double)r, den, num), h = 0.5 * den;
    const bool odd = ((int)r & 1) != 0;
    if (e > h || (e == h && odd)) r += 1.0f;
    if (e < -h || (e == -h && odd)) r -= 1.0f;
    r = fminf(fmaxf(r, -127.0f), 127.0f);
  }
  return r;
}

// Byte of x under scale s (inv = 1 / s, or 0 for s = 0).
template <int DT>
__device__ __forceinline__ uint32_t tile_byte(float x, float s, float inv) {
  if constexpr (DT == RKV_I8_BLOCK) {
    if (!(x == x) || s == 0.0f) return 0u;
    return (uint32_t)(int)exact_round(x * inv, (double)x, (double)s) & 0xffu;
  } else {
    if (x == x && s == 0.0f) return 0u;
    return e4m3_from_f32(x * inv);
  }
}

// Byte b of a tile of scale s_old under scale s >= s_old (ratio = s_old / s).
template <int DT>
__device__ __forceinline__ uint32_t tile_rebyte(uint32_t b, float s_old, float s, float ratio) {
  if constexpr (DT == RKV_I8_BLOCK) {
    const float v = (float)(int8_t)b;
    if (s == 0.0f) return 0u;
    return (uint32_t)(int)exact_round(v * ratio, (double)v * (double)s_old, (double)s) & 0xffu;
  } else {
    return e4m3_from_f32(f32_from_e4m3((uint8_t)b) * ratio);
  }
}

// The four bytes of a word so treated.
template <int DT>
__device__ __forceinline__ uint32_t tile_reword(uint32_t w, float s_old, float s, float ratio) {
  uint32_t o = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o |= tile_rebyte<DT>((w >> (8 * e)) & 0xffu, s_old, s, ratio) << (8 * e);
  return o;
}

}  // namespace rkv
