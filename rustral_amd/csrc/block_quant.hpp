// block_quant.hpp -- the arithmetic of the 8-bit pools with one scale for each
// (block, KV head) tile (RKV_I8_BLOCK, RKV_FP8_BLOCK): the scale a tile needs,
// a value's byte, and an older byte brought to a larger scale.
//
// Bytes are the exactly rounded quotients x / scale and byte * old / scale
// (nearest, ties to even), so they do not depend on how a quotient was
// approximated: an int8 product with the reciprocal or the ratio is within 2^-15 of the
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

// Whether y may be on the wrong side of the middle between two integers (y is within
// 2^-15 of the quotient it stands for; r = rintf(y)).
__device__ __forceinline__ bool near_middle(float y, float r) { return fabsf(y - r) > 0.4999f; }

// r, the rounding of a quotient's approximation, corrected to that of num / den.
__device__ __forceinline__ float exact_round(float r, double num, double den) {
  const double e = fma(-(double)r, den, num), h = 0.5 * den;
  const bool odd = ((int)r & 1) != 0;
  if (e > h || (e == h && odd)) r += 1.0f;
  if (e < -h || (e == -h && odd)) r -= 1.0f;
  return r;
}

// Four floats of at most 448 in magnitude as e4m3 bytes, round to nearest even:
// v_cvt_pk_fp8_f32, whose bytes are e4m3_from_f32's (checked on the GPU).  A NaN
// loses its sign on the way: its byte is taken from `nan`.
__device__ __forceinline__ uint32_t pack_e4m3x4(const float (&v)[4], uint32_t nan) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
  if (!(v[0] == v[0] && v[1] == v[1] && v[2] == v[2] && v[3] == v[3])) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = 0xffu << (8 * e);
      if (v[e] != v[e]) w = (int)(((uint32_t)w & ~m) | (nan & m));
    }
  }
  return (uint32_t)w;
}

// The bytes of four values under scale s (inv = 1 / s, or 0 for s = 0).
template <int DT>
__device__ __forceinline__ uint32_t tile_word(const float4& x, float s, float inv) {
  const float v[4] = {x.x, x.y, x.z, x.w};
  if constexpr (DT == RKV_I8_BLOCK) {
    float r[4];
    bool near = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = v[e] * inv;  // an infinity: clamped; a NaN (of x, or 0 times an infinity): 0
      r[e] = rintf(y);
      near = near || near_middle(y, r[e]);
      r[e] = y == y ? fminf(fmaxf(r[e], -127.0f), 127.0f) : 0.0f;
    }
    if (near) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (fabsf(v[e]) < INFINITY) r[e] = exact_round(r[e], (double)v[e], (double)s);
    }
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= ((uint32_t)(int)r[e] & 0xffu) << (8 * e);
    return w;
  } else {
    float y[4];
    uint32_t nan = 0x7f7f7f7fu;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      nan |= (__float_as_uint(v[e]) >> 31) << (8 * e + 7);
      const float c = s > 0.0f ? __builtin_amdgcn_fmed3f(v[e] * inv, -448.0f, 448.0f) : 0.0f;
      y[e] = v[e] == v[e] ? c : v[e];
    }
    return pack_e4m3x4(y, nan);
  }
}

// The four bytes of a word of a tile of scale s_old brought to scale s >= s_old,
// s > 0 (ratio = s_old / s).
template <int DT>
__device__ __forceinline__ uint32_t tile_reword(uint32_t w, float s_old, float s, float ratio) {
  if constexpr (DT == RKV_I8_BLOCK) {
    // byte + 128 converts in one instruction, and 128 * ratio comes off in the
    // product's rounding; adding 1.5 * 2^23 leaves the rounded integer in the low byte
    constexpr float kMagic = 12582912.0f;
    const uint32_t u = w ^ 0x80808080u;
    float z[4], far = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = fmaf((float)((u >> (8 * e)) & 0xffu), ratio, -128.0f * ratio);
      z[e] = y + kMagic;
      far = fmaxf(far, fabsf(y - (z[e] - kMagic)));
    }
    if (far > 0.4999f) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        z[e] = kMagic + exact_round(z[e] - kMagic, (double)((int32_t)(w << (24 - 8 * e)) >> 24) *
                                                       (double)s_old, (double)s);
    }
    const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(z[1]), __float_as_uint(z[0]), 0x0c0c0400u);
    const uint32_t c = __builtin_amdgcn_perm(__float_as_uint(z[3]), __float_as_uint(z[2]), 0x04000c0cu);
    return a | c;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    const float v[4] = {lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio};
    return pack_e4m3x4(v, w);
  }
}

}  // namespace rkv
