// The 8-bit form of a cached row: per (row, head) 128 codes in e4m3 and one fp32 scale,
//   scale = 2^e, e the least integer >= -60 with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3 number),
//   value = code * scale.
// A power of two costs no precision (e4m3 is a floating format: the relative step does not depend on the scale) and keeps the
// scaling exact: x / scale, ties included, and code * scale (four significant bits: a bf16 number).  A head of a row that holds
// a NaN or an infinity gets codes of zero and a NaN for its scale, so that it reads as NaN while no code ever is one: in a
// matrix product a key whose weight is zero then adds nothing, whatever its row holds.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace dyllm {

constexpr int kFp8MinExp = -60;       // floor of the scales: rows below 448 * 2^-60 share it (and keep value = 0 finite)

#ifdef __CUDACC__

// Two floats to two codes (the first in the low byte), to nearest even, saturating.
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two floats to two codes in e5m2.
__device__ __forceinline__ uint32_t fp8_pack2_e5m2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// The two codes in the low 16 bits as two half-precision numbers (exact).
__device__ __forceinline__ uint32_t fp8_to_half2(uint32_t codes) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(static_cast<uint16_t>(codes)));
  return d;
}
__device__ __forceinline__ float2 fp8_to_float2(uint32_t codes) {
  const uint32_t h = fp8_to_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Bits of the scale of a head whose largest magnitude has the bits `amax` (sign bit clear; NaN and infinity compare as larger
// than every number).  Adding 0x1fffff carries into the exponent exactly when the fraction is above 0.75.
__device__ __forceinline__ uint32_t fp8_scale_bits(uint32_t amax) {
  if (amax >= 0x7f800000u)
    return 0x7fc00000u;
  const int e = static_cast<int>((amax + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(e < 127 + kFp8MinExp ? 127 + kFp8MinExp : e) << 23;
}
// 1 / scale (exact), 0 for a NaN: finite inputs of such a head become codes of zero.
__device__ __forceinline__ float fp8_inverse(uint32_t scale_bits) {
  return scale_bits >= 0x7f800000u ? 0.f : __uint_as_float((254u << 23) - scale_bits);
}

// Largest magnitude of the eight threads that share a head, as bits.
__device__ __forceinline__ uint32_t fp8_amax8(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 4));
}

// Sixteen values of a thread to codes: x[0..7] and x[8..15] are eight neighbours each.  Returns the scale's bits.
__device__ __forceinline__ uint32_t fp8_quantise16(const float (&x)[16], uint2& lo, uint2& hi) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
  const uint32_t scale = fp8_scale_bits(fp8_amax8(m));
  const float inv = fp8_inverse(scale);
  if (scale >= 0x7f800000u) {       // infinity * 0 would be a NaN code
    lo = hi = make_uint2(0u, 0u);
    return scale;
  }
  lo.x = fp8_pack2(x[0] * inv, x[1] * inv) | fp8_pack2(x[2] * inv, x[3] * inv) << 16;
  lo.y = fp8_pack2(x[4] * inv, x[5] * inv) | fp8_pack2(x[6] * inv, x[7] * inv) << 16;
  hi.x = fp8_pack2(x[8] * inv, x[9] * inv) | fp8_pack2(x[10] * inv, x[11] * inv) << 16;
  hi.y = fp8_pack2(x[12] * inv, x[13] * inv) | fp8_pack2(x[14] * inv, x[15] * inv) << 16;
  return scale;
}

__device__ __forceinline__ void bf16x8_to_float(const uint4& v, float* x) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(p[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}
// Bits of the largest magnitude of eight bf16 numbers, as those of a float.
__device__ __forceinline__ uint32_t bf16x8_amax(const uint4& v) {
  const uint32_t w[4] = {v.x & 0x7fff7fffu, v.y & 0x7fff7fffu, v.z & 0x7fff7fffu, v.w & 0x7fff7fffu};
  const uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
  return max(m >> 16, m & 0xffffu) << 16;
}
__device__ __forceinline__ uint4 float_to_bf16x8(const float* x) {
  uint4 v;
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    p[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
  return v;
}
// Eight codes times the scale.
__device__ __forceinline__ void fp8x8_to_float(uint2 c, float scale, float* x) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 a = fp8_to_float2(w[j] & 0xffffu), b = fp8_to_float2(w[j] >> 16);
    x[4 * j] = a.x * scale;
    x[4 * j + 1] = a.y * scale;
    x[4 * j + 2] = b.x * scale;
    x[4 * j + 3] = b.y * scale;
  }
}

#endif  // __CUDACC__

}  // namespace dyllm
