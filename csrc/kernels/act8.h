// Activations in 8 bits: OCP e4m3 codes [M, N] and one power-of-two scale per row and 32 columns
// [M, ceil(N / 32)], stored as the biased exponent e + 127 (the scale's fp32 exponent byte).
#pragma once
#include "common.h"

constexpr int A8_BLOCK = 32;         // columns per scale
constexpr int A8_EMIN = -110, A8_EMAX = 120;

__device__ __forceinline__ float a8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Smallest e with amax <= 448 * 2^e: amax = m 2^x, m in [1, 2), 448 = 1.75 * 2^8.  (Zero and
// subnormal amax have x = -127 and end at A8_EMIN.)
__device__ __forceinline__ int a8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < A8_EMIN ? A8_EMIN : (e > A8_EMAX ? A8_EMAX : e);
}

// 4 values -> 4 codes.  `inv` = 2^-e.  A nonzero value that would round to zero takes the smallest
// code of its sign: the backward pass reads the relu / dropout mask from the codes, so which
// values are zero must not change.  Non-finite values become NaN.
__device__ __forceinline__ uint32_t a8_pack4(float a, float b, float c, float d, float inv) {
  const float v[4] = {a, b, c, d};
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = fabsf(v[i]) < INFINITY ? v[i] * inv : 0.f;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  uint32_t r = (uint32_t)w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t code = (r >> (8 * i)) & 0x7Fu;
    if (!(fabsf(v[i]) < INFINITY)) r |= 0x7Fu << (8 * i);
    else if (code == 0u && v[i] != 0.f) r |= ((v[i] < 0.f ? 0x81u : 0x01u) << (8 * i));
  }
  return r;
}

// 8 codes (two words) -> 8 fp32 values times the scale (exact: 4 significant bits)
__device__ __forceinline__ void a8_unpack8(uint2 w, float s, float (&f)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 p0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
  const f32x2 p2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), p3 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
  f[0] = p0[0] * s; f[1] = p0[1] * s; f[2] = p1[0] * s; f[3] = p1[1] * s;
  f[4] = p2[0] * s; f[5] = p2[1] * s; f[6] = p3[0] * s; f[7] = p3[1] * s;
}

// 2 codes (the low or high half of a word) -> 2 bf16 values times the scale, exact: one conversion
template <bool HI>
__device__ __forceinline__ uint32_t a8_pair_bf16(uint32_t w, float s) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI);
  return __builtin_bit_cast(uint32_t, v);
}

// whether a code stands for a value above zero (0x7F is NaN)
__device__ __forceinline__ bool a8_positive(uint32_t code) { return code - 1u < 0x7Eu; }
