// Activations in 8 bits: OCP e4m3 codes [M, N] and one power-of-two scale per row and 32 columns
// [M, ceil(N / 32)], stored as the biased exponent e + 127 (the scale's fp32 exponent byte).
//
// At the largest scale 2^120 magnitudes from 248 * 2^120 on have the code of 256, and 2^128 is past fp32 and
// bf16: that code reads as 240 there, the largest finite value of the format (at most 2^-4 off, half an e4m3 step).
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

// 4 codes with those of +-256 made 240 where their scale's byte is the largest: a byte of m is 0 for the code
// 0x78 of either sign, and only then (m + 0x7F) has no bit 7, without a carry to the next byte.
__device__ __forceinline__ uint32_t a8_finite(uint32_t w, uint32_t scale) {
  const uint32_t m = (w & 0x7F7F7F7Fu) ^ 0x78787878u;
  return w - ((~(m + 0x7F7F7F7Fu) >> 7) & (scale == A8_EMAX + 127 ? 0x01010101u : 0u));
}

// The same for 8 words of one scale (the scale itself, not its byte), with a wave's branch over it (no lane has that scale but for values next to the
// type's largest) that the compiler does not see, for loops whose registers do not survive a block (16384 x 4096 x 4096: 4 us
// of 450; by a8_finite it would be 56 instructions more in every step).
__device__ __forceinline__ void a8_finite_rare(uint32_t (&w)[8], float scale) {
  uint32_t t, one;
#define HFM_A8_WORD(i)                                                                                   \
  "v_and_b32 %8, 0x7f7f7f7f, %" #i "\n\tv_xor_b32 %8, 0x78787878, %8\n\tv_add_u32 %8, 0x7f7f7f7f, %8\n\t" \
  "v_not_b32 %8, %8\n\tv_lshrrev_b32 %8, 7, %8\n\tv_and_b32 %8, %9, %8\n\tv_sub_u32 %" #i ", %" #i ", %8\n\t"
  asm volatile(
      "v_cmp_eq_u32 vcc, %11, %10\n\ts_nop 4\n\ts_cmp_lg_u64 vcc, 0\n\ts_cbranch_scc0 .Lskip%=\n\t"
      "v_mov_b32 %9, 0x01010101\n\tv_cndmask_b32 %9, 0, %9, vcc\n\t"
      HFM_A8_WORD(0) HFM_A8_WORD(1) HFM_A8_WORD(2) HFM_A8_WORD(3)
      HFM_A8_WORD(4) HFM_A8_WORD(5) HFM_A8_WORD(6) HFM_A8_WORD(7)
      "s_nop 1\n.Lskip%=:"
      : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]), "+v"(w[4]), "+v"(w[5]), "+v"(w[6]), "+v"(w[7]), "=&v"(t), "=&v"(one)
      : "v"(scale), "s"((A8_EMAX + 127) << 23)
      : "vcc", "scc");
#undef HFM_A8_WORD
}

// 8 codes (two words) -> 8 fp32 values times their scale (its byte; exact: 4 significant bits)
__device__ __forceinline__ void a8_unpack8(uint2 w, uint32_t scale, float (&f)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float s = a8_scale(scale);
  w = make_uint2(a8_finite(w.x, scale), a8_finite(w.y, scale));
  const f32x2 p0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
  const f32x2 p2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), p3 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
  f[0] = p0[0] * s; f[1] = p0[1] * s; f[2] = p1[0] * s; f[3] = p1[1] * s;
  f[4] = p2[0] * s; f[5] = p2[1] * s; f[6] = p3[0] * s; f[7] = p3[1] * s;
}

// 2 codes (the low or high half of a word, after a8_finite) -> 2 bf16 values times the scale, exact: one conversion
template <bool HI>
__device__ __forceinline__ uint32_t a8_pair_bf16(uint32_t w, float s) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI);
  return __builtin_bit_cast(uint32_t, v);
}

// whether a code stands for a value above zero (0x7F is NaN)
__device__ __forceinline__ bool a8_positive(uint32_t code) { return code - 1u < 0x7Eu; }
