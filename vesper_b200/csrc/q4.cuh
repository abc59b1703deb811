// The 4-bit ring cache's format, shared by its write, read and attention kernels.
//
// Per (row, key head, slot) a key and a value of DK channels, DK a multiple of 16 up to 128, in
// groups of GS channels (32 where DK is a multiple of 32, else 16). A group keeps two bf16 numbers
// and a code of four bits per channel:
//   lo   = min rounded towards -inf to bf16,
//   step = (max - lo) / 15 rounded towards +inf to bf16,
//   code = rint((x - lo) / step), at most 15;   the value it stands for is lo + code * step.
// Because lo is rounded down and step up, [lo, lo + 15 step] covers the group and every value is at
// most step / 2 off, however large the group's common offset is. A group whose range is below
// 2^-100 has step 0 and codes 0 (all channels lo); one whose range is not finite has lo and step
// NaN and reads back as NaN. code * step has 12 significant bits, so lo + code * step is the same
// in one rounding or two.
//
// Buffers: codes [B, HKV, SLOTS, DK / 2] bytes, params [B, HKV, SLOTS, DK / GS] 32-bit words (step
// in the low half, lo in the high half), pos [B, SLOTS] int64 (-1: nothing written). SLOTS is the
// window rounded up to a multiple of 64; a token at position p lives in slot p % window. Channels are
// stored in the order in which the attention's matrix instructions hand them to lanes, two codes a
// byte, the first in the low half:
//   keys:   channel g GS + t GS/4 + i  at place  t DK/4 + g GS/4 + i   (t < 4: a lane's part of every group)
//   values: channel 16 i + 2 g + r     at place  g DK/8 + 2 i + r      (g < 8: a lane's part of every 16)
#pragma once
#include "common.cuh"

namespace vb {

constexpr int Q4_TILE = 64;  // slots are allocated and walked in tiles of 64
constexpr float Q4_FLAT = 7.888609052210118e-31f;  // 2^-100

__host__ __device__ constexpr int q4_group(int dk) { return dk % 32 == 0 ? 32 : 16; }
__host__ __device__ constexpr int q4_groups(int dk) { return dk / q4_group(dk); }

__device__ __forceinline__ int q4_key_place(int dk, int c) {
  const int gs = q4_group(dk), g = c / gs, rem = c - g * gs, t = rem / (gs / 4);
  return t * (dk / 4) + g * (gs / 4) + rem % (gs / 4);
}
__device__ __forceinline__ int q4_value_place(int dk, int c) {
  return ((c & 15) >> 1) * (dk / 8) + 2 * (c >> 4) + (c & 1);
}

// the smaller and the larger of two numbers, NaN if either is
__device__ __forceinline__ float min_nan(float x, float y) {
  float z;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
__device__ __forceinline__ float max_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// A group's step and lo (float values of bf16 numbers) and the correctly rounded reciprocal of step (0 for step 0) from
// its extremes. Quotients by Markstein's steps (IBM J. Res. Dev. 34, 1990): with r the rounded reciprocal of d, q = n r
// and one residual step q + (n - q d) r give the rounded n / d; and one step r + (1 - r d) r from an r within a unit in
// the last place gives the rounded reciprocal, d not having all its bits set. No operand here leaves the
// range in which the residuals are exact: spans lie between 2^-100 and 2^128.
__device__ __forceinline__ void q4_params(float low, float high, float& step, float& lo, float& inverse) {
  // bf16 is float32's upper half: with its lower half added up or cut off, the next number away from or towards zero
  const uint32_t bits = __float_as_uint(low);
  lo = __uint_as_float((bits + ((uint32_t)((int32_t)bits >> 31) & 0xffffu)) & 0xffff0000u);
  const float span = high - lo;
  constexpr float FIFTEENTH = 1.0f / 15.0f;
  const float q = __fmul_rn(span, FIFTEENTH);
  const float exact = __fmaf_rn(__fmaf_rn(-q, 15.0f, span), FIFTEENTH, q);
  step = span < Q4_FLAT ? 0.f : __uint_as_float((__float_as_uint(exact) + 0xffffu) & 0xffff0000u);
  if (!(fabsf(lo) < INFINITY && span < INFINITY)) lo = step = __uint_as_float(0x7fc00000u);  // also for a NaN
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(step));
  inverse = step > 0.f ? __fmaf_rn(__fmaf_rn(-step, r, 1.0f), r, r) : 0.f;
}
__device__ __forceinline__ uint32_t q4_pack_params(float step, float lo) {
  return (__float_as_uint(step) >> 16) | (__float_as_uint(lo) & 0xffff0000u);
}
__device__ __forceinline__ float q4_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float q4_lo(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// two floats side by side: Blackwell's packed float32 arithmetic, each half rounded for itself
__device__ __forceinline__ uint64_t pair_f32(float x, float y) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t z;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(x), "l"(y));
  return z;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t z;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(x), "l"(y));
  return z;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t w) {
  uint64_t z;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(z) : "l"(x), "l"(y), "l"(w));
  return z;
}

// The codes of eight channels, the first in the low four bits: rint of the correctly rounded quotient
// (x - lo) / step, which is at most 15 (step is not below span / 15). Adding 1.5 * 2^23 rounds to whole numbers, which
// then lie in the lowest bits of the float. Step 0 or NaN gives zeros.
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[8], float step, float lo, float inverse) {
  const uint64_t minus_lo = pair_f32(-lo, -lo), minus_step = pair_f32(-step, -step), r = pair_f32(inverse, inverse);
  const uint64_t whole = pair_f32(12582912.0f, 12582912.0f);
  uint32_t w0 = 0, w1 = 0;  // codes 0 to 3 and 4 to 7, in the low halves
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    const uint64_t t = add2(pair_f32(x[e], x[e + 4]), minus_lo);
    const uint64_t q = mul2(t, r);
    const uint64_t c = add2(fma2(fma2(q, minus_step, t), r, q), whole);
    uint32_t c0, c1;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(c0), "=r"(c1) : "l"(c));
    w0 = w0 * 16 + c0;
    w1 = w1 * 16 + c1;
  }
  return step > 0.f ? __byte_perm(w0, w1, 0x5410) : 0u;
}

// the values lo + code step of eight codes
__device__ __forceinline__ void q4_values(uint32_t w, float step, float lo, float (&x)[8]) {
  const uint64_t steps = pair_f32(step, step), los = pair_f32(lo, lo), back = pair_f32(-8388608.f, -8388608.f);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {  // 2^23 + code, less 2^23
    const uint64_t c = add2(pair_f32(__uint_as_float(((w >> (4 * e)) & 15u) | 0x4b000000u),
                                     __uint_as_float(((w >> (4 * e + 4)) & 15u) | 0x4b000000u)), back);
    const uint64_t y = fma2(c, steps, los);
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x[e]), "=f"(x[e + 1]) : "l"(y));
  }
}

}  // namespace vb
