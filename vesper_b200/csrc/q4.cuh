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

// a group's step and lo (float values of bf16 numbers) from its extremes
__device__ __forceinline__ void q4_params(float low, float high, float& step, float& lo) {
  lo = __bfloat162float(__float2bfloat16_rd(low));
  const float span = high - lo;
  step = span < Q4_FLAT ? 0.f : __bfloat162float(__float2bfloat16_ru(span / 15.0f));
  const bool fine = fabsf(lo) <= 3.4e38f && step <= 3.4e38f;  // false for NaN
  if (!fine) lo = step = __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t q4_pack_params(float step, float lo) {
  return (__float_as_uint(step) >> 16) | (__float_as_uint(lo) & 0xffff0000u);
}
__device__ __forceinline__ float q4_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float q4_lo(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// the code of x: rint of the correctly rounded quotient (x - lo) / step. With r = 1 / step rounded,
// q = t r and one residual step q + (t - q step) r is the rounded quotient (Markstein, IBM J. Res.
// Dev. 34, 1990); step 0 or NaN gives code 0
__device__ __forceinline__ uint32_t q4_code(float x, float step, float lo, float inverse) {
  const float t = __fsub_rn(x, lo);
  const float q = __fmul_rn(t, inverse);
  const float quotient = __fmaf_rn(__fmaf_rn(-q, step, t), inverse, q);
  return step > 0.f ? (uint32_t)min(__float2int_rn(quotient), 15) : 0u;
}

}  // namespace vb
