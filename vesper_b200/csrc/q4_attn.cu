// One decoding token per row attending over a 4-bit ring cache (vesper/attention.py:298-338
// attend_ring, over the format of q4.cuh): o_h = softmax_j(q_h . k_j / sqrt(DK)) v_j over the slots
// whose position lies in (p - W, p], the token itself written first.
//
// The bytes of the cache bound it: 0.625 per channel at DK a multiple of 32, which at the memory's rate
// leaves some three instructions per channel on the ordinary pipes, less than unpacking and one
// product per head would take. So the codes go to the matrix units as they are. A warp takes tiles of
// 64 slots (copied by the bulk engine, two tiles in flight per warp) and eight query heads of one key head:
//   scores  S[slot, head] = sum_g step[slot, g] (sum_{c in g} code q) + lo[slot, g] (sum_{c in g} q):
//     m16n8k16 in f16, slots as rows. A code in the low four bits of a half is the subnormal code 2^-24, one
//     in the next four bits 16 code 2^-24, both exact, so a word of eight codes needs one shift and
//     four ANDs; the queries are scaled per head by a power of two to fit f16 (an f32 query takes two terms) and
//     divided by 16 where their codes come 16-fold. The group's step and lo are applied to the float32 sums.
//   output  O[channel, head] = sum_slot (w step) (code - 8) + w (lo + 8 step): m16n8k16 in bf16 (whose range the
//     products w step need), channels as rows. A code becomes a bf16 number by OR (128 + code) and one subtraction
//     per pair; centred codes keep the rounding of w step and of the sums in proportion to the values. The weights cross from the scores' layout to the operand's by movmatrix. w step is rounded to
//     bf16 for bf16 and f16 inputs (2^-9, of both signs) and held in three bf16 terms for float32.
// Running maximum and sum per warp and head in float32; the warps' parts are joined in shared memory, those of the
// CTAs that share a long window by a second kernel, in a fixed order. A slot that is not seen has score -inf and its
// step and lo are read as zeros, whatever it holds.
#include <cmath>
#include <type_traits>

#include "launch.cuh"
#include "q4.cuh"
#include "umma.cuh"

namespace vb {
namespace {

constexpr int AW = 8;  // warps per CTA
constexpr int HEADS = 8;  // query heads of one key head per CTA

template <typename T, int DK>
struct Q4Attn {
  static constexpr int GS = q4_group(DK), NG = DK / GS;
  static constexpr int CODES = DK / 2, PAR = NG * 4;  // bytes per slot
  static constexpr int VC = Q4_TILE * CODES, KP = 2 * VC, VP = KP + Q4_TILE * PAR, POS = VP + Q4_TILE * PAR;
  static constexpr int TILE = POS + Q4_TILE * 8;
  static constexpr int STAGES = 2;
  static constexpr int SMEM = AW * STAGES * TILE;
  static constexpr int QT = sizeof(T) == 4 ? 2 : 1, PT = sizeof(T) == 4 ? 3 : 1;  // terms of queries, of weights
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float f16_value(float x) { return __half2float(__float2half_rn(x)); }

// the low four bits of each half as a pair of bf16 numbers code - 8
__device__ __forceinline__ uint32_t centred(uint32_t x) {
  uint32_t y;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"((x & 0x000f000fu) | 0x43004300u), "r"(0x43084308u));
  return y;
}

// BYTES consecutive bytes (aligned to their largest power-of-two divisor, 16 at most) as words
template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t (&w)[(BYTES + 3) / 4]) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  } else if constexpr (BYTES % 2 == 0) {
#pragma unroll
    for (int i = 0; i < (BYTES + 3) / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < BYTES / 2; ++i) w[i / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + 2 * i) << (16 * (i & 1));
  } else {
#pragma unroll
    for (int i = 0; i < (BYTES + 3) / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < BYTES; ++i) w[i / 4] |= (uint32_t)p[i] << (8 * (i & 3));
  }
}

struct Ring {
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  int64_t* pos;
};

// Partial layout: [(b * units + unit) * splits + z][HEADS][DK + 2], per head the unnormalised output, the base-2
// running maximum and the sum.
template <typename T, int DK>
__global__ void __launch_bounds__(AW * 32, DK <= 64 ? 2 : 1)
    q4_attn_kernel(const T* __restrict__ q, int64_t q_row, const T* __restrict__ k_new, int64_t k_row,
                   const T* __restrict__ v_new, int64_t v_row, const int64_t* __restrict__ pos, Ring ring,
                   T* __restrict__ o, float* __restrict__ part, int H, int HKV, int head_tiles, int W, int SLOTS,
                   float scale_log2, int* status) {
  using C = Q4Attn<T, DK>;
  constexpr int GS = C::GS, NG = C::NG, QT = C::QT, PT = C::PT, TILES = DK / 16, KSTEPS = GS / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[AW][C::STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int z = blockIdx.x, splits = gridDim.x, unit = blockIdx.y, kh = unit / head_tiles, ht = unit - kh * head_tiles;
  const int64_t b = blockIdx.z;
  const int G = H / HKV, h0 = kh * G + ht * HEADS, heads = min(HEADS, G - ht * HEADS);
  uint8_t* mine = smem + warp * C::STAGES * C::TILE;
  if (lane == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
  }
  __syncwarp();
  grid_wait();
  grid_release();
  const int64_t p = pos[b];
  const int nt = p < 0 ? 0 : (int)((min(p + 1, (int64_t)W) + Q4_TILE - 1) / Q4_TILE);  // tiles that can be seen
  const int lo_t = (int)((int64_t)nt * z / splits), hi_t = (int)((int64_t)nt * (z + 1) / splits);
  const int64_t base = (b * HKV + kh) * SLOTS;
  const int own = p < 0 ? -1 : (int)(p % W);
  auto copy = [&](int i) {  // tile lo_t + warp + 8 i into its stage
    const int tile = lo_t + warp + AW * i;
    if (tile >= hi_t) return;
    uint8_t* to = mine + (i % C::STAGES) * C::TILE;
    uint64_t* bar = &full[warp][i % C::STAGES];
    const int64_t s = base + (int64_t)tile * Q4_TILE;
    mbar_arrive_expect_tx(bar, C::TILE);
    bulk_load(to, ring.k_codes + s * C::CODES, C::VC, bar);
    bulk_load(to + C::KP, ring.k_params + s * NG, Q4_TILE * C::PAR, bar);
    bulk_load(to + C::POS, ring.pos + b * SLOTS + (int64_t)tile * Q4_TILE, Q4_TILE * 8, bar);
    bulk_load(to + C::VC, ring.v_codes + s * C::CODES, C::VC, bar);
    bulk_load(to + C::VP, ring.v_params + s * NG, Q4_TILE * C::PAR, bar);
  };
  if (lane == 0)
    for (int i = 0; i < C::STAGES; ++i) copy(i);

  // queries: thread (g, t) holds head g's channels of every group that the key codes of lane part t belong to
  uint32_t qb[NG][KSTEPS][QT][2];
  float qs[NG][2], f[2];
  {
    float x[NG][GS / 4], top = 0.f, sum[NG];
#pragma unroll
    for (int a = 0; a < NG; ++a)
#pragma unroll
      for (int i = 0; i < GS / 4; ++i) {
        x[a][i] = g < heads ? to_f32<T>(q[b * q_row + (int64_t)(h0 + g) * DK + a * GS + t * (GS / 4) + i]) : 0.f;
        top = fmaxf(top, fabsf(x[a][i]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the power of two that brings the largest magnitude to [2^14, 2^15), and its inverse times 2^24
    const int e = top > 0.f ? (int)(__float_as_uint(top) >> 23) : 127;
    const float up = __uint_as_float((uint32_t)min(268 - e, 254) << 23);
    const float down = ldexpf(1.0f, 24 - (min(268 - e, 254) - 127));
#pragma unroll
    for (int a = 0; a < NG; ++a) {
      sum[a] = 0.f;
#pragma unroll
      for (int i = 0; i < GS / 4; ++i) {
        x[a][i] *= up;
        sum[a] += x[a][i];
      }
      sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 1);
      sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 2);
      // nibbles (i, i + half) share a register: halves of a word of eight codes, or of four for groups of 16
      constexpr int HALF = GS / 8;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        float u[4] = {x[a][2 * s], x[a][2 * s + HALF], x[a][2 * s + 1] * 0.0625f, x[a][2 * s + 1 + HALF] * 0.0625f};
#pragma unroll
        for (int r = 0; r < QT; ++r) {
          qb[a][s][r][0] = pack_f16(u[0], u[1]);
          qb[a][s][r][1] = pack_f16(u[2], u[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] -= f16_value(u[i]);
        }
      }
    }
    // what the sums' layout needs: heads 2 t and 2 t + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int from = 4 * (2 * t + c);
      f[c] = scale_log2 * __shfl_sync(0xffffffffu, down, from);
#pragma unroll
      for (int a = 0; a < NG; ++a) qs[a][c] = __shfl_sync(0xffffffffu, sum[a], from) * 5.9604644775390625e-8f;  // 2^-24
    }
  }

  // the new token, in the warp whose tile holds its slot: lane c < 16 holds eight channels of the key, 16 + c of
  // the value
  const int own_at = own >= 0 ? own / Q4_TILE - lo_t : -1;
  const bool has_own = own_at >= 0 && own / Q4_TILE < hi_t && own_at % AW == warp;
  float tok[8];
  if (has_own) {
    const int c = (lane & 15) * 8;
    const T* src = lane < 16 ? k_new + b * k_row + (int64_t)kh * DK + c : v_new + b * v_row + (int64_t)kh * DK + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) tok[i] = c < DK ? to_f32<T>(src[i]) : 0.f;
  }

  float acc[TILES][4], low[NG][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
  for (int a = 0; a < NG; ++a) low[a][0] = low[a][1] = 0.f;
  // row r of a 16-slot step is slot r, pairs swapped in the upper half of each eight: keys and values are then both
  // read from shared memory without bank conflicts at DK 64
  const int krow = g ^ ((g >> 2) & 1), vrow0 = (2 * t) ^ (t >> 1), vrow1 = (2 * t + 1) ^ (t >> 1);

  for (int i = 0; lo_t + warp + AW * i < hi_t; ++i) {
    const int st = i % C::STAGES, tile = lo_t + warp + AW * i;
    uint8_t* at = mine + st * C::TILE;
    const bool landed = mbar_wait(&full[warp][st], (i / C::STAGES) & 1);
    if (!__all_sync(0xffffffffu, landed)) {
      if (lane == 0) atomicOr(status, 1);
      for (int j = i; j < i + C::STAGES && lo_t + warp + AW * j < hi_t; ++j)  // the copies that may still be in flight
        mbar_wait(&full[warp][j % C::STAGES], (j / C::STAGES) & 1, 200000000ull);
      break;
    }
    if (has_own && own_at == warp + AW * i) {
      // quantise the token and put it into its slot, here and (once per key head) in the ring
      const bool value = lane >= 16;
      const int c = (lane & 15) * 8, slot = own % Q4_TILE;
      float lowest = tok[0], highest = tok[0];
      bool nan = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lowest = fminf(lowest, tok[j]);
        highest = fmaxf(highest, tok[j]);
        nan |= tok[j] != tok[j];
      }
      if (nan) lowest = highest = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int s = 1; s < GS / 8; s <<= 1) {
        const float l2 = __shfl_xor_sync(0xffffffffu, lowest, s), h2 = __shfl_xor_sync(0xffffffffu, highest, s);
        const bool bad = lowest != lowest || l2 != l2;
        lowest = bad ? __uint_as_float(0x7fc00000u) : fminf(lowest, l2);
        highest = bad ? lowest : fmaxf(highest, h2);
      }
      float step, lo;
      q4_params(lowest, highest, step, lo);
      const float inverse = step > 0.f ? 1.0f / step : 0.f;
      if (c < DK) {
        uint8_t* codes = at + (value ? C::VC : 0) + slot * C::CODES;
        uint8_t* out = (value ? ring.v_codes : ring.k_codes) + (base + own) * C::CODES;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const uint8_t byte = (uint8_t)(q4_code(tok[j], step, lo, inverse) | q4_code(tok[j + 1], step, lo, inverse) << 4);
          const int place = (value ? q4_value_place(DK, c + j) : q4_key_place(DK, c + j)) / 2;
          codes[place] = byte;
          if (ht == 0) out[place] = byte;
        }
        if (c % GS == 0) {
          const uint32_t word = q4_pack_params(step, lo);
          reinterpret_cast<uint32_t*>(at + (value ? C::VP : C::KP))[slot * NG + c / GS] = word;
          if (ht == 0) (value ? ring.v_params : ring.k_params)[(base + own) * NG + c / GS] = word;
        }
      }
      if (unit == 0 && lane == 0) ring.pos[b * SLOTS + own] = p;
      fence_async_smem();  // before the stage is copied into again
      __syncwarp();
    }
    // which of the 64 slots are seen
    uint32_t seen[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int slot = tile * Q4_TILE + 32 * j + lane;
      const int64_t kp = reinterpret_cast<const int64_t*>(at + C::POS)[32 * j + lane];
      seen[j] = __ballot_sync(0xffffffffu, slot == own || (slot < W && kp >= 0 && kp <= p && kp > p - W));
    }
    // scores of slots (rows) by heads (columns), in base 2
    float s[4][4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      const int r0 = 16 * mt + krow;
      uint32_t c0[(DK / 8 + 3) / 4], c1[(DK / 8 + 3) / 4], p0[NG], p1[NG];
      load_bytes<DK / 8>(at + r0 * C::CODES + t * (DK / 8), c0);
      load_bytes<DK / 8>(at + (r0 + 8) * C::CODES + t * (DK / 8), c1);
      load_bytes<4 * NG>(at + C::KP + r0 * C::PAR, p0);
      load_bytes<4 * NG>(at + C::KP + (r0 + 8) * C::PAR, p1);
      float tot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int a = 0; a < NG; ++a) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w0, w1;
        if constexpr (GS == 32) {
          w0 = c0[a]; w1 = c1[a];
        } else {  // four codes: the upper two in the upper half
          w0 = (c0[a / 2] >> (16 * (a & 1))) & 0xffffu;
          w1 = (c1[a / 2] >> (16 * (a & 1))) & 0xffffu;
          w0 |= w0 << 8;
          w1 |= w1 << 8;
        }
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const uint32_t x0 = w0 >> (8 * k), x1 = w1 >> (8 * k);
#pragma unroll
          for (int r = 0; r < QT; ++r)
            mma_f16(d, x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, qb[a][k][r][0],
                    qb[a][k][r][1]);
        }
        tot[0] = fmaf(q4_step(p0[a]), d[0], fmaf(q4_lo(p0[a]), qs[a][0], tot[0]));
        tot[1] = fmaf(q4_step(p0[a]), d[1], fmaf(q4_lo(p0[a]), qs[a][1], tot[1]));
        tot[2] = fmaf(q4_step(p1[a]), d[2], fmaf(q4_lo(p1[a]), qs[a][0], tot[2]));
        tot[3] = fmaf(q4_step(p1[a]), d[3], fmaf(q4_lo(p1[a]), qs[a][1], tot[3]));
      }
      const uint32_t bits = seen[mt >> 1] >> (16 * (mt & 1) + krow);
      s[mt][0] = bits & 1u ? tot[0] * f[0] : -INFINITY;
      s[mt][1] = bits & 1u ? tot[1] * f[1] : -INFINITY;
      s[mt][2] = bits & 256u ? tot[2] * f[0] : -INFINITY;
      s[mt][3] = bits & 256u ? tot[3] * f[1] : -INFINITY;
    }
    // the running maximum and sum, and the weights
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float top = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) top = fmaxf(top, fmaxf(s[mt][c], s[mt][2 + c]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m[c]);
      const float from = top == -INFINITY ? 0.f : top, fade = exp2f(m[c] - from);
      m[c] = top;
      l[c] *= fade;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        s[mt][c] = exp2f(s[mt][c] - from);
        s[mt][2 + c] = exp2f(s[mt][2 + c] - from);
        l[c] += s[mt][c] + s[mt][2 + c];
      }
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        acc[j][c] *= fade;
        acc[j][2 + c] *= fade;
      }
#pragma unroll
      for (int a = 0; a < NG; ++a) low[a][c] *= fade;
    }
    // weights x values
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      constexpr int VB = DK / 16, VW = (VB + 3) / 4;
      const int r0 = 16 * mt + krow;
      uint32_t p0[NG], p1[NG], w[4][VW];
      load_bytes<4 * NG>(at + C::VP + r0 * C::PAR, p0);
      load_bytes<4 * NG>(at + C::VP + (r0 + 8) * C::PAR, p1);
      const uint8_t* vc = at + C::VC + 16 * mt * C::CODES + g * VB;
      load_bytes<VB>(vc + vrow0 * C::CODES, w[0]);
      load_bytes<VB>(vc + vrow1 * C::CODES, w[1]);
      load_bytes<VB>(vc + (vrow0 + 8) * C::CODES, w[2]);
      load_bytes<VB>(vc + (vrow1 + 8) * C::CODES, w[3]);
      const uint32_t bits = seen[mt >> 1] >> (16 * (mt & 1) + krow);
      const uint32_t on0 = 0u - (bits & 1u), on1 = 0u - ((bits >> 8) & 1u);
#pragma unroll
      for (int a = 0; a < NG; ++a) {
        const uint32_t q0 = p0[a] & on0, q1 = p1[a] & on1;  // zeros where the slot is not seen
        const float mid0 = fmaf(8.f, q4_step(q0), q4_lo(q0)), mid1 = fmaf(8.f, q4_step(q1), q4_lo(q1));
        low[a][0] = fmaf(s[mt][0], mid0, fmaf(s[mt][2], mid1, low[a][0]));
        low[a][1] = fmaf(s[mt][1], mid0, fmaf(s[mt][3], mid1, low[a][1]));
        float e[4] = {s[mt][0] * q4_step(q0), s[mt][1] * q4_step(q0), s[mt][2] * q4_step(q1), s[mt][3] * q4_step(q1)};
#pragma unroll
        for (int r = 0; r < PT; ++r) {
          const uint32_t e0 = pack_bf16(e[0], e[1]), e1 = pack_bf16(e[2], e[3]);
          if constexpr (PT > 1) {
            e[0] -= __uint_as_float(e0 << 16); e[1] -= __uint_as_float(e0 & 0xffff0000u);
            e[2] -= __uint_as_float(e1 << 16); e[3] -= __uint_as_float(e1 & 0xffff0000u);
          }
          const uint32_t b0 = transpose8(e0), b1 = transpose8(e1);
#pragma unroll
          for (int j = 0; j < GS / 16; ++j) {
            const int i16 = a * (GS / 16) + j;  // channels [16 i16, 16 i16 + 16): nibbles 2 i16 and 2 i16 + 1
            const int sh = 8 * (i16 & 1);
            const uint32_t sel = i16 & 2 ? 0x7632u : 0x5410u;
            const uint32_t x = __byte_perm(w[0][i16 / 4], w[1][i16 / 4], sel);
            const uint32_t y = __byte_perm(w[2][i16 / 4], w[3][i16 / 4], sel);
            mma_bf16(acc[i16], centred(x >> sh), centred(x >> (sh + 4)), centred(y >> sh), centred(y >> (sh + 4)), b0, b1);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) copy(i + C::STAGES);
  }

  // this warp's part: heads 2 t and 2 t + 1, channels 16 i + 2 g and 16 i + 2 g + 1
  __syncthreads();  // the stages are free
  float* parts = reinterpret_cast<float*>(smem);  // [AW][HEADS][DK + 2]
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
      for (int a = 0; a < NG; ++a) low[a][c] += __shfl_xor_sync(0xffffffffu, low[a][c], x);
    }
    float* row = parts + (warp * HEADS + 2 * t + c) * (DK + 2);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int a = i / (GS / 16);
      *reinterpret_cast<float2*>(row + 16 * i + 2 * g) = make_float2(acc[i][c] + low[a][c], acc[i][2 + c] + low[a][c]);
    }
    if (g == 0) {
      row[DK] = m[c];
      row[DK + 1] = l[c];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < heads * DK; e += AW * 32) {
    const int h = e / DK, c = e - h * DK;
    const float* col = parts + h * (DK + 2);
    float M = -INFINITY, L = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < AW; ++w) M = fmaxf(M, col[w * HEADS * (DK + 2) + DK]);
#pragma unroll
    for (int w = 0; w < AW; ++w) {
      const float* x = col + w * HEADS * (DK + 2);
      const float fade = x[DK] == -INFINITY ? 0.f : exp2f(x[DK] - M);
      L = fmaf(x[DK + 1], fade, L);
      out = fmaf(x[c], fade, out);
    }
    if (splits == 1) {
      o[(b * H + h0 + h) * DK + c] = from_f32<T>(p < 0 ? 0.f : out / L);
    } else {
      float* to = part + (((b * gridDim.y + unit) * splits + z) * HEADS + h) * (DK + 2);
      to[c] = out;
      if (c == 0) {
        to[DK] = M;
        to[DK + 1] = L;
      }
    }
  }
}

// joins the splits of a (row, unit) in order; a row that saw nothing (a negative position) is zero
template <typename T, int DK>
__global__ void __launch_bounds__(DK) q4_attn_join_kernel(const float* __restrict__ part, T* __restrict__ o, int H, int HKV,
                                                          int head_tiles, int units, int splits) {
  grid_wait();
  grid_release();
  const int unit = blockIdx.y, kh = unit / head_tiles, ht = unit - kh * head_tiles, h = blockIdx.x, c = threadIdx.x;
  const int64_t b = blockIdx.z;
  const int G = H / HKV, head = kh * G + ht * HEADS + h;
  if (ht * HEADS + h >= G) return;
  const float* from = part + ((b * units + unit) * splits * HEADS + h) * (DK + 2);
  constexpr int STEP = HEADS * (DK + 2);
  float M = -INFINITY, L = 0.f, out = 0.f;
  for (int z = 0; z < splits; ++z) M = fmaxf(M, from[(int64_t)z * STEP + DK]);
#pragma unroll 4
  for (int z = 0; z < splits; ++z) {
    const float* x = from + (int64_t)z * STEP;
    const float fade = x[DK] == -INFINITY ? 0.f : exp2f(x[DK] - M);
    L = fmaf(x[DK + 1], fade, L);
    out = fmaf(x[c], fade, out);
  }
  o[(b * H + head) * DK + c] = from_f32<T>(L == 0.f ? 0.f : out / L);
}

// CTAs per (row, unit): enough to fill the SMs some times over, each with work for all its warps
int split_count(int B, int units, int W) {
  const int tiles = (W + Q4_TILE - 1) / Q4_TILE;
  const int64_t want = (4 * 148 + (int64_t)B * units - 1) / ((int64_t)B * units);
  const int most = (tiles + 2 * AW - 1) / (2 * AW);
  return (int)(want < most ? want : most);
}

int head_tiles_of(int H, int HKV) { return (H / HKV + HEADS - 1) / HEADS; }

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" size_t vb_q4_attend_workspace(int B, int H, int HKV, int DK, int W) {
  if (B <= 0 || H <= 0 || HKV <= 0 || H % HKV || DK <= 0 || W <= 0) return 16;
  const int units = HKV * head_tiles_of(H, HKV), splits = split_count(B, units, W);
  return splits == 1 ? 16 : sizeof(float) * (size_t)B * units * splits * HEADS * (DK + 2);
}

extern "C" int vb_q4_attend(const void* q, int64_t q_row, const void* k_new, int64_t k_row, const void* v_new,
                            int64_t v_row, const int64_t* pos, void* k_codes, void* k_params, void* v_codes,
                            void* v_params, int64_t* ring_pos, void* o, void* workspace, int B, int H, int HKV, int DK,
                            int W, int SLOTS, int dtype, int* status, void* stream) {
  VB_REQUIRE(B >= 0 && H >= 1 && HKV >= 1 && W >= 1, "q4_attend: bad shape B=%d H=%d HKV=%d W=%d", B, H, HKV, W);
  VB_REQUIRE(H % HKV == 0, "q4_attend: %d query heads are not a multiple of %d key heads", H, HKV);
  VB_REQUIRE(DK >= 16 && DK <= 128 && DK % 16 == 0, "q4_attend: head dimension %d must be a multiple of 16 up to 128", DK);
  VB_REQUIRE(SLOTS % Q4_TILE == 0 && SLOTS >= W, "q4_attend: %d slots must be a multiple of %d holding the window %d",
             SLOTS, Q4_TILE, W);
  VB_REQUIRE(dtype_size(dtype) > 0, "q4_attend: unsupported dtype code %d", dtype);
  if (B == 0) return VB_OK;
  VB_REQUIRE(q && k_new && v_new && pos && k_codes && k_params && v_codes && v_params && ring_pos && o && workspace && status,
             "q4_attend: null pointer");
  VB_REQUIRE(aligned16(k_codes) && aligned16(k_params) && aligned16(v_codes) && aligned16(v_params) && aligned16(ring_pos),
             "q4_attend: the ring's buffers must start on 16-byte boundaries");
  const int head_tiles = head_tiles_of(H, HKV), units = HKV * head_tiles, splits = split_count(B, units, W);
  VB_REQUIRE(B <= 65535 && units <= 65535, "q4_attend: %d rows of %d head tiles exceed the grid", B, units);
  const Ring ring{(uint8_t*)k_codes, (uint32_t*)k_params, (uint8_t*)v_codes, (uint32_t*)v_params, ring_pos};
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)DK);
  cudaStream_t st = (cudaStream_t)stream;
  float* part = (float*)workspace;
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    auto run = [&](auto dk) -> int {
      constexpr int D = decltype(dk)::value;
      int rc = launch_early("q4_attend", q4_attn_kernel<T, D>, dim3(splits, units, B), AW * 32, Q4Attn<T, D>::SMEM, 1, st,
                            (const T*)q, q_row, (const T*)k_new, k_row, (const T*)v_new, v_row, pos, ring, (T*)o, part, H,
                            HKV, head_tiles, W, SLOTS, scale_log2, status);
      if (rc || splits == 1) return rc;
      return launch_early("q4_attend join", q4_attn_join_kernel<T, D>, dim3(HEADS, units, B), D, 0, 1, st,
                          (const float*)part, (T*)o, H, HKV, head_tiles, units, splits);
    };
    switch (DK) {
      case 16: return run(std::integral_constant<int, 16>{});
      case 32: return run(std::integral_constant<int, 32>{});
      case 48: return run(std::integral_constant<int, 48>{});
      case 64: return run(std::integral_constant<int, 64>{});
      case 80: return run(std::integral_constant<int, 80>{});
      case 96: return run(std::integral_constant<int, 96>{});
      case 112: return run(std::integral_constant<int, 112>{});
      default: return run(std::integral_constant<int, 128>{});
    }
  });
}
