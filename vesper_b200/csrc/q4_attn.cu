// One decoding token per row attending over a 4-bit ring cache (vesper/attention.py:298-338
// attend_ring, over the format of q4.cuh): o_h = softmax_j(q_h . k_j / sqrt(DK)) v_j over the slots
// whose position lies in (p - W, p], the token itself written first.
//
// The bytes of the cache bound it: 0.625 per channel at DK a multiple of 32, which at the memory's rate
// leaves some three instructions per channel on the ordinary pipes, less than unpacking and one
// product per head would take. So the codes go to the matrix units as they are. A warp takes tiles of
// 64 slots (copied 16 bytes a lane by cp.async, two tiles in flight per warp) and eight query heads of one key head:
//   scores  S[slot, head] = sum_g step[slot, g] (sum_{c in g} code q) + lo[slot, g] (sum_{c in g} q):
//     m16n8k16 in f16, slots as rows. A code in the low four bits of a half is the subnormal code 2^-24, one
//     in the next four bits 16 code 2^-24, both exact, so a word of eight codes needs one shift and
//     four ANDs; the queries are scaled per head by a power of two to fit f16 and
//     divided by 16 where their codes come 16-fold. The group's step and lo are applied to the float32 sums.
//   output  O[channel, head] = sum_slot (w step) code + w lo: m16n8k16 in f16, channels as rows, the codes again as
//     they are (those in the upper four bits make their rows of O 16-fold, taken off at the end). The products w step
//     are held in two f16 terms (22 bits), whose range they fit because the scores' reference is chosen with the largest
//     step in view. They cross from the scores' layout to the operand's by movmatrix.
//     The matrix unit cuts its sums off, always towards zero: with codes of one sign the loss of a long run would add up, to
//     15 times an f16 output's rounding where a warp has 50 tiles of equal weights. So every second step of 16 slots takes
//     15 - code (the complement, at no cost) with the products negated, and the sums stay near zero (1 to 2 % of the time).
// For float32 inputs queries and products are held in three bf16 terms and the codes as bf16 code - 7.5, around zero, and
// the matrix unit's sums, which are cut off rather than rounded, are short: the output is within 1e-6 of its norm.
// A reference r and the sum of the weights 2^(score - r) per warp and head in float32; r rises only when a weight
// times its tile's largest step (its slot's, where steps lie far apart) would pass 2^14, and then to 2^6, so that the
// sums are seldom rescaled. The warps' parts are joined in shared memory, those of the CTAs that share a long window by
// a second kernel, in a fixed order. A slot that is not seen has score -inf and its step and lo are read as zeros,
// whatever it holds.
//
// Measured (bf16, device): 8 rows of 6249 to 49999 positions, 32 query and 8 key heads of 128, 67 us (290 MB, 4.3
// TB/s, 66 % of a plain copy's rate); 8 x 32768 76 us (4.45 TB/s, 68 %). What keeps it from the copy's rate is
// latency: eight warps an SM (255 registers each at DK 128) issue in half of the cycles, and the last tiles of a unit, the
// joining of its warps and the next unit's first tiles follow one another. At DK 64, eight query heads to two key heads,
// 64 x 8192 take 33 us (88 MB, 41 %): half the bytes for each instruction. 64 rows of 512 positions take 5.7 us, the
// latency of position, tiles, two products and the joining. One float32 row of 100003 positions at DK 64,
// three products for one, takes 21.5 us. Of the first two figures some 8 % buy what 16-bit outputs keep: the second term of
// the products 4 us of the 76, sums and ranges 2.
#include <cmath>
#include <type_traits>

#include "launch.cuh"
#include "q4.cuh"
#include "umma.cuh"

namespace vb {
namespace {

constexpr int HEADS = 8;  // query heads of one key head per CTA

// resident CTAs: registers for DK above 64 leave room for one
__host__ __device__ constexpr int ctas_per_sm(int dk) { return dk <= 64 ? 2 : 1; }

template <typename T, int DK>
struct Q4Attn {
  static constexpr int GS = q4_group(DK), NG = DK / GS;
  static constexpr int CODES = DK / 2, PAR = NG * 4;  // bytes per slot
  static constexpr int TS = Q4_TILE, MT = TS / 16;     // slots of a warp's tile, and its steps of 16
  static constexpr int VC = TS * CODES, KP = 2 * VC, VP = KP + TS * PAR, POS = VP + TS * PAR;
  static constexpr int TILE = POS + TS * 8;
  static constexpr int AW = 8, STAGES = 2, CTAS = ctas_per_sm(DK);  // warps per CTA, tiles in flight per warp
  static constexpr int SMEM = AW * STAGES * TILE;
  // float32 throughout: queries and the weights' products in three bf16 terms, codes as code - 7.5. Else queries in one
  // f16 term, which a 16-bit query is (but for bf16 channels 2^28 below their head's largest: they lose their last bits, 2^-36
  // of the largest), and the products in two (with one, 17 % of a bf16 output's numbers are not the
  // rounded result, with two 0.4 %)
  static constexpr bool EXACT = sizeof(T) == 4;
  static constexpr int QT = EXACT ? 3 : 1, PT = EXACT ? 3 : 2;
  // the sum of lo times the queries' sums as one product in bf16: four groups, three terms
  static constexpr bool WIDE = std::is_same<T, __nv_bfloat16>::value;  // float32's range in 16 bits
  static constexpr bool LO_MMA = !EXACT && (NG == 1 || NG == 2 || NG == 4);
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float exp2_approx(float x) {  // within 2^-22; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// x and y plus m (an f16 number, as bits) times the f16 numbers of a pair, in float32
constexpr uint16_t F16_MINUS_ONE = 0xbc00;
__device__ __forceinline__ void less_f16(float& x, float& y, uint32_t pair, uint16_t m) {
  asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "fma.rn.f32.f16 %0, a, %3, %0;\n\tfma.rn.f32.f16 %1, b, %3, %1;\n\t}"
      : "+f"(x), "+f"(y)
      : "r"(pair), "h"(m));
}

// the low four bits of each half as a pair of bf16 numbers code - 7.5: 16 + code by their place in the mantissa, less 23.5
__device__ __forceinline__ uint32_t centred(uint32_t x) {
  uint32_t y;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(((x << 3) & 0x00780078u) | 0x41804180u), "r"(0x41bc41bcu));
  return y;
}

// the larger of two pairs of bf16 numbers, each half for itself; a NaN gives way to a number
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
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

// What a weight may be multiplied by, as a power of two, from a largest step and a largest magnitude of lo (as bits): a power
// above the step, between 2^-80 and 2^80, past which the weights' sum or the smaller weights would leave float32, and one by
// which lo is at most 2^86 larger, so that no sum overflows. Without any step the weights may be large, but not so large
// that a later tile's rescaling would lose them.
constexpr int MOST_STEP = 80;
__device__ __forceinline__ float size_of(uint32_t step, uint32_t lo) {
  const int of_step = step == 0 ? -40 : min(max((int)(step >> 23) - 126, -80), MOST_STEP);
  return (float)max(of_step, (int)(lo >> 23) - 212);
}

struct Ring {
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  int64_t* pos;
};

// tiles of a row that can be seen from position p
template <int TS>
__device__ __forceinline__ int tiles_of(int64_t p, int W) {
  return p < 0 ? 0 : (int)((min(p + 1, (int64_t)W) + TS - 1) / TS);
}

// What a unit counts when the work is shared: its tiles, and `opening` more for what its opening and closing cost (the
// queries, the first tiles' way from memory, the joining of the warps).
__device__ __forceinline__ int cost_of(int tiles, int opening) { return tiles > 0 ? tiles + opening : 0; }

// Where `at` lies among all rows' and units' costs, in that order: its row, where the row begins and its number of
// tiles (per unit). Called by whole warps.
template <int TS>
__device__ __forceinline__ void find_row(const int64_t* pos, int B, int units, int W, int opening, int64_t at,
                                         int64_t& row, int64_t& first, int& n) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int r0 = 0; r0 < B; r0 += 32) {
    const int mine = r0 + lane < B ? cost_of(tiles_of<TS>(pos[r0 + lane], W), opening) : 0;
    int upto = mine;  // 32 rows of at most 2^25 tiles
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, x);
      if (lane >= x) upto += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * units > at);
    if (past) {
      const int l = __ffs(past) - 1;
      row = r0 + l;
      const int cost = __shfl_sync(0xffffffffu, mine, l);
      n = cost - opening;
      first = (before + __shfl_sync(0xffffffffu, upto, l) - cost) * units;
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  row = B;
  first = before * units;
  n = 0;
}

// All rows' and units' costs, and how many of a launch's CTAs share them: as many as have a tile for each of their warps,
// but one for each unit that sees something if that is more. An opening counts 16 tiles where a CTA has over 32 (8
// streams of 6249 to 49999 positions, 8 key heads of 128, when this was chosen: 61 us, with none 67, with 40 63), none
// where it has fewer.
template <int TS, int AW>
__device__ __forceinline__ int64_t all_costs(const int64_t* pos, int B, int units, int W, int& ctas, int& opening) {
  int64_t sum = 0;
  int live = 0;
  for (int r = threadIdx.x & 31; r < B; r += 32) {
    const int n = tiles_of<TS>(pos[r], W);
    sum += n;
    live += n > 0;
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  live = __reduce_add_sync(0xffffffffu, live);
  ctas = (int)min((int64_t)ctas, max((sum * units + AW - 1) / AW, (int64_t)live * units));
  opening = sum * units > (int64_t)32 * ctas ? 16 : 0;
  return (sum + (int64_t)live * opening) * units;
}

// `total` in even parts: part i begins at floor(i total / parts)
struct Share {
  int64_t each;
  uint32_t rest, parts;
  __device__ __forceinline__ Share(int64_t total, int n) : parts((uint32_t)n) {
    if (total < ((int64_t)1 << 32)) {
      each = (uint32_t)total / parts;
      rest = (uint32_t)total % parts;
    } else {
      each = total / n;
      rest = (uint32_t)(total % n);
    }
  }
  __device__ __forceinline__ int64_t start(uint32_t i) const { return each * i + rest * i / parts; }
};

// A unit is eight query heads of one key head. With `shared` the CTAs divide all rows' and units' costs evenly between
// them, whatever the rows' lengths: CTA i takes what lies in [i T / n, (i + 1) T / n) and writes what it has of a unit it does
// not hold whole to its partials, [2 i] of the unit it starts within and [2 i + 1] of the one it ends within, each
// [HEADS][DK + 2]: per head the unnormalised output, the reference and the sum; span[row][unit] gets the first and
// the last CTA of a unit. Else a CTA per unit and row.
// PAIR: at most four heads to a key head. Columns 4 to 7 of the products then repeat the heads of columns 0 to 3, bit for bit,
// and take the second f16 term of the weights' products, so that two terms cost no second product (8 x 32768 positions, 32 /
// 8 heads of 128, when this was chosen: 75 us, with two products 82, a single term 71).
template <typename T, int DK, bool PAIR>
__global__ void __launch_bounds__(Q4Attn<T, DK>::AW * 32, (Q4Attn<T, DK>::CTAS))
    q4_attn_kernel(const T* __restrict__ q, int64_t q_row, int q_vec, const T* __restrict__ k_new, int64_t k_row,
                   const T* __restrict__ v_new, int64_t v_row, const int64_t* __restrict__ pos, Ring ring,
                   T* __restrict__ o, float* __restrict__ part, int2* __restrict__ span, int shared, int B, int H,
                   int HKV, int head_tiles, int W, int SLOTS, float scale_log2) {
  using C = Q4Attn<T, DK>;
  constexpr int GS = C::GS, NG = C::NG, QT = C::QT, PT = C::PT, TILES = DK / 16, KSTEPS = GS / 16, AW = C::AW;
  constexpr int TS = C::TS, MT = C::MT, PM = PAIR ? 1 : PT;  // PM: products for a step's terms
  static_assert(!(PAIR && C::EXACT), "three terms do not fit two columns");
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int units = HKV * head_tiles, G = H / HKV;
  uint8_t* mine = smem + warp * C::STAGES * C::TILE;
  grid_wait();
  grid_release();
  int64_t b = blockIdx.y, from = 0, until = 1, row_first = 0;  // this CTA's share, and where row b begins
  int opening = 0, n = 0, unit = blockIdx.x, lo_t = 0, hi_t = 0;  // tiles of a unit of row b, and those of them this CTA has
  if (shared) {
    int ctas = gridDim.x;
    const int64_t total = all_costs<TS, AW>(pos, B, units, W, ctas, opening);
    if (blockIdx.x >= ctas) return;
    const Share share(total, ctas);
    from = share.start(blockIdx.x);
    until = share.start(blockIdx.x + 1);
    find_row<TS>(pos, B, units, W, opening, from, b, row_first, n);
  }
  while (from < until) {
    int64_t p = 0;
    if (shared) {
      p = pos[b];
      const int cost = cost_of(n, opening);
      unit = from - row_first < ((int64_t)1 << 32) ? (int)((uint32_t)(from - row_first) / (uint32_t)cost)
                                                   : (int)((from - row_first) / cost);
      const int lo = (int)(from - row_first - (int64_t)unit * cost), hi = (int)min((int64_t)cost, lo + (until - from));
      from += hi - lo;
      lo_t = max(0, lo - opening);
      hi_t = max(0, hi - opening);
      if (lo_t >= hi_t) break;  // the share ends within a unit's opening
    } else {
      hi_t = SLOTS / TS;  // until the position has come: the first copies do not wait for it
      from = until;
    }
    const int kh = unit / head_tiles, ht = unit - kh * head_tiles, h0 = kh * G + ht * HEADS, heads = min(HEADS, G - ht * HEADS);
    const int64_t base = (b * HKV + kh) * SLOTS;
    const int column = PAIR ? g & 3 : g;  // the head whose query this thread holds
    // queries: thread (g, t) holds head g's channels of every group that the key codes of lane part t belong to. They and
    // the token are loaded before the cache's tiles, behind which they would wait
    __align__(16) T xraw[NG * (GS / 4)], tokraw[8];  // as they come: nothing waits for them before the copies are issued
    {
      const T* src = q + b * q_row + (int64_t)(h0 + min(column, heads - 1)) * DK + t * (GS / 4);
      constexpr int BYTES = GS / 4 * (int)sizeof(T);
      if (q_vec) {  // rows on 16-byte boundaries
#pragma unroll
        for (int a = 0; a < NG; ++a) {
          if constexpr (BYTES == 8) reinterpret_cast<uint2*>(xraw)[a] = __ldg(reinterpret_cast<const uint2*>(src + a * GS));
          else
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i)
              reinterpret_cast<uint4*>(xraw)[a * (BYTES / 16) + i] = __ldg(reinterpret_cast<const uint4*>(src + a * GS) + i);
        }
      } else {
#pragma unroll
        for (int a = 0; a < NG; ++a)
#pragma unroll
          for (int i = 0; i < GS / 4; ++i) xraw[a * (GS / 4) + i] = src[a * GS + i];
      }
    }
    // the token: lane c < 16 holds eight channels of the key, 16 + c of the value
    const bool tok_value = lane >= 16;
    const int tok_c = (lane & 15) * 8;
    if (tok_c < DK) {
      const T* src = tok_value ? v_new + b * v_row + (int64_t)kh * DK + tok_c : k_new + b * k_row + (int64_t)kh * DK + tok_c;
#pragma unroll
      for (int i = 0; i < 8; ++i) tokraw[i] = src[i];
    }
    auto copy = [&](int i) {  // tile lo_t + warp + 8 i into stage i mod 2; the group is committed even if it is empty
      const int tile = lo_t + warp + AW * i;
      if (tile < hi_t) {
        const uint32_t to = smem_u32(mine + (i % C::STAGES) * C::TILE) + 16 * lane;
        const int64_t s0 = base + (int64_t)tile * TS;
        const uint8_t* kc = ring.k_codes + s0 * C::CODES + 16 * lane;
        const uint8_t* vc = ring.v_codes + s0 * C::CODES + 16 * lane;
        const uint8_t* kp = reinterpret_cast<const uint8_t*>(ring.k_params + s0 * NG) + 16 * lane;
        const uint8_t* vp = reinterpret_cast<const uint8_t*>(ring.v_params + s0 * NG) + 16 * lane;
#pragma unroll
        for (int x = 0; x < C::VC; x += 512) cp_async16(to + x, kc + x, 16);
#pragma unroll
        for (int x = 0; x < TS * C::PAR; x += 512)
          if (x + 512 <= TS * C::PAR || x + 16 * lane < TS * C::PAR) {
            cp_async16(to + C::KP + x, kp + x, 16);
            cp_async16(to + C::VP + x, vp + x, 16);
          }
        cp_async16(to + C::POS, reinterpret_cast<const uint8_t*>(ring.pos + b * SLOTS + (int64_t)tile * TS) + 16 * lane, 16);
#pragma unroll
        for (int x = 0; x < C::VC; x += 512) cp_async16(to + C::VC + x, vc + x, 16);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < C::STAGES; ++i) copy(i);

    if (!shared) {
      p = pos[b];
      n = hi_t = tiles_of<TS>(p, W);
    }
    const int own = p < 0 ? -1 : p < ((int64_t)1 << 31) ? (int)((uint32_t)p % (uint32_t)W) : (int)(p % W);
    const int own_at = own >= 0 ? own / TS - lo_t : -1;  // the warp whose tile holds the token's slot has it
    const bool has_own = own_at >= 0 && own / TS < hi_t && own_at % AW == warp;

    uint32_t qb[NG][KSTEPS][QT][2], qlo[2] = {0u, 0u};
    float qs[NG][2], f[2];
    uint32_t huge = 0;  // bit c: the scores of column 2 t + c are still to be multiplied by 2^24
    {
      float x[NG][GS / 4], top = 0.f, sum[NG];
#pragma unroll
      for (int a = 0; a < NG; ++a)
#pragma unroll
        for (int i = 0; i < GS / 4; ++i) x[a][i] = column < heads ? to_f32<T>(xraw[a * (GS / 4) + i]) : 0.f;
#pragma unroll
      for (int a = 0; a < NG; ++a)
#pragma unroll
        for (int i = 0; i < GS / 4; ++i) top = fmaxf(top, fabsf(x[a][i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that brings the largest magnitude to [2^14, 2^15) (in float32 to [2, 4), which leaves the keys'
      // range to the sums), and its inverse over the products' unit (which comes later where both would leave float32:
      // queries from 2^104 on)
      const int e = top > 0.f ? (int)(__float_as_uint(top) >> 23) : 127;
      const bool apart = C::WIDE && e > 230;
      const int up_e = min((C::EXACT ? 255 : 268) - e, 254);
      const float up = __uint_as_float((uint32_t)up_e << 23);
      constexpr float UNIT = C::EXACT ? 1.f : 5.9604644775390625e-8f;  // what a product's code counts: 2^-24 in f16
      const float down = ldexpf(1.0f, (C::EXACT || apart ? 0 : 24) - (up_e - 127));
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
          float u[4] = {x[a][2 * s], x[a][2 * s + HALF], x[a][2 * s + 1], x[a][2 * s + 1 + HALF]};
          if constexpr (C::EXACT) {
#pragma unroll
            for (int r = 0; r < QT; ++r) {
              qb[a][s][r][0] = pack_bf16(u[0], u[1]);
              qb[a][s][r][1] = pack_bf16(u[2], u[3]);
#pragma unroll
              for (int i = 0; i < 4; ++i) u[i] -= __bfloat162float(__float2bfloat16_rn(u[i]));
            }
          } else {
            qb[a][s][0][0] = pack_f16(u[0], u[1]);
            qb[a][s][0][1] = pack_f16(u[2] * 0.0625f, u[3] * 0.0625f);
          }
        }
      }
      if constexpr (C::LO_MMA) {
        // k = 2 t holds a step (times zero), k = 2 t + 1, 2 t + 8 and 2 t + 9 the lo of group t, times the group's query sum
        // in three terms
        float mine_sum = 0.f, term[3];
#pragma unroll
        for (int a = 0; a < NG; ++a) mine_sum = t == a ? sum[a] * UNIT : mine_sum;
#pragma unroll
        for (int r = 0; r < 3; ++r) {
          term[r] = __bfloat162float(__float2bfloat16_rn(mine_sum));
          mine_sum -= term[r];
        }
        qlo[0] = pack_bf16(0.f, term[0]);
        qlo[1] = pack_bf16(term[2], term[1]);
      }
      // what the sums' layout needs: heads 2 t and 2 t + 1
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * t + c);
        f[c] = scale_log2 * __shfl_sync(0xffffffffu, down, from);
        if constexpr (C::WIDE) huge |= (uint32_t)__shfl_sync(0xffffffffu, (int)apart, from) << c;
#pragma unroll
        for (int a = 0; a < NG; ++a) qs[a][c] = __shfl_sync(0xffffffffu, sum[a], from) * UNIT;
      }
    }

    uint32_t tok_codes = 0, tok_params = 0;
    if (has_own) {  // quantised, and written to the ring once per key head
      float tok[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) tok[j] = tok_c < DK ? to_f32<T>(tokraw[j]) : 0.f;
      float lowest = tok[0], highest = tok[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        lowest = min_nan(lowest, tok[j]);
        highest = max_nan(highest, tok[j]);
      }
#pragma unroll
      for (int s = 1; s < GS / 8; s <<= 1) {
        lowest = min_nan(lowest, __shfl_xor_sync(0xffffffffu, lowest, s));
        highest = max_nan(highest, __shfl_xor_sync(0xffffffffu, highest, s));
      }
      float step, lo, inverse;
      q4_params(lowest, highest, step, lo, inverse);
      tok_params = q4_pack_params(step, lo);
      tok_codes = q4_codes(tok, step, lo, inverse);
      if (tok_c < DK && ht == 0) {
        uint8_t* out = (tok_value ? ring.v_codes : ring.k_codes) + (base + own) * C::CODES;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          out[(tok_value ? q4_value_place(DK, tok_c + 2 * j) : q4_key_place(DK, tok_c + 2 * j)) / 2] = (uint8_t)(tok_codes >> (8 * j));
        if (tok_c % GS == 0) (tok_value ? ring.v_params : ring.k_params)[(base + own) * NG + tok_c / GS] = tok_params;
      }
      if (unit == 0 && lane == 0) ring.pos[b * SLOTS + own] = p;
    }

    float acc[TILES][4], low[NG][2], ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int a = 0; a < NG; ++a) low[a][0] = low[a][1] = 0.f;
    const uint16_t second = t < 2 ? 0 : F16_MINUS_ONE;
    // row r of a 16-slot step is slot r, pairs swapped in the upper half of each eight: keys and values are then both
    // read from shared memory without bank conflicts at DK 64
    const int krow = g ^ ((g >> 2) & 1), vrow0 = (2 * t) ^ (t >> 1), vrow1 = (2 * t + 1) ^ (t >> 1);

    // Tiles from the i-th on, in f16 as far as it goes. That form stops at a tile where the reference is to rise and steps lie
    // more than 2^8 apart: from there on the products are held in three bf16 terms (X), whose range takes any steps, so that a
    // group of large ones takes nothing from the others of its slots. Where that has not come, every group has had products of
    // 2^-2 or more, beside which what f16 drops, 2^-25, is nothing. It stops too before a reference of 2^20, beside which the
    // rounding of the reference itself would begin to count, and before steps of 2^80. (Both forms in one loop cost 5 %,
    // whole scores in it 3 %.)
    int i = 0;
    auto walk = [&](auto exact) {
      constexpr bool X = decltype(exact)::value;
      constexpr int TERMS = X ? 3 : PM;
      for (; lo_t + warp + AW * i < hi_t; ++i) {
        const int tile = lo_t + warp + AW * i;
        uint8_t* at = mine + (i % C::STAGES) * C::TILE;
        cp_async_wait<C::STAGES - 1>();
        __syncwarp();
        if (has_own && own_at == warp + AW * i) {  // the token takes its slot here too
          if (tok_c < DK) {
            const int slot = own % TS;
            uint8_t* codes = at + (tok_value ? C::VC : 0) + slot * C::CODES;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              codes[(tok_value ? q4_value_place(DK, tok_c + 2 * j) : q4_key_place(DK, tok_c + 2 * j)) / 2] =
                  (uint8_t)(tok_codes >> (8 * j));
            if (tok_c % GS == 0)
              reinterpret_cast<uint32_t*>(at + (tok_value ? C::VP : C::KP))[slot * NG + tok_c / GS] = tok_params;
          }
          __syncwarp();
        }
        // which of the slots are seen
        uint32_t seen[TS / 32];
#pragma unroll
        for (int j = 0; j < TS / 32; ++j) {
          const int slot = tile * TS + 32 * j + lane;
          const int64_t kp = reinterpret_cast<const int64_t*>(at + C::POS)[32 * j + lane];
          seen[j] = __ballot_sync(0xffffffffu, slot == own || (slot < W && kp >= 0 && (uint64_t)(p - kp) < (uint64_t)W));
        }
        bool every = true;
#pragma unroll
        for (int j = 0; j < TS / 32; ++j) every &= seen[j] == 0xffffffffu;
        if (!every) {  // a slot that is not seen has step and lo 0, whatever it holds
#pragma unroll
          for (int x = 0; x < TS * NG / 32; ++x) {
            const int slot = (32 * x + lane) / NG;
            if (!((seen[slot >> 5] >> (slot & 31)) & 1u)) {
              reinterpret_cast<uint32_t*>(at + C::KP)[32 * x + lane] = 0;
              reinterpret_cast<uint32_t*>(at + C::VP)[32 * x + lane] = 0;
            }
          }
          __syncwarp();
        }
        // scores of slots (rows) by heads (columns)
        float s[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int r0 = 16 * mt + krow;
          uint32_t c0[(DK / 8 + 3) / 4], c1[(DK / 8 + 3) / 4], p0[NG], p1[NG];
          load_bytes<DK / 8>(at + r0 * C::CODES + t * (DK / 8), c0);
          load_bytes<DK / 8>(at + (r0 + 8) * C::CODES + t * (DK / 8), c1);
          load_bytes<4 * NG>(at + C::KP + r0 * C::PAR, p0);
          load_bytes<4 * NG>(at + C::KP + (r0 + 8) * C::PAR, p1);
          float tot[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (C::LO_MMA) {
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(at + C::KP + r0 * C::PAR + 4 * (t % NG));
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(at + C::KP + (r0 + 8) * C::PAR + 4 * (t % NG));
            mma_bf16_first(tot, w0, w1, __byte_perm(w0, w0, 0x3232), __byte_perm(w1, w1, 0x3232), qlo[0], qlo[1]);
          } else {
#pragma unroll
            for (int a = 0; a < NG; ++a) {
              // with codes as code - 7.5, lo + 7.5 step takes the place of lo
              const float lo0 = C::EXACT ? fmaf(7.5f, q4_step(p0[a]), q4_lo(p0[a])) : q4_lo(p0[a]);
              const float lo1 = C::EXACT ? fmaf(7.5f, q4_step(p1[a]), q4_lo(p1[a])) : q4_lo(p1[a]);
              tot[0] = fmaf(lo0, qs[a][0], tot[0]);
              tot[1] = fmaf(lo0, qs[a][1], tot[1]);
              tot[2] = fmaf(lo1, qs[a][0], tot[2]);
              tot[3] = fmaf(lo1, qs[a][1], tot[3]);
            }
          }
#pragma unroll
          for (int a = 0; a < NG; ++a) {
            float d[4];
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
              if constexpr (C::EXACT) {
                const uint32_t a0 = centred(x0), a1 = centred(x1), a2 = centred(x0 >> 4), a3 = centred(x1 >> 4);
#pragma unroll
                for (int r = 0; r < QT; ++r) {
                  if (k == 0 && r == 0) mma_bf16_first(d, a0, a1, a2, a3, qb[a][k][r][0], qb[a][k][r][1]);
                  else mma_bf16(d, a0, a1, a2, a3, qb[a][k][r][0], qb[a][k][r][1]);
                }
              } else {
                const uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
                if (k == 0) mma_f16_first(d, a0, a1, a2, a3, qb[a][k][0][0], qb[a][k][0][1]);
                else mma_f16(d, a0, a1, a2, a3, qb[a][k][0][0], qb[a][k][0][1]);
              }
            }
            const float s0 = q4_step(p0[a]), s1 = q4_step(p1[a]);
            tot[0] = fmaf(s0, d[0], tot[0]);
            tot[1] = fmaf(s0, d[1], tot[1]);
            tot[2] = fmaf(s1, d[2], tot[2]);
            tot[3] = fmaf(s1, d[3], tot[3]);
          }
          // X: whole scores, rounded here, so that the largest of them and the reference made of it differ by what they
          // should however large they are; else still to be multiplied by f
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][x] = X ? __fmul_rn(tot[x], f[x & 1]) : tot[x];
        }
        if (C::WIDE && huge) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (huge >> (x & 1) & 1u) s[mt][x] *= 16777216.f;
        }
        if (!every) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint32_t bits = seen[mt >> 1] >> (16 * (mt & 1) + krow);
            if (!(bits & 1u)) s[mt][0] = s[mt][1] = -INFINITY;
            if (!(bits & 256u)) s[mt][2] = s[mt][3] = -INFINITY;
          }
        }
        // the references, the weights and their sum
        {
          uint32_t big = 0;
#pragma unroll
          for (int x = 0; x < TS * NG / 32; ++x)
            big = max_bf16x2(big, reinterpret_cast<const uint32_t*>(at + C::VP)[32 * x + lane] & 0x7fff7fffu);
          const uint32_t far = __reduce_max_sync(0xffffffffu, big & 0xffff0000u);  // the largest lo,
          big = __reduce_max_sync(0xffffffffu, big << 16);                         // and the largest step
          if constexpr (!X)
            if (big >= (uint32_t)(127 + MOST_STEP) << 23) return;  // products of which f16 would overflow
          const float size = size_of(big, far);
          float top[2];
          bool rise = false;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            top[c] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) top[c] = fmaxf(top[c], fmaxf(s[mt][c], s[mt][2 + c]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], x));
            top[c] = fmaf(top[c], X ? 1.f : f[c], size);
            rise |= top[c] > ref[c] + 14.f;
          }
          if (__any_sync(0xffffffffu, rise)) {
            uint32_t small = 0xffffffffu;  // the smallest step of a slot that is seen
#pragma unroll
            for (int x = 0; x < TS * NG / 32; ++x) {
              const int slot = (32 * x + lane) / NG;
              if (every || ((seen[slot >> 5] >> (slot & 31)) & 1u))
                small = min(small, reinterpret_cast<const uint32_t*>(at + C::VP)[32 * x + lane] << 16);
            }
            const bool apart = (int)(big >> 23) - (int)(__reduce_min_sync(0xffffffffu, small) >> 23) > 8;
            if constexpr (!X) {  // nothing of this tile is counted yet
              const bool steep = (fabsf(top[0]) >= 0x1p20f && top[0] != -INFINITY) ||
                                 (fabsf(top[1]) >= 0x1p20f && top[1] != -INFINITY);
              if (__any_sync(0xffffffffu, apart || steep)) return;
            } else if (apart) {
              // steps far apart: every slot with its own, so that large values of little weight take no precision from others
              top[0] = top[1] = -INFINITY;
#pragma unroll
              for (int x = 0; x < 2 * MT; ++x) {
                uint32_t par[NG];
                load_bytes<4 * NG>(at + C::VP + (8 * x + krow) * C::PAR, par);
                float step = 0.f, lo = 0.f;
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                  step = fmaxf(step, q4_step(par[a]));
                  lo = fmaxf(lo, fabsf(q4_lo(par[a])));
                }
                const float slot_size = size_of(__float_as_uint(step), __float_as_uint(lo));
#pragma unroll
                for (int c = 0; c < 2; ++c) top[c] = fmaxf(top[c], s[x / 2][x % 2 * 2 + c] + slot_size);
              }
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], x));
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float next = top[c] > ref[c] + 14.f ? top[c] - 6.f : ref[c];
              const float fade = next == -INFINITY ? 1.f : exp2_approx(ref[c] - next);
              ref[c] = next;
              l[c] *= fade;
#pragma unroll
              for (int j = 0; j < TILES; ++j) {
                acc[j][c] *= fade;
                acc[j][2 + c] *= fade;
              }
#pragma unroll
              for (int a = 0; a < NG; ++a) low[a][c] *= fade;
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float r = ref[c] == -INFINITY ? 0.f : ref[c];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              s[mt][c] = exp2_approx(X ? s[mt][c] - r : fmaf(s[mt][c], f[c], -r));
              s[mt][2 + c] = exp2_approx(X ? s[mt][2 + c] - r : fmaf(s[mt][2 + c], f[c], -r));
              l[c] += s[mt][c] + s[mt][2 + c];
            }
          }
        }
        // weights x values
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
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
#pragma unroll
          for (int a = 0; a < NG; ++a) {
            // with codes as code - 7.5, lo + 7.5 step takes the place of lo. In f16 the odd steps of 16 slots take the codes
            // from the other end: value = lo + 15 step - step (15 - code)
            const float up = X ? 7.5f : mt & 1 ? 15.f : 0.f;
            const float lo0 = fmaf(up, q4_step(p0[a]), q4_lo(p0[a])), lo1 = fmaf(up, q4_step(p1[a]), q4_lo(p1[a]));
            const float st0 = !X && mt & 1 ? -q4_step(p0[a]) : q4_step(p0[a]);
            const float st1 = !X && mt & 1 ? -q4_step(p1[a]) : q4_step(p1[a]);
            low[a][0] = fmaf(s[mt][0], lo0, fmaf(s[mt][2], lo1, low[a][0]));
            low[a][1] = fmaf(s[mt][1], lo0, fmaf(s[mt][3], lo1, low[a][1]));
            float e[4] = {s[mt][0] * st0, s[mt][1] * st0, s[mt][2] * st1, s[mt][3] * st1};
            if constexpr (PAIR && X) {
              if (second) e[0] = e[1] = e[2] = e[3] = 0.f;  // columns 4 to 7 have no part in it
            } else if constexpr (PAIR) {  // columns 4 to 7: what the first term leaves
              less_f16(e[0], e[1], pack_f16(e[0], e[1]), second);
              less_f16(e[2], e[3], pack_f16(e[2], e[3]), second);
            }
            uint32_t b0[TERMS], b1[TERMS];
#pragma unroll
            for (int r = 0; r < TERMS; ++r) {
              const uint32_t e0 = X ? pack_bf16(e[0], e[1]) : pack_f16(e[0], e[1]);
              const uint32_t e1 = X ? pack_bf16(e[2], e[3]) : pack_f16(e[2], e[3]);
              b0[r] = transpose8(e0);
              b1[r] = transpose8(e1);
              if constexpr (X) {
                e[0] -= __uint_as_float(e0 << 16); e[1] -= __uint_as_float(e0 & 0xffff0000u);
                e[2] -= __uint_as_float(e1 << 16); e[3] -= __uint_as_float(e1 & 0xffff0000u);
              } else if constexpr (TERMS > 1) {
                less_f16(e[0], e[1], e0, F16_MINUS_ONE);
                less_f16(e[2], e[3], e1, F16_MINUS_ONE);
              }
            }
#pragma unroll
            for (int j = 0; j < GS / 16; ++j) {
              const int i16 = a * (GS / 16) + j;  // channels [16 i16, 16 i16 + 16): byte i16 of the lanes' parts
              const uint32_t sel = 0x4400u + 0x1111u * (i16 % 4);
              // that byte of two slots in the low bytes of the halves: low four bits for rows g, the others for rows g + 8
              const uint32_t x = __byte_perm(w[0][i16 / 4], w[1][i16 / 4], sel);
              const uint32_t y = __byte_perm(w[2][i16 / 4], w[3][i16 / 4], sel);
              if constexpr (X) {
                const uint32_t a0 = centred(x), a1 = centred(x >> 4), a2 = centred(y), a3 = centred(y >> 4);
                // the matrix unit's sums are cut off, not rounded: a short one, then a rounded addition
                float d[4];
                mma_bf16_first(d, a0, a1, a2, a3, b0[0], b1[0]);
#pragma unroll
                for (int r = 1; r < TERMS; ++r) mma_bf16(d, a0, a1, a2, a3, b0[r], b1[r]);
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2)
                  acc[i16][e2] = C::EXACT ? acc[i16][e2] + d[e2] : fmaf(d[e2], e2 < 2 ? 0x1p-24f : 0x1p-20f, acc[i16][e2]);
              } else {
                const uint32_t u = mt & 1 ? ~x : x, v = mt & 1 ? ~y : y;
                const uint32_t a0 = u & 0x000f000fu, a1 = u & 0x00f000f0u, a2 = v & 0x000f000fu, a3 = v & 0x00f000f0u;
#pragma unroll
                for (int r = 0; r < TERMS; ++r) mma_f16(acc[i16], a0, a1, a2, a3, b0[r], b1[r]);
              }
            }
          }
        }
        __syncwarp();
        copy(i + C::STAGES);
      }
    };
    if constexpr (!C::EXACT) walk(std::false_type{});
    walk(std::true_type{});

    // this warp's part: heads 2 t and 2 t + 1, channels 16 i + 2 g and 16 i + 2 g + 1
    cp_async_wait_all();  // also of copies that the position then made needless
    __syncthreads();      // the stages are free
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
        const float x = C::EXACT ? acc[i][c] : acc[i][c] * 16777216.f;        // f16: the codes' 2^-24
        const float y = C::EXACT ? acc[i][2 + c] : acc[i][2 + c] * 1048576.f;  // and 2^-20
        const float z = PAIR && t >= 2 ? 0.f : low[a][c];  // once per head
        *reinterpret_cast<float2*>(row + 16 * i + 2 * g) = make_float2(x + z, y + z);
      }
      if (g == 0) {
        row[DK] = ref[c];
        row[DK + 1] = l[c];
      }
    }
    __syncthreads();
    const bool whole = lo_t == 0 && hi_t == n;
    if (shared && threadIdx.x == 0) {
      if (lo_t == 0) span[b * units + unit].x = blockIdx.x;
      if (hi_t == n) span[b * units + unit].y = blockIdx.x;
    }
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
        out = fmaf(PAIR ? x[c] + x[4 * (DK + 2) + c] : x[c], fade, out);
      }
      if (whole) {
        o[(b * H + h0 + h) * DK + c] = from_f32<T>(p < 0 ? 0.f : out / L);
      } else {
        float* to = part + (2 * (int64_t)blockIdx.x + (lo_t == 0)) * HEADS * (DK + 2) + h * (DK + 2);
        to[c] = out;
        if (c == 0) {
          to[DK] = M;
          to[DK + 1] = L;
        }
      }
    }
    if (from >= until) break;
    // the next unit: its copies come into what was just read
    __syncthreads();
    if (hi_t == n && unit + 1 == units) {  // the next row that sees something
      row_first += (int64_t)cost_of(n, opening) * units;
      do n = tiles_of<TS>(pos[++b], W);
      while (n == 0);
    }
  }
}

// Joins the partials of each (row, unit) that several CTAs of a shared launch have had, in a fixed order; a row that sees
// nothing (a negative position) is zero. A CTA per head, row and unit, the partials spread over its threads.
constexpr int JOIN = 512;
template <typename T, int DK>
__global__ void __launch_bounds__(JOIN) q4_attn_join_kernel(const int64_t* __restrict__ pos, const float* __restrict__ part,
                                                           const int2* __restrict__ span, T* __restrict__ o, int H, int HKV,
                                                           int head_tiles) {
  constexpr int LANES = JOIN / DK;  // threads per channel
  __shared__ float tops[JOIN / 32], sums[LANES][DK + 1];
  const int units = HKV * head_tiles, G = H / HKV, unit = blockIdx.y, kh = unit / head_tiles, ht = unit - kh * head_tiles;
  const int h = blockIdx.x, tid = threadIdx.x;
  const int64_t b = blockIdx.z;
  if (ht * HEADS + h >= G) return;
  T* out = o + (b * H + kh * G + ht * HEADS + h) * DK;
  grid_wait();
  grid_release();
  const int2 ends = span[b * units + unit];
  if (pos[b] < 0) {
    if (tid < DK) out[tid] = from_f32<T>(0.f);
    return;
  }
  const int lo = ends.x, hi = ends.y;
  if (lo == hi) return;  // that CTA wrote the output
  // the first CTA ends within the unit (or with it), the others start within it
  auto row = [&](int i) { return part + ((2 * (int64_t)i + (i == lo)) * HEADS + h) * (DK + 2); };
  float top = -INFINITY;
  for (int i = lo + tid; i <= hi; i += JOIN) top = fmaxf(top, row(i)[DK]);
  top = warp_max(top);
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < JOIN / 32; ++i) top = fmaxf(top, tops[i]);
  const int c = tid % DK, lane = tid / DK;
  float acc = 0.f, L = 0.f;
  if (lane < LANES) {
#pragma unroll 4
    for (int i = lo + lane; i <= hi; i += LANES) {
      const float* x = row(i);
      const float fade = x[DK] == -INFINITY ? 0.f : exp2f(x[DK] - top);
      L = fmaf(x[DK + 1], fade, L);
      acc = fmaf(x[c], fade, acc);
    }
    sums[lane][c] = acc;
    if (c == 0) sums[lane][DK] = L;
  }
  __syncthreads();
  if (tid < DK) {
    acc = L = 0.f;
#pragma unroll
    for (int i = 0; i < LANES; ++i) {
      acc += sums[i][c];
      L += sums[i][DK];
    }
    out[c] = from_f32<T>(acc / L);
  }
}

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      v = 148;
    return v > 0 ? v : 148;
  }();
  return n;
}

// CTAs of a shared launch, 0 for a CTA per row and unit: a window of few tiles is one CTA's work, and many units
// fill the SMs by themselves
int shared_ctas(int B, int units, int DK, int W) {
  const int tiles = (W + Q4_TILE - 1) / Q4_TILE, slots = sm_count() * ctas_per_sm(DK);
  if (tiles <= 16 || (int64_t)B * units >= 8 * slots) return 0;
  return slots;
}

int head_tiles_of(int H, int HKV) { return (H / HKV + HEADS - 1) / HEADS; }

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" size_t vb_q4_attend_workspace(int B, int H, int HKV, int DK, int W) {
  if (B <= 0 || H <= 0 || HKV <= 0 || H % HKV || DK <= 0 || W <= 0) return 0;
  const int units = HKV * head_tiles_of(H, HKV), ctas = shared_ctas(B, units, DK, W);
  if (ctas == 0) return 0;
  return sizeof(int2) * (size_t)B * units + sizeof(float) * 2 * (size_t)ctas * HEADS * (DK + 2);
}

extern "C" int vb_q4_attend(const void* q, int64_t q_row, const void* k_new, int64_t k_row, const void* v_new,
                            int64_t v_row, const int64_t* pos, void* k_codes, void* k_params, void* v_codes,
                            void* v_params, int64_t* ring_pos, void* o, void* workspace, int B, int H, int HKV, int DK,
                            int W, int SLOTS, int dtype, void* stream) {
  VB_REQUIRE(B >= 0 && H >= 1 && HKV >= 1 && W >= 1, "q4_attend: bad shape B=%d H=%d HKV=%d W=%d", B, H, HKV, W);
  VB_REQUIRE(H % HKV == 0, "q4_attend: %d query heads are not a multiple of %d key heads", H, HKV);
  VB_REQUIRE(DK >= 16 && DK <= 128 && DK % 16 == 0, "q4_attend: head dimension %d must be a multiple of 16 up to 128", DK);
  VB_REQUIRE(SLOTS % Q4_TILE == 0 && SLOTS >= W, "q4_attend: %d slots must be a multiple of %d holding the window %d",
             SLOTS, Q4_TILE, W);
  VB_REQUIRE(dtype_size(dtype) > 0, "q4_attend: unsupported dtype code %d", dtype);
  if (B == 0) return VB_OK;
  VB_REQUIRE(q && k_new && v_new && pos && k_codes && k_params && v_codes && v_params && ring_pos && o,
             "q4_attend: null pointer");
  VB_REQUIRE(aligned16(k_codes) && aligned16(k_params) && aligned16(v_codes) && aligned16(v_params) && aligned16(ring_pos),
             "q4_attend: the ring's buffers must start on 16-byte boundaries");

  const int head_tiles = head_tiles_of(H, HKV), units = HKV * head_tiles, ctas = shared_ctas(B, units, DK, W);
  VB_REQUIRE(ctas == 0 || (workspace != nullptr && aligned16(workspace)),
             "q4_attend: a workspace of vb_q4_attend_workspace bytes must start on a 16-byte boundary");
  VB_REQUIRE(B <= 65535 && units <= 65535, "q4_attend: %d rows of %d head tiles exceed the grid", B, units);
  const Ring ring{(uint8_t*)k_codes, (uint32_t*)k_params, (uint8_t*)v_codes, (uint32_t*)v_params, ring_pos};
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)DK);
  const int q_vec = aligned16(q) && (q_row * dtype_size(dtype)) % 16 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  int2* span = (int2*)workspace;  // first, then the partials
  float* part = (float*)(span + (ctas ? (size_t)B * units : 0));
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    auto run = [&](auto dk) -> int {
      constexpr int D = decltype(dk)::value;
      auto attend = [&](auto pair) -> int {
        return launch_early("q4_attend", q4_attn_kernel<T, D, decltype(pair)::value>, ctas ? dim3(ctas) : dim3(units, B),
                            Q4Attn<T, D>::AW * 32, Q4Attn<T, D>::SMEM, 1, st, (const T*)q, q_row, q_vec, (const T*)k_new,
                            k_row, (const T*)v_new, v_row, pos, ring, (T*)o, part, span, ctas != 0, B, H, HKV, head_tiles,
                            W, SLOTS, scale_log2);
      };
      int rc;
      if constexpr (Q4Attn<T, D>::EXACT) rc = attend(std::false_type{});
      else rc = H / HKV <= HEADS / 2 ? attend(std::true_type{}) : attend(std::false_type{});
      if (rc || ctas == 0) return rc;
      return launch_early("q4_attend join", q4_attn_join_kernel<T, D>, dim3(HEADS, units, B), JOIN, 0, 1, st, pos,
                          (const float*)part, (const int2*)span, (T*)o, H, HKV, head_tiles);
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
