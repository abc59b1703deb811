// The 4-bit ring cache: tokens quantised as they are written, and read back at given positions
// (a RingKVCache, vesper/attention.py:63-139, whose keys and values take five bits a channel).
// The format is q4.cuh's. A CTA takes some tokens of one (row, key head) (16 at DK 128), keys and values: a group's
// extremes from a thread's registers and its neighbour's, and the codes by way of shared memory, where they find their
// places a byte or a word at a time and leave or arrive in 8-byte pieces of consecutive slots. HBM bound: 2 bytes in and
// 0.625 out per bf16 channel, or the reverse. 4 x 32701 tokens, 8 heads of 128, are written in 144 us (4.9 TB/s, 75 % of
// a plain copy's rate; instructions issue in 80 % of the cycles) and read back in 148 us (4.75 TB/s, 73 %; instructions
// issue in 72 % of the cycles, and memory would take more: float32, with half the codes for its bytes, is stored at 4.9 TB/s
// where this stores 3.6). float32 tokens, with twice the bytes for each, are written at 6.1
// TB/s (93 %). 64 x 2048 tokens into a window of 512, two heads of 64: 6.3 and 5.9 us.
#include <type_traits>

#include "launch.cuh"
#include "q4.cuh"

namespace vb {
namespace {

constexpr int NT = 128;  // more and smaller CTAs start and end in turn (with 256, read back: 4 x 32701 tokens of 8 heads of 128
                         // 151 us against 148, 4 x 16384 of 8 heads of 64 in float32 61 against 55)

// How a CTA's threads lie over its tokens. Writing: a thread per sixteen channels of a group, in two pieces of eight half a
// group apart, so that half of a group's work is a thread's own and two neighbours read 32 bytes of bf16 at a time (4 x
// 32701 tokens, 8 heads of 128: 144 us, with a thread per eight channels 175). Reading: a thread per eight channels, two
// passes over the tokens, whose float32 stores cover whole lines (4 x 16384 tokens of 8 heads of 64: 61 us, in two
// pieces 75). For codes a thread per 8 bytes, for parameters a thread per group.
template <int DK>
struct Layout {
  static constexpr int GS = q4_group(DK), NG = DK / GS, HALF = DK / 2;
  static constexpr int PER = DK / 16, ROWS = NT / PER;             // writing: threads per token, tokens per CTA
  static constexpr int GL = GS / 16, PIECE = GS / 2;               // threads per group, from one piece to the other
  static constexpr int PER8 = DK / 8, PASS = NT / PER8, READ_ROWS = 2 * PASS;  // reading
  static_assert(ROWS * (HALF / 8) <= NT && ROWS * NG <= NT && READ_ROWS <= ROWS, "one step each");
};

struct Q4Ring {
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  int64_t* pos;
};

__device__ __forceinline__ int slot_of(int64_t p, int W) {
  return p < ((int64_t)1 << 32) ? (int)((uint32_t)p % (uint32_t)W) : (int)(p % W);
}

// eight consecutive elements as they lie in memory; `vec`: on a 16-byte boundary
template <typename T>
struct __align__(16) Raw8 {
  T v[8];
  __device__ __forceinline__ void load(const T* __restrict__ p, int vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
  }
};

// the smallest and the largest of sixteen elements, NaN if one is; 16-bit types two at a time
__device__ __forceinline__ void extremes(const Raw8<float> (&raw)[2], float& low, float& high) {
  low = high = raw[0].v[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) {
    low = min_nan(low, raw[e / 8].v[e % 8]);
    high = max_nan(high, raw[e / 8].v[e % 8]);
  }
}
template <typename T2, typename T>
__device__ __forceinline__ void extremes2(const Raw8<T> (&raw)[2], float& low, float& high) {
  const T2 *w = reinterpret_cast<const T2*>(raw[0].v), *u = reinterpret_cast<const T2*>(raw[1].v);
  T2 l = __hmin2_nan(w[0], u[0]), h = __hmax2_nan(w[0], u[0]);
#pragma unroll
  for (int e = 1; e < 4; ++e) {
    l = __hmin2_nan(l, __hmin2_nan(w[e], u[e]));
    h = __hmax2_nan(h, __hmax2_nan(w[e], u[e]));
  }
  low = min_nan(__low2float(l), __high2float(l));
  high = max_nan(__low2float(h), __high2float(h));
}
__device__ __forceinline__ void extremes(const Raw8<__nv_bfloat16> (&raw)[2], float& low, float& high) {
  extremes2<__nv_bfloat162>(raw, low, high);
}
__device__ __forceinline__ void extremes(const Raw8<__half> (&raw)[2], float& low, float& high) {
  extremes2<__half2>(raw, low, high);
}

// Tokens [B, N] at positions pos, negative ones (padding, at either end of a row) not written. Of those that share a
// slot the last is kept: only the last W before a row's padding are looked at.
template <typename T, int DK>
__global__ void __launch_bounds__(NT) q4_write_kernel(Q4Ring ring, const T* __restrict__ k, int64_t kb, int64_t kt,
                                                      const T* __restrict__ v, int64_t vb_, int64_t vt,
                                                      const int64_t* __restrict__ pos, int vec, int N, int HKV,
                                                      int W, int SLOTS) {
  using L = Layout<DK>;
  constexpr int PER = L::PER, ROWS = L::ROWS, GS = L::GS, NG = L::NG, HALF = L::HALF, PIECE = L::PIECE;
  __shared__ __align__(16) uint8_t codes[2][ROWS][HALF];
  __shared__ uint32_t params[2][ROWS][NG];
  __shared__ int slots[ROWS];  // -1: not written
  // consecutive CTAs take consecutive tokens of a head, whose slots they fill side by side (4 x 32701 tokens, 8 heads of
  // 128: 144 us; with a token's heads next to each other 154)
  const int tid = threadIdx.x, block = blockIdx.x, kh = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int mine = tid / PER, c0 = tid % PER / L::GL * GS + tid % PER % L::GL * 8;
  const bool busy = ROWS * PER == NT || tid < ROWS * PER;
  grid_wait();
  grid_release();
  const int64_t* at = pos + b * N;
  Raw8<T> raw[2][2];       // [keys, values][piece]
  int end = N, first = 0;  // the tokens before the padding at the row's end, and the first of this CTA's
  int64_t p = -1;
  auto fetch = [&] {  // every load of the thread in flight before any is used
    first = max(0, end - W) + block * ROWS;
    if (tid < ROWS && first + tid < end) p = at[first + tid];
    if (!busy || first + mine >= end) return;
    const T* from[2] = {k + b * kb + (int64_t)(first + mine) * kt + (int64_t)kh * DK + c0,
                        v + b * vb_ + (int64_t)(first + mine) * vt + (int64_t)kh * DK + c0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      raw[0][i].load(from[0] + i * PIECE, vec);
      raw[1][i].load(from[1] + i * PIECE, vec);
    }
  };
  fetch();  // as if there were no padding at the end
  if (at[N - 1] < 0) {
    do {  // whole warps look for its beginning, 32 tokens at a time
      const int i = end - 1 - (tid & 31);
      const uint32_t found = __ballot_sync(0xffffffffu, i >= 0 && at[i] >= 0);
      if (found) {
        end -= __ffs(found) - 1;
        break;
      }
      end -= min(end, 32);
    } while (end > 0);
    p = -1;
    fetch();
  }
  if (first >= end) return;
  if (tid < ROWS) {
    slots[tid] = p >= 0 ? slot_of(p, W) : -1;
    if (kh == 0 && p >= 0) ring.pos[b * SLOTS + slots[tid]] = p;
  }
#pragma unroll
  for (int value = 0; value < 2; ++value) {
    // a token that is not written holds what it may here and is left out below
    float x[2][8], low, high;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = to_f32<T>(raw[value][i].v[e]);
    extremes(raw[value], low, high);
    if constexpr (L::GL == 2) {  // the other half of the group: a neighbour's (PER is even)
      low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, 1));
      high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, 1));
    }
    float step, lo, inverse;
    q4_params(low, high, step, lo, inverse);
    const uint32_t w0 = q4_codes(x[0], step, lo, inverse), w1 = q4_codes(x[1], step, lo, inverse);
    if (!busy) continue;
    uint8_t* to = codes[value][mine];
    if (value && GS == 32) {  // the two pieces' codes are neighbours
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<uint16_t*>(to + q4_value_place(DK, c0 + 2 * e) / 2) =
            (uint16_t)__byte_perm(w0, w1, e | (4 + e) << 4);
    } else if (value) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        to[q4_value_place(DK, c0 + 2 * e) / 2] = (uint8_t)(w0 >> (8 * e));
        to[q4_value_place(DK, c0 + PIECE + 2 * e) / 2] = (uint8_t)(w1 >> (8 * e));
      }
    } else if (GS == 32) {
      *reinterpret_cast<uint32_t*>(to + q4_key_place(DK, c0) / 2) = w0;
      *reinterpret_cast<uint32_t*>(to + q4_key_place(DK, c0 + PIECE) / 2) = w1;
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        *reinterpret_cast<uint16_t*>(to + q4_key_place(DK, c0 + 4 * e) / 2) = (uint16_t)(w0 >> (16 * e));
        *reinterpret_cast<uint16_t*>(to + q4_key_place(DK, c0 + PIECE + 4 * e) / 2) = (uint16_t)(w1 >> (16 * e));
      }
    }
    if (c0 % GS == 0) params[value][mine][c0 / GS] = q4_pack_params(step, lo);
  }
  __syncthreads();
  const int64_t base = (b * HKV + kh) * SLOTS;
  {
    const int row = tid / (HALF / 8), c = tid % (HALF / 8);
    if (row < ROWS && slots[row] >= 0) {
      const int64_t to = (base + slots[row]) * (HALF / 8) + c;
      reinterpret_cast<uint2*>(ring.k_codes)[to] = reinterpret_cast<const uint2*>(codes[0][row])[c];
      reinterpret_cast<uint2*>(ring.v_codes)[to] = reinterpret_cast<const uint2*>(codes[1][row])[c];
    }
  }
  const int row = tid / NG, g = tid % NG;
  if (row < ROWS && slots[row] >= 0) {
    const int64_t to = (base + slots[row]) * NG + g;
    ring.k_params[to] = params[0][row][g];
    ring.v_params[to] = params[1][row][g];
  }
}

template <typename T, int DK>
__global__ void __launch_bounds__(NT) q4_read_kernel(Q4Ring ring, const int64_t* __restrict__ pos, T* __restrict__ k,
                                                     T* __restrict__ v, uint8_t* __restrict__ held, int N, int HKV,
                                                     int W, int SLOTS) {
  using L = Layout<DK>;
  constexpr int PER = L::PER8, RP = L::PASS, ROWS = L::READ_ROWS, GS = L::GS, NG = L::NG, HALF = L::HALF;
  __shared__ __align__(16) uint8_t codes[2][ROWS][HALF];
  __shared__ uint32_t params[2][ROWS][NG];
  __shared__ int slots[ROWS];  // -1: no position that a ring could hold
  __shared__ bool have[ROWS];
  // consecutive CTAs take the heads of the same tokens, whose values lie side by side (the same, with 256 threads:
  // 151 us; by head 157)
  const int tid = threadIdx.x, block = blockIdx.x / HKV, kh = blockIdx.x - block * HKV, first = block * ROWS;
  const int64_t b = blockIdx.y;
  grid_wait();
  grid_release();
  const int64_t p = tid < ROWS && first + tid < N ? pos[b * N + first + tid] : -1;
  if (tid < ROWS) slots[tid] = p >= 0 ? slot_of(p, W) : -1;
  __syncthreads();
  const int64_t base = (b * HKV + kh) * SLOTS;
  // the slot is read before it is known to hold the position
  if (tid < ROWS) {
    have[tid] = p >= 0 && ring.pos[b * SLOTS + slots[tid]] == p;
    if (kh == 0 && first + tid < N) held[b * N + first + tid] = have[tid];
  }
  {
    const int row = tid / (HALF / 8), c = tid % (HALF / 8);
    if (row < ROWS && slots[row] >= 0) {
      const int64_t from = (base + slots[row]) * (HALF / 8) + c;
      reinterpret_cast<uint2*>(codes[0][row])[c] = reinterpret_cast<const uint2*>(ring.k_codes)[from];
      reinterpret_cast<uint2*>(codes[1][row])[c] = reinterpret_cast<const uint2*>(ring.v_codes)[from];
    }
  }
  {
    const int row = tid / NG, g = tid % NG;
    if (row < ROWS && slots[row] >= 0) {
      const int64_t from = (base + slots[row]) * NG + g;
      params[0][row][g] = ring.k_params[from];
      params[1][row][g] = ring.v_params[from];
    }
  }
  __syncthreads();
  const int row0 = tid / PER, c0 = tid % PER * 8;
  if (RP * PER < NT && tid >= RP * PER) return;
#pragma unroll
  for (int value = 0; value < 2; ++value)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + i * RP;
      if (first + row >= N) continue;
      float x[8];
      if (have[row]) {
        const uint8_t* from = codes[value][row];
        uint32_t w = 0;
        if (value) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w |= (uint32_t)from[q4_value_place(DK, c0 + 2 * e) / 2] << (8 * e);
        } else if constexpr (GS == 32) {
          w = *reinterpret_cast<const uint32_t*>(from + q4_key_place(DK, c0) / 2);
        } else {
          w = *reinterpret_cast<const uint16_t*>(from + q4_key_place(DK, c0) / 2) |
              (uint32_t)*reinterpret_cast<const uint16_t*>(from + q4_key_place(DK, c0 + 4) / 2) << 16;
        }
        const uint32_t pr = params[value][row][c0 / GS];
        q4_values(w, q4_step(pr), q4_lo(pr), x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      store_vec<T, 8>((value ? v : k) + ((b * N + first + row) * HKV + kh) * DK + c0, x);
    }
}

int check_ring(const char* what, int B, int N, int HKV, int DK, int W, int SLOTS, int dtype) {
  VB_REQUIRE(B >= 0 && N >= 0 && HKV >= 1 && W >= 1, "%s: bad shape B=%d N=%d HKV=%d W=%d", what, B, N, HKV, W);
  VB_REQUIRE(DK >= 16 && DK <= 128 && DK % 16 == 0, "%s: head dimension %d must be a multiple of 16 up to 128", what,
             DK);
  VB_REQUIRE(SLOTS % Q4_TILE == 0 && SLOTS >= W, "%s: %d slots must be a multiple of %d holding the window %d", what,
             SLOTS, Q4_TILE, W);
  VB_REQUIRE(dtype_size(dtype) > 0, "%s: unsupported dtype code %d", what, dtype);
  // a CTA's tokens more are still an int
  VB_REQUIRE(B <= 65535 && HKV <= 65535 && N <= 1 << 30 && (int64_t)N * HKV < (int64_t(1) << 31),
             "%s: %d rows of %d tokens x %d key heads exceed the grid", what, B, N, HKV);
  return VB_OK;
}

// runs f with DK as a compile-time constant
template <typename F>
int with_head_dim(int DK, F f) {
  switch (DK) {
    case 16: return f(std::integral_constant<int, 16>{});
    case 32: return f(std::integral_constant<int, 32>{});
    case 48: return f(std::integral_constant<int, 48>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 80: return f(std::integral_constant<int, 80>{});
    case 96: return f(std::integral_constant<int, 96>{});
    case 112: return f(std::integral_constant<int, 112>{});
    default: return f(std::integral_constant<int, 128>{});
  }
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_q4_write(void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t* ring_pos,
                           const void* k, int64_t k_batch, int64_t k_token, const void* v, int64_t v_batch,
                           int64_t v_token, const int64_t* pos, int B, int N, int HKV, int DK, int W, int SLOTS,
                           int dtype, void* stream) {
  int rc = check_ring("q4_write", B, N, HKV, DK, W, SLOTS, dtype);
  if (rc) return rc;
  if (B == 0 || N == 0) return VB_OK;
  VB_REQUIRE(k_codes && k_params && v_codes && v_params && ring_pos && k && v && pos, "q4_write: null pointer");
  const Q4Ring ring{(uint8_t*)k_codes, (uint32_t*)k_params, (uint8_t*)v_codes, (uint32_t*)v_params, ring_pos};
  VB_REQUIRE(aligned16(k_codes) && aligned16(k_params) && aligned16(v_codes) && aligned16(v_params),
             "q4_write: the ring's buffers must start on 16-byte boundaries");
  const int size = dtype_size(dtype);
  const int vec = aligned16(k) && aligned16(v) && k_batch * size % 16 == 0 && k_token * size % 16 == 0 &&
                  v_batch * size % 16 == 0 && v_token * size % 16 == 0;
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return with_head_dim(DK, [&](auto dk) -> int {
      constexpr int D = decltype(dk)::value, ROWS = Layout<D>::ROWS;
      return launch_early("q4_write", q4_write_kernel<T, D>, dim3((min(N, W) + ROWS - 1) / ROWS, HKV, B), NT, 0, 1,
                          (cudaStream_t)stream, ring, (const T*)k, k_batch, k_token, (const T*)v, v_batch, v_token, pos,
                          vec, N, HKV, W, SLOTS);
    });
  });
}

extern "C" int vb_q4_read(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                          const int64_t* ring_pos, const int64_t* pos, void* k, void* v, uint8_t* held, int B, int N,
                          int HKV, int DK, int W, int SLOTS, int dtype, void* stream) {
  int rc = check_ring("q4_read", B, N, HKV, DK, W, SLOTS, dtype);
  if (rc) return rc;
  if (B == 0 || N == 0) return VB_OK;
  VB_REQUIRE(k_codes && k_params && v_codes && v_params && ring_pos && pos && k && v && held, "q4_read: null pointer");
  const Q4Ring ring{(uint8_t*)k_codes, (uint32_t*)k_params, (uint8_t*)v_codes, (uint32_t*)v_params, (int64_t*)ring_pos};
  VB_REQUIRE(aligned16(k_codes) && aligned16(k_params) && aligned16(v_codes) && aligned16(v_params) && aligned16(k) &&
                 aligned16(v),
             "q4_read: the buffers must start on 16-byte boundaries");
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return with_head_dim(DK, [&](auto dk) -> int {
      constexpr int D = decltype(dk)::value, ROWS = Layout<D>::READ_ROWS;
      return launch_early("q4_read", q4_read_kernel<T, D>, dim3((N + ROWS - 1) / ROWS * HKV, B), NT, 0, 1,
                          (cudaStream_t)stream, ring, pos, (T*)k, (T*)v, held, N, HKV, W, SLOTS);
    });
  });
}
