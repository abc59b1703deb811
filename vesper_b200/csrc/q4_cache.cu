// The 4-bit ring cache: tokens quantised as they are written, and read back at given positions
// (a RingKVCache, vesper/attention.py:63-139, whose keys and values take five bits a channel).
// The format is q4.cuh's. One thread per eight channels of a token's key or value: a group's lanes
// share its extremes by shuffles. HBM bound: 2 bytes in and 0.625 out per bf16 channel.
#include "q4.cuh"

namespace vb {
namespace {

constexpr int NT = 256;

struct Q4Ring {
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  int64_t* pos;
};

// tokens [B, N] at positions pos; a token is written when its position is not negative and no
// later token of the chunk takes its slot (positions being consecutive, the one W later)
template <typename T>
__global__ void __launch_bounds__(NT) q4_write_kernel(Q4Ring ring, const T* __restrict__ k, int64_t kb, int64_t kt,
                                                      const T* __restrict__ v, int64_t vb_, int64_t vt,
                                                      const int64_t* __restrict__ pos, int64_t rows, int N, int HKV,
                                                      int DK, int W, int SLOTS) {
  const int per = DK / 8, gs = q4_group(DK), ng = DK / gs;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t row = id / per;  // (b, token, head)
  const int c0 = (int)(id - row * per) * 8;
  const bool value = blockIdx.y;
  const bool inside = row < rows;
  const int64_t token = inside ? row / HKV : 0;
  const int kh = inside ? (int)(row - token * HKV) : 0;
  const int64_t b = token / N;
  const int i = (int)(token - b * N);
  const int64_t p = inside ? pos[token] : -1;
  const bool live = p >= 0 && !(i + W < N && pos[token + W] >= 0);
  float x[8];
  const T* src = value ? v + b * vb_ + i * vt + (int64_t)kh * DK + c0 : k + b * kb + i * kt + (int64_t)kh * DK + c0;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = live ? to_f32<T>(src[e]) : 0.f;
  float low = x[0], high = x[0];
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    low = fminf(low, x[e]);
    high = fmaxf(high, x[e]);
    nan |= x[e] != x[e];
  }
  if (nan) low = high = __uint_as_float(0x7fc00000u);
  // the lanes of a group are neighbours (DK / 8 is a multiple of a group's lanes)
  for (int o = 1; o < gs / 8; o <<= 1) {
    const float l2 = __shfl_xor_sync(0xffffffffu, low, o), h2 = __shfl_xor_sync(0xffffffffu, high, o);
    const bool bad = low != low || l2 != l2;
    low = bad ? __uint_as_float(0x7fc00000u) : fminf(low, l2);
    high = bad ? low : fmaxf(high, h2);
  }
  if (!live) return;
  float step, lo;
  q4_params(low, high, step, lo);
  const float inverse = step > 0.f ? 1.0f / step : 0.f;
  const int slot = (int)(p % W);
  const int64_t at = (b * HKV + kh) * SLOTS + slot;
  uint8_t* codes = (value ? ring.v_codes : ring.k_codes) + at * (DK / 2);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t byte = q4_code(x[e], step, lo, inverse) | q4_code(x[e + 1], step, lo, inverse) << 4;
    codes[(value ? q4_value_place(DK, c0 + e) : q4_key_place(DK, c0 + e)) / 2] = (uint8_t)byte;
  }
  if (c0 % gs == 0) (value ? ring.v_params : ring.k_params)[at * ng + c0 / gs] = q4_pack_params(step, lo);
  if (!value && kh == 0 && c0 == 0) ring.pos[b * SLOTS + slot] = p;
}

template <typename T>
__global__ void __launch_bounds__(NT) q4_read_kernel(Q4Ring ring, const int64_t* __restrict__ pos, T* __restrict__ k,
                                                     T* __restrict__ v, uint8_t* __restrict__ held, int64_t rows, int N,
                                                     int HKV, int DK, int W, int SLOTS) {
  const int per = DK / 8, gs = q4_group(DK), ng = DK / gs;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t row = id / per;
  if (row >= rows) return;
  const int c0 = (int)(id - row * per) * 8;
  const bool value = blockIdx.y;
  const int64_t token = row / HKV;
  const int kh = (int)(row - token * HKV);
  const int64_t b = token / N, p = pos[token];
  const int slot = p >= 0 ? (int)(p % W) : 0;
  const bool have = p >= 0 && ring.pos[b * SLOTS + slot] == p;
  const int64_t at = (b * HKV + kh) * SLOTS + slot;
  const uint8_t* codes = (value ? ring.v_codes : ring.k_codes) + at * (DK / 2);
  const uint32_t pr = (value ? ring.v_params : ring.k_params)[at * ng + c0 / gs];
  T* dst = (value ? v : k) + row * DK + c0;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t byte = codes[(value ? q4_value_place(DK, c0 + e) : q4_key_place(DK, c0 + e)) / 2];
    dst[e] = from_f32<T>(have ? fmaf((float)(byte & 15u), q4_step(pr), q4_lo(pr)) : 0.f);
    dst[e + 1] = from_f32<T>(have ? fmaf((float)(byte >> 4), q4_step(pr), q4_lo(pr)) : 0.f);
  }
  if (!value && kh == 0 && c0 == 0) held[token] = have ? 1 : 0;
}

int check_ring(const char* what, int B, int N, int HKV, int DK, int W, int SLOTS, int dtype) {
  VB_REQUIRE(B >= 0 && N >= 0 && HKV >= 1 && W >= 1, "%s: bad shape B=%d N=%d HKV=%d W=%d", what, B, N, HKV, W);
  VB_REQUIRE(DK >= 16 && DK <= 128 && DK % 16 == 0, "%s: head dimension %d must be a multiple of 16 up to 128", what,
             DK);
  VB_REQUIRE(SLOTS % Q4_TILE == 0 && SLOTS >= W, "%s: %d slots must be a multiple of %d holding the window %d", what,
             SLOTS, Q4_TILE, W);
  VB_REQUIRE(dtype_size(dtype) > 0, "%s: unsupported dtype code %d", what, dtype);
  const int64_t blocks = ((int64_t)B * N * HKV * (DK / 8) + NT - 1) / NT;
  VB_REQUIRE(blocks < (int64_t(1) << 31), "%s: %d x %d tokens exceed the grid", what, B, N);
  return VB_OK;
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
  const int64_t rows = (int64_t)B * N * HKV;
  const dim3 grid((unsigned)((rows * (DK / 8) + NT - 1) / NT), 2);
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    q4_write_kernel<T><<<grid, NT, 0, (cudaStream_t)stream>>>(ring, (const T*)k, k_batch, k_token, (const T*)v, v_batch,
                                                              v_token, pos, rows, N, HKV, DK, W, SLOTS);
    VB_LAUNCH_CHECK("q4_write");
    return VB_OK;
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
  const int64_t rows = (int64_t)B * N * HKV;
  const dim3 grid((unsigned)((rows * (DK / 8) + NT - 1) / NT), 2);
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    q4_read_kernel<T><<<grid, NT, 0, (cudaStream_t)stream>>>(ring, pos, (T*)k, (T*)v, held, rows, N, HKV, DK, W, SLOTS);
    VB_LAUNCH_CHECK("q4_read");
    return VB_OK;
  });
}
