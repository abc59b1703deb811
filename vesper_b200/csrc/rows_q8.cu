// Rows in 8 bits with a float32 scale per row: RMSNorm (with the residual's addition) straight to
// int8 codes, plain rows and squared-ReLU rows to int8 codes, and codes back to values. They feed
// the int8 product of linear_q8.cu; the norm is the column's (vesper/column.py:159-188).
//
// With s the row (x, or x + r), c = max(max|s|, floor) and z = s / c, the norm is
// y = z / sqrt(mean z^2 + eps / c^2) * g. The codes are rint(127 y / max|y|), in which the root
// cancels: with m = max|z g| they are rint(z g * (127 / m)) and the scale is m / (127 rms). So one
// read of the row gives everything: max|s| first, then the sum of z^2 and m together, then the
// codes, the row held in registers throughout. Magnitudes are compared as the bit patterns of
// |v| (unsigned order, infinities above every number and NaN above infinities), so a row holding
// a value that is not finite is seen as such: it gets zero codes and a NaN scale and stands for
// NaN in every place, as the norm of such a row is. Rows of magnitude below 1e-35 are zero.
//
// HBM bound: 4 + 2 + 4 + 1 bytes per channel for a float32 stream with a bf16 addend. Measured, in turn with other
// inputs: 32768 x 512 in 29.7 us (6.2 TB/s, 95 % of a plain copy's rate), 8192 x 5000 in 72 us (6.2 TB/s), 16384 x 2048
// in 56.5 us (6.5 TB/s); a kernel that reads the row anew for every step takes 108, 113 and 84. 64 x 512 takes 1.8 us,
// the latency of one load, two reductions and a launch. Plain rows: 64 x 512 of bf16 1.5 us, 64 x 1536 with the squared ReLU
// 1.7, 32768 x 512 10.1 (5.0 TB/s), 32768 x 1536 with the squared ReLU 37 (4.0 TB/s), 8192 x 4096 of float32 25 (6.7 TB/s).
#include <type_traits>

#include "launch.cuh"

namespace vb {
namespace {

constexpr float TINY_ROW = 1e-35f;
enum { ROW_ADD_NORM = 0, ROW_NORM = 1, ROW_PLAIN = 2, ROW_RELU2 = 3 };

// nearest integer (ties to even) of v, |v| < 2^22, as the low byte of the result
__device__ __forceinline__ uint32_t code_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.0f)) & 0xffu; }

__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (NT > 32) {
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) v = max(v, shared[i]);
  }
  return v;
}
// the sum of `s` and the maximum of `v`
template <int NT>
__device__ __forceinline__ void block_sum_max(float& s, uint32_t& v, float* sums, uint32_t* tops) {
  s = warp_sum(s);
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (NT > 32) {
    if ((threadIdx.x & 31) == 0) {
      sums[threadIdx.x >> 5] = s;
      tops[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      s += sums[i];
      v = max(v, tops[i]);
    }
  }
}

// a row's scale and the factor that makes codes of its values, from their largest magnitude m (as bits) and what the
// values are still to be multiplied by
__device__ __forceinline__ float code_factor(uint32_t top, uint32_t m, float factor, float& scale) {
  const float amax = __uint_as_float(m) * factor;
  const bool finite = top < 0x7f800000u && mag_bits(amax) < 0x7f800000u;
  const bool live = finite && fminf(amax, __uint_as_float(m)) >= TINY_ROW;  // 127 / m stays finite
  scale = live ? amax / 127.0f : finite ? 0.f : __uint_as_float(0x7fc00000u);
  return live ? 127.0f / __uint_as_float(m) : 0.f;
}

// E elements of T (16 or 8 bytes) as floats and back
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* __restrict__ p, float (&x)[E]) {
  if constexpr (E * sizeof(T) == 16) {
    load_vec<T, E>(p, x);
  } else if constexpr (E * sizeof(T) == 32) {
    load_vec<T, E>(p, x);
  } else {
    const uint2 raw = __ldg(reinterpret_cast<const uint2*>(p));
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = to_f32<T>(e[i]);
  }
}

// NT threads per row, each holding VPL pieces of four channels (8 of a 16-bit input) from one read to the codes.
// RPC rows per CTA (more than one only where a warp has a row).
template <typename TX, typename TR, int MODE, int NT, int VPL, int RPC>
__global__ void __launch_bounds__(NT* RPC) rows_q8_kernel(const TX* __restrict__ x, int64_t ldx, const TR* __restrict__ r,
                                                          const float* __restrict__ w, float* __restrict__ sum,
                                                          int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                          int64_t rows, int width, float floor_, float eps) {
  constexpr bool NORM = MODE == ROW_ADD_NORM || MODE == ROW_NORM;
  constexpr int E = sizeof(TX) == 4 ? 4 : 8;
  __shared__ float sums[NT / 32];
  __shared__ uint32_t tops[2][NT / 32];
  const int64_t row = (int64_t)blockIdx.x * RPC + threadIdx.x / NT;
  const int tid = threadIdx.x % NT, nv = width / E;
  grid_wait();
  grid_release();
  if (row >= rows) return;
  float v[VPL][E];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int c = (tid + NT * i) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) v[i][e] = 0.f;
    if (tid + NT * i < nv) load_e<TX, E>(x + row * ldx + c, v[i]);
  }
  if constexpr (MODE == ROW_ADD_NORM) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int64_t c = row * width + (tid + NT * i) * E;
      if (tid + NT * i < nv) {
        float a[E];
        load_e<TR, E>(r + c, a);
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] += a[e];
        store_vec<float, E>(sum + c, v[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (MODE == ROW_RELU2) v[i][e] = v[i][e] < 0.f ? 0.f : v[i][e] * v[i][e];  // a NaN stays one
      top = max(top, mag_bits(v[i][e]));
    }
  top = block_max<NT>(top, tops[0]);
  uint32_t m = top;
  float factor = 1.f;
  if constexpr (NORM) {
    const float c = fmaxf(__uint_as_float(top), floor_), rscale = 1.0f / c;
    float ss = 0.f;
    m = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      float g[E];
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = 0.f;
      if (tid + NT * i < nv) load_e<float, E>(w + (tid + NT * i) * E, g);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = v[i][e] * rscale;
        ss += z * z;
        v[i][e] = z * g[e];
        m = max(m, mag_bits(v[i][e]));
      }
    }
    block_sum_max<NT>(ss, m, sums, tops[1]);
    factor = 1.0f / sqrtf(ss / (float)width + eps / (c * c));
  }
  float s;
  const float by = code_factor(top, m, factor, s);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if (tid + NT * i >= nv) continue;
    uint32_t word[E / 4];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(v[i][e + j], by), 12582912.0f));
      word[e / 4] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
      // a row that stands for NaN has NaN products: its codes are zero
      if (by == 0.f) word[e / 4] = 0;
    }
    uint32_t* to = reinterpret_cast<uint32_t*>(q + row * ldq + (tid + NT * i) * E);
    if constexpr (E == 4) to[0] = word[0];
    else *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[E / 4 - 1]);
  }
  if (tid == 0) scale[row] = s;
}

// Any width, any alignment: a CTA per row, the row read once per step, the second and third time from L2 (8192 x 4096:
// 82 us, in registers 56; 8192 x 9000, wider than registers hold, 239 us for the 124 of its bytes).
template <typename TX, typename TR, int MODE>
__global__ void __launch_bounds__(256) rows_q8_any_kernel(const TX* __restrict__ x, int64_t ldx,
                                                          const TR* __restrict__ r, const float* __restrict__ w,
                                                          float* __restrict__ sum, int8_t* __restrict__ q, int64_t ldq,
                                                          float* __restrict__ scale, int width, float floor_,
                                                          float eps) {
  constexpr bool NORM = MODE == ROW_ADD_NORM || MODE == ROW_NORM;
  __shared__ float sums[8];
  __shared__ uint32_t tops[2][8];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  grid_wait();
  grid_release();
  auto value = [&](int j) {
    float v = to_f32<TX>(x[row * ldx + j]);
    if constexpr (MODE == ROW_ADD_NORM) v += to_f32<TR>(r[row * width + j]);
    if constexpr (MODE == ROW_RELU2) v = v < 0.f ? 0.f : v * v;
    return v;
  };
  uint32_t top = 0;
  for (int j = tid; j < width; j += 256) {
    const float v = value(j);
    if constexpr (MODE == ROW_ADD_NORM) sum[row * width + j] = v;
    top = max(top, mag_bits(v));
  }
  top = block_max<256>(top, tops[0]);
  uint32_t m = top;
  float factor = 1.f, rscale = 1.f;
  if constexpr (NORM) {
    const float c = fmaxf(__uint_as_float(top), floor_);
    rscale = 1.0f / c;
    float ss = 0.f;
    m = 0;
    for (int j = tid; j < width; j += 256) {
      const float z = value(j) * rscale;
      ss += z * z;
      m = max(m, mag_bits(z * w[j]));
    }
    block_sum_max<256>(ss, m, sums, tops[1]);
    factor = 1.0f / sqrtf(ss / (float)width + eps / (c * c));
  }
  float s;
  const float by = code_factor(top, m, factor, s);
  for (int j = tid; j < width; j += 256) {
    float v = value(j);
    if constexpr (NORM) v = v * rscale * w[j];
    q[row * ldq + j] = by == 0.f ? (int8_t)0 : (int8_t)code_bits(__fmul_rn(v, by));
  }
  if (tid == 0) scale[row] = s;
}

// codes back to values, HBM bound (32768 x 512 to bf16: 9.7 us, 5.2 TB/s); `vec`: eight
// channels at a time, rows and widths allowing
template <typename T>
__global__ void __launch_bounds__(256) rows_q8_values_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                             const float* __restrict__ scale, T* __restrict__ y,
                                                             int64_t rows, int width, int vec) {
  const int per = vec ? width / 8 : width;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = rows * per < ((int64_t)1 << 32) ? (int64_t)((uint32_t)id / (uint32_t)per) : id / per;
  const int c = (int)(id - row * per);
  grid_wait();
  grid_release();
  if (row >= rows) return;
  const float s = scale[row];
  if (vec) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(q + row * ldq) + c);
    const int8_t* e = reinterpret_cast<const int8_t*>(&w);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)e[i] * s;
    store_vec<T, 8>(y + row * width + 8 * c, x);
  } else {
    y[row * width + c] = from_f32<T>((float)q[row * ldq + c] * s);
  }
}

template <typename TX, typename TR, int MODE>
int launch_rows(const char* what, const void* x, int64_t ldx, const void* r, const float* w, float* sum, int8_t* q,
                int64_t ldq, float* scale, int64_t rows, int width, float floor_, float eps, cudaStream_t st) {
  constexpr int E = sizeof(TX) == 4 ? 4 : 8;
  const int nv = width / E;
  const bool vec = width % E == 0 && aligned16(x) && aligned16(r) && aligned16(w) && aligned16(sum) &&
                   ldx * (int64_t)sizeof(TX) % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
  auto run = [&](auto nt, auto vpl) -> int {
    constexpr int NT = decltype(nt)::value, VPL = decltype(vpl)::value, RPC = NT == 32 ? 4 : 1;
    return launch_early(what, rows_q8_kernel<TX, TR, MODE, NT, VPL, RPC>, dim3((unsigned)((rows + RPC - 1) / RPC)), NT * RPC, 0,
                        1, st, (const TX*)x, ldx, (const TR*)r, w, sum, q, ldq, scale, rows, width, floor_, eps);
  };
  using std::integral_constant;
  // A warp per row while it holds the row in four pieces a lane (32768 x 512: 29.7 us, with 128 threads a row 36.5), but
  // 128 threads for the longest of these when rows are few and their latency counts (64 x 512: 1.8 us against 2.4, 2048 x
  // 512: 3.7 and 3.1). Longer rows get as many threads as keep them in four to eight pieces (16384 x 1024: 29.1 us with
  // 128, 38.8 with 256, 30.9 with 32; 8192 x 5000: 101 with 128, 72 with 256).
  if (vec && nv <= 32) return run(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (vec && nv <= 64) return run(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  if (vec && nv <= 128 && rows <= 1024) return run(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (vec && nv <= 128) return run(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  if (vec && nv <= 256) return run(integral_constant<int, 128>{}, integral_constant<int, 2>{});
  if (vec && nv <= 512) return run(integral_constant<int, 128>{}, integral_constant<int, 4>{});
  if (vec && nv <= 1024) return run(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  if (vec && nv <= 1280) return run(integral_constant<int, 256>{}, integral_constant<int, 5>{});
  if (vec && nv <= 1536) return run(integral_constant<int, 256>{}, integral_constant<int, 6>{});
  if (vec && nv <= 2048) return run(integral_constant<int, 256>{}, integral_constant<int, 8>{});
  return launch_early(what, rows_q8_any_kernel<TX, TR, MODE>, dim3((unsigned)rows), 256, 0, 1, st, (const TX*)x, ldx,
                      (const TR*)r, w, sum, q, ldq, scale, width, floor_, eps);
}

int check_rows(const char* what, int64_t rows, int width, int64_t ldq) {
  VB_REQUIRE(rows >= 0 && width > 0 && ldq >= width, "%s: bad shape rows=%lld width=%d row pitch=%lld", what,
             (long long)rows, width, (long long)ldq);
  VB_REQUIRE(rows < (int64_t(1) << 31), "%s: %lld rows exceed 2^31", what, (long long)rows);
  VB_REQUIRE(width <= 1 << 30, "%s: rows of %d channels exceed 2^30", what, width);  // a step further is still an int
  return VB_OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_rms_norm_q8(const void* x, const void* r, const float* weight, float* sum, int8_t* q, int64_t ldq,
                              float* scale, int64_t rows, int width, float floor_, float eps, int x_dtype, int r_dtype,
                              void* stream) {
  int rc = check_rows("rms_norm_q8", rows, width, ldq);
  if (rc) return rc;
  VB_REQUIRE(dtype_size(x_dtype) > 0, "rms_norm_q8: unsupported dtype code %d", x_dtype);
  VB_REQUIRE((r == nullptr) == (sum == nullptr), "rms_norm_q8: the addend and the sum come together");
  VB_REQUIRE(r == nullptr || x_dtype == VB_F32, "rms_norm_q8: with an addend the stream is float32, got dtype code %d",
             x_dtype);
  if (rows == 0) return VB_OK;
  VB_REQUIRE(x && weight && q && scale, "rms_norm_q8: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  if (r != nullptr)
    return VB_DISPATCH_DTYPE(r_dtype, TR, [&]() -> int {
      return launch_rows<float, TR, ROW_ADD_NORM>("rms_norm_q8", x, width, r, weight, sum, q, ldq, scale, rows, width,
                                                  floor_, eps, st);
    });
  return VB_DISPATCH_DTYPE(x_dtype, TX, [&]() -> int {
    return launch_rows<TX, float, ROW_NORM>("rms_norm_q8", x, width, nullptr, weight, nullptr, q, ldq, scale, rows,
                                            width, floor_, eps, st);
  });
}

extern "C" int vb_quantize_rows_q8(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                                   int width, int relu_square, int dtype, void* stream) {
  int rc = check_rows("quantize_rows_q8", rows, width, ldq);
  if (rc) return rc;
  VB_REQUIRE(ldx >= width, "quantize_rows_q8: row pitch %lld below the width %d", (long long)ldx, width);
  VB_REQUIRE(dtype_size(dtype) > 0, "quantize_rows_q8: unsupported dtype code %d", dtype);
  if (rows == 0) return VB_OK;
  VB_REQUIRE(x && q && scale, "quantize_rows_q8: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return VB_DISPATCH_DTYPE(dtype, TX, [&]() -> int {
    if (relu_square)
      return launch_rows<TX, float, ROW_RELU2>("quantize_rows_q8", x, ldx, nullptr, nullptr, nullptr, q, ldq, scale,
                                               rows, width, 0.f, 0.f, st);
    return launch_rows<TX, float, ROW_PLAIN>("quantize_rows_q8", x, ldx, nullptr, nullptr, nullptr, q, ldq, scale,
                                             rows, width, 0.f, 0.f, st);
  });
}

extern "C" int vb_dequantize_rows_q8(const int8_t* q, int64_t ldq, const float* scale, void* y, int64_t rows, int width,
                                     int dtype, void* stream) {
  int rc = check_rows("dequantize_rows_q8", rows, width, ldq);
  if (rc) return rc;
  VB_REQUIRE(dtype_size(dtype) > 0, "dequantize_rows_q8: unsupported dtype code %d", dtype);
  if (rows == 0) return VB_OK;
  VB_REQUIRE(q && scale && y, "dequantize_rows_q8: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    const int vec = width % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0 && aligned16(y);
    const int64_t blocks = (rows * (vec ? width / 8 : width) + 255) / 256;
    VB_REQUIRE(blocks < (int64_t(1) << 31), "dequantize_rows_q8: %lld x %d values exceed the grid", (long long)rows, width);
    return launch_early("dequantize_rows_q8", rows_q8_values_kernel<T>, dim3((unsigned)blocks), 256, 0, 1, st, q, ldq, scale,
                        (T*)y, rows, width, vec);
  });
}
