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
// HBM bound: 4 + 2 + 4 + 1 bytes per channel for a float32 stream with a bf16 addend.
#include "common.cuh"

namespace vb {
namespace {

constexpr float TINY_ROW = 1e-35f;
enum { ROW_ADD_NORM = 0, ROW_NORM = 1, ROW_PLAIN = 2, ROW_RELU2 = 3 };

// nearest integer (ties to even) of v, |v| < 2^22, as the low byte of the result
__device__ __forceinline__ uint32_t code_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.0f)) & 0xffu; }

__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Any width, any alignment: a CTA per row, the row read once per step from L2.
template <typename TX, typename TR, int MODE>
__global__ void __launch_bounds__(256) rows_q8_any_kernel(const TX* __restrict__ x, int64_t ldx,
                                                          const TR* __restrict__ r, const float* __restrict__ w,
                                                          float* __restrict__ sum, int8_t* __restrict__ q, int64_t ldq,
                                                          float* __restrict__ scale, int width, float floor_,
                                                          float eps) {
  constexpr bool NORM = MODE == ROW_ADD_NORM || MODE == ROW_NORM;
  __shared__ float red[2][8];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto value = [&](int j) {
    float v = to_f32<TX>(x[row * ldx + j]);
    if constexpr (MODE == ROW_ADD_NORM) v += to_f32<TR>(r[row * width + j]);
    if constexpr (MODE == ROW_RELU2) v = v < 0.f ? 0.f : v * v;  // a NaN stays one
    return v;
  };
  uint32_t top = 0;
  for (int j = tid; j < width; j += 256) {
    const float v = value(j);
    if constexpr (MODE == ROW_ADD_NORM) sum[row * width + j] = v;
    top = max(top, mag_bits(v));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) red[0][warp] = __uint_as_float(top);
  __syncthreads();
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(red[0][i]));
  __syncthreads();
  float m = __uint_as_float(top), factor = 1.f, rscale = 1.f;
  if constexpr (NORM) {
    const float c = fmaxf(__uint_as_float(top), floor_);
    rscale = 1.0f / c;
    float ss = 0.f;
    uint32_t mz = 0;
    for (int j = tid; j < width; j += 256) {
      const float z = value(j) * rscale;
      ss += z * z;
      mz = max(mz, mag_bits(z * w[j]));
    }
    ss = warp_sum(ss);
    mz = __reduce_max_sync(0xffffffffu, mz);
    if (lane == 0) { red[0][warp] = ss; red[1][warp] = __uint_as_float(mz); }
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < 8; ++i) { ss += red[0][i]; mz = max(mz, __float_as_uint(red[1][i])); }
    factor = 1.0f / sqrtf(ss / (float)width + eps / (c * c));
    m = __uint_as_float(mz);
  }
  const bool finite = top < 0x7f800000u && __float_as_uint(m) < 0x7f800000u;
  const float amax = m * factor;
  const bool live = finite && amax >= TINY_ROW;
  const float inverse = live ? 127.0f / m : 0.f;
  for (int j = tid; j < width; j += 256) {
    float v = value(j);
    if constexpr (NORM) v = v * rscale * w[j];
    q[row * ldq + j] = live ? (int8_t)code_bits(__fmul_rn(v, inverse)) : (int8_t)0;
  }
  if (tid == 0) scale[row] = live ? amax / 127.0f : finite ? 0.f : __uint_as_float(0x7fc00000u);
}

template <typename T>
__global__ void __launch_bounds__(256) rows_q8_values_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                             const float* __restrict__ scale, T* __restrict__ y,
                                                             int64_t rows, int width) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float s = scale[row];
  for (int j = threadIdx.x & 31; j < width; j += 32) y[row * width + j] = from_f32<T>((float)q[row * ldq + j] * s);
}

template <typename TX, typename TR, int MODE>
int launch_rows(const char* what, const void* x, int64_t ldx, const void* r, const float* w, float* sum, int8_t* q,
                int64_t ldq, float* scale, int64_t rows, int width, float floor_, float eps, cudaStream_t st) {
  rows_q8_any_kernel<TX, TR, MODE><<<(unsigned)rows, 256, 0, st>>>((const TX*)x, ldx, (const TR*)r, w, sum, q, ldq,
                                                                   scale, width, floor_, eps);
  VB_LAUNCH_CHECK(what);
  return VB_OK;
}

int check_rows(const char* what, int64_t rows, int width, int64_t ldq) {
  VB_REQUIRE(rows >= 0 && width > 0 && ldq >= width, "%s: bad shape rows=%lld width=%d row pitch=%lld", what,
             (long long)rows, width, (long long)ldq);
  VB_REQUIRE(rows < (int64_t(1) << 31), "%s: %lld rows exceed 2^31", what, (long long)rows);
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
    rows_q8_values_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(q, ldq, scale, (T*)y, rows, width);
    VB_LAUNCH_CHECK("dequantize_rows_q8");
    return VB_OK;
  });
}
