// The int8 product of a quantised linear layer: y[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n],
// the sum exact in int32 (K <= 131056), the scales applied in float32 and the result rounded once.
//
// A CTA of 256 threads per 64 x 64 tile of y: 16-byte pieces of 64 rows of each operand staged in
// shared memory, 4 x 4 outputs per thread by four-way byte dot products.
#include "common.cuh"

namespace vb {
namespace {

constexpr int TILE = 64, KS = 64, PITCH = KS + 4;

template <typename T>
__global__ void __launch_bounds__(256) linear_q8_dp4a_kernel(const int8_t* __restrict__ x, int64_t ldx,
                                                             const float* __restrict__ xs,
                                                             const int8_t* __restrict__ w, int64_t ldw,
                                                             const float* __restrict__ ws, T* __restrict__ y, int M,
                                                             int N, int K) {
  __shared__ __align__(16) int8_t sx[TILE][PITCH], sw[TILE][PITCH];
  const int64_t m0 = (int64_t)blockIdx.y * TILE, n0 = (int64_t)blockIdx.x * TILE;
  const int tid = threadIdx.x, tm = tid / 16, tn = tid % 16;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += KS) {
    for (int e = tid; e < TILE * KS; e += 256) {
      const int row = e / KS, k = e % KS;
      sx[row][k] = m0 + row < M && k0 + k < K ? x[(m0 + row) * ldx + k0 + k] : (int8_t)0;
      sw[row][k] = n0 + row < N && k0 + k < K ? w[(n0 + row) * ldw + k0 + k] : (int8_t)0;
    }
    __syncthreads();
    for (int k = 0; k < KS; k += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __dp4a(*reinterpret_cast<const int*>(&sx[tm + 16 * i][k]),
                             *reinterpret_cast<const int*>(&sw[tn + 16 * j][k]), acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m < M && n < N) y[m * N + n] = from_f32<T>((float)acc[i][j] * xs[m] * ws[n]);
    }
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_linear_q8(const int8_t* xq, int64_t ldx, const float* xs, const int8_t* wq, int64_t ldw,
                            const float* ws, void* y, int M, int N, int K, int dtype, int* status, void* stream) {
  VB_REQUIRE(M >= 0 && N > 0 && K > 0 && ldx >= K && ldw >= K, "linear_q8: bad shape M=%d N=%d K=%d pitches %lld, %lld",
             M, N, K, (long long)ldx, (long long)ldw);
  VB_REQUIRE(K <= 131056, "linear_q8: K=%d exceeds 131056, above which a sum may leave int32", K);
  VB_REQUIRE(dtype_size(dtype) > 0, "linear_q8: unsupported dtype code %d", dtype);
  if (M == 0) return VB_OK;
  VB_REQUIRE(xq && xs && wq && ws && y && status, "linear_q8: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((N + TILE - 1) / TILE, (M + TILE - 1) / TILE);
  VB_REQUIRE(grid.y <= 65535, "linear_q8: %d rows exceed the grid", M);
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    linear_q8_dp4a_kernel<T><<<grid, 256, 0, st>>>(xq, ldx, xs, wq, ldw, ws, (T*)y, M, N, K);
    VB_LAUNCH_CHECK("linear_q8");
    return VB_OK;
  });
}
