// Host-side construction of TMA tensor maps (cuTensorMapEncodeTiled through the runtime's driver
// entry point, so the library needs no link against libcuda).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"
#include "tmap.cuh"

namespace vb {
namespace {
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;
void find_encode() {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
}
}  // namespace

int make_byte_map(CUtensorMap* map, const void* base, int64_t rows, int64_t width, int64_t pitch, int box_rows) {
  find_encode();
  VB_REQUIRE(g_encode != nullptr, "cuTensorMapEncodeTiled is not available from the driver");
  VB_REQUIRE(aligned16(base) && pitch % 16 == 0, "byte map: base or row pitch not 16-byte aligned");
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VB_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) for [%lld,%lld] bytes", (int)r, (long long)rows,
             (long long)width);
  return VB_OK;
}

int make_out_map(CUtensorMap* map, void* base, int64_t rows, int64_t width, int box_width, int box_rows, int dtype) {
  find_encode();
  VB_REQUIRE(g_encode != nullptr, "cuTensorMapEncodeTiled is not available from the driver");
  const int64_t pitch = width * dtype_size(dtype);
  VB_REQUIRE(aligned16(base) && pitch % 16 == 0, "output map: base or row pitch not 16-byte aligned");
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_width, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(map, dtype_size(dtype) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                              2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VB_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) for [%lld,%lld] outputs", (int)r, (long long)rows,
             (long long)width);
  return VB_OK;
}

int make_token_map(CUtensorMap* map, const void* base, int B, int T, int H, int D, bool f16) {
  find_encode();
  VB_REQUIRE(g_encode != nullptr, "cuTensorMapEncodeTiled is not available from the driver");
  VB_REQUIRE(aligned16(base) && (D * 2) % 16 == 0, "token map: base or row pitch not 16-byte aligned");
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)H * D * 2, (cuuint64_t)T * H * D * 2};
  const cuuint32_t box[4] = {64, 1, 64, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = g_encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
                              box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VB_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) for [%d,%d,%d,%d]", (int)r, B, T, H, D);
  return VB_OK;
}

}  // namespace vb
