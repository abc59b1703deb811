// One decoding token per row attending over a 4-bit ring cache (vesper/attention.py:298-338
// attend_ring, over the format of q4.cuh): o_h = softmax_j(q_h . k_j / sqrt(DK)) v_j over the slots
// whose position lies in (p - window, p].
//
// A CTA of eight warps per (row, head): a warp walks every eighth slot, its lanes holding channels
// lane, lane + 32, ..., with the running maximum and sum of its softmax; the warps' parts are joined
// in warp order. A row with a negative position attends nothing: its output is zero.
#include <cmath>

#include "q4.cuh"

namespace vb {
namespace {

template <typename T>
__global__ void __launch_bounds__(256) q4_attn_simple_kernel(const T* __restrict__ q, int64_t q_row,
                                                             const int64_t* __restrict__ pos,
                                                             const uint8_t* __restrict__ k_codes,
                                                             const uint32_t* __restrict__ k_params,
                                                             const uint8_t* __restrict__ v_codes,
                                                             const uint32_t* __restrict__ v_params,
                                                             const int64_t* __restrict__ ring_pos, T* __restrict__ o,
                                                             int H, int HKV, int DK, int W, int SLOTS, float scale) {
  __shared__ float part[8][128 + 2];
  const int b = blockIdx.x, h = blockIdx.y, kh = h / (H / HKV), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t p = pos[b];
  const int gs = q4_group(DK), ng = DK / gs;
  float qv[4], acc[4] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    qv[e] = lane + 32 * e < DK ? to_f32<T>(q[b * q_row + (int64_t)h * DK + lane + 32 * e]) * scale : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int s = warp; s < W; s += 8) {
    const int64_t kp = ring_pos[(int64_t)b * SLOTS + s];
    if (!(kp >= 0 && kp <= p && kp > p - W)) continue;
    const int64_t at = ((int64_t)b * HKV + kh) * SLOTS + s;
    float vv[4], dot = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = lane + 32 * e;
      vv[e] = 0.f;
      if (c < DK) {
        const int kp_ = q4_key_place(DK, c), vp = q4_value_place(DK, c);
        const uint32_t pk = k_params[at * ng + c / gs], pv = v_params[at * ng + c / gs];
        const float kc = (float)(k_codes[at * (DK / 2) + kp_ / 2] >> (4 * (kp_ & 1)) & 15);
        const float vc = (float)(v_codes[at * (DK / 2) + vp / 2] >> (4 * (vp & 1)) & 15);
        dot = fmaf(qv[e], fmaf(kc, q4_step(pk), q4_lo(pk)), dot);
        vv[e] = fmaf(vc, q4_step(pv), q4_lo(pv));
      }
    }
    dot = warp_sum(dot);
    const float m2 = fmaxf(m, dot), f = expf(m - m2), w = expf(dot - m2);
    m = m2;
    l = fmaf(l, f, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(acc[e], f, w * vv[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < DK) part[warp][lane + 32 * e] = acc[e];
  if (lane == 0) { part[warp][128] = m; part[warp][129] = l; }
  __syncthreads();
  for (int c = threadIdx.x; c < DK; c += 256) {
    float M = -INFINITY, L = 0.f, out = 0.f;
    for (int w = 0; w < 8; ++w) M = fmaxf(M, part[w][128]);
    for (int w = 0; w < 8; ++w) {
      const float f = part[w][128] == -INFINITY ? 0.f : expf(part[w][128] - M);
      L = fmaf(part[w][129], f, L);
      out = part[w][128] == -INFINITY ? out : fmaf(part[w][c], f, out);
    }
    o[((int64_t)b * H + h) * DK + c] = from_f32<T>(p >= 0 ? out / L : 0.f);
  }
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" size_t vb_q4_attend_workspace(int B, int H, int HKV, int DK, int W) {
  (void)B; (void)H; (void)HKV; (void)DK; (void)W;
  return 16;
}

extern "C" int vb_q4_attend(const void* q, int64_t q_row, const void* k_new, int64_t k_row, const void* v_new,
                            int64_t v_row, const int64_t* pos, void* k_codes, void* k_params, void* v_codes,
                            void* v_params, int64_t* ring_pos, void* o, void* workspace, int B, int H, int HKV, int DK,
                            int W, int SLOTS, int dtype, void* stream) {
  VB_REQUIRE(H >= 1 && HKV >= 1 && H % HKV == 0, "q4_attend: %d query heads are not a multiple of %d key heads", H, HKV);
  int rc = vb_q4_write(k_codes, k_params, v_codes, v_params, ring_pos, k_new, k_row, 0, v_new, v_row, 0, pos, B, 1, HKV,
                       DK, W, SLOTS, dtype, stream);
  if (rc) return rc;
  if (B == 0) return VB_OK;
  VB_REQUIRE(q && o && workspace, "q4_attend: null pointer");
  VB_REQUIRE(H <= 65535, "q4_attend: %d heads exceed the grid", H);
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    q4_attn_simple_kernel<T><<<dim3(B, H), 256, 0, (cudaStream_t)stream>>>(
        (const T*)q, q_row, pos, (const uint8_t*)k_codes, (const uint32_t*)k_params, (const uint8_t*)v_codes,
        (const uint32_t*)v_params, ring_pos, (T*)o, H, HKV, DK, W, SLOTS, 1.0f / sqrtf((float)DK));
    VB_LAUNCH_CHECK("q4_attend");
    return VB_OK;
  });
}
