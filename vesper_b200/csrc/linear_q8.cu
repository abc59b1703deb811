// The int8 product of a quantised linear layer: y[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n],
// the sum exact in int32 (K <= 131056), the scales applied in float32 and the result rounded once.
//
// Operand tiles of 128 bytes x rows arrive by TMA in the 128-byte swizzle (zero past the edges, so no
// size needs a case of its own); the products run on tcgen05 (kind::i8, 32 bytes of K each) into int32 in TMEM.
//
// linear_q8_split_kernel: few tokens. The weights' rows (output channels) lie on the accumulator's lanes and the
//   tokens on its columns, so one token costs a tile of 16 columns. A cluster of S CTAs per tile of 128
//   channels x BN tokens, each over its part of K; the parts are added through distributed shared memory, whole
//   numbers, so the order does not matter. The weights are read once, and S spreads their bytes over the SMs: 1 x 4096 x
//   8192 in 8.7 us, 3.9 TB/s (59 % of a plain copy's rate; half the rest is the copies' start, the products' end and
//   the clusters' sum). Small weights are bound by those alone: 64 x 512 x 1544 in 4.1 us.
// linear_q8_tile_kernel: many tokens, on the lanes; persistent over tiles of 128 tokens x BN channels, or of 256 x 256
//   on CTA pairs (cta_group::2), each CTA copying half of either operand (32 KB per 128 bytes of K, against 48 KB for
//   a single CTA's 128 x 256). Accumulators are double-buffered in TMEM, so that the storing warps' loads,
//   scaling and TMA stores run under the next tile's products. 8192 x 4096 x 8192 in 184 us, 2.98 POP/s, the tensor
//   pipe active 75 % of the time (before the pairs 236 us, before the doubled accumulators 271). Longer K adds 43 ns a
//   byte of it, 3.14 POP/s, so some 15 us are the kernel's start, its last tiles and their stores; 777 x 1040 x 2001,
//   112 tiles of nine blocks of K on 148 SMs, in 8.8 us: the latency of one tile.
#include <cmath>

#include "launch.cuh"
#include "tmap.cuh"
#include "umma.cuh"

namespace vb {
namespace {

constexpr int KB = 128;    // bytes of K per stage
constexpr int ROWS = 128;  // channels per CTA

// kind::i8 instruction descriptor: signed x signed -> int32, both operands K-major
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// k-step s (32 bytes) of a swizzled tile of 128-byte rows
__device__ __forceinline__ uint64_t desc_bytes(uint32_t tile, int s) { return sdesc(tile + 32u * s, 16u, 1024u); }

template <int GROUP>
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (GROUP == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate));
}

__device__ __forceinline__ void tma_load_2d(void* dst, const void* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// ---- clusters -------------------------------------------------------------------------------
constexpr uint32_t LEADER = 0xFEFFFFFFu;  // clears a shared::cluster address's odd-CTA bit within a pair

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the shared::cluster address of `local` in CTA `rank`
__device__ __forceinline__ uint32_t in_cta(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void st_cluster4(uint32_t remote, int x, int y, int z, int w) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
// this CTA's tile into its own shared memory, completing on the pair leader's barrier
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar) & LEADER), "r"(x), "r"(y)
      : "memory");
}
// when this thread's products are done: one arrival on the barrier of both CTAs of the pair
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & LEADER) : "memory");
}

constexpr uint64_t LATE_NS = 200000000ull;  // the limit of waits that only tidy up

__device__ __forceinline__ void gave_up(int* status) { atomicOr(status, 1); }

template <typename T>
__device__ __forceinline__ T scaled(int acc, float sw, float sx) {
  return from_f32<T>((float)acc * sx * sw);
}

// ---- few tokens: K split over a cluster -------------------------------------------------------
template <int BN>
struct Split {
  static constexpr int STAGE = (ROWS + BN) * KB;
  static constexpr int PARTS = ROWS * BN * 4;  // the partial sums this CTA receives
  static constexpr int STAGES = (104 * 1024 - PARTS) / STAGE;  // two CTAs share an SM
  static constexpr int SMEM = STAGES * STAGE + PARTS + 1024;
  static constexpr int COLS = BN < 32 ? 32 : BN;
};

template <int BN, typename T>
__global__ void __launch_bounds__(128, 2)
    linear_q8_split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                           const float* __restrict__ xs, const float* __restrict__ ws, T* __restrict__ y, int M, int N,
                           int kblocks, int S, int* status) {
  using C = Split<BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], done;
  __shared__ uint32_t tmem_at;
  __shared__ float sxs[BN], sws[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  if (S > 1) cluster_arrive();
  const int n0 = (int)(blockIdx.x / S) * ROWS, m0 = blockIdx.y * BN;
  const int k_lo = (int)((int64_t)kblocks * rank / S), blocks = (int)((int64_t)kblocks * (rank + 1) / S) - k_lo;
  auto load = [&](int i) {
    const int st = i % C::STAGES;
    mbar_arrive_expect_tx(&full[st], C::STAGE);
    tma_load_2d(smem + st * C::STAGE, &wmap, &full[st], (k_lo + i) * KB, n0);
    tma_load_2d(smem + st * C::STAGE + ROWS * KB, &xmap, &full[st], (k_lo + i) * KB, m0);
  };
  if (tid == 0) {  // the first copies leave before anything else is set up
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    mbar_fence_init();
    prefetch_tmap(&wmap);
    prefetch_tmap(&xmap);
    grid_wait();
    for (int i = 0; i < min(blocks, C::STAGES); ++i) load(i);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_at, C::COLS);
    tmem_relinquish();
  }
  grid_wait();
  if (tid >= 64)
    for (int i = tid - 64; i < BN + ROWS; i += 64) {
      if (i < BN) sxs[i] = m0 + i < M ? xs[m0 + i] : 0.f;
      else sws[i - BN] = n0 + i - BN < N ? ws[n0 + i - BN] : 0.f;
    }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_release();  // the next kernel comes once this one has its tensor memory
  const uint32_t tmem = tmem_at;
  if (tid == 0) {
    for (int i = C::STAGES; i < blocks; ++i) {
      if (!mbar_wait(&empty[i % C::STAGES], ((i / C::STAGES) - 1) & 1)) {
        gave_up(status);
        break;
      }
      load(i);
    }
  } else if (tid == 32) {
    bool ok = true;
    int i = 0;
    for (; i < blocks; ++i) {
      const int st = i % C::STAGES;
      if (!(ok = mbar_wait(&full[st], (i / C::STAGES) & 1))) break;
      const uint32_t a = smem_u32(smem + st * C::STAGE), b = a + ROWS * KB;
#pragma unroll
      for (int s = 0; s < KB / 32; ++s)
        umma_i8<1>(tmem, desc_bytes(a, s), desc_bytes(b, s), idesc_i8(ROWS, BN), i > 0 || s > 0);
      umma_commit(&empty[st]);
    }
    if (!ok) {
      gave_up(status);
      for (int j = i; j < min(i + C::STAGES, blocks); ++j)  // the copies that may still be in flight
        mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, LATE_NS);
    }
    umma_commit(&done);
  }
  __syncwarp();
  if (!mbar_wait(&done, 0)) gave_up(status);
  tc_fence_after();
  __syncwarp();
  if (S > 1) cluster_wait();  // the others have begun: their shared memory may be written
  // rank r adds and stores the channels [128 r / S, 128 (r + 1) / S): each CTA sends it their sums, in
  // pieces of four columns of one channel, [sender][column / 4][channel]
  const int per = ROWS / S, row = warp * 32 + lane, owner = row / per;
  int4* parts = reinterpret_cast<int4*>(smem + C::STAGES * C::STAGE);
  const uint32_t to = S > 1 ? in_cta(smem_u32(parts + (rank * (BN / 4)) * per + row - owner * per), owner) : 0;
#pragma unroll
  for (int c = 0; c < BN; c += 16) {
    if (m0 + c >= M) break;
    int v[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr(tmem, warp * 32, c)));
    tmem_wait_ld();
    if (S > 1) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) st_cluster4(to + (c + j) / 4 * per * 16, v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else if (n0 + row < N) {
      const float sw = sws[row];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (m0 + c + j < M) y[(int64_t)(m0 + c + j) * N + n0 + row] = scaled<T>(v[j], sw, sxs[c + j]);
    }
  }
  if (S > 1) {
    cluster_sync();  // every sum has arrived, and nothing else crosses between the CTAs
    const int cols = min(BN, M - m0);
    for (int e = tid; e < per * ((cols + 3) / 4); e += 128) {
      const int c = e / per, r = e - c * per;
      int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < S) {
          const int4 v = parts[(i * (BN / 4) + c) * per + r];
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
      const int n = n0 + rank * per + r;
      if (n >= N) continue;
      const float sw = sws[rank * per + r];
      T* out = y + (int64_t)(m0 + 4 * c) * N + n;
      out[0] = scaled<T>(sum.x, sw, sxs[4 * c]);
      if (4 * c + 1 < cols) out[N] = scaled<T>(sum.y, sw, sxs[4 * c + 1]);
      if (4 * c + 2 < cols) out[2 * (int64_t)N] = scaled<T>(sum.z, sw, sxs[4 * c + 2]);
      if (4 * c + 3 < cols) out[3 * (int64_t)N] = scaled<T>(sum.w, sw, sxs[4 * c + 3]);
    }
  }
  if (tid == 0)  // every commit has arrived before this CTA can end
    for (int j = max(0, blocks - C::STAGES); j < blocks; ++j)
      mbar_wait(&empty[j % C::STAGES], (j / C::STAGES) & 1, LATE_NS);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::COLS);
}

// ---- many tokens: persistent tiles -------------------------------------------------------------
// GROUP CTAs per tile of 128 GROUP tokens x BN channels
template <int GROUP, int BN>
struct Tile {
  static constexpr int BROWS = BN / GROUP;  // channels whose weights a CTA copies
  static constexpr int STAGE = (ROWS + BROWS) * KB;
  static constexpr int WARPS = BN >= 128 ? 8 : 4;     // storing warps, each over SPAN columns of 32 lanes
  static constexpr int SPAN = BN / (WARPS / 4);
  static constexpr int THREADS = 64 + 32 * WARPS;     // warp 0 copies, warp 1 multiplies, the others store
  static constexpr int OUT = WARPS * 2 * 32 * 128;    // per storing warp two buffers of 32 rows x 128 bytes
  static constexpr int STAGES = (220 * 1024 - OUT) / STAGE < 6 ? (220 * 1024 - OUT) / STAGE : 6;
  static constexpr int SMEM = STAGES * STAGE + OUT + 1024;
  static constexpr int COLS = 2 * BN;  // two accumulators
};
// waits for this thread's TMEM loads, of which v is one: v is not read, moved or kept before
__device__ __forceinline__ void tmem_wait_ld32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                 "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

// tile t: tokens vary fastest within bands of eight channel tiles
__device__ __forceinline__ void tile_at(int t, int tiles_n, int tiles_m, int& tn, int& tm) {
  const int band = t / (8 * tiles_m), first = band * 8, width = min(8, tiles_n - first);
  const int r = t - band * 8 * tiles_m;
  tm = r / width;
  tn = first + r - tm * width;
}

template <int GROUP, int BN, typename T>
__global__ void __launch_bounds__(Tile<GROUP, BN>::THREADS, 1)
    linear_q8_tile_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                          const __grid_constant__ CUtensorMap ymap, int by_tma, const float* __restrict__ xs,
                          const float* __restrict__ ws, T* __restrict__ y, int M, int N, int kblocks, int tiles_n,
                          int tiles_m, int* status) {
  using C = Tile<GROUP, BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], tfull[2], tempty[2];
  __shared__ uint32_t tmem_at;
  __shared__ __align__(16) float sws[2][BN];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = GROUP == 2 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / GROUP, stride = gridDim.x / GROUP, tiles = tiles_n * tiles_m;
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);   // the expected bytes (in a pair: the leader's, both CTAs' copies complete on it)
      mbar_init(&empty[i], 1);  // the commit (in a pair: the leader's, on both CTAs)
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], C::WARPS * GROUP);  // the storing warps
    }
    mbar_fence_init();
    prefetch_tmap(&wmap);
    prefetch_tmap(&xmap);
  }
  if (warp == 0) {
    if constexpr (GROUP == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)),
                   "r"(C::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&tmem_at, C::COLS);
      tmem_relinquish();
    }
  }
  __syncthreads();
  if constexpr (GROUP == 2) cluster_sync();  // both CTAs' barriers and TMEM are ready
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  grid_wait();
  grid_release();
  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += stride) {
        int tn, tm;
        tile_at(t, tiles_n, tiles_m, tn, tm);
        const int m0 = (tm * GROUP + rank) * ROWS, n0 = tn * BN + rank * C::BROWS;
        for (int k = 0; k < kblocks; ++k, ++i) {
          const int st = i % C::STAGES;
          if (i >= C::STAGES && !(ok = mbar_wait(&empty[st], ((i / C::STAGES) - 1) & 1))) break;
          uint8_t* a = smem + st * C::STAGE;
          if (rank == 0) mbar_arrive_expect_tx(&full[st], GROUP * C::STAGE);
          if constexpr (GROUP == 2) {
            tma_load_2d_pair(a, &xmap, &full[st], k * KB, m0);
            tma_load_2d_pair(a + ROWS * KB, &wmap, &full[st], k * KB, n0);
          } else {
            tma_load_2d(a, &xmap, &full[st], k * KB, m0);
            tma_load_2d(a + ROWS * KB, &wmap, &full[st], k * KB, n0);
          }
        }
      }
      if (!ok) gave_up(status);
      for (int j = max(0, i - C::STAGES); j < i; ++j)  // the copies are read and every commit has arrived
        mbar_wait(&empty[j % C::STAGES], (j / C::STAGES) & 1, ok ? 2000000000ull : LATE_NS);
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      int i = 0, n = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += stride, ++n) {
        const int buf = n & 1;
        if (n >= 2 && !(ok = mbar_wait(&tempty[buf], ((n >> 1) - 1) & 1))) break;
        tc_fence_after();
        for (int k = 0; k < kblocks; ++k, ++i) {
          const int st = i % C::STAGES;
          if (!(ok = mbar_wait(&full[st], (i / C::STAGES) & 1))) break;
          const uint32_t a = smem_u32(smem + st * C::STAGE), b = a + ROWS * KB;
#pragma unroll
          for (int s = 0; s < KB / 32; ++s)
            umma_i8<GROUP>(tmem + buf * BN, desc_bytes(a, s), desc_bytes(b, s), idesc_i8(GROUP * ROWS, BN),
                           k > 0 || s > 0);
          if constexpr (GROUP == 2) umma_commit_pair(&empty[st]);
          else umma_commit(&empty[st]);
        }
        if constexpr (GROUP == 2) umma_commit_pair(&tfull[buf]);
        else umma_commit(&tfull[buf]);
      }
      if (!ok) gave_up(status);
    }
  } else {
    constexpr int PER = 128 / (int)sizeof(T);  // channels of one 128-byte output row piece
    constexpr int CHUNKS = C::SPAN / 32, SCALES = (BN + 32 * C::WARPS - 1) / (32 * C::WARPS);
    const int quad = warp & 3, col0 = ((warp - 2) / 4) * C::SPAN;
    uint8_t* stage = smem + C::STAGES * C::STAGE + (warp - 2) * 2 * 32 * 128;
    if (lane == 0 && by_tma) prefetch_tmap(&ymap);
    // a tile's scales, loaded while the tile before it is stored: this thread's token's, and the channels', which
    // the storing warps share in shared memory
    float sx, wreg[SCALES];
    auto load_scales = [&](int t) {
      int tn, tm;
      tile_at(min(t, tiles - 1), tiles_n, tiles_m, tn, tm);
      const int m = (tm * GROUP + rank) * ROWS + quad * 32 + lane;
      sx = m < M ? __ldg(xs + m) : 0.f;
#pragma unroll
      for (int i = 0; i < SCALES; ++i) {
        const int c = tid - 64 + i * 32 * C::WARPS;
        wreg[i] = c < BN && tn * BN + c < N ? __ldg(ws + tn * BN + c) : 0.f;
      }
    };
    load_scales(first);
    int n = 0, piece = 0;
    bool ok = true;  // a warp that gave up stores nothing more but keeps to the barriers of its tiles
    for (int t = first; t < tiles; t += stride, ++n) {
      const int buf = n & 1;
      int tn, tm;
      tile_at(t, tiles_n, tiles_m, tn, tm);
      const int m0 = (tm * GROUP + rank) * ROWS + quad * 32, n0 = tn * BN;
#pragma unroll
      for (int i = 0; i < SCALES; ++i) {
        const int c = tid - 64 + i * 32 * C::WARPS;
        if (c < BN) sws[buf][c] = wreg[i];
      }
      const float sxt = sx;
      bar_sync_named(1, 32 * C::WARPS);
      load_scales(t + stride);
      if (ok && !(ok = mbar_wait(&tfull[buf], (n >> 1) & 1))) gave_up(status);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        continue;
      }
      tc_fence_after();
      float v2[2][32];  // one chunk of 32 columns is scaled and stored while the next is on its way from TMEM
      tmem_ld32(taddr(tmem, quad * 32, buf * BN + col0), v2[0]);
      uint8_t* out = stage;
#pragma unroll
      for (int q = 0; q < CHUNKS; ++q) {
        float(&v)[32] = v2[q & 1];
        const int c0 = col0 + 32 * q;
        tmem_wait_ld32(v);
        if (q + 1 < CHUNKS) {
          tmem_ld32(taddr(tmem, quad * 32, buf * BN + c0 + 32), v2[(q + 1) & 1]);
        } else {  // this warp's part of the accumulator is read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (GROUP == 2) mbar_arrive_leader(&tempty[buf]);
            else mbar_arrive(&tempty[buf]);
          }
        }
        if (32 * q % PER == 0) {
          out = stage + (piece++ & 1) * 32 * 128;
          // the buffer's previous store has been read out of shared memory
          if (lane == 0 && by_tma) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(&sws[buf][c0 + j]);
          v[j] = (float)__float_as_int(v[j]) * sxt * w4.x;
          v[j + 1] = (float)__float_as_int(v[j + 1]) * sxt * w4.y;
          v[j + 2] = (float)__float_as_int(v[j + 2]) * sxt * w4.z;
          v[j + 3] = (float)__float_as_int(v[j + 3]) * sxt * w4.w;
        }
        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
        for (int j = 0; j < 32; j += E) {  // 16-byte chunk i of row `lane` at i ^ (lane mod 8)
          float e[E];
#pragma unroll
          for (int i = 0; i < E; ++i) e[i] = v[j + i];
          store_vec<T, E>(reinterpret_cast<T*>(out + lane * 128 + (((((32 * q) % PER + j) / E) ^ (lane & 7)) << 4)), e);
        }
        if ((32 * q + 32) % PER != 0) continue;
        const int p0 = n0 + c0 + 32 - PER;  // the piece's first channel
        if (by_tma) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (m0 < M && p0 < N)
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&ymap),
                           "r"(smem_u32(out)), "r"(p0), "r"(m0)
                           : "memory");
            bulk_commit();
          }
        } else {
          __syncwarp();
          for (int r = 0; r < min(32, M - m0); ++r)
#pragma unroll
            for (int c = lane; c < PER; c += 32)
              if (p0 + c < N)
                y[(int64_t)(m0 + r) * N + p0 + c] = *reinterpret_cast<const T*>(
                    out + r * 128 + (((c * (int)sizeof(T) / 16) ^ (r & 7)) << 4) + (c * (int)sizeof(T)) % 16);
          __syncwarp();
        }
      }
    }
    if (lane == 0 && by_tma) bulk_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (GROUP == 2) cluster_sync();  // no CTA leaves while its pair's copies, products or arrivals may still reach it
  if (warp == 0) {
    if constexpr (GROUP == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    else
      tmem_dealloc(tmem, C::COLS);
  }
}

// ---- launches ---------------------------------------------------------------------------------
struct Args {
  const int8_t* xq;
  int64_t ldx;
  const float* xs;
  const int8_t* wq;
  int64_t ldw;
  const float* ws;
  void* y;
  int M, N, K;
  int* status;
  cudaStream_t st;
};

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      v = 148;
    return v > 1 ? v : 148;
  }();
  return n;
}

template <int BN, typename T>
int launch_split(const Args& a) {
  const int kblocks = (a.K + KB - 1) / KB, tiles_n = (a.N + ROWS - 1) / ROWS, tiles_m = (a.M + BN - 1) / BN;
  // K over S CTAs: one per SM, or two where each still has two blocks of K to itself (1 x 4096 x 8192: 8.7 us with
  // two, 10.1 with one; 1 x 1024 x 8192: 4.9 and 5.4; 1 x 1024 x 4096, whose CTAs would be left one block: 5.0 and 4.3)
  int S = 1;
  while (S < 8 && 2 * S <= kblocks && 2LL * S * tiles_n * tiles_m <= (long long)sm_count() * (kblocks / (2 * S) >= 2 ? 2 : 1))
    S *= 2;
  CUtensorMap wmap, xmap;
  int rc = make_byte_map(&wmap, a.wq, a.N, a.K, a.ldw, ROWS);
  if (!rc) rc = make_byte_map(&xmap, a.xq, a.M, a.K, a.ldx, BN);
  if (rc) return rc;
  VB_REQUIRE(tiles_m <= 65535, "linear_q8: %d rows exceed the grid", a.M);
  return launch_early("linear_q8", linear_q8_split_kernel<BN, T>, dim3(tiles_n * S, tiles_m), 128, Split<BN>::SMEM, S, a.st, wmap, xmap,
                a.xs, a.ws, (T*)a.y, a.M, a.N, kblocks, S, a.status);
}

template <int GROUP, int BN, typename T>
int launch_tile(const Args& a) {
  using C = Tile<GROUP, BN>;
  const int kblocks = (a.K + KB - 1) / KB;
  const int tiles_n = (a.N + BN - 1) / BN, tiles_m = (a.M + GROUP * ROWS - 1) / (GROUP * ROWS);
  VB_REQUIRE((int64_t)tiles_n * tiles_m < (int64_t(1) << 28), "linear_q8: %d x %d outputs exceed the grid", a.M, a.N);
  CUtensorMap wmap, xmap, ymap = {};
  int rc = make_byte_map(&wmap, a.wq, a.N, a.K, a.ldw, C::BROWS);
  if (!rc) rc = make_byte_map(&xmap, a.xq, a.M, a.K, a.ldx, ROWS);
  // y leaves by TMA where its rows start on 16-byte boundaries, else by the warps' own stores
  const int by_tma = aligned16(a.y) && ((int64_t)a.N * sizeof(T)) % 16 == 0;
  if (!rc && by_tma) rc = make_out_map(&ymap, a.y, a.M, a.N, 128 / (int)sizeof(T), 32, sizeof(T) == 4 ? VB_F32 : VB_BF16);
  if (rc) return rc;
  const int groups = min(tiles_n * tiles_m, sm_count() / GROUP);
  return launch_early("linear_q8", linear_q8_tile_kernel<GROUP, BN, T>, dim3(GROUP * groups), C::THREADS, C::SMEM, GROUP, a.st, wmap, xmap,
                ymap, by_tma, a.xs, a.ws, (T*)a.y, a.M, a.N, kblocks, tiles_n, tiles_m, a.status);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_linear_q8(const int8_t* xq, int64_t ldx, const float* xs, const int8_t* wq, int64_t ldw,
                            const float* ws, void* y, int M, int N, int K, int dtype, int* status, void* stream) {
  VB_REQUIRE(M >= 0 && N > 0 && K > 0 && ldx >= K && ldw >= K, "linear_q8: bad shape M=%d N=%d K=%d pitches %lld, %lld",
             M, N, K, (long long)ldx, (long long)ldw);
  VB_REQUIRE(K <= 131056, "linear_q8: K=%d exceeds 131056, above which a sum may leave int32", K);
  constexpr int MOST = INT32_MAX - 255;  // a tile more is still an int
  VB_REQUIRE(M <= MOST && N <= MOST, "linear_q8: %d x %d outputs, of at most %d rows and columns", M, N, MOST);
  VB_REQUIRE(dtype_size(dtype) > 0, "linear_q8: unsupported dtype code %d", dtype);
  if (M == 0) return VB_OK;
  VB_REQUIRE(xq && xs && wq && ws && y && status, "linear_q8: null pointer");
  VB_REQUIRE(aligned16(xq) && aligned16(wq) && ldx % 16 == 0 && ldw % 16 == 0,
             "linear_q8: operands must start on 16-byte boundaries with pitches a multiple of 16");
  const Args a{xq, ldx, xs, wq, ldw, ws, y, M, N, K, status, (cudaStream_t)stream};
  return VB_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    // Few tokens: the split kernel, whose time is the weights' bytes. Tiles of 32 tokens rather than 64 where the
    // weights are small and CTAs few (64 x 1536 x 512: 4.2 us against 4.7; 64 x 4096 x 8192: 12.9 against 10.8). Up to
    // 256 tokens while K is long (256 x 4096 x 4096: 12.1 us, in tiles 13.7; 256 x 512 x 1544: 6.0 and 4.2).
    const int64_t kb = (K + KB - 1) / KB;
    if (M <= 16) return launch_split<16, T>(a);
    if (M <= 32 || (M <= 64 && (int64_t)N * K <= (4 << 20))) return launch_split<32, T>(a);
    if (M <= 64 || (M <= 256 && kb > 16)) return launch_split<64, T>(a);
    // Else the tile that the measured times of one wave favour, in tenths of a microsecond per wave of tiles: the
    // larger of its products' time per block of K and its store's. 1024 x 4096 x 4096: 17.0 us on pairs, 25.5 with
    // 128 channels, 45.4 with 64; 4096 x 512 x 1536: 9.3, 8.6, 12.4; 1024 x 1024 x 1024: 7.7, 6.1, 5.6.
    const int sms = sm_count();
    auto waves = [&](int tm, int tn, int slots) { return ((int64_t)((M + tm - 1) / tm) * ((N + tn - 1) / tn) + slots - 1) / slots; };
    const double pair = 40 + waves(256, 256, sms / 2) * fmax(4.1 * kb, 34.0);
    const double wide = 35 + waves(128, 128, sms) * fmax(3.57 * kb, 19.0);
    const double narrow = 32 + waves(128, 64, sms) * fmax(3.3 * kb, 16.0);
    if (narrow <= wide && narrow <= pair) return launch_tile<1, 64, T>(a);
    return wide <= pair ? launch_tile<1, 128, T>(a) : launch_tile<2, 256, T>(a);
  });
}
