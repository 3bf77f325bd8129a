// Linear layers with their epilogue, bf16 in / fp32 accumulate / bf16 out, for sm_100a:
//   y = residual + gate * act(x w^T + bias)          x [m, k], w [n, k], bias / gate [n], residual / y [m, n]
// and their gradients:  dz = gate dy act'(z) (z = x w^T + bias, which the forward keeps for it), dx = dz w, dw = dz^T x,
// db = sum dz, dgate = sum dy act(z).
//
// gemm_kernel computes C = A B^T over operands whose contraction dimension is contiguous (K-major) or not (MN-major:
// the tcgen05 descriptors read such tiles transposed), so dx and dw need no transposed copies. Persistent and warp
// specialised: warp 0 streams 64-deep A and B tiles by TMA into a ring, warp 1 issues the MMAs into one of two TMEM
// accumulators, four or eight warps drain the other: bias, activation, gate, residual and the bf16 stores run under the
// next tile's MMAs. kCtas = 2: a cluster of two CTAs owns a 256 x 256 tile (tcgen05 cta_group::2): each holds half of A's
// rows and half of B's, so an SM reads 64 bytes of shared memory per clock where a 128 x 256 tile of its own would read
// 96 and fill as much again. Its epilogue moves 32-row x 64-column pieces through shared memory: the residual comes in
// and y (and z) go out by TMA, whole 128-byte lines at a time (stored from the registers, a row per lane, the epilogue of
// 9540 x 2048 -> 8192 with z took longer than the product: 319 us instead of 222). kCtas = 1 serves problems too small
// for that, down to a few rows. Rows and columns past the ends are zeros (TMA fill) and are not stored.
// Every mbarrier wait is bounded (ptx.cuh); the epilogue warps' have one verdict per warp.
//
// Measured (device time): 22260 x 8192 -> 2048 with bias, gate and residual 490 to 520 us a launch by itself, 1.43 to 1.52
// PFLOP/s, 0.88 to 0.93 of a library product's burst rate; 610 us (1.22 PFLOP/s) in a row, under the power cap. 9540 x 2048
// -> 8192 with gelu 238 us keeping z, dx 234, dw 219, dz and db 99 + 4. Few rows: 1 x 2048 -> 24576 19.4 us, 0.79 of the
// memory's copy rate; 77 x 2048 -> 8192 11.4 us (the weight alone 5.4), where neither the memory nor the tensor pipe is
// busy: a block's chain of loads, products and epilogue is.
//
// Rounded to bf16 are the outputs, z and dz: dz as the operand of two tensor-core products, z because it is m n values to
// store and read again (act' and act of the rounded z move dz and dgate by half a step of z at most).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "column_sum.cuh"
#include "orl_common.h"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace orl {

// ------------------------------------------------------------------------------------------------ activations
// With t = 1 / (1 + exp(-a)): silu a = z, gelu_tanh a = 2 sqrt(2 / pi) (z + 0.044715 z^3) (tanh(u) = 2 sigmoid(2u) - 1);
// act = z t in both, act' = t + z a' t (1 - t). z^2 is capped where t has long been 0 or 1, so that a and a' stay finite.
constexpr float kMinusLog2e = -1.4426950408889634f;
constexpr float kGelu = 1.5957691216057308f;          // 2 sqrt(2 / pi)
constexpr float kGelu3 = 0.044715f;

template <int kAct>
__device__ __forceinline__ float gate_of(float z, float z2) {
  const float a = kAct == ORL_ACT_GELU_TANH ? z * fmaf(kMinusLog2e * kGelu * kGelu3, z2, kMinusLog2e * kGelu)
                                            : z * kMinusLog2e;
  return __fdividef(1.0f, 1.0f + ex2(a));
}

template <int kAct>
__device__ __forceinline__ float activate(float z) {
  if (kAct == ORL_ACT_NONE) return z;
  return z * gate_of<kAct>(z, fminf(z * z, 1e4f));
}

// act(z) and act'(z)
template <int kAct>
__device__ __forceinline__ float2 activate_slope(float z) {
  if (kAct == ORL_ACT_NONE) return make_float2(z, 1.0f);
  const float z2 = fminf(z * z, 1e4f);
  const float t = gate_of<kAct>(z, z2);
  const float s = fmaf(-t, t, t);                      // t (1 - t): 0 far out
  const float d = kAct == ORL_ACT_GELU_TANH ? fmaf(3.0f * kGelu * kGelu3, z2, kGelu) * s : s;
  return make_float2(z * t, fmaf(z, d, t));
}

__device__ __forceinline__ void unpack8(uint4 r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// what happens to a product on its way out; null pointers: not there
struct Epilogue {
  const __nv_bfloat16* bias;
  const __nv_bfloat16* gate;
  const __nv_bfloat16* residual;
  long long ldr;
  __nv_bfloat16* y;        // [m, n]
  __nv_bfloat16* z;        // [m, n]: x w^T + bias, kept for the backward pass
  int act;
};

// eight columns n0.. of a row: f = products in, y out, z = their bf16 sums with the bias; res: the residual's values or
// null
__device__ __forceinline__ void finish8(const Epilogue& ep, int n0, float (&f)[8], uint4& z, const uint4* res) {
  float t[8];
  if (ep.bias != nullptr) {
    unpack8(__ldg(reinterpret_cast<const uint4*>(ep.bias + n0)), t);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += t[i];
  }
  z = pack8(f);
  if (ep.act == ORL_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = activate<ORL_ACT_GELU_TANH>(f[i]);
  } else if (ep.act == ORL_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = activate<ORL_ACT_SILU>(f[i]);
  }
  if (ep.gate != nullptr) {
    unpack8(__ldg(reinterpret_cast<const uint4*>(ep.gate + n0)), t);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= t[i];
  }
  if (res != nullptr) {
    unpack8(*res, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += t[i];
  }
}

// the same with its loads and stores straight from memory
__device__ __forceinline__ void finish8_global(const Epilogue& ep, long long row, int n0, int n, float (&f)[8]) {
  uint4 z, r;
  if (ep.residual != nullptr) r = *reinterpret_cast<const uint4*>(ep.residual + row * ep.ldr + n0);
  finish8(ep, n0, f, z, ep.residual != nullptr ? &r : nullptr);
  if (ep.z != nullptr) *reinterpret_cast<uint4*>(ep.z + row * n + n0) = z;
  *reinterpret_cast<uint4*>(ep.y + row * n + n0) = pack8(f);
}

// ------------------------------------------------------------------------------------------------ matrix product

constexpr int kBk = 64;                                // contraction depth of a stage: one 128-byte swizzle row

template <int kCtas, int BN>
struct GemmCfg {
  static constexpr int kTileM = 128 * kCtas;           // rows of C per cluster
  static constexpr int kBRows = BN / kCtas;            // columns of C whose B each CTA holds
  static constexpr int kABytes = 128 * kBk * 2;
  static constexpr int kBBytes = kBRows * kBk * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // kCtas = 2: eight epilogue warps, two per 32 rows that take pieces by turns (with four, bias, gelu and z of a 256 x 256
  // tile at k = 2048 took longer than its product); staging of two pieces each: y (the residual first) and z, or y twice
  static constexpr bool kStaged = kCtas == 2;
  static constexpr int kEpiWarps = kStaged ? 8 : 4;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kPiece = 32 * 128;
  static constexpr int kStagingBytes = kStaged ? kEpiWarps * 2 * kPiece : 0;
  static constexpr int kStages = (224 * 1024 - kStagingBytes) / kStageBytes;
  static constexpr int kStagingOff = kStages * kStageBytes;
  static constexpr int kBarOff = kStagingOff + kStagingBytes;
  static constexpr int kBarFull = 0;
  static constexpr int kBarEmpty = kStages;
  static constexpr int kBarAccFull = 2 * kStages;      // + accumulator
  static constexpr int kBarAccEmpty = kBarAccFull + 2;
  static constexpr int kBarRes = kBarAccEmpty + 2;     // residual piece landed, per epilogue warp and buffer
  static constexpr int kBarDrain = kBarRes + 2 * kEpiWarps;
  static constexpr int kNumBars = kBarDrain + 1;
  static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16 + 1024;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
  static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols >= 32 && kTmemCols <= 512, "TMEM allocation size");
  static_assert(kStageBytes % 1024 == 0 && (!kStaged || BN % 64 == 0), "tile alignment");
};

struct GemmShape {
  int m, n, k;             // C [m, n], contraction k
  int tiles_m, tiles_n;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// arrive on the barrier at the same shared-memory offset in CTA 0 of the cluster
__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [ra];\n\t}" ::"r"(bar)
      : "memory");
}
// 2-D tiled load (no multicast) into this CTA whose bytes complete on the barrier of the pair's CTA 0 (the address
// with the CTA's bit cleared)
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y,
                                                 uint64_t cache_hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y), "l"(cache_hint)
      : "memory");
}
__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on the barrier at this offset in both CTAs of the pair once the MMAs issued before have completed
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

struct GemmShared {
  uint32_t sbase, bar0;
  volatile int* abort_flag;
  __device__ uint32_t bar(int i) const { return bar0 + 8u * i; }
};

// tile -> (tile row, tile column): groups of eight tile rows, columns outermost in a group, so that the tiles in flight
// share A and B tiles in L2
__device__ __forceinline__ int2 tile_at(const GemmShape& g, int t) {
  constexpr int kGroup = 8;
  const int per = kGroup * g.tiles_n;
  const int first = (t / per) * kGroup;
  const int rows = min(kGroup, g.tiles_m - first);
  const int r = t % per;
  return make_int2(first + r % rows, r / rows);
}

template <int kCtas, int BN, bool kAmn, bool kBmn>
__global__ void __launch_bounds__(GemmCfg<kCtas, BN>::kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_z,
                const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ GemmShape g, const __grid_constant__ Epilogue ep, int* __restrict__ err) {
  using C = GemmCfg<kCtas, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOff + C::kNumBars * 8);
  GemmShared sh;
  sh.sbase = smem_u32(smem);
  sh.bar0 = sh.sbase + C::kBarOff;
  sh.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kCtas == 2 ? static_cast<int>(cluster_rank()) : 0;
  const int cluster = blockIdx.x / kCtas, n_clusters = gridDim.x / kCtas;
  const int n_tiles = g.tiles_m * g.tiles_n;
  const int n_k = (g.k + kBk - 1) / kBk;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(sh.bar(C::kBarFull + s), 1);
      mbar_init(sh.bar(C::kBarEmpty + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sh.bar(C::kBarAccFull + i), 1);
      mbar_init(sh.bar(C::kBarAccEmpty + i), C::kEpiWarps * kCtas);
    }
    for (int i = 0; i < 2 * C::kEpiWarps; ++i) mbar_init(sh.bar(C::kBarRes + i), 1);
    mbar_init(sh.bar(C::kBarDrain), 1);
    *sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if (kCtas == 2) {
      tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
    } else {
      tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kCtas == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      tma_prefetch_map(&tm_a);
      tma_prefetch_map(&tm_b);
      const uint64_t pol = policy_evict_last();
      auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
        if (kCtas == 2) tma_load_2d_pair(dst, map, bar, x, y, pol);
        else tma_load_2d(dst, map, bar, x, y, pol);
      };
      int it = 0;
      bool ok = true;
      for (int t = cluster; ok && t < n_tiles; t += n_clusters) {
        const int2 at = tile_at(g, t);
        const int m0 = at.x * C::kTileM + 128 * rank, n0 = at.y * BN + C::kBRows * rank;
        for (int kb = 0; kb < n_k; ++kb, ++it) {
          const int s = it % C::kStages;
          if (it >= C::kStages && !mbar_wait(sh.bar(C::kBarEmpty + s), ((it / C::kStages) - 1) & 1, sh.abort_flag)) {
            atomicOr(err, kErrTimeoutLoad);
            ok = false;
            break;
          }
          const uint32_t a = sh.sbase + s * C::kStageBytes, b = a + C::kABytes, bar = sh.bar(C::kBarFull + s);
          if (rank == 0) mbar_expect_tx(bar, kCtas * C::kStageBytes);
          const int k0 = kb * kBk;
          if (kAmn) {
            for (int c = 0; c < 2; ++c) load(a + c * 8192, &tm_a, bar, m0 + 64 * c, k0);
          } else {
            load(a, &tm_a, bar, k0, m0);
          }
          if (kBmn) {
            for (int c = 0; c < C::kBRows / 64; ++c) load(b + c * 8192, &tm_b, bar, n0 + 64 * c, k0);
          } else {
            load(b, &tm_b, bar, k0, n0);
          }
        }
      }
      if (*sh.abort_flag && rank == 0) {
        // wind down: the copies in flight (both CTAs' complete on CTA 0's barriers) land before shared memory goes
        for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i) {
          const unsigned long long t0 = global_ns();
          while (!mbar_try_wait(sh.bar(C::kBarFull + i % C::kStages), (i / C::kStages) & 1))
            if (global_ns() - t0 > kWaitLimitNs) {
              atomicOr(err, kErrTimeoutDrain);
              break;
            }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (CTA 0 of a pair)
    if (rank == 0 && elect_one()) {
      constexpr uint32_t kIdesc = idesc_bf16(C::kTileM, BN, kAmn, kBmn);
      auto commit = [&](uint32_t bar) {
        if (kCtas == 2) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      int it = 0, n = 0;
      bool ok = true;
      for (int t = cluster; ok && t < n_tiles; t += n_clusters, ++n) {
        const int buf = n & 1;
        if (n >= 2) ok = mbar_wait(sh.bar(C::kBarAccEmpty + buf), ((n >> 1) - 1) & 1, sh.abort_flag);
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int kb = 0; ok && kb < n_k; ++kb, ++it) {
          const int s = it % C::kStages;
          ok = mbar_wait(sh.bar(C::kBarFull + s), (it / C::kStages) & 1, sh.abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = sh.sbase + s * C::kStageBytes, b = a + C::kABytes;
#pragma unroll
          for (int kk = 0; kk < kBk / 16; ++kk) {
            // K-major: 16 columns on; MN-major: 16 rows of 128 bytes on, 64-column blocks 8 KiB apart
            const uint64_t da = kAmn ? smem_desc_sw128(a + kk * 2048, 8192, 1024) : smem_desc_sw128(a + kk * 32, 16, 1024);
            const uint64_t db = kBmn ? smem_desc_sw128(b + kk * 2048, 8192, 1024) : smem_desc_sw128(b + kk * 32, 16, 1024);
            if (kCtas == 2) mma_ss_pair(d, da, db, kIdesc, (kb | kk) ? 1u : 0u);
            else mma_ss(d, da, db, kIdesc, (kb | kk) ? 1u : 0u);
          }
          commit(sh.bar(C::kBarEmpty + s));
        }
        if (ok) commit(sh.bar(C::kBarAccFull + buf));
      }
      if (!ok) {
        atomicOr(err, kErrTimeoutMma);
        commit(sh.bar(C::kBarDrain));
        const unsigned long long t0 = global_ns();
        while (!mbar_try_wait(sh.bar(C::kBarDrain), 0))
          if (global_ns() - t0 > kWaitLimitNs) {
            atomicOr(err, kErrTimeoutDrain);
            break;
          }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue: one row per thread
    const int ew = warp - 4;
    const uint32_t lanes = static_cast<uint32_t>(32 * (ew & 3)) << 16;
    const bool res = ep.residual != nullptr, two = ep.z == nullptr;    // two: both pieces are y's, by turns
    uint8_t* staging = smem + C::kStagingOff + ew * 2 * C::kPiece;
    const uint32_t staging_s = sh.sbase + C::kStagingOff + ew * 2 * C::kPiece;
    int n = 0, piece = 0;                                              // pieces done by this warp
    bool ok = true;
    for (int t = cluster; ok && t < n_tiles; t += n_clusters, ++n) {
      const int buf = n & 1;
      const int2 at = tile_at(g, t);
      const int row0 = at.x * C::kTileM + 128 * rank + 32 * (ew & 3);
      const int n0 = at.y * BN;
      const uint32_t acc = tmem + buf * BN + lanes;
      if constexpr (C::kStaged) {
        // piece p goes into buffer b: free once the store that used it last has read it; then its residual comes in
        auto prepare = [&](int p, int c) {
          const int b = two ? p & 1 : 0;
          if (lane == 0) {
            if (two) bulk_wait_read<1>();
            else bulk_wait_read<0>();
            if (res) {
              mbar_expect_tx(sh.bar(C::kBarRes + 2 * ew + b), C::kPiece);
              tma_load_2d(staging_s + b * C::kPiece, &tm_r, sh.bar(C::kBarRes + 2 * ew + b), n0 + c, row0,
                          policy_evict_first());
            }
          }
          __syncwarp();
        };
        const int half = ew >> 2;                // this warp's pieces: half, half + 2, ...
        const int n_pieces = row0 < g.m ? (min(BN, g.n - n0) + 63) / 64 : 0;
        if (half < n_pieces) prepare(piece, 64 * half);
        ok = mbar_wait_warp(sh.bar(C::kBarAccFull + buf), (n >> 1) & 1, sh.abort_flag);
        if (ok) tc_fence_after();
#pragma unroll 1
        for (int i = half; ok && i < n_pieces; i += 2, ++piece) {
          const int b = two ? piece & 1 : 0;
          uint32_t v[64];
          tmem_ld32(acc + 64 * i, *reinterpret_cast<uint32_t(*)[32]>(v));
          tmem_ld32(acc + 64 * i + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
          tmem_wait_ld();
          if (res) {
            ok = mbar_wait_warp(sh.bar(C::kBarRes + 2 * ew + b), (two ? piece >> 1 : piece) & 1, sh.abort_flag);
            if (!ok) break;
          }
          uint8_t* y = staging + b * C::kPiece + lane * 128;
          uint8_t* z = staging + C::kPiece + lane * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const int col = n0 + 64 * i + 8 * c;
            uint4* dst = reinterpret_cast<uint4*>(y + ((c ^ (lane & 7)) << 4));      // the 128-byte swizzle
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[8 * c + e]);
            uint4 zz;
            const uint4 r = res ? *dst : make_uint4(0u, 0u, 0u, 0u);
            finish8(ep, min(col, g.n - 8), f, zz, res ? &r : nullptr);               // columns past the end: not stored
            *dst = pack8(f);
            if (!two) *reinterpret_cast<uint4*>(z + ((c ^ (lane & 7)) << 4)) = zz;
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tm_y, staging_s + b * C::kPiece, n0 + 64 * i, row0);
            if (!two) tma_store_2d(&tm_z, staging_s + C::kPiece, n0 + 64 * i, row0);
            bulk_commit();
          }
          if (i + 2 < n_pieces) prepare(piece + 1, 64 * (i + 2));
        }
      } else {
        ok = mbar_wait_warp(sh.bar(C::kBarAccFull + buf), (n >> 1) & 1, sh.abort_flag);
        if (ok) tc_fence_after();
        const long long row = row0 + lane;
#pragma unroll 1
        for (int c = 0; ok && c < BN; c += 32) {
          if (n0 + c >= g.n) break;
          uint32_t v[32];
          tmem_ld32(acc + c, v);
          tmem_wait_ld();
          if (row < g.m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (n0 + c + 8 * i < g.n) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[8 * i + e]);
                finish8_global(ep, row, n0 + c + 8 * i, g.n, f);
              }
            }
          }
        }
      }
      if (!ok) {
        atomicOr(err, kErrTimeoutSoftmax);
        break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kCtas == 2) mbar_arrive_leader(sh.bar(C::kBarAccEmpty + buf));
        else mbar_arrive(sh.bar(C::kBarAccEmpty + buf));
      }
    }
    if (C::kStaged && lane == 0) {
      if (!ok && res) {                          // a residual piece may be in flight: it lands before shared memory goes
        const unsigned long long t0 = global_ns();
        while (!mbar_try_wait(sh.bar(C::kBarRes + 2 * ew + (two ? piece & 1 : 0)), (two ? piece >> 1 : piece) & 1))
          if (global_ns() - t0 > kWaitLimitNs) {
            atomicOr(err, kErrTimeoutDrain);
            break;
          }
      }
      bulk_wait_read<0>();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (kCtas == 2) cluster_sync();           // the peer may still arrive on, or read, this CTA's shared memory
  if (warp == 1) {
    tc_fence_after();
    if (kCtas == 2) tmem_dealloc_pair(tmem, C::kTmemCols);
    else tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// m <= kRowsMax rows: the weight is read once and little else happens, so tensor-core tiles would leave most SMs idle
// (n / 64 CTAs). A block of eight warps takes eight output columns; the warps split the depth and read their parts of the
// eight weight rows with 16-byte loads, all of them in flight at once; sums meet in shared memory.
constexpr int kRowsMax = 4;

template <int M>
__global__ void __launch_bounds__(256) linear_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx,
                                                          const __nv_bfloat16* __restrict__ w, long long ldw, int n,
                                                          int k, Epilogue ep) {
  __shared__ float part[M * 8][9];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = 8 * blockIdx.x;                        // n is a multiple of 8
  const __nv_bfloat16* w0 = w + static_cast<long long>(n0) * ldw;
  float acc[M][8];
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[r][c] = 0.f;
  for (int e = 256 * warp + 8 * lane; e < k; e += 2048) {
    uint4 wr[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) wr[c] = __ldcs(reinterpret_cast<const uint4*>(w0 + c * ldw + e));
    float xf[M][8];
#pragma unroll
    for (int r = 0; r < M; ++r) unpack8(__ldg(reinterpret_cast<const uint4*>(x + r * ldx + e)), xf[r]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float wf[8];
      unpack8(wr[c], wf);
#pragma unroll
      for (int r = 0; r < M; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][c] = fmaf(xf[r][i], wf[i], acc[r][c]);
    }
  }
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r][c] += __shfl_xor_sync(0xffffffffu, acc[r][c], o);
      if (lane == 0) part[8 * r + c][warp] = acc[r][c];
    }
  __syncthreads();
  const int r = threadIdx.x;
  if (r < M) {
    float f[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      f[c] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[c] += part[8 * r + c][i];
    }
    finish8_global(ep, r, n0, n, f);
  }
}

// Their gradients, likewise bound by the weight-sized tensor: dx [m, k] = dz w reads w once (a block takes 256 columns of a
// strip of w's rows, its sums are one partial row of m k values), dw [n, k] = dz^T x writes dw once.
constexpr int kRowsDxBlocks = 592;                       // at most, over columns and strips: 4 per SM

template <int M>
__global__ void __launch_bounds__(256) linear_rows_dx_kernel(const __nv_bfloat16* __restrict__ dz, long long lddz,
                                                             const __nv_bfloat16* __restrict__ w, long long ldw, int n,
                                                             int k, float* __restrict__ part) {
  __shared__ float red[8][M][257];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = 256 * blockIdx.x + 8 * lane;
  const int per = (n + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = min(n, lo + per);
  float acc[M][8];
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[r][i] = 0.f;
  if (col < k) {
    for (int j0 = lo + warp; j0 < hi; j0 += 32) {
      uint4 wr[4];                                       // four rows' loads in flight
#pragma unroll
      for (int u = 0; u < 4; ++u)
        wr[u] = j0 + 8 * u < hi ? __ldcs(reinterpret_cast<const uint4*>(w + (j0 + 8 * u) * ldw + col))
                                : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = min(j0 + 8 * u, hi - 1);
        float wf[8];
        unpack8(wr[u], wf);
#pragma unroll
        for (int r = 0; r < M; ++r) {
          const float g = j0 + 8 * u < hi ? __bfloat162float(dz[r * lddz + j]) : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(g, wf[i], acc[r][i]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int i = 0; i < 8; ++i) red[warp][r][8 * lane + i] = acc[r][i];
  __syncthreads();
  const int c = 256 * blockIdx.x + threadIdx.x;
  if (c < k) {
#pragma unroll
    for (int r = 0; r < M; ++r) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a += red[i][r][threadIdx.x];
      part[(static_cast<long long>(blockIdx.y) * M + r) * k + c] = a;
    }
  }
}

template <int M>
__global__ void __launch_bounds__(256) linear_rows_dw_kernel(const __nv_bfloat16* __restrict__ dz, long long lddz,
                                                             const __nv_bfloat16* __restrict__ x, long long ldx, int n,
                                                             int k, __nv_bfloat16* __restrict__ dw) {
  // one 16-byte vector of a row of dw per thread; a block's rows follow each other
  const int vecs = k / 8;
  const long long total = static_cast<long long>(n) * vecs;
  for (long long v = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; v < total;
       v += static_cast<long long>(gridDim.x) * 256) {
    const int j = static_cast<int>(v / vecs), c = 8 * static_cast<int>(v - static_cast<long long>(j) * vecs);
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < M; ++r) {
      const float g = __bfloat162float(dz[r * lddz + j]);
      float xf[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(x + r * ldx + c)), xf);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = fmaf(g, xf[i], f[i]);
    }
    __stcs(reinterpret_cast<uint4*>(dw) + v, pack8(f));
  }
}

static int rows_dx_strips(int n, int k) {
  return std::max(1, std::min((n + 63) / 64, kRowsDxBlocks / std::max(1, (k + 255) / 256)));
}

template <int M>
static int rows_gradients(const void* dz, long long lddz, const void* x, long long ldx, const void* w, long long ldw,
                          void* dx, void* dw, float* scratch, int n, int k, cudaStream_t stream) {
  auto bf = [](const void* p) { return static_cast<const __nv_bfloat16*>(p); };
  if (dx != nullptr) {
    const int strips = rows_dx_strips(n, k);
    linear_rows_dx_kernel<M><<<dim3((k + 255) / 256, strips), 256, 0, stream>>>(bf(dz), lddz, bf(w), ldw, n, k, scratch);
    if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
    const int rc = column_sum(scratch, strips, M * k, static_cast<long long>(M) * k, dx, stream);
    if (rc != ORL_OK) return rc;
  }
  if (dw != nullptr) {
    const long long blocks = std::min<long long>(8 * 148, (static_cast<long long>(n) * (k / 8) + 255) / 256);
    linear_rows_dw_kernel<M><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(bf(dz), lddz, bf(x), ldx, n, k,
                                                                               static_cast<__nv_bfloat16*>(dw));
    if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  }
  return ORL_OK;
}

// ------------------------------------------------------------------------------------------------ dz and column sums
// dz = gate * dy * act'(z), with the column sums of dz (bias) and of dy * act(z) (gate). Memory bound. A block covers
// 256 columns (8 per thread, 32 threads across) and a strip of rows (8 at a time); its sums are one partial row.
constexpr int kDzBlocks = 1184;                          // at most, over rows and columns: 8 per SM

template <int kAct, bool kGateGrad>
__global__ void __launch_bounds__(256, 4) linear_dz_kernel(const __nv_bfloat16* __restrict__ dy, long long lddy,
                                                        const __nv_bfloat16* __restrict__ z,
                                                        const __nv_bfloat16* __restrict__ gate, int m, int n,
                                                        __nv_bfloat16* __restrict__ dz, float* __restrict__ part_b,
                                                        float* __restrict__ part_g) {
  __shared__ float red[8][257];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = 256 * blockIdx.x + 8 * tx;
  const bool on = col < n;
  float sb[8], sg[8], gf[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sb[i] = sg[i] = 0.f;
    gf[i] = 1.f;
  }
  if (on && gate != nullptr) unpack8(__ldg(reinterpret_cast<const uint4*>(gate + col)), gf);
  if (on) {
    const int stride = 8 * gridDim.y;
    const bool slope = z != nullptr;
    for (int r0 = 8 * blockIdx.y + ty; r0 < m; r0 += 2 * stride) {
      uint4 rd[2], rz[2];                                // two rows' loads in flight
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = r0 + u * stride;
        rd[u] = rz[u] = make_uint4(0u, 0u, 0u, 0u);
        if (r < m) {
          rd[u] = __ldcs(reinterpret_cast<const uint4*>(dy + r * lddy + col));
          if (slope) rz[u] = __ldcs(reinterpret_cast<const uint4*>(z + static_cast<long long>(r) * n + col));
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = r0 + u * stride;
        if (r >= m) break;                               // no 0 * gate where the gate is infinite
        float d[8];
        unpack8(rd[u], d);
        if (slope) {
          float h[8];
          unpack8(rz[u], h);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 a = activate_slope<kAct>(h[i]);
            if (kGateGrad) sg[i] += d[i] * a.x;
            d[i] *= gf[i] * a.y;
          }
        } else if (gate != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] *= gf[i];
        }
        if (dz != nullptr) *reinterpret_cast<uint4*>(dz + static_cast<long long>(r) * n + col) = pack8(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) sb[i] += d[i];
      }
    }
  }
#pragma unroll 1
  for (int which = 0; which < (kGateGrad ? 2 : 1); ++which) {
    float* part = which == 0 ? part_b : part_g;
    if (part == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[ty][8 * tx + i] = which == 0 ? sb[i] : sg[i];
    __syncthreads();
    const int c = threadIdx.x;
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a += red[i][c];
    if (256 * blockIdx.x + c < n) part[static_cast<long long>(blockIdx.y) * n + 256 * blockIdx.x + c] = a;
  }
}

static int dz_strips(int m, int n) {
  const int cols = (n + 255) / 256;
  return std::max(1, std::min((m + 7) / 8, kDzBlocks / cols));
}

// ------------------------------------------------------------------------------------------------ host side

template <int kCtas, int BN, bool kAmn, bool kBmn>
static int launch_gemm(const void* a, long long lda, const void* b, long long ldb, GemmShape g, const Epilogue& ep,
                       int* err, cudaStream_t stream) {
  using C = GemmCfg<kCtas, BN>;
  g.tiles_m = (g.m + C::kTileM - 1) / C::kTileM;
  g.tiles_n = (g.n + BN - 1) / BN;
  if (static_cast<long long>(g.tiles_m) * g.tiles_n > 0x7fffffffLL) return ORL_ERR_ARG;
  CUtensorMap ma, mb;
  int rc;
  rc = kAmn ? make_rows_map(&ma, a, g.k, g.m, lda, kBk) : make_rows_map(&ma, a, g.m, g.k, lda, 128);
  if (rc != ORL_OK) return rc;
  rc = kBmn ? make_rows_map(&mb, b, g.k, g.n, ldb, kBk) : make_rows_map(&mb, b, g.n, g.k, ldb, C::kBRows);
  if (rc != ORL_OK) return rc;
  CUtensorMap my = ma, mz = ma, mr = ma;                 // used where there is a z, a residual
  if (C::kStaged) {
    if ((rc = make_rows_map(&my, ep.y, g.m, g.n, g.n, 32)) != ORL_OK) return rc;
    if (ep.z != nullptr && (rc = make_rows_map(&mz, ep.z, g.m, g.n, g.n, 32)) != ORL_OK) return rc;
    if (ep.residual != nullptr && (rc = make_rows_map(&mr, ep.residual, g.m, g.n, ep.ldr, 32)) != ORL_OK) return rc;
  }
  auto kernel = gemm_kernel<kCtas, BN, kAmn, kBmn>;
  static std::mutex mu;
  static int clusters[kMaxDevices] = {};                 // clusters resident at once
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int most;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (clusters[dev] == 0) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != cudaSuccess)
        return ORL_ERR_LAUNCH;
      cfg.gridDim = dim3(kCtas);
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) return ORL_ERR_LAUNCH;
      clusters[dev] = n;
    }
    most = clusters[dev];
  }
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * std::min(most, g.tiles_m * g.tiles_n)));
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, my, mz, mr, g, ep, err) == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
}

// Tile choice: the largest tile that still occupies the GPU. The pair's 256 x 256 tile reads the least shared memory per
// MMA, 256 x 128 has twice the tiles; below that one CTA takes 128 x 64, or 128 x 32 where few rows leave the streaming of
// the weight to too few SMs. Measured on both sides (us, k = 2048 unless given, events resolve 2 us):
//   256 x 256 from 60 tiles on: 300 x 8192 (64 tiles) 25 against 27 with 256 x 128, 1800 x 2048 (64) 23 and 23; below,
//     1001 x 2048 (32) 20 against 16, 1537 x 2048 (56) 23 and 23, 1001 x 2048 for dw of depth 1001 (32) 16 against 12.
//   256 x 128 from 48 on: 513 x 2048 (48) 16 against 18 with 128 x 64, 2000 x 1024 at k = 8192 (64) 41 against 53; below,
//     300 x 2048 (32) 14 against 12, 1024 x 1024 for dw of depth 1001 (32) 12 against 10.
//   128 x 64 from 80 on: 300 x 2048 (96) 13 against 17 with 128 x 32, 77 x 8192 (128) 14 against 18; below, 200 x 2048 (64) 12
//     and 12, with silu, gate and residual at k = 1024 13 against 11, 77 x 2048 at k = 8192 (32) 29 against 27.
// Streaming kernels against 128 x 64 tiles: 1 x 2048 -> 24576 23 against 49, 3 rows 39 against 49, 4 rows 59 against 49 (and
// 10 against 14 at 2048 -> 2048); dx of one row, 24576 -> 2048, 35 against 84, of four 59 against 68.
template <bool kAmn, bool kBmn>
static int gemm(const void* a, long long lda, const void* b, long long ldb, int m, int n, int k, const Epilogue& ep,
                int* err, cudaStream_t stream) {
  GemmShape g{m, n, k, 0, 0};
  auto tiles = [&](int tm, int tn) { return (static_cast<long long>(m) + tm - 1) / tm * ((n + tn - 1) / tn); };
  if (m > 128 && tiles(256, 256) >= 60) return launch_gemm<2, 256, kAmn, kBmn>(a, lda, b, ldb, g, ep, err, stream);
  if (m > 128 && tiles(256, 128) >= 48) return launch_gemm<2, 128, kAmn, kBmn>(a, lda, b, ldb, g, ep, err, stream);
  if (kBmn || tiles(128, 64) >= 80) return launch_gemm<1, 64, kAmn, kBmn>(a, lda, b, ldb, g, ep, err, stream);
  if constexpr (!kBmn) return launch_gemm<1, 32, kAmn, kBmn>(a, lda, b, ldb, g, ep, err, stream);
  return ORL_ERR_UNSUPPORTED;
}

static bool lin_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int check_linear(long long m, long long n, long long k) {
  // rows and columns are counted in 32 bits, a step of a strip's rows past the end and kRowsMax rows' columns included
  if (m < 0 || n <= 0 || k <= 0 || m > 0x7fff0000LL || n > (1LL << 28) || k > (1LL << 28)) return ORL_ERR_ARG;
  if ((n & 7) || (k & 7)) return ORL_ERR_ALIGN;
  return ORL_OK;
}

}  // namespace orl

using namespace orl;

extern "C" int orl_linear(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                          const void* gate, const void* residual, long long ldr, void* y, void* z, long long m,
                          long long n, long long k, int act, int* err_dev, void* stream_ptr) {
  int rc = check_linear(m, n, k);
  if (rc != ORL_OK) return rc;
  if (act < ORL_ACT_NONE || act > ORL_ACT_SILU || w == nullptr || err_dev == nullptr) return ORL_ERR_ARG;
  if (m > 0 && (x == nullptr || y == nullptr)) return ORL_ERR_ARG;
  if (ldx < k || ldw < k || (residual != nullptr && ldr < n)) return ORL_ERR_ARG;
  if ((ldx & 7) || (ldw & 7) || (residual != nullptr && (ldr & 7))) return ORL_ERR_ALIGN;
  for (const void* p : {x, w, bias, gate, residual, static_cast<const void*>(y), static_cast<const void*>(z)})
    if (!lin_aligned(p)) return ORL_ERR_ALIGN;
  if (m == 0) return ORL_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  auto bf = [](const void* p) { return static_cast<const __nv_bfloat16*>(p); };
  const Epilogue ep{bf(bias), bf(gate), bf(residual), ldr, static_cast<__nv_bfloat16*>(y),
                    static_cast<__nv_bfloat16*>(z), act};
  if (m <= kRowsMax) {
    const unsigned grid = static_cast<unsigned>(n / 8);
    const int nn = static_cast<int>(n), kk = static_cast<int>(k);
    switch (m) {
      case 1: linear_rows_kernel<1><<<grid, 256, 0, stream>>>(bf(x), ldx, bf(w), ldw, nn, kk, ep); break;
      case 2: linear_rows_kernel<2><<<grid, 256, 0, stream>>>(bf(x), ldx, bf(w), ldw, nn, kk, ep); break;
      case 3: linear_rows_kernel<3><<<grid, 256, 0, stream>>>(bf(x), ldx, bf(w), ldw, nn, kk, ep); break;
      default: linear_rows_kernel<4><<<grid, 256, 0, stream>>>(bf(x), ldx, bf(w), ldw, nn, kk, ep);
    }
    return cudaGetLastError() == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
  }
  return gemm<false, false>(x, ldx, w, ldw, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), ep, err_dev,
                            stream);
}

extern "C" long long orl_linear_bwd_scratch(long long m, long long n, long long k) {
  if (check_linear(m, n, k) != ORL_OK) return ORL_ERR_ARG;
  const long long sums = 2ll * dz_strips(static_cast<int>(m), static_cast<int>(n)) * n;
  // few rows: the partial rows of dx, which follow the column sums on the stream and may take their place
  const long long rows = m <= kRowsMax ? m * k * rows_dx_strips(static_cast<int>(n), static_cast<int>(k)) : 0;
  return std::max(sums, rows);
}

extern "C" int orl_linear_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* w,
                              long long ldw, const void* z, const void* gate, int act, void* dz, void* dx, void* dw,
                              void* dbias, void* dgate, float* scratch, long long m, long long n, long long k,
                              int* err_dev, void* stream_ptr) {
  int rc = check_linear(m, n, k);
  if (rc != ORL_OK) return rc;
  if (act < ORL_ACT_NONE || act > ORL_ACT_SILU || err_dev == nullptr || lddy < n) return ORL_ERR_ARG;
  if (m > 0 && (dy == nullptr || (dw != nullptr && x == nullptr))) return ORL_ERR_ARG;
  if ((dw != nullptr && ldx < k) || (dx != nullptr && (w == nullptr || ldw < k))) return ORL_ERR_ARG;
  // an activation's slope and a gate's gradient need z; with it or a gate, dz is not dy and needs room
  if ((act != ORL_ACT_NONE || dgate != nullptr) && z == nullptr && m > 0) return ORL_ERR_ARG;
  const bool products = dx != nullptr || dw != nullptr, sums = dbias != nullptr || dgate != nullptr;
  const bool own_dz = z != nullptr || gate != nullptr;
  if ((own_dz && products && dz == nullptr && m > 0) ||
      ((sums || (dx != nullptr && m <= kRowsMax)) && scratch == nullptr))
    return ORL_ERR_ARG;
  if ((lddy & 7) || (dw != nullptr && (ldx & 7)) || (dx != nullptr && (ldw & 7))) return ORL_ERR_ALIGN;
  for (const void* p : {dy, x, w, z, gate, static_cast<const void*>(dz), static_cast<const void*>(dx),
                        static_cast<const void*>(dw)})
    if (!lin_aligned(p)) return ORL_ERR_ALIGN;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int mm = static_cast<int>(m), nn = static_cast<int>(n), kk = static_cast<int>(k);
  if (sums || (own_dz && products)) {
    const int strips = dz_strips(mm, nn);
    float* part_b = dbias != nullptr ? scratch : nullptr;
    float* part_g = dgate != nullptr ? scratch + static_cast<long long>(strips) * n : nullptr;
    const dim3 grid(static_cast<unsigned>((n + 255) / 256), static_cast<unsigned>(strips));
    auto kernel = act == ORL_ACT_GELU_TANH ? (part_g ? linear_dz_kernel<ORL_ACT_GELU_TANH, true> : linear_dz_kernel<ORL_ACT_GELU_TANH, false>)
                  : act == ORL_ACT_SILU    ? (part_g ? linear_dz_kernel<ORL_ACT_SILU, true> : linear_dz_kernel<ORL_ACT_SILU, false>)
                                           : (part_g ? linear_dz_kernel<ORL_ACT_NONE, true> : linear_dz_kernel<ORL_ACT_NONE, false>);
    kernel<<<grid, 256, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(dy), lddy, static_cast<const __nv_bfloat16*>(z),
        static_cast<const __nv_bfloat16*>(gate), mm, nn,
        own_dz && products ? static_cast<__nv_bfloat16*>(dz) : nullptr, part_b, part_g);
    if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
    if (part_b != nullptr) rc = column_sum(part_b, strips, nn, n, dbias, stream, part_g, dgate);
    else if (part_g != nullptr) rc = column_sum(part_g, strips, nn, n, dgate, stream);
    if (rc != ORL_OK) return rc;
  }
  const void* g = own_dz ? dz : dy;
  const long long ldg = own_dz ? n : lddy;
  if (m > 0 && m <= kRowsMax) {
    auto run = m == 1 ? rows_gradients<1> : m == 2 ? rows_gradients<2> : m == 3 ? rows_gradients<3> : rows_gradients<4>;
    return run(g, ldg, x, ldx, w, ldw, dx, dw, scratch, nn, kk, stream);
  }
  if (dx != nullptr && m > 0) {
    const Epilogue ep{nullptr, nullptr, nullptr, 0, static_cast<__nv_bfloat16*>(dx), nullptr, ORL_ACT_NONE};
    if ((rc = gemm<false, true>(g, ldg, w, ldw, mm, kk, nn, ep, err_dev, stream)) != ORL_OK) return rc;
  }
  if (dw != nullptr) {
    if (m == 0)
      return cudaMemsetAsync(dw, 0, 2 * static_cast<size_t>(n) * k, stream) == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
    const Epilogue ep{nullptr, nullptr, nullptr, 0, static_cast<__nv_bfloat16*>(dw), nullptr, ORL_ACT_NONE};
    return gemm<true, true>(g, ldg, x, ldx, nn, kk, mm, ep, err_dev, stream);
  }
  return ORL_OK;
}
