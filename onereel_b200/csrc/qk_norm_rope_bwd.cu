// Gradients of the fused q/k RMSNorm + rotary embedding (qk_norm_rope.cu), bf16 in / bf16 out, HBM-bound.
//
// Forward, per row (or per head of a row) of G elements: inv = rsqrt(mean(x^2) + eps), n = x * inv * w, y = R n with R
// the pairwise rotation. With u = R^T dy (the rotation by the opposite angle):
//   dw = sum over rows (and heads, for a per-head weight) of u * x * inv
//   dx = inv * (w u) - x * inv^3 * mean(w u x)
// x and dy are read once and dx written once; a row's two sums (x^2 and w u x) are kept in fp32. What keeps such a kernel
// from the memory's rate is the reduction between a row's loads and its stores, and the instructions that it takes. So a
// warp has up to 2048 elements of a row, 64 to a lane: the sums are a lane's own for the most part and one shuffle tree
// ends both, no barrier of a block stands between rows, and the arithmetic works on pairs (f32x2). Rows of more elements
// are shared by up to four warps. Every warp has its own shared-memory ring, filled by bulk copies rows ahead. Lanes keep
// their weight sums in registers over all their rows, so the weight gradient costs a partial row per block; column_sum
// adds the partial rows in a fixed order.
// 22260 rows of 2048: 56 us, 0.80 of the measured copy rate (a block of 256 threads to a row, eight elements each and two
// barriers of the block: 77 us); with the column sums 64 us, over heads 78 us, rows of 5120 over three warps 199 us (0.54).
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

constexpr int kNrMaxStages = 8, kNrWarps = 8, kNrChunk = 256, kNrMaxChunks = 8;

// two bf16 values as a pair of floats (the bits moved up)
__device__ __forceinline__ F2 widen(uint32_t x) {
  return f2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// Values that the compiler is to widen again where they are used, not to keep widened: 64 elements of a row, of its
// gradient and of the weight fit a lane's registers only as bf16.
__device__ __forceinline__ void keep_packed(uint4& x) {
  asm volatile("" : "+r"(x.x), "+r"(x.y), "+r"(x.z), "+r"(x.w));
}
// R^T on a pair: (g.x c + g.y s, g.y c - g.x s), with cc = (c, c) and sn = (s, -s)
__device__ __forceinline__ F2 unrotate(uint32_t g, F2 cc, F2 sn) {
  const float lo = __uint_as_float(g << 16), hi = __uint_as_float(g & 0xffff0000u);
  return ffma2(f2(hi, lo), sn, fmul2(f2(lo, hi), cc));
}
__device__ __forceinline__ void table_pairs(const float* cr, const float* sr, int shift, F2* cc, F2* sn) {
  const float4 c0 = *reinterpret_cast<const float4*>(cr), c1 = *reinterpret_cast<const float4*>(cr + 4);
  const float4 s0 = *reinterpret_cast<const float4*>(sr), s1 = *reinterpret_cast<const float4*>(sr + 4);
  const float c[4] = {c0.x, c0.z, c1.x, c1.z};
  const float s[4] = {shift ? s0.y : s0.x, shift ? s0.w : s0.z, shift ? s1.y : s1.x, shift ? s1.w : s1.z};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cc[i] = f2(c[i], c[i]);
    sn[i] = f2(s[i], -s[i]);
  }
}

// How a lane's chunks (eight elements each, 256 apart) meet the heads. kSame: head_dim divides 256, so all of them have the
// same place in a head and one set of table values serves them. kHead: the same, and the norm is over each head. kAny: the
// table values are read for each chunk, from global memory.
enum { kSame, kHead, kAny };

// `split` warps per row, each with `chunks` chunks of 256 columns (the last one with what is left). A stage of a warp's
// ring holds its part of a row of x and of dy, and the row's tables.
template <int kNC, int kMode>
__global__ void __launch_bounds__(32 * kNrWarps) qk_norm_rope_bwd_kernel(
    const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ weight,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, __nv_bfloat16* __restrict__ dx,
    float* __restrict__ part, long long rows, int hidden, int head_dim, float eps, int shift, long long rope_ld, int split,
    int chunks, int stages, int* __restrict__ err) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kNrWarps * kNrMaxStages];
  __shared__ float2 red[2][kNrWarps];
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / split, groups = (blockDim.x >> 5) / split, wr = warp % split;
  const int col0 = wr * chunks * kNrChunk, cols = min(hidden - col0, chunks * kNrChunk);
  const int d = (8 * lane) % head_dim;     // a lane's place in a head (kSame, kHead)
  const int part_bytes = 2 * kNrChunk * chunks, tab_bytes = kMode == kAny ? 0 : 4 * head_dim;
  const int stage_bytes = 2 * (part_bytes + tab_bytes);
  uint8_t* ring = smem + warp * stages * stage_bytes;
  const uint32_t bar0 = smem_u32(bars + warp * kNrMaxStages), ring0 = smem_u32(ring);
  const long long step = static_cast<long long>(gridDim.x) * groups;
  const long long first = static_cast<long long>(group) * gridDim.x + blockIdx.x;   // few rows go to as many SMs
  // lane 0: the copies of the warp's next row into stage s
  long long row_next = first;
  const uint64_t pol = policy_evict_first();
  auto load = [&](int s) {
    if (row_next >= rows) return false;
    const uint32_t bar = bar0 + 8 * s, dst = ring0 + s * stage_bytes;
    mbar_expect_tx(bar, 2 * (2 * cols + tab_bytes));
    bulk_load(dst, x + row_next * hidden + col0, 2 * cols, bar, pol);
    bulk_load(dst + part_bytes, dy + row_next * hidden + col0, 2 * cols, bar, pol);
    if (kMode != kAny) {
      bulk_load(dst + 2 * part_bytes, cos_t + row_next * rope_ld, tab_bytes, bar, pol);
      bulk_load(dst + 2 * part_bytes + tab_bytes, sin_t + row_next * rope_ld, tab_bytes, bar, pol);
    }
    row_next += step;
    return true;
  };
  long long issued = 0;                    // lane 0: rows whose copies were started
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_mbar_init();
    while (issued < stages && load(static_cast<int>(issued))) ++issued;
  }
  constexpr int kW = kMode == kHead ? 1 : kNC;
  uint4 w[kW];                             // bf16 pairs
  F2 acc[kW][4];
#pragma unroll
  for (int c = 0; c < kW; ++c) {
    const int e = kNrChunk * c + 8 * lane;
    w[c] = make_uint4(0u, 0u, 0u, 0u);
    if (kMode == kHead || e < cols)
      w[c] = __ldg(reinterpret_cast<const uint4*>(weight + (kMode == kHead ? d : col0 + e)));
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[c][i] = f2(0.f, 0.f);
  }
  const float inv_n = 1.0f / (kMode == kHead ? head_dim : hidden);
  __syncthreads();                         // the barriers and the flag are there
  int s = 0, phase = 0, turn = 0;
  bool ok = true;                          // after a wait that ran out the rows are gone through without data
  for (long long row = first; row < rows; row += step) {
    ok = ok && mbar_wait(bar0 + 8 * s, phase, &abort_flag);
    if (!ok) atomicOr(err, kErrTimeoutLoad);
    __syncwarp();
    const uint8_t* st = ring + s * stage_bytes;
    uint4 rx[kNC], ry[kNC];
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      const int e = kNrChunk * c + 8 * lane;
      rx[c] = ry[c] = make_uint4(0u, 0u, 0u, 0u);
      if (e < cols) {
        rx[c] = *reinterpret_cast<const uint4*>(st + 2 * e);
        ry[c] = *reinterpret_cast<const uint4*>(st + part_bytes + 2 * e);
      }
    }
    F2 cc[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cc[i] = sn[i] = f2(0.f, 0.f);
    if (kMode != kAny) {
      const float* tab = reinterpret_cast<const float*>(st + 2 * part_bytes);
      table_pairs(tab + d, tab + head_dim + d, shift, cc, sn);
    }
    auto tables = [&](int c) {
      if (kMode == kAny && kNrChunk * c + 8 * lane < cols) {
        const long long at = row * rope_ld + (col0 + kNrChunk * c + 8 * lane) % head_dim;
        table_pairs(cos_t + at, sin_t + at, shift, cc, sn);
      }
    };
    __syncwarp();                          // the warp has read the stage
    if (lane == 0 && ok && load(s)) ++issued;
    // sums of one chunk: x^2 and w u x in pairs
    auto sums = [&](int c, F2& xx, F2& wux) {
      const int cw = kMode == kHead ? 0 : c;
      if (kMode != kHead) keep_packed(w[cw]);
      const uint32_t ax[4] = {rx[c].x, rx[c].y, rx[c].z, rx[c].w}, ay[4] = {ry[c].x, ry[c].y, ry[c].z, ry[c].w};
      const uint32_t aw[4] = {w[cw].x, w[cw].y, w[cw].z, w[cw].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 v = widen(ax[i]), u = unrotate(ay[i], cc[i], sn[i]);
        xx = ffma2(v, v, xx);
        wux = ffma2(fmul2(widen(aw[i]), u), v, wux);
      }
    };
    // dx and the weight sums of one chunk from its row's (or head's) sums
    auto finish = [&](int c, float sum_xx, float sum_wux) {
      // Over heads, lanes past the row's end have sums of their own, all 0: without their factor of 0 (eps = 0: infinite
      // times their zeros) they would put NaN into the weight sums that they share with the row's lanes.
      const float inv = kMode == kHead && kNrChunk * c + 8 * lane >= cols ? 0.f : rsqrtf(sum_xx * inv_n + eps);
      const float back = -inv * inv * inv * inv_n * sum_wux;
      const F2 inv2 = f2(inv, inv), back2 = f2(back, back);
      const int cw = kMode == kHead ? 0 : c;
      if (kMode != kHead) {
        keep_packed(rx[c]);
        keep_packed(ry[c]);
        keep_packed(w[cw]);
      }
      const uint32_t ax[4] = {rx[c].x, rx[c].y, rx[c].z, rx[c].w}, ay[4] = {ry[c].x, ry[c].y, ry[c].z, ry[c].w};
      const uint32_t aw[4] = {w[cw].x, w[cw].y, w[cw].z, w[cw].w};
      uint4 packed;
      uint32_t* o = &packed.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 v = widen(ax[i]), a = fmul2(unrotate(ay[i], cc[i], sn[i]), inv2);
        acc[cw][i] = ffma2(a, v, acc[cw][i]);
        const float2 r = f2_split(ffma2(v, back2, fmul2(a, widen(aw[i]))));
        o[i] = pack_bf16x2(r.x, r.y);
      }
      const int e = kNrChunk * c + 8 * lane;
      if (ok && e < cols) *reinterpret_cast<uint4*>(dx + row * hidden + col0 + e) = packed;
    };
    // One tree for both sums over a group of 2 half lanes: the first exchange leaves the lower half of the group with
    // x^2 and the upper half with w u x.
    auto tree = [&](F2 xx, F2 wux, int half) {
      const float2 a = f2_split(xx), b = f2_split(wux);
      float2 mine = make_float2(a.x + a.y, b.x + b.y);
      if (half == 0) return mine;
      const bool upper = (lane & half) != 0;
      float one = upper ? mine.y : mine.x;
      one += __shfl_xor_sync(0xffffffffu, upper ? mine.x : mine.y, half);
      for (int o = half >> 1; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
      mine.x = __shfl_sync(0xffffffffu, one, lane & ~half);
      mine.y = __shfl_sync(0xffffffffu, one, lane | half);
      return mine;
    };
    if (kMode == kHead) {
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        if (kNrChunk * c >= cols) break;
        F2 xx = f2(0.f, 0.f), wux = xx;
        sums(c, xx, wux);
        const float2 sum = tree(xx, wux, head_dim >> 4);
        finish(c, sum.x, sum.y);
      }
    } else {
      F2 xx = f2(0.f, 0.f), wux = xx;
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        tables(c);
        sums(c, xx, wux);
      }
      float2 sum = tree(xx, wux, 16);
      if (split > 1) {
        // the row's other warps, in their order; two buffers by turns
        if (lane == 0) red[turn][warp] = sum;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * split) : "memory");
        sum = make_float2(0.f, 0.f);
        for (int i = 0; i < split; ++i) {
          const float2 r = red[turn][group * split + i];
          sum.x += r.x;
          sum.y += r.y;
        }
        turn ^= 1;
      }
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        if (kNrChunk * c >= cols) break;
        tables(c);
        finish(c, sum.x, sum.y);
      }
    }
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  if (lane == 0 && !ok) {
    // copies in flight land before shared memory goes
    for (long long i = issued > stages ? issued - stages : 0; i < issued; ++i) {
      const unsigned long long t0 = global_ns();
      while (!mbar_try_wait(bar0 + 8 * static_cast<uint32_t>(i % stages), (i / stages) & 1))
        if (global_ns() - t0 > kWaitLimitNs) {
          atomicOr(err, kErrTimeoutDrain);
          break;
        }
    }
  }
  __syncthreads();
  // this block's partial row: its groups, and the heads of a per-head weight, added in order
  float* wsum = reinterpret_cast<float*>(smem);
  const int wcols = kMode == kHead ? kNrChunk : chunks * kNrChunk;
#pragma unroll
  for (int c = 0; c < kW; ++c) {
    if (kNrChunk * c >= wcols) break;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float2*>(wsum + warp * wcols + kNrChunk * c + 8 * lane + 2 * i) = f2_split(acc[c][i]);
  }
  __syncthreads();
  const int out = kMode == kHead ? head_dim : hidden;
  for (int col = threadIdx.x; col < out; col += blockDim.x) {
    float a = 0.f;
    if (kMode == kHead) {
      for (int h = col; h < groups * split * kNrChunk; h += head_dim) a += wsum[h];
    } else {
      for (int g = 0; g < groups; ++g) a += wsum[(g * split + col / wcols) * wcols + col % wcols];
    }
    part[static_cast<long long>(blockIdx.x) * out + col] = a;
  }
}

struct NrShape {
  int split, chunks, warps, blocks, cols, stages, smem, mode;
};

// A block per SM with as many rows at a time as eight warps take; each warp's ring takes its share of shared memory (three
// stages for 2048 columns: some 200 KB on their way per SM).
static NrShape nr_shape(long long rows, int heads, int head_dim, int per_head) {
  NrShape s;
  const int hidden = heads * head_dim, all = (hidden + kNrChunk - 1) / kNrChunk;
  s.split = (all + kNrMaxChunks - 1) / kNrMaxChunks;
  s.chunks = (all + s.split - 1) / s.split;
  s.warps = kNrWarps / s.split * s.split;
  s.blocks = static_cast<int>(std::max<long long>(1, std::min<long long>(148, rows)));
  s.cols = per_head ? head_dim : hidden;
  s.mode = per_head ? kHead : kNrChunk % head_dim == 0 ? kSame : kAny;
  const int stage = 2 * (2 * kNrChunk * s.chunks + (s.mode == kAny ? 0 : 4 * head_dim));
  s.stages = std::min(kNrMaxStages, 220 * 1024 / (s.warps * stage));
  s.smem = std::max(s.warps * s.stages * stage, s.warps * 4 * kNrChunk * (per_head ? 1 : s.chunks));
  return s;
}

template <int kNC, int kMode>
static int nr_launch(const NrShape& s, const void* x, const void* dy, const void* weight, const float* cos_t,
                     const float* sin_t, void* dx, float* part, long long rows, int hidden, int head_dim, float eps,
                     int shift, long long rope_ld, int* err, cudaStream_t stream) {
  static std::mutex mu;
  static int set[kMaxDevices] = {};                      // largest opt-in so far
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (set[dev] < s.smem) {
      if (cudaFuncSetAttribute(qk_norm_rope_bwd_kernel<kNC, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               s.smem) != cudaSuccess)
        return ORL_ERR_LAUNCH;
      set[dev] = s.smem;
    }
  }
  qk_norm_rope_bwd_kernel<kNC, kMode><<<s.blocks, 32 * s.warps, s.smem, stream>>>(
      static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(dy),
      static_cast<const __nv_bfloat16*>(weight), cos_t, sin_t, static_cast<__nv_bfloat16*>(dx), part, rows, hidden,
      head_dim, eps, shift, rope_ld, s.split, s.chunks, s.stages, err);
  return cudaGetLastError() == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
}

}  // namespace orl

using namespace orl;

extern "C" long long orl_qk_norm_rope_bwd_scratch(long long rows, int heads, int head_dim, int per_head) {
  if (rows < 0 || heads <= 0 || head_dim <= 0 || static_cast<long long>(heads) * head_dim > 8192) return ORL_ERR_ARG;
  const NrShape s = nr_shape(rows, heads, head_dim, per_head);
  return static_cast<long long>(s.blocks) * s.cols;
}

extern "C" int orl_qk_norm_rope_bwd(const void* x, const void* dy, const void* weight, const float* cos_t,
                                    const float* sin_t, void* dx, void* dweight, float* scratch, long long rows,
                                    int heads, int head_dim, int per_head, float eps, int sin_shift, long long rope_ld,
                                    int* err_dev, void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (rows < 0 || heads <= 0 || head_dim <= 0 || (head_dim & 7) || sin_shift < 0 || sin_shift > 1 ||
      rope_ld < head_dim || weight == nullptr || dweight == nullptr || err_dev == nullptr)
    return ORL_ERR_ARG;
  if (rows > 0 && (x == nullptr || dy == nullptr || cos_t == nullptr || sin_t == nullptr || dx == nullptr ||
                   scratch == nullptr))
    return ORL_ERR_ARG;
  if (static_cast<long long>(heads) * head_dim > 8192) return ORL_ERR_UNSUPPORTED;
  if (per_head && ((head_dim >> 3) > 32 || ((head_dim >> 3) & ((head_dim >> 3) - 1)) != 0)) return ORL_ERR_UNSUPPORTED;
  if ((rope_ld & 3) || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dy) |
                         reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(weight) |
                         reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) & 15u))
    return ORL_ERR_ALIGN;
  const NrShape s = nr_shape(rows, heads, head_dim, per_head);
  if (rows == 0)
    return cudaMemsetAsync(dweight, 0, 2 * s.cols, stream) == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
  const auto launch = s.chunks <= 4 ? (s.mode == kSame   ? nr_launch<4, kSame>
                                       : s.mode == kHead ? nr_launch<4, kHead>
                                                         : nr_launch<4, kAny>)
                                    : (s.mode == kSame   ? nr_launch<8, kSame>
                                       : s.mode == kHead ? nr_launch<8, kHead>
                                                         : nr_launch<8, kAny>);
  const int rc = launch(s, x, dy, weight, cos_t, sin_t, dx, scratch, rows, heads * head_dim, head_dim, eps, sin_shift,
                        rope_ld, err_dev, stream);
  if (rc != ORL_OK) return rc;
  return column_sum(scratch, s.blocks, s.cols, s.cols, dweight, stream);
}
