// Gradients of the fused q/k RMSNorm + rotary embedding (qk_norm_rope.cu), bf16 in / bf16 out, HBM-bound.
//
// Forward, per row (or per head of a row) of G elements: inv = rsqrt(mean(x^2) + eps), n = x * inv * w, y = R n with R
// the pairwise rotation. With u = R^T dy (the rotation by the opposite angle):
//   dw = sum over rows (and heads, for a per-head weight) of u * x * inv
//   dx = inv * (w u) - x * inv^3 * mean(w u x)
// x and dy are read once and dx written once; both sums of a row (x^2 and w u x) are reduced together, in fp32. What keeps
// such a kernel from the memory's rate is the reduction between a row's loads and its stores, so the rows (and their rows
// of the tables) are brought into a shared-memory ring by bulk copies several rows ahead; then the instructions count (340
// per thread and row kept the issue slots 65 % busy at 0.57 of the memory's rate), so the arithmetic works on pairs
// (f32x2) and one shuffle tree carries both sums. A block takes rows in strides
// and keeps its dw sums in registers (8 columns per thread), so the weight gradient costs one partial row per block;
// column_sum adds the partial rows in a fixed order.
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

constexpr int kNrMaxStages = 8;

// two bf16 values as a pair of floats (the bits moved up)
__device__ __forceinline__ F2 widen(uint32_t x) { return f2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }

// tpr threads per row (hidden / 8, rounded up to whole warps), n_lanes = blockDim.x / tpr rows at a time. A stage of the
// ring holds n_lanes rows of x, of dy, of cos and of sin. Thread 0 fills it: a warp of its own for that took 82 us where
// this takes 77 (24000 rows of 2048).
template <int kThreads, int kShift>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(
    const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ weight,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, __nv_bfloat16* __restrict__ dx,
    float* __restrict__ part, long long rows, int hidden, int head_dim, int per_head, float eps, long long rope_ld,
    int tpr, int stages, int* __restrict__ err) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kNrMaxStages];
  __shared__ __align__(16) float2 red[2][32];
  __shared__ int abort_flag;
  const int t = threadIdx.x, lane_row = t / tpr, tr = t % tpr;
  const int n_lanes = blockDim.x / tpr;
  const int e = 8 * tr;                    // first element of this thread in a row
  const bool active = e < hidden;
  const int d = active ? e % head_dim : 0;
  const int row_bytes = 2 * hidden, tab_bytes = 4 * head_dim;
  const int stage_bytes = n_lanes * 2 * (row_bytes + tab_bytes);
  const uint32_t bar0 = smem_u32(bars), base = smem_u32(smem);
  const long long step = static_cast<long long>(gridDim.x) * n_lanes;
  const long long first = static_cast<long long>(blockIdx.x) * n_lanes;
  // thread 0: the copies of the next turn into stage s
  long long row_next = first;
  const __nv_bfloat16 *x_next = x + first * hidden, *dy_next = dy + first * hidden;
  const float *cos_next = cos_t + first * rope_ld, *sin_next = sin_t + first * rope_ld;
  const uint64_t pol = policy_evict_first();
  auto load = [&](int s) {
    if (row_next >= rows) return false;
    const int n = static_cast<int>(min(static_cast<long long>(n_lanes), rows - row_next));
    const uint32_t bar = bar0 + 8 * s, dst = base + s * stage_bytes, tab = dst + 2 * n_lanes * row_bytes;
    mbar_expect_tx(bar, n * 2 * (row_bytes + tab_bytes));
    bulk_load(dst, x_next, n * row_bytes, bar, pol);
    bulk_load(dst + n_lanes * row_bytes, dy_next, n * row_bytes, bar, pol);
    for (int i = 0; i < n; ++i) {
      bulk_load(tab + i * tab_bytes, cos_next + i * rope_ld, tab_bytes, bar, pol);
      bulk_load(tab + (n_lanes + i) * tab_bytes, sin_next + i * rope_ld, tab_bytes, bar, pol);
    }
    row_next += step;
    x_next += step * hidden;
    dy_next += step * hidden;
    cos_next += step * rope_ld;
    sin_next += step * rope_ld;
    return true;
  };
  long long issued = 0;                    // thread 0: turns whose copies were started
  if (t == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(bar0 + 8 * s, 1);
    abort_flag = 0;
    fence_mbar_init();
    while (issued < stages && load(static_cast<int>(issued))) ++issued;
  }
  F2 w[4], acc[4];
  {
    const uint4 raw = active ? __ldg(reinterpret_cast<const uint4*>(weight + (per_head ? d : e)))
                             : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = widen(r[i]);
      acc[i] = f2(0.f, 0.f);
    }
  }
  const float inv_n = 1.0f / (per_head ? head_dim : hidden);
  const int wpr = tpr >> 5;
  __syncthreads();                         // the barriers are there
  int s = 0, phase = 0;
  long long it = 0;
  for (long long row0 = first; row0 < rows; row0 += step, ++it) {
    const long long row = row0 + lane_row;
    const bool on = active && row < rows;
    if (!mbar_wait(bar0 + 8 * s, phase, &abort_flag)) {
      if (t == 0) atomicOr(err, kErrTimeoutLoad);
      break;
    }
    uint4 rx = make_uint4(0u, 0u, 0u, 0u), ry = rx;
    float4 c0 = make_float4(0.f, 0.f, 0.f, 0.f), c1 = c0, s0 = c0, s1 = c0;
    if (on) {
      const uint8_t* st = smem + s * stage_bytes;
      rx = *reinterpret_cast<const uint4*>(st + lane_row * row_bytes + 16 * tr);
      ry = *reinterpret_cast<const uint4*>(st + (n_lanes + lane_row) * row_bytes + 16 * tr);
      const float4* cr = reinterpret_cast<const float4*>(st + 2 * n_lanes * row_bytes + lane_row * tab_bytes + 4 * d);
      const float4* sr = cr + n_lanes * tab_bytes / 16;
      c0 = cr[0];
      c1 = cr[1];
      s0 = sr[0];
      s1 = sr[1];
    }
    const float c[4] = {c0.x, c0.z, c1.x, c1.z};
    const float sn[4] = {kShift ? s0.y : s0.x, kShift ? s0.w : s0.z, kShift ? s1.y : s1.x, kShift ? s1.w : s1.z};
    const uint32_t ax[4] = {rx.x, rx.y, rx.z, rx.w}, ay[4] = {ry.x, ry.y, ry.z, ry.w};
    F2 v[4], u[4], xx = f2(0.f, 0.f), wux = xx;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = widen(ax[i]);
      const F2 g = widen(ay[i]);
      const float2 gs = f2_split(g);
      u[i] = ffma2(f2(gs.y, -gs.x), f2(sn[i], sn[i]), fmul2(g, f2(c[i], c[i])));
      xx = ffma2(v[i], v[i], xx);
      wux = ffma2(fmul2(w[i], u[i]), v[i], wux);
    }
    const float2 a2 = f2_split(xx), b2 = f2_split(wux);
    const float2 mine = make_float2(a2.x + a2.y, b2.x + b2.y);        // x^2, w u x of this thread's elements
    // One tree for both sums over a group of lanes (a head's head_dim / 8, or a warp): the first exchange leaves the
    // lower half of the group with x^2 and the upper half with w u x.
    const int half = per_head ? (head_dim >> 4) : 16;
    const bool upper = (t & half) != 0;
    float one = mine.x;
    if (half > 0) {
      one = upper ? mine.y : mine.x;
      one += __shfl_xor_sync(0xffffffffu, upper ? mine.x : mine.y, half);
      for (int o = half >> 1; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
    }
    const bool across = !per_head && tpr > 32;
    // across warps: through shared memory, two buffers by turns
    if (across && (t & 15) == 0) (upper ? red[it & 1][t >> 5].y : red[it & 1][t >> 5].x) = one;
    __syncthreads();                       // the partial sums are there, and everyone has read the stage
    if (t == 0 && load(s)) issued = it + stages + 1;
    float2 sum;
    if (across) {
      F2 total = f2(0.f, 0.f);
      const float2* r = red[it & 1] + lane_row * wpr;
      for (int i = 0; i < wpr; ++i) total = fadd2(total, f2(r[i].x, r[i].y));
      sum = f2_split(total);
    } else if (half > 0) {
      sum.x = __shfl_sync(0xffffffffu, one, t & 31 & ~half);
      sum.y = __shfl_sync(0xffffffffu, one, (t & 31) | half);
    } else {
      sum = mine;
    }
    const float inv = rsqrtf(sum.x * inv_n + eps);
    const float back = -inv * inv * inv * inv_n * sum.y;
    const F2 inv2 = f2(inv, inv), back2 = f2(back, back);
    uint4 packed;
    uint32_t* o = &packed.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F2 a = fmul2(u[i], inv2);
      acc[i] = ffma2(a, v[i], acc[i]);
      const float2 r = f2_split(ffma2(v[i], back2, fmul2(a, w[i])));
      o[i] = pack_bf16x2(r.x, r.y);
    }
    if (on) *reinterpret_cast<uint4*>(dx + row * hidden + e) = packed;
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  if (t == 0 && abort_flag) {
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
  // this block's partial row: its row lanes, and the heads of a per-head weight, added in order
  float* wsum = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(wsum + t * 8 + 2 * i) = f2_split(acc[i]);
  __syncthreads();
  const int cols = per_head ? head_dim : hidden;
  for (int col = t; col < cols; col += blockDim.x) {
    float a = 0.f;
    for (int l = 0; l < n_lanes; ++l)
      for (int h = col; h < hidden; h += cols) a += wsum[l * tpr * 8 + h];
    part[static_cast<long long>(blockIdx.x) * cols + col] = a;
  }
}

struct NrShape {
  int tpr, threads, blocks, cols, stages, smem;
};

// Blocks of 256 threads, or of one row where it is longer; small rows share a block. Three blocks of 256 threads per SM, with
// a third of its shared memory each, keep 20 rows of 2048 elements on their way; one block where a row needs more threads.
static NrShape nr_shape(long long rows, int heads, int head_dim, int per_head) {
  NrShape s;
  const int hidden = heads * head_dim;
  s.tpr = ((hidden / 8 + 31) / 32) * 32;
  const int lanes = std::max(1, 256 / s.tpr);
  s.threads = s.tpr * lanes;
  const int per_sm = s.threads <= 256 ? 3 : 1;
  s.blocks = static_cast<int>(std::min<long long>(148 * per_sm, (rows + lanes - 1) / lanes));
  s.cols = per_head ? head_dim : hidden;
  const int stage = lanes * (4 * hidden + 8 * head_dim);
  s.stages = std::max(2, std::min(kNrMaxStages, (per_sm == 3 ? 70 * 1024 : 200 * 1024) / stage));
  s.smem = std::max(s.stages * stage, 32 * s.threads);
  return s;
}

template <int kThreads, int kShift>
static int nr_attributes(int smem) {
  static std::mutex mu;
  static int set[kMaxDevices] = {};                      // largest opt-in so far
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  std::lock_guard<std::mutex> lock(mu);
  if (set[dev] < smem) {
    if (cudaFuncSetAttribute(qk_norm_rope_bwd_kernel<kThreads, kShift>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem) != cudaSuccess)
      return ORL_ERR_LAUNCH;
    set[dev] = smem;
  }
  return ORL_OK;
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
  const bool small = s.threads <= 256;
  const int rc = sin_shift ? (small ? nr_attributes<256, 1>(s.smem) : nr_attributes<1024, 1>(s.smem))
                           : (small ? nr_attributes<256, 0>(s.smem) : nr_attributes<1024, 0>(s.smem));
  if (rc != ORL_OK) return rc;
  auto kernel = sin_shift ? (small ? qk_norm_rope_bwd_kernel<256, 1> : qk_norm_rope_bwd_kernel<1024, 1>)
                          : (small ? qk_norm_rope_bwd_kernel<256, 0> : qk_norm_rope_bwd_kernel<1024, 0>);
  kernel<<<s.blocks, s.threads, s.smem, stream>>>(
      static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(dy),
      static_cast<const __nv_bfloat16*>(weight), cos_t, sin_t, static_cast<__nv_bfloat16*>(dx), scratch, rows,
      heads * head_dim, head_dim, per_head, eps, rope_ld, s.tpr, s.stages, err_dev);
  if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  return column_sum(scratch, s.blocks, s.cols, s.cols, dweight, stream);
}
