// Gradients of the fused q/k RMSNorm + rotary embedding (qk_norm_rope.cu), bf16 in / bf16 out, HBM-bound.
//
// Forward, per row (or per head of a row) of G elements: inv = rsqrt(mean(x^2) + eps), n = x * inv * w, y = R n with R
// the pairwise rotation. With u = R^T dy (the rotation by the opposite angle):
//   dw = sum over rows (and heads, for a per-head weight) of u * x * inv
//   dx = inv * (w u) - x * inv^3 * mean(w u x)
// x and dy are read once and dx written once; both sums of a row (x^2 and w u x) are reduced together, in fp32. What keeps
// such a kernel from the memory's rate is the reduction between a row's loads and its stores, so the rows (and their rows
// of the tables) are brought into a shared-memory ring by bulk copies several rows ahead. A block takes rows in strides
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

// tpr threads per row (hidden / 8, rounded up to whole warps), n_lanes = blockDim.x / tpr rows at a time. A stage of the
// ring holds n_lanes rows of x, of dy, of cos and of sin.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(
    const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ weight,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, __nv_bfloat16* __restrict__ dx,
    float* __restrict__ part, long long rows, int hidden, int head_dim, int per_head, float eps, int sin_shift,
    long long rope_ld, int tpr, int stages, int* __restrict__ err) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kNrMaxStages];
  __shared__ float2 red[2][32];
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
  // thread 0: the copies of turn `it` into stage s
  auto load = [&](long long it, int s) {
    const long long row0 = first + it * step;
    if (row0 >= rows) return false;
    const int n = static_cast<int>(min(static_cast<long long>(n_lanes), rows - row0));
    const uint32_t bar = bar0 + 8 * s, dst = base + s * stage_bytes, tab = dst + 2 * n_lanes * row_bytes;
    const uint64_t pol = policy_evict_first();
    mbar_expect_tx(bar, n * 2 * (row_bytes + tab_bytes));
    bulk_load(dst, x + row0 * hidden, n * row_bytes, bar, pol);
    bulk_load(dst + n_lanes * row_bytes, dy + row0 * hidden, n * row_bytes, bar, pol);
    for (int i = 0; i < n; ++i) {
      bulk_load(tab + i * tab_bytes, cos_t + (row0 + i) * rope_ld, tab_bytes, bar, pol);
      bulk_load(tab + (n_lanes + i) * tab_bytes, sin_t + (row0 + i) * rope_ld, tab_bytes, bar, pol);
    }
    return true;
  };
  long long issued = 0;                    // thread 0: turns whose copies were started
  if (t == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(bar0 + 8 * s, 1);
    abort_flag = 0;
    fence_mbar_init();
    while (issued < stages && load(issued, static_cast<int>(issued))) ++issued;
  }
  float w[8], acc[8];
  {
    const uint4 raw = active ? __ldg(reinterpret_cast<const uint4*>(weight + (per_head ? d : e)))
                             : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r[i]));
      w[2 * i] = f.x;
      w[2 * i + 1] = f.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
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
    const float sn[4] = {sin_shift ? s0.y : s0.x, sin_shift ? s0.w : s0.z, sin_shift ? s1.y : s1.x,
                         sin_shift ? s1.w : s1.z};
    const uint32_t ax[4] = {rx.x, rx.y, rx.z, rx.w}, ay[4] = {ry.x, ry.y, ry.z, ry.w};
    float v[8], u[8];
    float2 sum = make_float2(0.f, 0.f);    // x^2, w u x
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ax[i]));
      const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ay[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
      u[2 * i] = g.x * c[i] + g.y * sn[i];
      u[2 * i + 1] = g.y * c[i] - g.x * sn[i];
      sum.x += f.x * f.x + f.y * f.y;
      sum.y += w[2 * i] * u[2 * i] * f.x + w[2 * i + 1] * u[2 * i + 1] * f.y;
    }
    // per head: its head_dim / 8 consecutive lanes; whole row: its warps, through shared memory (two buffers by turns)
    for (int o = per_head ? (head_dim >> 4) : 16; o > 0; o >>= 1) {
      sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
      sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
    }
    const bool across = !per_head && tpr > 32;
    if (across && (t & 31) == 0) red[it & 1][t >> 5] = sum;
    __syncthreads();                       // the partial sums are there, and everyone has read the stage
    if (t == 0 && load(it + stages, s)) issued = it + stages + 1;
    if (across) {
      sum = make_float2(0.f, 0.f);
      for (int i = 0; i < wpr; ++i) {
        const float2 p = red[it & 1][lane_row * wpr + i];
        sum.x += p.x;
        sum.y += p.y;
      }
    }
    const float inv = rsqrtf(sum.x * inv_n + eps);
    const float back = inv * inv * inv * inv_n * sum.y;
    uint4 packed;
    uint32_t* o = &packed.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = u[2 * i] * inv, b = u[2 * i + 1] * inv;
      acc[2 * i] += a * v[2 * i];
      acc[2 * i + 1] += b * v[2 * i + 1];
      const __nv_bfloat162 r = __floats2bfloat162_rn(a * w[2 * i] - v[2 * i] * back,
                                                     b * w[2 * i + 1] - v[2 * i + 1] * back);
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
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
  for (int i = 0; i < 8; ++i) wsum[t * 8 + i] = acc[i];
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

template <int kThreads>
static int nr_attributes(int smem) {
  static std::mutex mu;
  static int set[kMaxDevices] = {};                      // largest opt-in so far
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  std::lock_guard<std::mutex> lock(mu);
  if (set[dev] < smem) {
    if (cudaFuncSetAttribute(qk_norm_rope_bwd_kernel<kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
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
  const int rc = s.threads <= 256 ? nr_attributes<256>(s.smem) : nr_attributes<1024>(s.smem);
  if (rc != ORL_OK) return rc;
  auto kernel = s.threads <= 256 ? qk_norm_rope_bwd_kernel<256> : qk_norm_rope_bwd_kernel<1024>;
  kernel<<<s.blocks, s.threads, s.smem, stream>>>(
      static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(dy),
      static_cast<const __nv_bfloat16*>(weight), cos_t, sin_t, static_cast<__nv_bfloat16*>(dx), scratch, rows,
      heads * head_dim, head_dim, per_head, eps, sin_shift, rope_ld, s.tpr, s.stages, err_dev);
  if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  return column_sum(scratch, s.blocks, s.cols, s.cols, dweight, stream);
}
