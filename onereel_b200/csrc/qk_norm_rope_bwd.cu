// Gradients of the fused q/k RMSNorm + rotary embedding (qk_norm_rope.cu), bf16 in / bf16 out, HBM-bound.
//
// Forward, per row (or per head of a row) of G elements: inv = rsqrt(mean(x^2) + eps), n = x * inv * w, y = R n with R
// the pairwise rotation. With u = R^T dy (the rotation by the opposite angle):
//   dw = sum over rows (and heads, for a per-head weight) of u * x * inv
//   dx = inv * (w u) - x * inv^3 * mean(w u x)
// x and dy are read once and dx written once; both sums of a row (x^2 and w u x) are reduced together, in fp32. A block
// takes rows in strides and keeps its dw sums in registers (8 columns per thread), so the weight gradient costs one
// partial row per block; column_sum adds the partial rows in a fixed order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "column_sum.cuh"
#include "orl_common.h"

namespace orl {

constexpr int kNrBlocks = 592;             // at most: 148 SMs x 4 blocks of 256 threads
constexpr int kNrRows = 2;                 // rows in flight per thread

// tpr threads per row (hidden / 8, rounded up to whole warps), blockDim.x / tpr rows at a time
__global__ void __launch_bounds__(1024) qk_norm_rope_bwd_kernel(
    const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ weight,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, __nv_bfloat16* __restrict__ dx,
    float* __restrict__ part, long long rows, int hidden, int head_dim, int per_head, float eps, int sin_shift,
    long long rope_ld, int tpr) {
  __shared__ float2 red[2][kNrRows][32];
  extern __shared__ float wsum[];          // [blockDim.x][8] at the end
  const int t = threadIdx.x, lane_row = t / tpr, tr = t % tpr;
  const int n_lanes = blockDim.x / tpr;
  const int e = 8 * tr;                    // first element of this thread in a row
  const bool active = e < hidden;
  const int d = active ? e % head_dim : 0;
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
  const long long step = static_cast<long long>(gridDim.x) * n_lanes;
  int turn = 0;
  for (long long row0 = static_cast<long long>(blockIdx.x) * n_lanes; row0 < rows; row0 += kNrRows * step, turn ^= 1) {
    // the rows' loads are all in flight before anything is reduced; the rows stay packed meanwhile
    uint4 rx[kNrRows], ry[kNrRows];
    float c[kNrRows][4], s[kNrRows][4];
#pragma unroll
    for (int k = 0; k < kNrRows; ++k) {
      const long long row = row0 + k * step + lane_row;
      rx[k] = ry[k] = make_uint4(0u, 0u, 0u, 0u);
      float4 c0 = make_float4(0.f, 0.f, 0.f, 0.f), c1 = c0, s0 = c0, s1 = c0;
      if (active && row < rows) {
        rx[k] = __ldcs(reinterpret_cast<const uint4*>(x + row * hidden + e));
        ry[k] = __ldcs(reinterpret_cast<const uint4*>(dy + row * hidden + e));
        const float4* cr = reinterpret_cast<const float4*>(cos_t + row * rope_ld + d);
        const float4* sr = reinterpret_cast<const float4*>(sin_t + row * rope_ld + d);
        c0 = __ldg(cr);
        c1 = __ldg(cr + 1);
        s0 = __ldg(sr);
        s1 = __ldg(sr + 1);
      }
      c[k][0] = c0.x, c[k][1] = c0.z, c[k][2] = c1.x, c[k][3] = c1.z;
      s[k][0] = sin_shift ? s0.y : s0.x, s[k][1] = sin_shift ? s0.w : s0.z;
      s[k][2] = sin_shift ? s1.y : s1.x, s[k][3] = sin_shift ? s1.w : s1.z;
    }
    // pair i of row k: x, u = R^T dy
    auto pair = [&](int k, int i, float2& v, float2& u) {
      const uint32_t ax = i == 0 ? rx[k].x : i == 1 ? rx[k].y : i == 2 ? rx[k].z : rx[k].w;
      const uint32_t ay = i == 0 ? ry[k].x : i == 1 ? ry[k].y : i == 2 ? ry[k].z : ry[k].w;
      v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ax));
      const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ay));
      u = make_float2(g.x * c[k][i] + g.y * s[k][i], g.y * c[k][i] - g.x * s[k][i]);
    };
    float2 sum[kNrRows];                   // x^2, w u x
#pragma unroll
    for (int k = 0; k < kNrRows; ++k) {
      sum[k] = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v, u;
        pair(k, i, v, u);
        sum[k].x += v.x * v.x + v.y * v.y;
        sum[k].y += w[2 * i] * u.x * v.x + w[2 * i + 1] * u.y * v.y;
      }
    }
    // per head: its head_dim / 8 consecutive lanes; whole row: its warps, through shared memory (two buffers by turns,
    // so that one barrier per turn is enough)
    for (int o = per_head ? (head_dim >> 4) : 16; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < kNrRows; ++k) {
        sum[k].x += __shfl_xor_sync(0xffffffffu, sum[k].x, o);
        sum[k].y += __shfl_xor_sync(0xffffffffu, sum[k].y, o);
      }
    }
    if (!per_head && tpr > 32) {
      if ((t & 31) == 0) {
#pragma unroll
        for (int k = 0; k < kNrRows; ++k) red[turn][k][t >> 5] = sum[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kNrRows; ++k) {
        sum[k] = make_float2(0.f, 0.f);
        for (int i = 0; i < wpr; ++i) {
          const float2 p = red[turn][k][lane_row * wpr + i];
          sum[k].x += p.x;
          sum[k].y += p.y;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kNrRows; ++k) {
      const long long row = row0 + k * step + lane_row;
      const float inv = rsqrtf(sum[k].x * inv_n + eps);
      const float back = inv * inv * inv * inv_n * sum[k].y;
      uint4 packed;
      uint32_t* o = &packed.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v, u;
        pair(k, i, v, u);
        const float a = u.x * inv, b = u.y * inv;
        acc[2 * i] += a * v.x;
        acc[2 * i + 1] += b * v.y;
        const __nv_bfloat162 r = __floats2bfloat162_rn(a * w[2 * i] - v.x * back, b * w[2 * i + 1] - v.y * back);
        o[i] = *reinterpret_cast<const uint32_t*>(&r);
      }
      if (active && row < rows) *reinterpret_cast<uint4*>(dx + row * hidden + e) = packed;
    }
  }
  // this block's partial row: its row lanes, and the heads of a per-head weight, added in order
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
  int tpr, threads, blocks, cols;
};

static NrShape nr_shape(long long rows, int heads, int head_dim, int per_head) {
  NrShape s;
  const int hidden = heads * head_dim;
  s.tpr = ((hidden / 8 + 31) / 32) * 32;
  // small rows share a block, so that a block has 256 threads or one row
  const int lanes = std::max(1, 256 / s.tpr);
  s.threads = s.tpr * lanes;
  s.blocks = static_cast<int>(std::min<long long>(std::max(1, kNrBlocks * 256 / std::max(256, s.threads)),
                                                  (rows + lanes - 1) / lanes));
  s.cols = per_head ? head_dim : hidden;
  return s;
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
                                    void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (rows < 0 || heads <= 0 || head_dim <= 0 || (head_dim & 7) || sin_shift < 0 || sin_shift > 1 ||
      rope_ld < head_dim || weight == nullptr || dweight == nullptr)
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
  qk_norm_rope_bwd_kernel<<<s.blocks, s.threads, 32 * s.threads, stream>>>(
      static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(dy),
      static_cast<const __nv_bfloat16*>(weight), cos_t, sin_t, static_cast<__nv_bfloat16*>(dx), scratch, rows,
      heads * head_dim, head_dim, per_head, eps, sin_shift, rope_ld, s.tpr);
  if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  return column_sum(scratch, s.blocks, s.cols, s.cols, dweight, stream);
}
