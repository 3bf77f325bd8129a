// Column sums of fp32 partial rows, in a fixed order (no atomics): out[c] = bf16(sum_r part[r * ld + c]). The second
// stage of every parameter gradient that sums over rows: a block per 32 columns, 32 row lanes, each adding rows
// lane, lane + 32, ... ; then a tree over the lanes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "orl_common.h"

namespace orl {

// Two such sums may share a launch: blockIdx.y = 1 takes part1 and out1.
static __global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part0, int rows, int cols,
                                                                 long long ld, __nv_bfloat16* __restrict__ out0,
                                                                 const float* __restrict__ part1,
                                                                 __nv_bfloat16* __restrict__ out1) {
  const float* part = blockIdx.y == 0 ? part0 : part1;
  __nv_bfloat16* out = blockIdx.y == 0 ? out0 : out1;
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = 32 * blockIdx.x + x;
  float a = 0.f, b = 0.f;
  if (c < cols) {
    int r = y;
    for (; r + 32 < rows; r += 64) {
      a += part[r * ld + c];
      b += part[(r + 32) * ld + c];
    }
    if (r < rows) a += part[r * ld + c];
  }
  s[y][x] = a + b;
  __syncthreads();
  // warp y adds column y's 32 lanes
  float v = s[x][y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int cc = 32 * blockIdx.x + y;
  if (x == 0 && cc < cols) out[cc] = __float2bfloat16_rn(v);
}

// part1 / out1: a second sum of the same shape, or NULL
inline int column_sum(const float* part, int rows, int cols, long long ld, void* out, cudaStream_t stream,
                      const float* part1 = nullptr, void* out1 = nullptr) {
  column_sum_kernel<<<dim3((cols + 31) / 32, part1 != nullptr ? 2 : 1), 1024, 0, stream>>>(
      part, rows, cols, ld, static_cast<__nv_bfloat16*>(out), part1, static_cast<__nv_bfloat16*>(out1));
  return cudaGetLastError() == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
}

}  // namespace orl
