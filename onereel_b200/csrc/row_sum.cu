// Gradient of a pack: dst row i = sum of the packed rows that are copies of it (bf16 in and out, summed in fp32 in list
// order: no atomics). HBM-bound: every packed row is read once, every source row written once; rows without copies get
// zeros. One block per row and plane, 16 bytes per thread. The copies' gradients come as the attention backward rounded them
// to bf16 (as torch's gradient of a gather does): a source row's sum has one rounding for each of its copies besides its own;
// fp32 copies would cost twice the memory of the packed dk and dv. 22260 rows of 2048 in two planes from 50880 copies: 160 us,
// 0.57 of the measured copy rate (a row's copies lie far apart, and most rows have two).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "orl_common.h"

namespace orl {

constexpr int kRowSumPlanes = 3;

struct RowSumBases {
  const uint8_t* src[kRowSumPlanes];
  uint8_t* dst[kRowSumPlanes];
};

__global__ void __launch_bounds__(256) row_sum_kernel(RowSumBases b, const int32_t* __restrict__ offsets,
                                                      const int32_t* __restrict__ rows, long long row_bytes) {
  const long long i = blockIdx.x;
  const uint8_t* src = b.src[blockIdx.y];
  uint8_t* dst = b.dst[blockIdx.y] + i * row_bytes;
  const int lo = __ldg(offsets + i), hi = __ldg(offsets + i + 1);
  for (long long o = 16ll * threadIdx.x; o < row_bytes; o += 16ll * blockDim.x) {
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = lo; j < hi; j += 4) {
      uint4 r[4];                                        // four copies' loads in flight
#pragma unroll
      for (int u = 0; u < 4; ++u)
        r[u] = j + u < hi ? __ldcs(reinterpret_cast<const uint4*>(src + __ldg(rows + j + u) * row_bytes + o))
                          : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
          s[2 * e] += f.x;
          s[2 * e + 1] += f.y;
        }
      }
    }
    uint4 out;
    uint32_t* w = &out.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(s[2 * e], s[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&p);
    }
    *reinterpret_cast<uint4*>(dst + o) = out;
  }
}

}  // namespace orl

extern "C" int orl_row_sum(const void* const* src, void* const* dst, int planes, const int32_t* offsets_dev,
                           const int32_t* rows_dev, long long n_rows, long long row_bytes, void* stream_ptr) {
  using namespace orl;
  if (src == nullptr || dst == nullptr || planes < 1 || planes > kRowSumPlanes || n_rows < 0 || row_bytes <= 0 ||
      n_rows > 0x7fffffffLL)
    return ORL_ERR_ARG;
  if (row_bytes & 15) return ORL_ERR_ALIGN;
  if (n_rows == 0) return ORL_OK;
  if (offsets_dev == nullptr) return ORL_ERR_ARG;
  RowSumBases b{};
  for (int p = 0; p < planes; ++p) {
    if (dst[p] == nullptr || (src[p] == nullptr && rows_dev != nullptr)) return ORL_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(src[p]) | reinterpret_cast<uintptr_t>(dst[p])) & 15u) return ORL_ERR_ALIGN;
    b.src[p] = static_cast<const uint8_t*>(src[p]);
    b.dst[p] = static_cast<uint8_t*>(dst[p]);
  }
  const int threads = static_cast<int>(row_bytes / 16 >= 256 ? 256 : (row_bytes / 16 + 31) / 32 * 32);
  row_sum_kernel<<<dim3(static_cast<unsigned>(n_rows), planes), threads, 0, static_cast<cudaStream_t>(stream_ptr)>>>(
      b, offsets_dev, rows_dev, row_bytes);
  return cudaGetLastError() == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
}
