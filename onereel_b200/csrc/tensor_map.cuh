// TMA tensor maps over row-major bf16 matrices (host side), shared by the attention and linear kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "orl_common.h"

namespace orl {

constexpr int kMaxDevices = 64;

// cuTensorMapEncodeTiled (driver API, cuda.h), fetched through the runtime so the library needs no -lcuda.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// 2-D bf16 map over rows x row_elems (row stride ld_elems) with box_rows x 64-column boxes, 128-byte swizzle, zero
// fill out of bounds.
inline int make_rows_map(CUtensorMap* map, const void* base, long long rows, long long row_elems, long long ld_elems,
                         int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return ORL_ERR_DRIVER;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_elems), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld_elems) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  auto encode = [&] {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encode()) return ORL_OK;
  // A driver call: unlike the runtime's it does not bind the device's context to a thread that has made no call yet (a
  // server's worker, autograd's thread in a process's first backward pass). cudaSetDevice does.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return ORL_ERR_LAUNCH;
  return encode() ? ORL_OK : ORL_ERR_TENSOR_MAP;
}

}  // namespace orl
