// Internal: descriptions of matrices in device memory for tiled copies.
#pragma once
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "dfa3d_b200.h"

namespace dfa3d {

// cuTensorMapEncodeTiled by way of the runtime, so that the library does not link the driver's.
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 f = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return f;
}

// A thread that has made no call of the runtime yet (autograd's, at its first backward) has no context, without which no map is made.
inline cudaError_t bind_context() {
  int device = 0;
  const cudaError_t rc = cudaGetDevice(&device);
  return rc == cudaSuccess ? cudaSetDevice(device) : rc;
}

// Boxes of box_cols x box_rows of a row-major matrix (rows, cols) of `pitch` elements a row.  What a box has outside of the matrix is
// read as 0 and not written.  In shared memory a box is rows of 64 or 128 bytes whose 16-byte pieces are permuted within 512 or
// 1024 bytes, so that eight rows' pieces of one column lie in different banks.
inline bool describe_matrix(CUtensorMap &map, int dtype, const void *data, long long rows, long long cols, long long pitch, int box_cols,
                            int box_rows) {
  const int size = dtype == DFA3D_DTYPE_F32 ? 4 : 2;
  const cuuint64_t extent[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t stride[1] = {(cuuint64_t)pitch * size};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUtensorMapDataType type = dtype == DFA3D_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == DFA3D_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const auto encode = tensor_map_encoder();
  return encode && encode(&map, type, 2, const_cast<void *>(data), extent, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          box_cols * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Two CTAs of these kernels on one SM, each of a pair that holds tensor memory on the other one's second SM, would wait for each other:
// each takes more than half of an SM's shared memory.
constexpr bool one_an_sm(int bytes) { return 2 * (bytes + 1024) > 228 * 1024; }

// Shared memory beyond 48 KB is a setting of a kernel on a device, made once for each of the first 64.
template <auto KERNEL> cudaError_t allow_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int device = 0;
  cudaError_t rc = cudaGetDevice(&device);
  if (rc != cudaSuccess) return rc;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  rc = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}

// A launch whose CTAs may be set up while the last ones of the kernel before it in the stream end.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), int grid, int threads, int shared, cudaStream_t s, const A &...args) {
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = shared;
  c.stream = s;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &early;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

}  // namespace dfa3d
