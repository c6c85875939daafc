// Host-side TMA descriptors of the kernels that describe their operands themselves.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>
#include <mutex>
#include <string>
#include "common.cuh"

// Argument checks with numbers in their message. The message is built by std::string: c10's own
// formatting of several arguments goes through a string stream, which crashes in an extension whose
// libstdc++ is not the one torch was built with.
#define B200_REQUIRE(cond, msg)                        \
  do {                                                 \
    if (!(cond)) TORCH_CHECK(false, std::string(msg)); \
  } while (0)
#define B200_REQUIRE_CUDA(expr)                                                                      \
  do {                                                                                               \
    const cudaError_t e_ = (expr);                                                                   \
    B200_REQUIRE(e_ == cudaSuccess, std::string("CUDA error: ") + cudaGetErrorString(e_));           \
  } while (0)

namespace b200 {

typedef CUresult (*TmaEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline TmaEncodeFn tma_encode_fn() {
  static TmaEncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    B200_REQUIRE_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q));
    TORCH_CHECK(q == cudaDriverEntryPointSuccess && ptr, "cuTensorMapEncodeTiled not available");
    fn = reinterpret_cast<TmaEncodeFn>(ptr);
  });
  return fn;
}

// bf16 tensor of `rank` dims (innermost first), byte strides of dims 1.., 128-byte swizzled boxes;
// the innermost box is 64 elements (128 bytes). Rows outside the tensor read as zero.
inline CUtensorMap tma_bf16(const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                            const uint32_t* box) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(base) % 16 == 0, "TMA base must be 16-byte aligned");
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], es[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    es[i] = 1;
    if (i) {
      TORCH_CHECK(strides[i - 1] % 16 == 0, "TMA strides must be multiples of 16 bytes");
      st[i - 1] = strides[i - 1];
    }
  }
  CUtensorMap m;
  const CUresult r = tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                                     d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B200_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return m;
}

}  // namespace b200
