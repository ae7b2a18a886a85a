// Tensor maps for TMA tile copies: two-dimensional row-major tensors, zero fill past the edges.
// No counterpart in the reference (it has no tensor maps).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace purlin {

void setError(const std::string& e);

using TensorMapEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                       const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                       CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline TensorMapEncodeFn tensorMapEncodeFn() {
  static TensorMapEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<TensorMapEncodeFn>(p);
  }();
  return fn;
}

// [rows, rowBytes] row-major, rows `pitch` bytes apart; box = boxRows x 128 bytes with the 128-byte swizzle. `type`: bf16 or bytes.
inline bool makeTensorMap(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, uint64_t rows, uint64_t rowBytes, uint64_t pitch, uint32_t boxRows) {
  const TensorMapEncodeFn fn = tensorMapEncodeFn();
  if (!fn) { setError("cuTensorMapEncodeTiled is not available from this driver"); return false; }
  if (reinterpret_cast<uintptr_t>(ptr) % 16 || pitch % 16) { setError("TMA operands need 16-byte aligned base and row pitch"); return false; }
  const uint64_t size = type == CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 ? 2 : 1;
  const cuuint64_t dims[2] = {rowBytes / size, rows};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {uint32_t(128 / size), boxRows};
  const cuuint32_t elem[2] = {1, 1};
  auto encode = [&] {
    return fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {     // a thread that has made no runtime call that binds its context yet (autograd's backward thread)
    int device = 0;
    if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
  }
  if (r != CUDA_SUCCESS) { setError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r))); return false; }
  return true;
}

}  // namespace purlin
