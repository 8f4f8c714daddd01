// dev_call.cuh — what the argument-block entry points share: element types,
// the check that tensors are device-readable, and the device they run on.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "common.cuh"

namespace armai {

inline int dtype_size(int dtype) { return dtype == ARMAI_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == ARMAI_F32 || dtype == ARMAI_F16 || dtype == ARMAI_BF16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Makes the device of the call's tensors current, and the caller's again at
// the end of the scope.
class DeviceScope {
 public:
  explicit DeviceScope(const char* op) : op_(op) {}
  ~DeviceScope() {
    if (prev_ >= 0) cudaSetDevice(prev_);
  }
  // Refuses a pointer that is no multiple of its values' size or that the device
  // cannot read; the first device pointer decides the device, the others have to
  // be on the same one.
  int check(const char* what, const void* p, int value_size) {
    if (reinterpret_cast<uintptr_t>(p) % value_size)
      return fail(ARMAI_E_INVALID, std::string(op_) + ": " + what + " is not aligned to its values of " +
                                       std::to_string(value_size) + " bytes");
    cudaPointerAttributes a;
    ARMAI_CUDA(cudaPointerGetAttributes(&a, p));
    if (a.type == cudaMemoryTypeUnregistered)
      return fail(ARMAI_E_INVALID, std::string(op_) + ": " + what + " is not device memory");
    if (a.type != cudaMemoryTypeDevice) return ARMAI_OK;
    if (dev_ < 0) {
      dev_ = a.device;
      int cur = 0;
      ARMAI_CUDA(cudaGetDevice(&cur));
      if (cur != dev_) {
        ARMAI_CUDA(cudaSetDevice(dev_));
        prev_ = cur;
      }
    } else if (a.device != dev_) {
      return fail(ARMAI_E_INVALID, std::string(op_) + ": " + what + " is on another device than the tensors before it");
    }
    return ARMAI_OK;
  }

 private:
  const char* op_;
  int dev_ = -1, prev_ = -1;
};

}  // namespace armai
