// device_ops.h -- what the operators on device tensors share: error text, the device of a call, element types.
#ifndef LINMT_DEVICE_OPS_H_
#define LINMT_DEVICE_OPS_H_
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/linmt_decoder.h"

namespace linmt {
namespace ops {

// Text of the thread's last refused call (beam_ops.cu).
char* op_error_text();
constexpr int kOpErrorBytes = 256;

inline int op_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(op_error_text(), kOpErrorBytes, fmt, ap);
  va_end(ap);
  return code;
}
// A launch that was refused: its error is taken out of the runtime, or the caller's next check finds it again.
inline int op_cuda(cudaError_t e, const char* what) {
  cudaGetLastError();
  return op_fail(LINMT_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

// What every call on a pool checks of it (pages4_ops.cu).
int check_pages4(const linmt_pages4& p, const char* what);

// Makes `device` current for a call and puts the caller's back.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err = cudaGetDevice(&before_);
    if (err == cudaSuccess && before_ != device) {
      err = cudaSetDevice(device);
      switched_ = err == cudaSuccess;
    }
    if (err != cudaSuccess) cudaGetLastError();
  }
  ~OnDevice() { if (switched_) cudaSetDevice(before_); }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  cudaError_t err;

 private:
  int before_ = 0;
  bool switched_ = false;
};

inline bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline int dtype_bytes(int dtype) { return dtype == LINMT_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == LINMT_F32 || dtype == LINMT_BF16 || dtype == LINMT_F16; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

}  // namespace ops
}  // namespace linmt
#endif
