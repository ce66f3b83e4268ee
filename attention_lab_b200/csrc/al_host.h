// Host helpers shared by the library's translation units: error messages, per-device facts, kernel attributes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/attention_lab_b200.h"

namespace al {

struct DeviceInfo {
  int sms = 0;
  int max_smem_optin = 0;
  unsigned* err = nullptr;   // the kernels' error bits
};

#pragma GCC visibility push(hidden)
// Store the message of a failing call (al_last_error) and return its status code.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* where);
// The current device's facts (looked up once per device).
int device_info(DeviceInfo** out);
// Allow `smem` bytes of dynamic shared memory and non-portable cluster sizes (set once per kernel and device).
int prepare_kernel_ptr(const void* kernel, size_t smem);
#pragma GCC visibility pop

template <typename K>
int prepare_kernel(K kernel, size_t smem) {
  return prepare_kernel_ptr(reinterpret_cast<const void*>(kernel), smem);
}

inline int plain_launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  return AL_OK;
}

inline bool dtype_ok(int t) { return t == AL_F32 || t == AL_BF16; }
inline int esize(int t) { return t == AL_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace al
