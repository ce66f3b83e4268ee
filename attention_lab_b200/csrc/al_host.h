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
// Whether the current device can schedule a cluster of `cs` CTAs of the kernel as cfg launches it (asked once per kernel,
// size, shared memory and device).
int cluster_schedulable(const void* kernel, const cudaLaunchConfig_t& cfg, int cs, bool* ok);
#pragma GCC visibility pop

template <typename K>
int prepare_kernel(K kernel, size_t smem) {
  return prepare_kernel_ptr(reinterpret_cast<const void*>(kernel), smem);
}

// The largest cluster size of cs, cs / 2, ..., 1 (cs a power of two) for which fits(size, &ok) says ok, into *out; a size
// of one needs no asking. fits returns a status code, and a failing one ends the search.
template <typename F>
int fitting_cluster(int cs, F&& fits, int* out) {
  for (; cs > 1; cs >>= 1) {
    bool ok = false;
    const int rc = fits(cs, &ok);
    if (rc != AL_OK) return rc;
    if (ok) break;
  }
  *out = cs;
  return AL_OK;
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
