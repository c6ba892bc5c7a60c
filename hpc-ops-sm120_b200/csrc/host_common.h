// host_common.h -- what the translation units of the library share on the
// host: the error message, the device check, the TMA descriptor encoder and
// the launch counter (all defined in decode_capi.cu).
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>

namespace adb_host {

// Keeps the message for adb_last_error on this thread and returns `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

// ADB_ERR_DEVICE unless `device` is a compute-capability 10.x GPU.
int sm_count(int device, int* sms);

int get_encoder(PFN_cuTensorMapEncodeTiled_v12000* fn);

void count_launch();

// The error word of each translation unit on the current device (and clears it).
cudaError_t cache_error_word(int* word, bool reset);
cudaError_t prefill_error_word(int* word, bool reset);

struct DeviceGuard {
  int previous = -1;
  bool switched = false;
  cudaError_t error = cudaSuccess;
  explicit DeviceGuard(int device) {
    error = cudaGetDevice(&previous);
    if (error == cudaSuccess && previous != device) {
      error = cudaSetDevice(device);
      switched = error == cudaSuccess;
    }
  }
  ~DeviceGuard() {
    if (switched) cudaSetDevice(previous);
  }
};

inline bool is_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace adb_host
