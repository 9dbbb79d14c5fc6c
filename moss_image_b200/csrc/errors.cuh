// Host-side error plumbing for the C ABI: a thread-local message and helpers that turn
// CUDA failures into MOSS_ERR_* codes.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/moss_w8.h"

namespace moss {

std::string& last_error_slot();

// Device-visible address of the current device's host-visible status copy (set up by
// moss_status_mirror), or nullptr when the caller has not asked for one.
int* status_mirror_for_current_device();

// Whether the calling thread asked for a debug stall of its next GEMM
// (moss_debug_stall_next_gemm); the request is consumed by this call.
bool take_debug_stall();

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  last_error_slot() = buf;
  return code;
}

inline int check_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return MOSS_OK;
  return fail(MOSS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// SMs of the current device (148, a B200's, where there is none), asked for once per device.
inline int device_sm_count() {
  static std::atomic<int> known[64];
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0) {
    cudaGetLastError();
    return 148;
  }
  if (device < 64 && (n = known[device].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

// What a kernel needs set up once on each device (function attributes belong to a device): `run` returns its error, and may
// leave a number in `value` that later calls read. One static object per kernel.
class DeviceSetup {
 public:
  static constexpr int kDevices = 64;
  template <typename F>
  int operator()(const char* what, int* value, const F& run) {
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return check_cuda(e, "cudaGetDevice");
    if (device < 0 || device >= kDevices) return fail(MOSS_ERR_UNSUPPORTED, "device %d is past the first %d", device, kDevices);
    Slot& slot = slots_[device];
    std::call_once(slot.once, [&] { slot.error = run(&slot.value); });
    if (value != nullptr) *value = slot.value;
    return check_cuda(slot.error, what);
  }

 private:
  struct Slot {
    std::once_flag once;
    cudaError_t error = cudaSuccess;
    int value = 0;
  };
  Slot slots_[kDevices];
};

// Makes the current device's context current on this thread, as a kernel launch would. A thread
// that has made no CUDA call yet (an autograd worker's first backward) has none, and the
// driver's tensor-map encoder refuses to work without one.
inline int bind_context() {
  int device = 0;
  const int rc = check_cuda(cudaGetDevice(&device), "cudaGetDevice");
  return rc != MOSS_OK ? rc : check_cuda(cudaSetDevice(device), "cudaSetDevice");
}

// Launches a kernel that may start while the one before it in the stream ends (it calls pdl_wait).
template <typename... Params, typename... Args>
inline int launch_dependent(const char* what, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                            cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...), what);
}

inline int clear_ok() {
  last_error_slot().clear();
  return MOSS_OK;
}

inline bool is_float_kind(int k) {
  return k == MOSS_DTYPE_F16 || k == MOSS_DTYPE_BF16 || k == MOSS_DTYPE_F32;
}

inline int dtype_size(int k) { return k == MOSS_DTYPE_F32 ? 4 : 2; }

}  // namespace moss

#define MOSS_CUDA_TRY(expr)                               \
  do {                                                    \
    int _rc = ::moss::check_cuda((expr), #expr);          \
    if (_rc != MOSS_OK) return _rc;                       \
  } while (0)
