// Host-side plumbing shared by the translation units of libbtp_sm100.so: error text, launch counter, per-device
// launch facts and the launch itself.  No torch types here.
#pragma once

#include "../../include/btp_sm100.h"

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <mutex>

namespace btp_host {

inline thread_local char tls_error[512] = "";
inline std::atomic<unsigned long long> g_launches{0};

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(tls_error, sizeof(tls_error), fmt, ap);
  va_end(ap);
  return code;
}

#define BTP_CUDA_TRY(expr)                                                                      \
  do {                                                                                          \
    cudaError_t _e = (expr);                                                                    \
    if (_e != cudaSuccess) return fail(BTP_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e));  \
  } while (0)

// ------------------------------------------------------------------ per-device launch facts, computed once
struct DeviceInfo {
  bool ready = false;
  int sms = 0;
  int cc_major = 0;
};
inline DeviceInfo g_dev[64];
inline std::mutex g_dev_mutex;

inline int device_info(int* dev_out, DeviceInfo* info) {
  int dev = 0;
  BTP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(BTP_ERR_CUDA, "device ordinal %d out of range", dev);
  // Binds the device's primary context to the calling thread: the descriptor encoder is a driver entry point
  // and threads that have made no runtime call yet (autograd's backward thread) have no current context.
  // Once per thread and device; later calls find the binding in place.
  thread_local int tls_bound_device = -1;
  thread_local DeviceInfo tls_info;
  if (tls_bound_device != dev) {
    BTP_CUDA_TRY(cudaSetDevice(dev));
    std::lock_guard<std::mutex> lock(g_dev_mutex);
    if (!g_dev[dev].ready) {
      BTP_CUDA_TRY(cudaDeviceGetAttribute(&g_dev[dev].sms, cudaDevAttrMultiProcessorCount, dev));
      BTP_CUDA_TRY(cudaDeviceGetAttribute(&g_dev[dev].cc_major, cudaDevAttrComputeCapabilityMajor, dev));
      g_dev[dev].ready = true;
    }
    tls_info = g_dev[dev];
    tls_bound_device = dev;
  }
  *dev_out = dev;
  *info = tls_info;
  if (info->cc_major != 10) {
    return fail(BTP_ERR_UNSUPPORTED_DEVICE, "device %d has compute capability %d.x; this library is built for 10.x only",
                dev, info->cc_major);
  }
  return BTP_OK;
}

// Launch with programmatic stream serialization: the launch of this kernel is processed while the previous
// kernel of the stream still runs; its CTAs start when that kernel's CTAs have all exited and wait in pdl_wait()
// until its memory is visible.  That hides the launch latency (-2 % on the forward+backward step at
// B=1024, H=32, L=128).  The kernels do NOT release their successor early (griddepcontrol.launch_dependents at
// kernel start was measured 9 % slower: the successor's CTAs then occupy SMs while the stragglers finish;
// at the end of each warp's work it was measured within 0.6 % of not doing it).
// BTP_SM100_PDL=0 launches the plain way.
inline bool use_pdl() {
  static const bool v = [] {
    const char* e = getenv("BTP_SM100_PDL");
    return e ? atoi(e) != 0 : true;
  }();
  return v;
}

template <class... Params, class... Args>
cudaError_t launch_kernel(void (*kernel)(Params...), int grid, int threads, int smem_bytes, cudaStream_t stream,
                          const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = use_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

inline bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace btp_host
