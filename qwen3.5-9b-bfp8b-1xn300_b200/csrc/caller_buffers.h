// caller_buffers.h — what the calls that work on the caller's own device buffers
// share (rope.cu, kv8.cu): the checks, every one of which refuses before anything
// is launched, and the launch.
#pragma once

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

#include "../../include/qcache.h"
#include "kernels.h"

namespace qc {

// Sets qc_last_error(NULL) and returns `code`.
inline int refuse(int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_thread_error(buf);
  return code;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A kernel launched here may follow `p`: it is device memory of the current
// device (a host pointer, or one of another device, would fault the kernel).
inline int check_device_pointer(const char* call, const char* name, const void* p) {
  if (!p) return refuse(QC_ERR_ARG, "%s: %s is null", call, name);
  int dev = 0;
  cudaPointerAttributes at{};
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return refuse(QC_ERR_CUDA, "%s: %s: %s", call, name, cudaGetErrorString(e));
  }
  if (at.type == cudaMemoryTypeManaged) return QC_OK;
  if (at.type != cudaMemoryTypeDevice)
    return refuse(QC_ERR_ARG, "%s: %s is not device memory", call, name);
  if (at.device != dev)
    return refuse(QC_ERR_ARG, "%s: %s is on device %d, the current one is %d", call, name,
                  at.device, dev);
  return QC_OK;
}

// Launch as a programmatic dependent of the kernel before: it may start early and
// waits (griddepcontrol.wait) before it reads or writes memory.
template <typename... A>
cudaError_t launch_dependent(void (*k)(A...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                             const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

}  // namespace qc
