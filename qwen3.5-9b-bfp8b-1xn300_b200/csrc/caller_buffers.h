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

// Sets qc_last_error(NULL) and returns `code`.  The runtime keeps the last error of a
// thread until someone takes it: left there, a launch that failed here would be found
// by the next call's own check.
inline int refuse(int code, const char* fmt, ...) {
  if (code == QC_ERR_CUDA) cudaGetLastError();
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_thread_error(buf);
  return code;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// The buffers of a call, each of which a kernel launched here may follow: device
// memory of the current device (a host pointer, or one of another device, would
// fault the kernel).  The first one that is not decides what check() returns.
class BufferCheck {
 public:
  explicit BufferCheck(const char* call) : call_(call) {}
  BufferCheck& need(const char* name, const void* p) {
    if (rc_) return *this;
    if (!p) return fail(QC_ERR_ARG, name, "is null");
    return maybe(name, p);
  }
  BufferCheck& maybe(const char* name, const void* p) {  // null is fine
    if (rc_ || !p) return *this;
    cudaPointerAttributes at{};
    cudaError_t e = dev_ < 0 ? cudaGetDevice(&dev_) : cudaSuccess;
    if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) return fail(QC_ERR_CUDA, name, cudaGetErrorString(e));
    if (at.type == cudaMemoryTypeManaged) return *this;
    if (at.type != cudaMemoryTypeDevice) return fail(QC_ERR_ARG, name, "is not device memory");
    if (at.device != dev_) return fail(QC_ERR_ARG, name, "is not on the current device");
    return *this;
  }
  int check() const { return rc_; }

 private:
  BufferCheck& fail(int code, const char* name, const char* why) {
    rc_ = refuse(code, "%s: %s %s", call_, name, why);
    return *this;
  }
  const char* call_;
  int dev_ = -1, rc_ = QC_OK;
};

// Launch as a programmatic dependent of the kernel before: it may start early and
// waits (griddepcontrol.wait) before it reads or writes memory.
template <typename... A, typename... B>
cudaError_t launch_dependent(void (*k)(A...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                             const B&... args) {
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
  return cudaLaunchKernelEx(&cfg, k, A(args)...);
}

}  // namespace qc
