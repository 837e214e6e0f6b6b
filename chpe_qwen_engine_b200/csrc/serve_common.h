// serve_common.h -- argument checks shared by the entry points that work on a
// caller's device buffers for a batch of sequences (qk_rope.cu,
// attention_paged.cu, logits.cu).
//
// Every entry point checks each pointer on the host before it launches: a host
// address, a freed one, or one on another GPU is answered with -1 instead of a
// fault on the device.  The launch goes to the device that holds the buffers,
// which need not be the current one; the current device is left as it was.
// Buffers that the call writes must not overlap the others, but for what an entry
// point allows.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/chpe.h"
#include "buffer_rows.h"
#include "engine.h"

namespace chpe {

struct ServeCall {
  const char* name;
  int device = -1;    // of the first checked pointer
  int rc = 0;         // first failure
  char msg[192] = {};

  explicit ServeCall(const char* n) : name(n) {}

  int fail(int code, const char* what, long long a = 0, long long b = 0) {
    if (rc == 0) {
      rc = code;
      snprintf(msg, sizeof(msg), what, a, b);
    }
    return rc;
  }
  // p: device memory of this call's device, aligned to `align` bytes (a power of two).
  void ptr(const void* p, const char* what, uintptr_t align) {
    if (rc) return;
    if (!p) {
      snprintf(msg, sizeof(msg), "%s is NULL", what);
      rc = -1;
      return;
    }
    if (reinterpret_cast<uintptr_t>(p) & (align - 1)) {
      snprintf(msg, sizeof(msg), "%s is not aligned to %d bytes", what, (int)align);
      rc = -1;
      return;
    }
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
      cudaGetLastError();
      snprintf(msg, sizeof(msg), "%s: no usable CUDA device or not a CUDA address", what);
      rc = -1;
      return;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
      snprintf(msg, sizeof(msg), "%s is not device memory", what);
      rc = -1;
      return;
    }
    if (at.type == cudaMemoryTypeManaged) return;
    if (device < 0) device = at.device;
    else if (device != at.device) {
      snprintf(msg, sizeof(msg), "%s lies on device %d, other buffers on %d", what, at.device, device);
      rc = -1;
    }
  }
  void ptr_or_null(const void* p, const char* what, uintptr_t align) {
    if (p) ptr(p, what, align);
  }
  // out: rows that the call writes; other: rows that it reads, or writes too.  For checked
  // pointers, behind the checks of strides.
  void apart(const Rows& out, const Rows& other) {
    if (rc || !out.meets(other)) return;
    snprintf(msg, sizeof(msg), "%s overlaps %s", out.name, other.name);
    rc = -1;
  }
  // The device to launch on: that of the buffers, or the current one for managed memory.
  int launch_device() {
    if (device < 0 && cudaGetDevice(&device) != cudaSuccess) device = 0;
    return device;
  }
  // Ends the call: keeps the message for chpe_last_error(NULL).
  int done() const {
    try {
      set_thread_error(rc ? std::string(name) + ": " + msg : std::string());
    } catch (...) {  // no memory for the message: the code alone
    }
    return rc;
  }
};

// Makes `device` current for one launch and restores the previous one.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device < 0 || cudaGetDevice(&prev_) != cudaSuccess || prev_ == device) return;
    changed_ = cudaSetDevice(device) == cudaSuccess;
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int prev_ = -1;
  bool changed_ = false;
};

// Launch attributes: the kernel may be started while the one before it in the
// stream ends (programmatic dependent launch); each kernel here waits for that one before it
// reads or writes anything.
struct ServeLaunch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  ServeLaunch(dim3 grid, unsigned threads, size_t smem, cudaStream_t s, unsigned cluster = 1) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
      at[1].id = cudaLaunchAttributeClusterDimension;
      at[1].val.clusterDim.x = cluster;
      at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
  }
};

inline size_t dtype_size(int t) { return t == CHPE_F32 ? 4 : (t == CHPE_F16 || t == CHPE_BF16) ? 2 : 0; }

}  // namespace chpe
