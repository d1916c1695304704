// Host-side helpers shared by the translation units of libgdsq.so: the
// calling thread's error text, cached device attributes, the launch wrapper
// and the tensor-map encoder.  Defined in gdsq.cu unless inline.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <stdint.h>
#include <string>
#include <utility>

namespace gdsq {

extern thread_local std::string t_last_error;
extern int g_pdl_enabled;

// Records the error text of this thread and returns `status`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int cuda_fail(cudaError_t e, const char* what);

struct DeviceInfo {
  bool ready = false;
  int ordinal = 0;
  int sms = 0;
  int smem_optin = 0;
};

constexpr int kMaxDevices = 64;

int device_info(const DeviceInfo** out);
int get_encoder(PFN_cuTensorMapEncodeTiled_v12000* out);

// ORs a translation unit's own device error word into *bits.
cudaError_t serve_error_bits(bool clear, int* bits);
cudaError_t attend_error_bits(bool clear, int* bits);

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                   cudaStream_t stream, bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Raises a kernel's dynamic shared-memory limit when a launch needs more than
// was last set for that (kernel, device).
cudaError_t ensure_smem_limit(const void* kernel, int bytes, int device);

template <typename K>
cudaError_t ensure_smem(K kernel, int bytes, int device) {
  return ensure_smem_limit(reinterpret_cast<const void*>(kernel), bytes, device);
}

}  // namespace gdsq
