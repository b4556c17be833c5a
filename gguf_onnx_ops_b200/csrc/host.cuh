// Host side shared by the library's translation units: the error channel, launches and argument checks.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/gguf_ops.h"

namespace gguf_b200 {

int set_error(int code, const std::string& msg);  // records the message for gguf_last_error, returns code
void clear_error();
bool pdl_enabled();
int device_sms(int* sms);  // of the current device

// The device error word of the translation unit of the KV-cache ops, read and cleared.
cudaError_t kv_device_error(int* error, int* site);

inline int set_cuda_error(const char* op, cudaError_t e) {
  return set_error(GGUF_ERR_CUDA, std::string(op) + ": " + cudaGetErrorString(e));
}
inline bool is_aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A launch on `s` with the programmatic-dependent attribute the library's kernels use.
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  if (pdl_enabled()) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace gguf_b200
