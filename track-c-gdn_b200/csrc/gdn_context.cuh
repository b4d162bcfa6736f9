// gdn_context.cuh -- the CUDA context that is current for the calling thread:
// the device's primary one as a rule, one of the caller's own (cuCtxCreate) in
// programs on the driver interface.  The runtime's calls work in either.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace gdn {

// A function of the driver, or null.
template <typename F>
F driver_function(const char *name) {
  void *p = nullptr;
  cudaDriverEntryPointQueryResult q;
  const bool found = cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) == cudaSuccess &&
                     q == cudaDriverEntryPointSuccess;
  return found ? reinterpret_cast<F>(p) : nullptr;
}

// Null: the thread has none.
inline CUcontext current_context() {
  static const auto get = driver_function<CUresult (*)(CUcontext *)>("cuCtxGetCurrent");
  CUcontext ctx = nullptr;
  return get != nullptr && get(&ctx) == CUDA_SUCCESS ? ctx : nullptr;
}

// A number that no other context of the process has or had; 0 for none.
inline unsigned long long current_context_id() {
  static const auto get = driver_function<CUresult (*)(CUcontext, unsigned long long *)>("cuCtxGetId");
  unsigned long long id = 0;
  const CUcontext ctx = current_context();
  return ctx != nullptr && get != nullptr && get(ctx, &id) == CUDA_SUCCESS ? id : 0;
}

}  // namespace gdn
