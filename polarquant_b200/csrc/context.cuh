// The id of the current context, for what is kept per context: a
// cudaDeviceReset re-creates the device's primary context, and with it go the
// addresses of device arrays and the attributes set on kernels.  The driver's
// cuCtxGetCurrent and cuCtxGetId are reached through cudaGetDriverEntryPoint.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace pqb {

// Id of the calling thread's current context, 0 when there is none (or the
// driver cannot say).
inline unsigned long long current_ctx_id() {
  struct Entries {
    CUresult (*get_current)(CUcontext*) = nullptr;
    CUresult (*get_id)(CUcontext, unsigned long long*) = nullptr;
    Entries() {
      void* p = nullptr;
      cudaDriverEntryPointQueryResult q;
      if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q) == cudaSuccess &&
          q == cudaDriverEntryPointSuccess)
        get_current = reinterpret_cast<CUresult (*)(CUcontext*)>(p);
      p = nullptr;
      if (cudaGetDriverEntryPoint("cuCtxGetId", &p, cudaEnableDefault, &q) == cudaSuccess &&
          q == cudaDriverEntryPointSuccess)
        get_id = reinterpret_cast<CUresult (*)(CUcontext, unsigned long long*)>(p);
    }
  };
  static const Entries driver;
  if (!driver.get_current || !driver.get_id) return 0;
  CUcontext ctx = nullptr;
  unsigned long long id = 0;
  if (driver.get_current(&ctx) != CUDA_SUCCESS || ctx == nullptr) return 0;
  if (driver.get_id(ctx, &id) != CUDA_SUCCESS) return 0;
  return id;
}

}  // namespace pqb
