// Host-side helpers shared by the translation units of libmh3_b200.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "mh3_b200.h"

namespace mh3 {

// Record ``msg`` as this thread's last error and return ``code``.
int fail(int code, const char* msg);
// Record a CUDA error with context and return it as a positive code.
int fail_cuda(cudaError_t e, const char* what);

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link
// dependency on libcuda).  Returns MH3_OK or MH3_ERR_DRIVER.
int encode_tiled(CUtensorMap* map, CUtensorMapDataType dtype, uint32_t rank, void* base, const cuuint64_t* dims,
                 const cuuint64_t* strides_bytes, const cuuint32_t* box, const cuuint32_t* elem_strides,
                 CUtensorMapSwizzle swizzle);

// The library's device error word on the current device.
int* device_error_word();

// Lets kernel K take up to ``most`` bytes of dynamic shared memory on the current device.  The
// limit belongs to the device's function, which all host threads share, so a call sets the most
// that K ever takes, not its own need: a lower value between another thread's call and its
// launch would fail that launch.
template <auto K>
cudaError_t allow_smem(size_t most) {
  static std::atomic<uint64_t> set{0};  // a bit for each device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (set.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e == cudaSuccess) set.fetch_or(bit, std::memory_order_release);
  return e;
}

// The calling thread's current CUDA context (CUcontext), or null; through
// the runtime's driver entry point, so the library does not link libcuda.
void* current_context();

// NVTX range named after a C entry point, over its host-side work (argument
// checks and launches), so a profiler can attribute kernels to entry points
// (e.g. ncu --nvtx --nvtx-include "mh3_fp8_attention_fwd/").  NVTX3 is
// header-only: without an attached tool a push/pop is a pointer check, and
// the library gains no link dependency.
struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

}  // namespace mh3
