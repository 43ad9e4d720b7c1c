// What the library's translation units share on the host: the calling thread's error text, the launch count, device facts.
// Defined in amsim.cu.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/amsim.h"

namespace amsim {

int host_fail(int code, const char* fmt, ...);  // records the text, returns code
void host_count_launch();
int host_sm_count(int device);
int host_device();
// A word in host memory that a kernel on `device` sets when a bounded wait of its warps has run out; reported, once, as
// AMSIM_ERR_CUDA by the next call that asks.
int host_stuck_word(int device, unsigned** word);
int host_report_stuck(int device);
bool host_no_tries();  // AMSIM_CODES_SPIN=0: bounded waits give up at once (for the test of the report)

// Lets `kernel` take up to `bytes` of dynamic shared memory: asked for once per device and kernel (`done`: a word of the
// kernel's own, one bit a device).
template <typename K>
cudaError_t host_allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  const int device = host_device();
  const unsigned long long bit = device >= 0 && device < 64 ? 1ull << device : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace amsim

#define AMSIM_HOST_TRY(...)                                                                                                  \
  do {                                                                                                                       \
    cudaError_t e_ = (__VA_ARGS__);                                                                                          \
    if (e_ != cudaSuccess) return amsim::host_fail(AMSIM_ERR_CUDA, "%s: %s", __func__, cudaGetErrorString(e_)); \
  } while (0)
