// What the library's translation units share on the host: the calling thread's error text, the launch count, device facts.
// Defined in amsim.cu.
#pragma once
#include <cuda_runtime.h>

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

}  // namespace amsim

#define AMSIM_HOST_TRY(expr)                                                                                        \
  do {                                                                                                              \
    cudaError_t e_ = (expr);                                                                                        \
    if (e_ != cudaSuccess) return amsim::host_fail(AMSIM_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)
