// The norms around a residual block on bfloat16 (amsim_norm.cuh).
#include "amsim_norm.cuh"

namespace amsim {
namespace normk {

template cudaError_t launch_type<__nv_bfloat16>(NormParams&, bool, bool, bool, int, int, cudaStream_t, const Plan*);
template cudaError_t launch_reduce<__nv_bfloat16>(const NormParams&, const Plan&, cudaStream_t);

}  // namespace normk
}  // namespace amsim
