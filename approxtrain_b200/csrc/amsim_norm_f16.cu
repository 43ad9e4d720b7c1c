// The norms around a residual block on half (amsim_norm.cuh).
#include "amsim_norm.cuh"

namespace amsim {
namespace normk {

template cudaError_t launch_type<__half>(NormParams&, bool, bool, bool, int, int, cudaStream_t, const Plan*);
template cudaError_t launch_reduce<__half>(const NormParams&, const Plan&, cudaStream_t);

}  // namespace normk
}  // namespace amsim
