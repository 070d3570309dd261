// Layer norm's kernels for one element type.
#include "norm_kernels.h"

namespace za {
namespace norm {
template hipError_t launch_forward<mma::T_F32>(const Args&, const Shape&, hipStream_t);
template hipError_t launch_backward<mma::T_F32>(const Args&, const ZenoAmdNormGradients&, const Shape&, hipStream_t);
}  // namespace norm
}  // namespace za
