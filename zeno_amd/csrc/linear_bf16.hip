// Linear attention's kernels for one element type.
#include "linear_kernels.h"

namespace za {
namespace linear {
template hipError_t launch_walk<mma::T_BF16>(Walk, Kind, bool, hipStream_t);
template hipError_t launch_gradients<mma::T_BF16>(Walk, Walk, Walk, uint32_t*, hipStream_t);
template hipError_t launch_share<mma::T_BF16>(const ZenoAmdLinearInputs&, const float*, const float*, const ZenoAmdLinearGradients&, hipStream_t);
template hipError_t launch_step<mma::T_BF16>(const ZenoAmdLinearInputs&, void*, const int64_t*, float*, hipStream_t);
}  // namespace linear
}  // namespace za
