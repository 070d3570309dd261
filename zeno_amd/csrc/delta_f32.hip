// The gated delta rule's kernels for one element type.
#include "delta_kernels.h"

namespace za {
namespace delta {
template hipError_t launch_forward<T_F32>(const Args&, const Shape&, hipStream_t);
template hipError_t launch_backward<T_F32>(const Args&, const Shape&, hipStream_t);
template hipError_t launch_step<T_F32>(const Args&, float*, hipStream_t);
}  // namespace delta
}  // namespace za
