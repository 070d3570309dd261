// Newton-Schulz orthogonalisation of matrix updates: host side.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/zeno_amd_ext.h"

namespace za {
namespace orth {

std::string check(const ZenoAmdOrthogonalize* a);
bool out_overlaps(const ZenoAmdOrthogonalize& a);         // two of its values in one place
uint64_t workspace_bytes(const ZenoAmdOrthogonalize& a);  // of checked arguments
hipError_t run(const ZenoAmdOrthogonalize& a, void* workspace, hipStream_t stream);

}  // namespace orth
}  // namespace za
