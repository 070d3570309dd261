// Layer norm: host side (argument checks, launch shapes) and the kernels' arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/zeno_amd_ext.h"

namespace za {
namespace norm {

struct Args {
    ZenoAmdNormInputs in;
    uint32_t rows;           // all of them
    bool flat;               // one stride leads from row to row
    void *y, *sum;           // sum: null without a residual
    int64_t y_stride[3], sum_stride[3];
    // backward
    const void *d_y, *d_sum;  // d_sum: null without a residual's, d_y never
    void* d_x;                // null: not wanted
    int64_t d_y_stride[3], d_sum_stride[3], d_x_stride[3];
    float* parts;             // [blocks, 2, dim]: each workgroup's sums for the weight and the bias; null: not wanted
};

// Launch shape: `lanes` lanes hold a row in vectors of eight elements, `vectors` each. A workgroup of
// `threads` takes threads / lanes rows at a time and goes on with those `blocks` workgroups further.
struct Shape {
    int lanes, vectors, threads;
    uint32_t blocks;
};
Shape shape_of(const ZenoAmdNormInputs& in, bool train);
uint64_t workspace_floats(const ZenoAmdNormInputs& in);

// One translation unit per element type.
template <int TY> hipError_t launch_forward(const Args& a, const Shape& s, hipStream_t stream);
template <int TY> hipError_t launch_backward(const Args& a, const ZenoAmdNormGradients& grad, const Shape& s, hipStream_t stream);

// Entry points behind the C ABI. A non-empty message means that nothing was launched.
std::string check(const ZenoAmdNormInputs* in);
std::string check_forward(const ZenoAmdNormInputs& in, const void* y, const int64_t* y_stride, const void* sum, const int64_t* sum_stride);
std::string check_backward(const ZenoAmdNormInputs& in, const ZenoAmdNormGradients& grad);
hipError_t forward(const ZenoAmdNormInputs& in, void* y, const int64_t* y_stride, void* sum, const int64_t* sum_stride, hipStream_t stream);
hipError_t backward(const ZenoAmdNormInputs& in, const ZenoAmdNormGradients& grad, float* workspace, hipStream_t stream);

}  // namespace norm
}  // namespace za
