// Layer norm: argument checks, launch shapes and dispatch by element type.
#include "norm.h"

#include <algorithm>
#include <cmath>
#include <vector>

#include "mma.h"
#include "overlap.h"

namespace za {
namespace norm {

using mma::T_BF16;
using mma::T_F16;
using mma::T_F32;

namespace {

int64_t bytes_of(uint32_t dtype) { return dtype == T_F32 ? 4 : 2; }
uint64_t rows_of(const ZenoAmdNormInputs& in) { return (uint64_t)in.rows[0] * in.rows[1] * in.rows[2]; }

Memory rows_in(const ZenoAmdNormInputs& in, const void* p, const int64_t* stride) {
    const int64_t n[3] = {in.rows[0], in.rows[1], in.rows[2]};
    return Memory(p, stride, n, 3, in.dim, bytes_of(in.dtype));
}
Memory weights_in(const ZenoAmdNormInputs& in, const void* p) {
    const int64_t none[1] = {0}, one[1] = {1};
    return Memory(p, none, one, 1, in.dim, bytes_of(in.weight_dtype));
}

std::string check_outputs(const std::vector<Memory>& inputs, const std::vector<Memory>& outputs) {
    for (size_t i = 0; i < outputs.size(); ++i) {
        if (!outputs[i].apart_from_itself()) return "an output overlaps itself";
        for (const Memory& x : inputs)
            if (!apart(outputs[i], x)) return "an output overlaps an input";
        for (size_t j = 0; j < i; ++j)
            if (!apart(outputs[i], outputs[j])) return "outputs overlap";
    }
    return "";
}

// Dimensions that follow on one another in every array become one: a row's place then takes one
// product, where it takes divisions otherwise.
void flatten(uint32_t* n, int64_t* const* stride, int arrays) {
    auto nest = [&](int outer) {
        const int inner = outer + 1;
        bool yes = true;
        for (int i = 0; i < arrays; ++i) yes = yes && (n[outer] == 1 || n[inner] == 1 || stride[i][outer] == stride[i][inner] * (int64_t)n[inner]);
        if (!yes) return false;
        for (int i = 0; i < arrays; ++i)
            if (n[inner] == 1) stride[i][inner] = stride[i][outer];
        n[inner] *= n[outer];
        n[outer] = 1;
        return true;
    };
    if (nest(1)) {
        std::swap(n[0], n[1]);
        for (int i = 0; i < arrays; ++i) stride[i][1] = stride[i][0];
        nest(1);
    } else {
        nest(0);
    }
}

void set_strides(int64_t* to, const int64_t* from) {
    for (int i = 0; i < 3; ++i) to[i] = from ? from[i] : 0;
}

}  // namespace

// A row of up to 1024 features is held by part of a wave or a wave, one or two vectors a lane; a wider
// one by a workgroup. Of 65536 rows of 1024, bfloat16, the norm takes 43 us and the gradients 95, by a workgroup of 256 to the row 85
// and 154; of 16384 rows of 4096 by 256 threads 45 and 100, by 1024 95 and 179; of 524288 rows of 64 by 8 lanes 23 us, by 16 39.
// Workgroups as fill the device several times over, each with several rows, as each reads the weights and leaves sums. Gradients
// (us; with half as many, with twice as many): 131072 rows of 512 86 (122, 92), 32768 of 2048 88 (119, 93), 8192 of 8192 116 (200,
// 121), 65536 of 1024 95 (87, 90), 16384 of 4096 101 (93, 99), 524288 of 64 71 (68, 71), 131072 of 200 73 (70, 71); float32: 16384 of
// 2500 177 (160, 152), 65536 of 1000 162 (155, 166).
Shape shape_of(const ZenoAmdNormInputs& in, bool train) {
    Shape s;
    const uint32_t n = in.dim;
    s.lanes = n <= 64 ? 8 : n <= 128 ? 16 : n <= 256 ? 32 : n <= 1024 ? 64 : n <= 4096 ? 256 : 1024;
    s.vectors = (n + 8 * s.lanes - 1) / (8 * s.lanes);
    s.threads = std::max(s.lanes, 256);
    const uint64_t each = s.threads / s.lanes, need = (rows_of(in) + each - 1) / each;
    s.blocks = (uint32_t)std::min<uint64_t>(need, (train ? 1024 : 2048) * 256 / s.threads);
    return s;
}

uint64_t workspace_floats(const ZenoAmdNormInputs& in) { return 2ull * shape_of(in, true).blocks * in.dim; }

std::string check(const ZenoAmdNormInputs* p) {
    if (!p) return "null arguments";
    const ZenoAmdNormInputs& in = *p;
    if (in.dtype > T_BF16) return "dtype is none of float32, float16, bfloat16";
    if (in.weight_dtype != in.dtype && in.weight_dtype != T_F32) return "weight_dtype is neither dtype nor float32";
    if (!in.rows[0] || !in.rows[1] || !in.rows[2]) return "there are no rows";
    if (!in.dim || in.dim > ZENO_AMD_NORM_MAX_DIM) return "dim must be 1 to " + std::to_string(ZENO_AMD_NORM_MAX_DIM);
    if ((uint64_t)in.rows[0] * in.rows[1] > 0x7fffffffull || rows_of(in) > 0x7fffffffull) return "too many rows";
    if (!std::isfinite(in.eps) || in.eps < 0.0f) return "eps must be finite and not negative";
    return "";
}

std::string check_forward(const ZenoAmdNormInputs& in, const void* y, const int64_t* y_stride, const void* sum, const int64_t* sum_stride) {
    if (!in.x) return "null input";
    if (!y || !y_stride) return "null output";
    if (!in.residual != !sum || (sum && !sum_stride)) return "a residual and its sum come together";
    std::vector<Memory> reads{rows_in(in, in.x, in.x_stride)}, writes{rows_in(in, y, y_stride)};
    if (in.residual) reads.push_back(rows_in(in, in.residual, in.residual_stride));
    if (in.weight) reads.push_back(weights_in(in, in.weight));
    if (in.bias) reads.push_back(weights_in(in, in.bias));
    if (sum) writes.push_back(rows_in(in, sum, sum_stride));
    return check_outputs(reads, writes);
}

std::string check_backward(const ZenoAmdNormInputs& in, const ZenoAmdNormGradients& grad) {
    if (!in.x || !grad.d_y) return "null input";
    if (!grad.d_x && !grad.d_weight && !grad.d_bias) return "no gradient is wanted";
    std::vector<Memory> reads{rows_in(in, in.x, in.x_stride), rows_in(in, grad.d_y, grad.d_y_stride)}, writes;
    if (grad.d_sum) reads.push_back(rows_in(in, grad.d_sum, grad.d_sum_stride));
    if (in.weight) reads.push_back(weights_in(in, in.weight));
    if (grad.d_x) writes.push_back(rows_in(in, grad.d_x, grad.d_x_stride));
    if (grad.d_weight) writes.push_back(weights_in(in, grad.d_weight));
    if (grad.d_bias) writes.push_back(weights_in(in, grad.d_bias));
    return check_outputs(reads, writes);
}

hipError_t forward(const ZenoAmdNormInputs& in, void* y, const int64_t* y_stride, void* sum, const int64_t* sum_stride, hipStream_t stream) {
    Args a{};
    a.in = in;
    a.rows = (uint32_t)rows_of(in);
    a.y = y;
    a.sum = sum;
    set_strides(a.y_stride, y_stride);
    set_strides(a.sum_stride, sum_stride);
    int64_t* const strides[] = {a.in.x_stride, a.y_stride, a.in.residual_stride, a.sum_stride};
    flatten(a.in.rows, strides, sum ? 4 : 2);
    a.flat = a.in.rows[0] == 1 && a.in.rows[1] == 1;
    const Shape s = shape_of(in, false);
    return in.dtype == T_F32   ? launch_forward<T_F32>(a, s, stream)
           : in.dtype == T_F16 ? launch_forward<T_F16>(a, s, stream)
                               : launch_forward<T_BF16>(a, s, stream);
}

hipError_t backward(const ZenoAmdNormInputs& in, const ZenoAmdNormGradients& grad, float* workspace, hipStream_t stream) {
    Args a{};
    a.in = in;
    a.rows = (uint32_t)rows_of(in);
    a.d_y = grad.d_y;
    a.d_sum = grad.d_sum;
    a.d_x = grad.d_x;
    set_strides(a.d_y_stride, grad.d_y_stride);
    set_strides(a.d_x_stride, grad.d_x ? grad.d_x_stride : grad.d_y_stride);
    set_strides(a.d_sum_stride, grad.d_sum ? grad.d_sum_stride : grad.d_y_stride);
    int64_t* const strides[] = {a.in.x_stride, a.d_y_stride, a.d_x_stride, a.d_sum_stride};
    flatten(a.in.rows, strides, 4);
    a.flat = a.in.rows[0] == 1 && a.in.rows[1] == 1;
    a.parts = grad.d_weight || grad.d_bias ? workspace : nullptr;
    const Shape s = shape_of(in, true);
    return in.dtype == T_F32   ? launch_backward<T_F32>(a, grad, s, stream)
           : in.dtype == T_F16 ? launch_backward<T_F16>(a, grad, s, stream)
                               : launch_backward<T_BF16>(a, grad, s, stream);
}

}  // namespace norm
}  // namespace za
