// The gated delta rule: host side (argument checks, launch shapes) and the kernels' arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/zeno_amd_ext.h"

namespace za {
namespace delta {

// What a kernel reads and writes. Strides are in elements: sequence, token, head.
struct Args {
    ZenoAmdDeltaInputs in;
    void* o;
    int64_t o_stride[3];
    float* last;                 // [batch, value_heads, key_dim, value_dim]
    float* saved;                // states inside the sequences (training), see saved_floats
    uint32_t chunks;             // chunks of the grid that a sequence has
    // A long sequence is cut into segments that run side by side. Between them: the states and
    // their gradients [batch, value_heads, segments - 1, DK, 16 waves], and of each segment but the
    // last (unused for the first) the matrix that takes the state over it, as operands of three
    // 16-bit parts, and its transpose (3 DK DK + 4 floats).
    uint32_t segments;
    int segment_length;          // tokens, whole chunks
    float *starts, *jumps, *d_starts;
    uint32_t share;              // value heads per key head
    bool q_vec, k_vec;           // eight elements of a row are aligned to 16 bytes (32 of fp32)
    bool v_vec, o_vec, s_vec, last_vec;  // four elements are aligned to their size
    bool full;                   // heads as wide as the launch shape, everything aligned
    // backward
    const void* d_o;
    int64_t d_o_stride[3];
    bool d_o_vec;
    const float* d_last;         // null: zeros
    void *dq, *dk, *dv;
    int64_t dq_stride[3], dk_stride[3], dv_stride[3];
    bool dq_vec, dk_vec, dv_vec, d_last_vec, d_state_vec;
    float *dg, *dbeta;
    int64_t dg_stride[3], dbeta_stride[3];
    float* d_state;              // null: not wanted
    float *part_q, *part_k;      // gradients per value head where heads share keys: [batch, length, value_heads, key_dim]
};

// Launch shape of the chunked kernels, by sizes and type alone.
struct Shape {
    int dk;      // key columns held: 64 or 128
    int waves;   // of 16 value columns each: 4 or 8
    int tiles;   // chunk of 16 or 32 tokens
    int segments, segment_length;
};
Shape shape_of(const ZenoAmdDeltaInputs& in, bool train);
// What a forward call leaves for its gradients (states inside the sequences, matrices over
// segments), and what either call needs beside that.
uint64_t saved_floats(const ZenoAmdDeltaInputs& in);
uint64_t workspace_floats(const ZenoAmdDeltaInputs& in);

// One translation unit per element type.
template <int TY> hipError_t launch_forward(const Args& a, const Shape& s, hipStream_t stream);
template <int TY> hipError_t launch_backward(const Args& a, const Shape& s, hipStream_t stream);
template <int TY> hipError_t launch_step(const Args& a, float* state, hipStream_t stream);

// Of the single step: a wave holds all rows of 4 `lanes` columns of a head.
inline int step_lanes(const ZenoAmdDeltaInputs& in) { return in.key_dim <= 32 || in.key_dim > 64 ? 8 : 16; }
inline uint64_t step_waves(const ZenoAmdDeltaInputs& in) {
    const uint32_t cols = 4 * step_lanes(in);
    return (uint64_t)in.batch * in.value_heads * ((in.value_dim + cols - 1) / cols);
}
inline uint64_t step_threads(const ZenoAmdDeltaInputs& in) { return (step_waves(in) + 3) / 4 * 256; }

// Entry points behind the C ABI. A non-empty message means that nothing was launched.
std::string check_sizes(const ZenoAmdDeltaInputs& in, bool step);
std::string check(const ZenoAmdDeltaInputs* in, bool step);
// Outputs of a step or a forward call (`state`: of either) that overlap themselves, each other or an
// input. o may be v itself, value by value: the wave that writes a value has read it.
std::string check_overlap(const ZenoAmdDeltaInputs& in, const void* o, const int64_t* o_stride, const float* state, bool step);
hipError_t forward(const ZenoAmdDeltaInputs& in, void* o, const int64_t* o_stride, float* last, float* saved, float* workspace,
                   hipStream_t stream);
hipError_t backward(const ZenoAmdDeltaInputs& in, const float* saved, const ZenoAmdDeltaGradients& grad, float* workspace,
                    hipStream_t stream);
hipError_t step(const ZenoAmdDeltaInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream);

}  // namespace delta
}  // namespace za
