// Linear attention with a decay for each head: host side (argument checks, launch shapes) and the
// kernels' arguments.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/zeno_amd_ext.h"

namespace za {
namespace linear {

constexpr int kChunk = 32;  // tokens, at most: segments are multiples of it

// Rows of one of the inputs. Strides are in elements: sequence, token, head.
struct Rows {
    const void* at;
    int64_t stride[3];
    uint32_t share;  // heads that read one of these
};

// One walk over the sequences, forward or back. With A, B and C three of the rows and S a state
// [da, dc]: the outputs of a token are sums over the tokens behind it in the walk's direction,
//     out_i = scale sum_j exp(g |i - j|) (A_i . B_j) C_j + A_i S,   S <- exp(g) S + B_i C_i^T
// The operator itself is the walk forward of q, k, v; its gradients are those of d_o, v, k (forward:
// d_q), of k, q, d_o (back: d_v) and of v, d_o, q (back: d_k).
struct Walk {
    Rows a, b, c, q;             // q: what the outputs of d_q are multiplied with for the gradient of g
    int da, dc;
    uint32_t batch, heads;       // value heads
    int length;
    float scale;
    const float* g;
    const uint8_t* reset;
    int64_t reset_stride[2];
    void* out;
    int64_t out_stride[3];
    bool out_f32;                // part sums per value head, where heads share one
    const float* first;          // the state that the walk begins with; null: zeros
    float* last;                 // the state that it ends with; null: not wanted
    int ld;                      // a state in memory: rows of this many values, its rows or (turned) its columns
    bool turned;
    int64_t size;                // of a state
    // A long sequence is cut into segments that are walked side by side. Between them: states (and
    // slopes, see the kernels) [batch, heads, segments - 1, size], and whether a state passes the
    // segment, [batch, heads, segments - 1].
    uint32_t segments;
    int segment_length;          // tokens, whole chunks
    float *starts, *slopes, *passes;
    const float* d_last;         // for the gradient of g; null: zeros
    double* parts;               // of it: [batch, heads, segments, waves]
    uint32_t blocks;             // waves that share the columns, set at the launch
};

// Two waves a SIMD. Sequences are cut into segments for as many waves (of 32 columns) at most, and waves of 64 columns are
// taken where there are as many of those, which fill their columns: never of a sequence that is cut, so the states between
// segments have no kernel for them.
constexpr int kWaves = 2048;
inline bool wide(uint64_t walks, int blocks, int halves) { return 2 * blocks == halves && walks * blocks >= kWaves; }  // of 64 columns and of 32

// A wave holds 32 times 1, 2 or 4 rows of a state.
inline int steps_of(int da) { return da <= 32 ? 1 : da <= 64 ? 2 : 4; }
// Tiles of 16 columns of a wave of the decays' gradient, which carries the state and its slope; `js` is of the waves beside it. Two
// where there are many waves and the registers bear it: by themselves those of 4096 sequences of 32 tokens, four heads of
// 64 x 64, bfloat16, take 233 us, with one tile 271; of 300 of 200, float32, 154 and 179. With few waves one (19 of 333, four heads of
// 24 x 48, float32: 25 us, 36), and with 32 rows (300 of 200, 32 x 32, bfloat16: 37, 39); with 128 rows two spill 145 registers.
constexpr int slope_tiles(int steps, int js) { return steps == 2 && js == 4 ? 2 : 1; }
struct Segments {
    uint32_t count;
    int length;
};
Segments segments_of(const ZenoAmdLinearInputs& in);
uint64_t saved_floats(const ZenoAmdLinearInputs& in);
uint64_t workspace_floats(const ZenoAmdLinearInputs& in, bool train);

// What a walk is for: its outputs, the gradient of g, the states between segments, or those with their slopes,
// which the gradient of g needs.
enum Kind { OUTPUTS, SLOPES, STATES, STATES_SLOPE };

// One translation unit per element type.
template <int TY> hipError_t launch_walk(Walk w, Kind kind, bool back, hipStream_t stream);
template <int TY> hipError_t launch_gradients(Walk v, Walk k, Walk q, uint32_t* slopes, hipStream_t stream);
template <int TY> hipError_t launch_share(const ZenoAmdLinearInputs& in, const float* part_q, const float* part_k, const ZenoAmdLinearGradients& grad, hipStream_t stream);
template <int TY> hipError_t launch_step(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream);

// Of the single step: a wave holds all rows of 4 `lanes` columns of a head.
inline int step_lanes(const ZenoAmdLinearInputs& in) { return in.key_dim <= 32 || in.key_dim > 64 ? 8 : 16; }
inline uint64_t step_waves(const ZenoAmdLinearInputs& in) {
    const uint32_t cols = 4 * step_lanes(in);
    return (uint64_t)in.batch * in.value_heads * ((in.value_dim + cols - 1) / cols);
}

// Entry points behind the C ABI. A non-empty message means that nothing was launched.
std::string check_sizes(const ZenoAmdLinearInputs& in, bool step);
std::string check(const ZenoAmdLinearInputs* in, bool step);
std::string check_overlap(const ZenoAmdLinearInputs& in, const void* o, const int64_t* o_stride, const float* state, bool step);
std::string check_gradients(const ZenoAmdLinearInputs& in, const ZenoAmdLinearGradients& grad);
hipError_t forward(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* last, float* saved, float* workspace, hipStream_t stream);
hipError_t backward(const ZenoAmdLinearInputs& in, const float* saved, const ZenoAmdLinearGradients& grad, float* workspace, hipStream_t stream);
hipError_t step(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream);

}  // namespace linear
}  // namespace za
