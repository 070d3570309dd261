// The gated delta rule: argument checks, launch shapes and dispatch by element type.
#include "delta.h"

#include <algorithm>
#include <cmath>

#include "mma.h"
#include "overlap.h"

namespace za {
namespace delta {

using mma::T_BF16;
using mma::T_F16;
using mma::T_F32;

namespace {

uint32_t element_bytes(uint32_t dtype) { return dtype == T_F32 ? 4 : 2; }

// Whether every row begins at a multiple of `unit` bytes: the base and every stride that is used.
bool vectors(const void* p, const int64_t* stride, uint32_t batch, uint32_t length, uint32_t heads, uint32_t bytes, uint32_t unit) {
    const int64_t n[3] = {batch, length, heads};
    if ((uintptr_t)p % unit) return false;
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && stride[i] * bytes % unit) return false;
    return true;
}
bool state_vectors(const void* state, const ZenoAmdDeltaInputs& in) { return in.value_dim % 4 == 0 && (uintptr_t)state % 16 == 0; }

hipError_t by_type(uint32_t dtype, hipError_t (*f32)(const Args&, const Shape&, hipStream_t), hipError_t (*f16)(const Args&, const Shape&, hipStream_t),
                   hipError_t (*bf16)(const Args&, const Shape&, hipStream_t), const Args& a, const Shape& s, hipStream_t stream) {
    return (dtype == T_F32 ? f32 : dtype == T_F16 ? f16 : bf16)(a, s, stream);
}

Args common(const ZenoAmdDeltaInputs& in, const Shape& s) {
    Args a{};
    a.in = in;
    a.share = in.value_heads / in.key_heads;
    a.chunks = (in.length + 16 * s.tiles - 1) / (16 * s.tiles);
    a.segments = s.segments;
    a.segment_length = s.segment_length;
    const uint32_t eb = element_bytes(in.dtype);
    a.q_vec = vectors(in.q, in.q_stride, in.batch, in.length, in.key_heads, eb, 16);
    a.k_vec = vectors(in.k, in.k_stride, in.batch, in.length, in.key_heads, eb, 16);
    a.v_vec = vectors(in.v, in.v_stride, in.batch, in.length, in.value_heads, eb, 4 * eb);
    a.s_vec = state_vectors(in.state, in);
    return a;
}

void set_strides(int64_t* to, const int64_t* from) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

}  // namespace

// 16 tokens a chunk where 32 do not fit the 160 KB of a CU in the gradients' kernel. Segments:
// with fewer heads than 256 workgroups of eight waves or 512 of four, as many as make up those, of at least
// three chunks (4 heads of 1000 tokens forward: 40 us with three, 64 with eight, 125 in one segment; 76 heads
// of 333 with gradients 251 and 352). The gradients' kernel of four waves fits a CU twice in bfloat16 (76 KB)
// and once in float16 (119) and float32 (143), where the other kernels' gain still pays for segments that
// take turns (128 heads of 1024 x 64 x 64 with gradients: bfloat16 278 us, 560 with room for 256; float16 410
// and 635; float32 475 and 670). The additional pass over the tokens costs more than it saves where fewer than
// three segments come of it (111 heads of 211 tokens of 40 x 72, float32, inputs in cache: 48 us in one, 53 in
// two; of 64 x 64, bfloat16, 34 and 43).
Shape shape_of(const ZenoAmdDeltaInputs& in, bool train) {
    Shape s;
    s.dk = in.key_dim <= 64 ? 64 : 128;
    s.waves = s.dk == 128 || in.value_dim > 64 ? 8 : 4;
    s.tiles = train && s.waves == 8 && (in.dtype == T_F32 || (in.dtype == T_F16 && s.dk == 128)) ? 1 : 2;
    const int64_t chunk = 16 * s.tiles, chunks = (in.length + chunk - 1) / chunk;
    const int64_t heads = (int64_t)in.batch * in.value_heads, room = s.waves == 8 ? 256 : 512;
    int64_t want = room / heads;
    if (want > chunks / 3) want = chunks / 3;
    if (want < 3) want = 1;
    const int64_t each = (chunks + want - 1) / want;
    s.segment_length = (int)(each * chunk);
    s.segments = (int)((chunks + each - 1) / each);
    return s;
}

namespace {
uint64_t heads_of(const ZenoAmdDeltaInputs& in) { return (uint64_t)in.batch * in.value_heads; }
uint64_t states_floats(const ZenoAmdDeltaInputs& in, const Shape& s) {  // between segments
    return heads_of(in) * (s.segments - 1) * s.dk * (16 * s.waves);
}
uint64_t jumps_floats(const ZenoAmdDeltaInputs& in, const Shape& s) { return heads_of(in) * (s.segments - 1) * (3 * s.dk * s.dk + 4); }
uint64_t inner_floats(const ZenoAmdDeltaInputs& in, const Shape& s) {
    const uint64_t chunks = (in.length + 16 * s.tiles - 1) / (16 * s.tiles);
    return heads_of(in) * (chunks - 1) * s.dk * (16 * s.waves);
}
uint64_t share_floats(const ZenoAmdDeltaInputs& in) {
    return in.key_heads == in.value_heads ? 0 : (2ull * in.batch * in.length * in.value_heads * in.key_dim + 3) / 4 * 4;
}
}  // namespace

uint64_t saved_floats(const ZenoAmdDeltaInputs& in) {
    const Shape s = shape_of(in, true);
    return inner_floats(in, s) + jumps_floats(in, s);
}
uint64_t workspace_floats(const ZenoAmdDeltaInputs& in) {
    const Shape run = shape_of(in, false), train = shape_of(in, true);
    return std::max(states_floats(in, run) + jumps_floats(in, run), share_floats(in) + states_floats(in, train));
}

std::string check_sizes(const ZenoAmdDeltaInputs& in, bool step) {
    if (in.dtype > T_BF16) return "dtype is none of float32, float16, bfloat16";
    if (!in.batch || !in.length || !in.key_heads || !in.value_heads) return "batch, length and head counts must be positive";
    if (in.value_heads % in.key_heads) return "value_heads is not a multiple of key_heads";
    if (!in.key_dim || in.key_dim > ZENO_AMD_DELTA_MAX_DIM || !in.value_dim || in.value_dim > ZENO_AMD_DELTA_MAX_DIM)
        return "key_dim and value_dim must be 1 to " + std::to_string(ZENO_AMD_DELTA_MAX_DIM);
    // A launch takes less than 2^32 threads: 64 to 512 for each sequence and head (step_threads: see there).
    const uint64_t heads = (uint64_t)in.batch * in.value_heads;
    if (in.length > 0x7fffff00u || heads > 0x7fffffffull / 64 || (step ? step_threads(in) : heads * 64 * shape_of(in, false).waves) > 0xffffffffull)
        return "too many sequences or tokens";
    if ((uint64_t)in.batch * in.length * in.key_heads > 0x7fffffffull) return "too many tokens";
    return "";
}

std::string check(const ZenoAmdDeltaInputs* p, bool step) {
    if (!p) return "null arguments";
    const ZenoAmdDeltaInputs& in = *p;
    const std::string why = check_sizes(in, step);
    if (!why.empty()) return why;
    if (step && in.length != 1) return "a step takes one token";
    if (!in.q || !in.k || !in.v || !in.g || !in.beta) return "null input";
    if (!std::isfinite(in.scale)) return "scale is not finite";
    return "";
}

std::string check_overlap(const ZenoAmdDeltaInputs& in, const void* o, const int64_t* o_stride, const float* state, bool step) {
    const int64_t eb = element_bytes(in.dtype), keys[3] = {in.batch, in.length, in.key_heads}, values[3] = {in.batch, in.length, in.value_heads};
    const int64_t none[1] = {0}, one[1] = {1}, states = (int64_t)in.batch * in.value_heads * in.key_dim * in.value_dim;
    const Memory out(o, o_stride, values, 3, in.value_dim, eb), kept(state, none, one, 1, states, 4), v(in.v, in.v_stride, values, 3, in.value_dim, eb);
    const Memory inputs[] = {Memory(in.q, in.q_stride, keys, 3, in.key_dim, eb), Memory(in.k, in.k_stride, keys, 3, in.key_dim, eb),
                             Memory(in.g, in.g_stride, values, 3, 1, 4), Memory(in.beta, in.beta_stride, values, 3, 1, 4)};
    if (!out.apart_from_itself()) return "o overlaps itself";
    if (!apart(out, kept)) return "o overlaps the state";
    bool same = o == in.v;
    for (int i = 0; i < 3; ++i) same = same && (values[i] == 1 || o_stride[i] == in.v_stride[i]);
    if (!same && !apart(out, v)) return "o overlaps v and is not v itself";
    bool clear = apart(kept, v);
    for (const Memory& x : inputs) {
        if (!apart(out, x)) return "o overlaps an input";
        clear = clear && apart(kept, x);
    }
    if (in.reset) {
        const Memory reset(in.reset, in.reset_stride, values, 2, 1, 1);
        if (!apart(out, reset)) return "o overlaps an input";
        clear = clear && apart(kept, reset);
    }
    if (!step && in.state) {
        const Memory before(in.state, none, one, 1, states, 4);
        if (!apart(out, before)) return "o overlaps an input";
        clear = clear && apart(kept, before);
    }
    return clear ? "" : "the state overlaps an input";
}

hipError_t forward(const ZenoAmdDeltaInputs& in, void* o, const int64_t* o_stride, float* last, float* saved, float* workspace,
                   hipStream_t stream) {
    const Shape s = shape_of(in, saved != nullptr);
    Args a = common(in, s);
    a.o = o;
    set_strides(a.o_stride, o_stride);
    a.o_vec = vectors(o, o_stride, in.batch, in.length, in.value_heads, element_bytes(in.dtype), 4 * element_bytes(in.dtype));
    a.last = last;
    a.last_vec = state_vectors(last, in);
    a.saved = saved;
    a.starts = workspace;
    a.jumps = saved ? saved + inner_floats(in, s) : workspace + states_floats(in, s);
    a.full = in.key_dim == (uint32_t)s.dk && in.value_dim == 16u * s.waves && a.q_vec && a.k_vec && a.v_vec && a.o_vec && a.s_vec && a.last_vec;
    return by_type(in.dtype, launch_forward<T_F32>, launch_forward<T_F16>, launch_forward<T_BF16>, a, s, stream);
}

hipError_t backward(const ZenoAmdDeltaInputs& in, const float* saved, const ZenoAmdDeltaGradients& grad, float* workspace,
                    hipStream_t stream) {
    const Shape s = shape_of(in, true);
    Args a = common(in, s);
    const uint32_t eb = element_bytes(in.dtype);
    a.saved = const_cast<float*>(saved);
    a.jumps = a.saved + inner_floats(in, s);
    a.d_starts = workspace + share_floats(in);
    a.d_o = grad.d_o;
    set_strides(a.d_o_stride, grad.d_o_stride);
    a.d_o_vec = vectors(grad.d_o, grad.d_o_stride, in.batch, in.length, in.value_heads, eb, 16);
    a.d_last = grad.d_last;
    a.d_last_vec = state_vectors(grad.d_last, in);
    a.dq = grad.d_q;
    a.dk = grad.d_k;
    a.dv = grad.d_v;
    set_strides(a.dq_stride, grad.d_q_stride);
    set_strides(a.dk_stride, grad.d_k_stride);
    set_strides(a.dv_stride, grad.d_v_stride);
    a.dq_vec = vectors(grad.d_q, grad.d_q_stride, in.batch, in.length, in.key_heads, eb, 16);
    a.dk_vec = vectors(grad.d_k, grad.d_k_stride, in.batch, in.length, in.key_heads, eb, 16);
    a.dv_vec = vectors(grad.d_v, grad.d_v_stride, in.batch, in.length, in.value_heads, eb, 4 * eb);
    a.dg = grad.d_g;
    a.dbeta = grad.d_beta;
    set_strides(a.dg_stride, grad.d_g_stride);
    set_strides(a.dbeta_stride, grad.d_beta_stride);
    a.d_state = grad.d_state;
    a.d_state_vec = state_vectors(grad.d_state, in);
    a.full = in.key_dim == (uint32_t)s.dk && in.value_dim == 16u * s.waves && a.q_vec && a.k_vec && a.v_vec && a.s_vec && a.d_o_vec &&
             a.dq_vec && a.dk_vec && a.dv_vec && a.d_last_vec && a.d_state_vec;
    if (a.share > 1) {
        a.part_q = workspace;
        a.part_k = workspace + (uint64_t)in.batch * in.length * in.value_heads * in.key_dim;
    }
    return by_type(in.dtype, launch_backward<T_F32>, launch_backward<T_F16>, launch_backward<T_BF16>, a, s, stream);
}

hipError_t step(const ZenoAmdDeltaInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream) {
    Args a{};
    a.in = in;
    a.share = in.value_heads / in.key_heads;
    a.o = o;
    set_strides(a.o_stride, o_stride);
    return in.dtype == T_F32   ? launch_step<T_F32>(a, state, stream)
           : in.dtype == T_F16 ? launch_step<T_F16>(a, state, stream)
                               : launch_step<T_BF16>(a, state, stream);
}

}  // namespace delta
}  // namespace za
