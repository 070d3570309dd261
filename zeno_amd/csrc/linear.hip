// Linear attention with a decay for each head: argument checks, launch shapes and dispatch by element type.
#include "linear.h"

#include <algorithm>
#include <cmath>
#include <vector>

#include "mma.h"
#include "overlap.h"

namespace za {
namespace linear {

using mma::T_BF16;
using mma::T_F16;
using mma::T_F32;

namespace {

// The gradient of g: the walks' parts of each head, in order, in 64 bits. Bound by the wait for each read, so eight are
// read at once, by as many threads as a workgroup has.
__global__ __launch_bounds__(1024) void linear_decay_kernel(const double* parts, uint32_t batch, uint32_t heads, uint32_t each, float* d_g) {
    __shared__ double all[1024];
    const uint32_t h = blockIdx.x;
    const int64_t n = (int64_t)batch * each;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
        double x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t at = i + 1024 * k;
            x[k] = at < n ? parts[(at / each * heads + h) * each + at % each] : 0.0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += x[k];
    }
    all[threadIdx.x] = sum;
    __syncthreads();
    for (int d = 512; d; d >>= 1) {
        if ((int)threadIdx.x < d) all[threadIdx.x] += all[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) d_g[h] = (float)all[0];
}

uint32_t blocks_of(uint32_t columns) { return (columns + 31) / 32; }
int64_t bytes_of(uint32_t dtype) { return dtype == T_F32 ? 4 : 2; }
uint64_t heads_of(const ZenoAmdLinearInputs& in) { return (uint64_t)in.batch * in.value_heads; }
uint64_t even(uint64_t floats) { return (floats + 3) / 4 * 4; }  // 16 bytes
int64_t state_size(const ZenoAmdLinearInputs& in) { return (int64_t)in.key_dim * in.value_dim; }
uint64_t between(const ZenoAmdLinearInputs& in) { return heads_of(in) * (segments_of(in).count - 1); }
uint64_t states_floats(const ZenoAmdLinearInputs& in) { return even(between(in) * state_size(in)); }
uint64_t share_floats(const ZenoAmdLinearInputs& in) {  // gradients of q (or k) by value head
    return in.key_heads == in.value_heads ? 0 : even((uint64_t)in.batch * in.length * in.value_heads * in.key_dim);
}
uint64_t parts_floats(const ZenoAmdLinearInputs& in) { return in.decay_gradient ? even(2 * heads_of(in) * segments_of(in).count * 2 * blocks_of(in.key_dim)) : 0; }

void set_strides(int64_t* to, const int64_t* from) {
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}
Rows rows_of(const void* at, const int64_t* stride, uint32_t share) {
    Rows r{};
    r.at = at;
    set_strides(r.stride, stride);
    r.share = share;
    return r;
}

hipError_t launch(uint32_t dtype, const Walk& w, Kind kind, bool back, hipStream_t stream) {
    auto run = dtype == T_F32 ? launch_walk<T_F32> : dtype == T_F16 ? launch_walk<T_F16> : launch_walk<T_BF16>;
    return run(w, kind, back, stream);
}

// A walk over states [key_dim, value_dim], or (turned) over them transposed.
Walk walk_of(const ZenoAmdLinearInputs& in, bool turned) {
    Walk w{};
    w.da = turned ? in.value_dim : in.key_dim;
    w.dc = turned ? in.key_dim : in.value_dim;
    w.ld = in.value_dim;
    w.turned = turned;
    w.size = state_size(in);
    w.batch = in.batch;
    w.heads = in.value_heads;
    w.length = in.length;
    w.scale = in.scale;
    w.g = in.g;
    w.reset = in.reset;
    w.reset_stride[0] = in.reset_stride[0];
    w.reset_stride[1] = in.reset_stride[1];
    const Segments s = segments_of(in);
    w.segments = s.count;
    w.segment_length = s.length;
    return w;
}

std::string check_outputs(const std::vector<Memory>& inputs, const std::vector<Memory>& outputs) {
    for (size_t i = 0; i < outputs.size(); ++i) {
        if (!outputs[i].apart_from_itself()) return "a gradient overlaps itself";
        for (const Memory& x : inputs)
            if (!apart(outputs[i], x)) return "a gradient overlaps an input";
        for (size_t j = 0; j < i; ++j)
            if (!apart(outputs[i], outputs[j])) return "gradients overlap";
    }
    return "";
}

}  // namespace

// With fewer waves than two a SIMD, as many segments as make up those, of at least two chunks of 32. (Kernels of one sequence of
// 16384, 8 heads of 128 x 128, float16: 168 us, with one wave a SIMD 200, with four 193; of 2 of 4096 with gradients, bfloat16: 305,
// 299 and 391; of 19 of 333 tokens, four heads of 24 x 48, float32, with gradients: 101, in segments of at least four chunks 139.)
Segments segments_of(const ZenoAmdLinearInputs& in) {
    const int64_t chunks = ((int64_t)in.length + kChunk - 1) / kChunk;
    const int64_t waves = (int64_t)heads_of(in) * blocks_of(in.value_dim);
    const int64_t want = std::max<int64_t>(std::min(kWaves / waves, chunks / 2), 1), each = (chunks + want - 1) / want;
    return Segments{(uint32_t)((chunks + each - 1) / each), (int)(each * kChunk)};
}

uint64_t saved_floats(const ZenoAmdLinearInputs& in) { return states_floats(in) * (in.decay_gradient ? 2 : 1); }
uint64_t workspace_floats(const ZenoAmdLinearInputs& in, bool train) {
    return even(between(in)) + states_floats(in) + (train ? 2 * share_floats(in) + parts_floats(in) : 0);
}

std::string check_sizes(const ZenoAmdLinearInputs& in, bool step) {
    if (in.dtype > T_BF16) return "dtype is none of float32, float16, bfloat16";
    if (!in.batch || !in.length || !in.key_heads || !in.value_heads) return "batch, length and head counts must be positive";
    if (in.value_heads % in.key_heads) return "value_heads is not a multiple of key_heads";
    if (!in.key_dim || in.key_dim > ZENO_AMD_LINEAR_MAX_DIM || !in.value_dim || in.value_dim > ZENO_AMD_LINEAR_MAX_DIM)
        return "key_dim and value_dim must be 1 to " + std::to_string(ZENO_AMD_LINEAR_MAX_DIM);
    // A launch takes less than 2^32 threads, and is rounded up to 32 waves. Most is what gradients take of a sequence and head, with
    // waves of 32 columns for three and of 16 for the decays': 4 + 4 + 4 + 8, and with dimensions to 64 and 32 values 1 + 2 + 2 + 4
    // (64 x 64 has waves of 64 where there are many).
    const uint64_t waves = std::max(in.key_dim, in.value_dim) > 64 ? 20 : 9;
    if (in.length > 0x7fffff00u || heads_of(in) > ((1ull << 32) / 64 - 32) / waves) return "too many sequences or tokens";
    if (step && in.length != 1) return "a step takes one token";
    return "";
}

std::string check(const ZenoAmdLinearInputs* p, bool step) {
    if (!p) return "null arguments";
    const std::string why = check_sizes(*p, step);
    if (!why.empty()) return why;
    if (!p->q || !p->k || !p->v || !p->g) return "null input";
    if (!std::isfinite(p->scale)) return "scale is not finite";
    return "";
}

namespace {
struct Places {  // what a call's arrays cover
    int64_t eb, keys[3], values[3], states, none[1] = {0}, one[1] = {1};
    explicit Places(const ZenoAmdLinearInputs& in)
        : eb(bytes_of(in.dtype)), keys{in.batch, in.length, in.key_heads}, values{in.batch, in.length, in.value_heads}, states((int64_t)heads_of(in) * state_size(in)) {}
    Memory key(const ZenoAmdLinearInputs& in, const void* p, const int64_t* stride) const { return Memory(p, stride, keys, 3, in.key_dim, eb); }
    Memory value(const ZenoAmdLinearInputs& in, const void* p, const int64_t* stride) const { return Memory(p, stride, values, 3, in.value_dim, eb); }
    Memory floats(const void* p, int64_t n) const { return Memory(p, none, one, 1, n, 4); }
    std::vector<Memory> inputs(const ZenoAmdLinearInputs& in, bool with_state) const {
        std::vector<Memory> m{key(in, in.q, in.q_stride), key(in, in.k, in.k_stride), floats(in.g, in.value_heads)};
        if (in.reset) m.push_back(Memory(in.reset, in.reset_stride, values, 2, 1, 1));
        if (with_state && in.state) m.push_back(floats(in.state, states));
        return m;
    }
};
}  // namespace

std::string check_overlap(const ZenoAmdLinearInputs& in, const void* o, const int64_t* o_stride, const float* state, bool step) {
    const Places at(in);
    const Memory out = at.value(in, o, o_stride), kept = at.floats(state, at.states), v = at.value(in, in.v, in.v_stride);
    if (!out.apart_from_itself()) return "o overlaps itself";
    if (!apart(out, kept)) return "o overlaps the state";
    // A step's o may be v itself, value by value: the wave that writes a value has read it.
    bool same = step && o == in.v;
    for (int i = 0; i < 3; ++i) same = same && (at.values[i] == 1 || o_stride[i] == in.v_stride[i]);
    if (!same && !apart(out, v)) return "o overlaps v";
    bool clear = apart(kept, v);
    for (const Memory& x : at.inputs(in, !step)) {
        if (!apart(out, x)) return "o overlaps an input";
        clear = clear && apart(kept, x);
    }
    return clear ? "" : "the state overlaps an input";
}

std::string check_gradients(const ZenoAmdLinearInputs& in, const ZenoAmdLinearGradients& grad) {
    if (!grad.d_o || !grad.d_q || !grad.d_k || !grad.d_v) return "null gradient";
    if (!in.decay_gradient != !grad.d_g) return "d_g comes with decay_gradient";
    const Places at(in);
    std::vector<Memory> reads = at.inputs(in, true), writes{at.key(in, grad.d_q, grad.d_q_stride), at.key(in, grad.d_k, grad.d_k_stride), at.value(in, grad.d_v, grad.d_v_stride)};
    reads.push_back(at.value(in, in.v, in.v_stride));
    reads.push_back(at.value(in, grad.d_o, grad.d_o_stride));
    if (grad.d_last) reads.push_back(at.floats(grad.d_last, at.states));
    if (grad.d_g) writes.push_back(at.floats(grad.d_g, in.value_heads));
    if (grad.d_state) writes.push_back(at.floats(grad.d_state, at.states));
    return check_outputs(reads, writes);
}

hipError_t forward(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* last, float* saved, float* workspace, hipStream_t stream) {
    const uint32_t share = in.value_heads / in.key_heads;
    Walk w = walk_of(in, false);
    w.a = rows_of(in.q, in.q_stride, share);
    w.b = rows_of(in.k, in.k_stride, share);
    w.c = rows_of(in.v, in.v_stride, 1);
    w.out = o;
    set_strides(w.out_stride, o_stride);
    w.first = in.state;
    w.last = last;
    w.passes = workspace;
    w.starts = saved ? saved : workspace + even(between(in));
    if (w.segments > 1) {
        const bool slope = saved && in.decay_gradient;
        if (slope) w.slopes = saved + states_floats(in);
        if (const hipError_t e = launch(in.dtype, w, slope ? STATES_SLOPE : STATES, false, stream)) return e;
    }
    return launch(in.dtype, w, OUTPUTS, false, stream);
}

hipError_t backward(const ZenoAmdLinearInputs& in, const float* saved, const ZenoAmdLinearGradients& grad, float* workspace, hipStream_t stream) {
    const uint32_t share = in.value_heads / in.key_heads;
    const Rows q = rows_of(in.q, in.q_stride, share), k = rows_of(in.k, in.k_stride, share), v = rows_of(in.v, in.v_stride, 1),
               d_o = rows_of(grad.d_o, grad.d_o_stride, 1);
    float* passes = workspace;
    float* d_starts = passes + even(between(in));
    float* parts = d_starts + states_floats(in);
    float* part_q = parts + parts_floats(in);
    float* part_k = part_q + share_floats(in);
    const int64_t part_stride[3] = {(int64_t)in.length * in.value_heads * in.key_dim, (int64_t)in.value_heads * in.key_dim, in.key_dim};
    auto key_out = [&](Walk& w, void* to, const int64_t* stride, float* part) {
        w.out = share > 1 ? part : to;
        set_strides(w.out_stride, share > 1 ? part_stride : stride);
        w.out_f32 = share > 1;
    };

    Walk wv = walk_of(in, false), wk = walk_of(in, true), wq = walk_of(in, true);
    wv.a = k, wv.b = q, wv.c = d_o;
    wk.a = v, wk.b = d_o, wk.c = q;
    wq.a = d_o, wq.b = v, wq.c = k, wq.q = q;
    wv.out = grad.d_v;
    set_strides(wv.out_stride, grad.d_v_stride);
    key_out(wk, grad.d_k, grad.d_k_stride, part_k);
    key_out(wq, grad.d_q, grad.d_q_stride, part_q);
    wv.first = wk.first = wq.d_last = grad.d_last;
    wv.last = grad.d_state;
    wv.starts = wk.starts = d_starts;
    wv.passes = passes;
    wq.first = in.state;
    wq.starts = const_cast<float*>(saved);
    wq.slopes = wq.starts + states_floats(in);
    wq.parts = grad.d_g ? reinterpret_cast<double*>(parts) : nullptr;

    hipError_t e;
    if (wv.segments > 1 && (e = launch(in.dtype, wv, STATES, true, stream))) return e;
    auto gradients = in.dtype == T_F32 ? launch_gradients<T_F32> : in.dtype == T_F16 ? launch_gradients<T_F16> : launch_gradients<T_BF16>;
    uint32_t slopes;
    if ((e = gradients(wv, wk, wq, &slopes, stream))) return e;
    if (grad.d_g) linear_decay_kernel<<<in.value_heads, 1024, 0, stream>>>(wq.parts, in.batch, in.value_heads, wq.segments * slopes, grad.d_g);
    if (share > 1) {
        auto add = in.dtype == T_F32 ? launch_share<T_F32> : in.dtype == T_F16 ? launch_share<T_F16> : launch_share<T_BF16>;
        return add(in, part_q, part_k, grad, stream);
    }
    return hipGetLastError();
}

hipError_t step(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream) {
    return in.dtype == T_F32   ? launch_step<T_F32>(in, o, o_stride, state, stream)
           : in.dtype == T_F16 ? launch_step<T_F16>(in, o, o_stride, state, stream)
                               : launch_step<T_BF16>(in, o, o_stride, state, stream);
}

}  // namespace linear
}  // namespace za
