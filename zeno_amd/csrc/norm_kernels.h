// Kernels of layer norm, forward and backward.
//
// Of a row s of n features (s = x, or x + residual rounded to its type), with d = s - mean:
//     y = u w + b,   u = (d - d') r,   d' = mean of d,   r = 1 / sqrt(mean of d^2 - d'^2 + eps)
// d' is what rounding left of the mean: without it a row far off zero is off by 2^-24 of its
// distance. With e = w dy the gradients are
//     ds = r (e - mean of e - u mean of (e u)) (+ the gradient of s itself)
//     dw = sum over rows of dy u,   db = sum over rows of dy
// The backward pass finds mean and r again from s, which it has to read anyway: two sums of values
// in registers for 8 bytes a row less each way.
//
// Bound by memory. Forward, bfloat16: 524288 rows of 64 23 us, 131072 of 512 45, 16384 of 4096 45, that is 5.7 to 6.0 TB/s;
// 65536 of 1000 in float32 106, 4.9. Narrower rows less, 524288 of 32 22 us, 3.1. Gradients, whose sums by column hold twice
// the registers and so fewer waves: 131072 of 512 86 us, 4.7 TB/s; 65536 of 1000 in float32 162, 4.8; 16384 of 4096 101, 4.0; 8192 of
// 8192 116, 3.5 (two barriers a row of 1024 threads). Those of narrow rows are bound by waits, for a row's two reads and then for sums across
// lanes that follow on one another, with no other row in flight: 524288 of 64 71 us, 2.8 TB/s, 131072 of 200 73, 2.2, 524288 of 32 71,
// 1.4; and 16384 of 2500 in float32 177, 2.8, fill 61 % of their lanes' 4096 places.
//
// A row is held in registers by LANES lanes of a wave (or by a workgroup), V vectors of eight
// elements each, so memory is read once. A lane keeps its columns from row to row: the weights stay
// in registers and the sums of dw and db too, until each workgroup writes its own and a second
// kernel adds those in order. All sums are fp32; results are bitwise reproducible.
#pragma once
#include "norm.h"
#include "rows.h"

namespace za {
namespace norm {

using namespace mma;

__device__ __forceinline__ int64_t row_at(const Args& a, uint32_t row, const int64_t* stride) {
    if (a.flat) return row * stride[2];
    const uint32_t n2 = a.in.rows[2], n1 = a.in.rows[1], r = row / n2;
    return (r / n1) * stride[0] + (r % n1) * stride[1] + (row % n2) * stride[2];
}

// Sums over a row's lanes; every lane gets them.
template <int LANES> __device__ __forceinline__ float sum_lanes(float x) {
    static_assert(LANES == 8 || LANES == 16 || LANES == 32 || LANES == 64, "part of a wave");
    if constexpr (LANES == 8) {
        x += dpp<0x141>(x);  // the mirror image within eight
        x += dpp<0x1b>(x);   // lanes 3 2 1 0 of four
        return x + dpp<0xb1>(x);  // lanes 1 0 3 2
    } else if constexpr (LANES == 16) {
        return sum16(x);
    } else if constexpr (LANES == 32) {
        x = sum16(x);
        const uint32_t b = __float_as_uint(x);
        const auto rows = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        return __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    } else {
        return sum64(x);
    }
}

// The same where a row is held by a whole workgroup: `at` is LDS of its own for each sum of a row
// and of the next row, so one barrier a sum is enough.
template <int LANES, int N> __device__ __forceinline__ void sum_row(float* x, float* at) {
    if constexpr (LANES <= 64) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = sum_lanes<LANES>(x[i]);
    } else {
        constexpr int waves = LANES / 64;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = sum64(x[i]);
            if (threadIdx.x % 64 == 0) at[i * waves + threadIdx.x / 64] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < waves; ++w) x[i] += at[i * waves + w];
        }
    }
}

// A product that is rounded before it meets anything else: both places that use e have the same one,
// so what cancels between them does (all of it, of rows of one feature).
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// u of a row in x (zeros behind its end), and r.
template <int LANES, int V, bool FULL> __device__ __forceinline__ float normalise(float* x, const int* left, float inv_n, float eps, float* at) {
    float m[1] = {0.0f}, s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) m[0] += x[i];
    sum_row<LANES, 1>(m, at);
    const float mean = m[0] * inv_n;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
        x[i] = FULL || i % 8 < left[i / 8] ? x[i] - mean : 0.0f;
        s[0] += x[i];
        s[1] += x[i] * x[i];
    }
    sum_row<LANES, 2>(s, at + LANES / 64);
    const float rest = s[0] * inv_n, r = 1.0f / sqrtf(fmaxf(s[1] * inv_n - rest * rest, 0.0f) + eps);
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) x[i] = FULL || i % 8 < left[i / 8] ? (x[i] - rest) * r : 0.0f;
    return r;
}

template <int TY, int V, bool FULL> __device__ __forceinline__ void load_row(Eight<TY>* x, const void* from, int64_t at, int e, int step, const int* left) {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v].template load<FULL>((const typename Elem<TY>::type*)from + at + e + v * step, left[v]);
}
template <int TY, int V, bool FULL> __device__ __forceinline__ void store_row(void* to, int64_t at, int e, int step, const int* left, const float* x) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        Eight<TY> y;
        y.set(x + 8 * v);
        y.template store<FULL>((typename Elem<TY>::type*)to + at + e + v * step, left[v]);
    }
}
template <int TY, int V> __device__ __forceinline__ void values(const Eight<TY>* raw, float* x) {
#pragma unroll
    for (int v = 0; v < V; ++v) raw[v].get(x + 8 * v);
}
// This lane's columns of the weight or the bias, or `missing` where there is none.
template <int WTY, int V, bool FULL> __device__ __forceinline__ void load_weight(float* w, const void* from, int e, int step, const int* left, float missing) {
    Eight<WTY> raw[V];
    if (from) {
        load_row<WTY, V, FULL>(raw, from, 0, e, step, left);
        values<WTY, V>(raw, w);
    } else {
#pragma unroll
        for (int i = 0; i < 8 * V; ++i) w[i] = missing;
    }
}

template <int LANES> constexpr int threads_of = LANES <= 64 ? 256 : LANES;
template <int LANES> constexpr int sums_of = LANES <= 64 ? 1 : 2 * 5 * (LANES / 64);  // LDS floats of five sums of two rows

template <int TY, int WTY, int LANES, int V, bool FULL>
__global__ __launch_bounds__(threads_of<LANES>) void norm_forward_kernel(const Args a) {
    constexpr int rows = threads_of<LANES> / LANES, step = 8 * LANES;
    __shared__ float sums[sums_of<LANES>];
    const int e = 8 * (threadIdx.x % LANES), n = a.in.dim;
    int left[V];
#pragma unroll
    for (int v = 0; v < V; ++v) left[v] = n - e - v * step;
    const float inv_n = 1.0f / n;
    float w[8 * V], b[8 * V];
    load_weight<WTY, V, FULL>(w, a.in.weight, e, step, left, 1.0f);
    load_weight<WTY, V, FULL>(b, a.in.bias, e, step, left, 0.0f);
    int turn = 0;
    for (uint64_t row = (uint64_t)blockIdx.x * rows + threadIdx.x / LANES; row < a.rows; row += (uint64_t)gridDim.x * rows) {
        Eight<TY> raw[V];
        float x[8 * V];
        load_row<TY, V, FULL>(raw, a.in.x, row_at(a, row, a.in.x_stride), e, step, left);
        if (a.in.residual) {
            Eight<TY> more[V];
            float z[8 * V];
            load_row<TY, V, FULL>(more, a.in.residual, row_at(a, row, a.in.residual_stride), e, step, left);
            values<TY, V>(raw, x);
            values<TY, V>(more, z);
#pragma unroll
            for (int i = 0; i < 8 * V; ++i) x[i] += z[i];
            const int64_t at = row_at(a, row, a.sum_stride);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                raw[v].set(x + 8 * v);
                raw[v].template store<FULL>((typename Elem<TY>::type*)a.sum + at + e + v * step, left[v]);
            }
        }
        values<TY, V>(raw, x);
        normalise<LANES, V, FULL>(x, left, inv_n, a.in.eps, sums + turn);
#pragma unroll
        for (int i = 0; i < 8 * V; ++i) x[i] = x[i] * w[i] + b[i];
        store_row<TY, V, FULL>(a.y, row_at(a, row, a.y_stride), e, step, left, x);
        if (LANES > 64) turn = 5 * (LANES / 64) - turn;
    }
}

template <int TY, int WTY, int LANES, int V, bool FULL>
__global__ __launch_bounds__(threads_of<LANES>) void norm_backward_kernel(const Args a) {
    constexpr int threads = threads_of<LANES>, rows = threads / LANES, step = 8 * LANES, waves = threads / 64;
    __shared__ float sums[sums_of<LANES>];
    const int e = 8 * (threadIdx.x % LANES), n = a.in.dim;
    int left[V];
#pragma unroll
    for (int v = 0; v < V; ++v) left[v] = n - e - v * step;
    const float inv_n = 1.0f / n;
    float w[8 * V], dw[8 * V], db[8 * V];
    load_weight<WTY, V, FULL>(w, a.in.weight, e, step, left, 1.0f);
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) dw[i] = db[i] = 0.0f;
    int turn = 0;
    for (uint64_t row = (uint64_t)blockIdx.x * rows + threadIdx.x / LANES; row < a.rows; row += (uint64_t)gridDim.x * rows) {
        Eight<TY> raw_x[V], raw_d[V];
        float x[8 * V], d[8 * V];
        load_row<TY, V, FULL>(raw_x, a.in.x, row_at(a, row, a.in.x_stride), e, step, left);
        load_row<TY, V, FULL>(raw_d, a.d_y, row_at(a, row, a.d_y_stride), e, step, left);
        values<TY, V>(raw_x, x);
        const float r = normalise<LANES, V, FULL>(x, left, inv_n, a.in.eps, sums + turn);
        values<TY, V>(raw_d, d);
        float m[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 8 * V; ++i) {
            db[i] += d[i];
            dw[i] += d[i] * x[i];
            d[i] = rounded_product(d[i], w[i]);
            m[0] += d[i];
            m[1] += d[i] * x[i];
        }
        if (a.d_x) {
            sum_row<LANES, 2>(m, sums + turn + 3 * (LANES / 64));
            const float along = m[0] * inv_n, across = m[1] * inv_n;
#pragma unroll
            for (int i = 0; i < 8 * V; ++i) d[i] = r * (d[i] - along - x[i] * across);
            if (a.d_sum) {
                load_row<TY, V, FULL>(raw_d, a.d_sum, row_at(a, row, a.d_sum_stride), e, step, left);
                values<TY, V>(raw_d, x);
#pragma unroll
                for (int i = 0; i < 8 * V; ++i) d[i] += x[i];
            }
            store_row<TY, V, FULL>(a.d_x, row_at(a, row, a.d_x_stride), e, step, left, d);
        }
        if (LANES > 64) turn = 5 * (LANES / 64) - turn;
    }
    if (!a.parts) return;
    float* to = a.parts + (int64_t)blockIdx.x * 2 * n;
    if constexpr (LANES > 64) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            Eight<T_F32> y;
            y.set(dw + 8 * v);
            y.template store<FULL>(to + e + v * step, left[v]);
            y.set(db + 8 * v);
            y.template store<FULL>(to + n + e + v * step, left[v]);
        }
    } else {
        // The rows of a wave, then those of the workgroup's waves.
        __shared__ float all[waves][2][8 * V][LANES];
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
        for (int i = 0; i < 8 * V; ++i) {
#pragma unroll
            for (int far = LANES; far < 64; far *= 2) {
                dw[i] += __shfl_xor(dw[i], far);
                db[i] += __shfl_xor(db[i], far);
            }
            if (lane < LANES) {
                all[wave][0][i][lane] = dw[i];
                all[wave][1][i][lane] = db[i];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * 8 * V * LANES; c += threads) {
            const int which = c / (8 * V * LANES), col = c % (8 * V * LANES), i = col % 8 + 8 * (col / step), at = col % step / 8;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < waves; ++k) sum += all[k][which][i][at];
            if (FULL || col < n) to[which * n + col] = sum;
        }
    }
}

// Adds the workgroups' sums, 32 columns a workgroup: 32 threads a column, each every 32nd
// part in order, then those in order.
template <int WTY> __global__ __launch_bounds__(1024) void norm_weights_kernel(const float* parts, uint32_t blocks, int n, void* d_weight, void* d_bias) {
    __shared__ float all[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x % 32, slice = threadIdx.x / 32;
    void* to = blockIdx.y ? d_bias : d_weight;
    if (!to) return;
    float sum = 0.0f;
    if (col < n) {
        const float* from = parts + (int64_t)blockIdx.y * n + col;
#pragma unroll 4
        for (uint32_t b = slice; b < blocks; b += 32) sum += from[(int64_t)b * 2 * n];
    }
    all[slice][threadIdx.x % 32] = sum;
    __syncthreads();
    if (slice || col >= n) return;
#pragma unroll
    for (int s = 1; s < 32; ++s) sum += all[s][threadIdx.x];
    ((typename Elem<WTY>::type*)to)[col] = Elem<WTY>::put(sum);
}

// ---- launches ------------------------------------------------------------------------------
template <int TY, int WTY, int LANES, int V> void run_forward(const Args& a, const Shape& s, hipStream_t stream) {
    if (a.in.dim == 8 * LANES * V) norm_forward_kernel<TY, WTY, LANES, V, true><<<s.blocks, threads_of<LANES>, 0, stream>>>(a);
    else norm_forward_kernel<TY, WTY, LANES, V, false><<<s.blocks, threads_of<LANES>, 0, stream>>>(a);
}
template <int TY, int WTY, int LANES, int V> void run_backward(const Args& a, const Shape& s, hipStream_t stream) {
    if (a.in.dim == 8 * LANES * V) norm_backward_kernel<TY, WTY, LANES, V, true><<<s.blocks, threads_of<LANES>, 0, stream>>>(a);
    else norm_backward_kernel<TY, WTY, LANES, V, false><<<s.blocks, threads_of<LANES>, 0, stream>>>(a);
}
template <int TY, int WTY> void pick_forward(const Args& a, const Shape& s, hipStream_t stream) {
    switch (s.lanes * s.vectors) {
        case 8: return run_forward<TY, WTY, 8, 1>(a, s, stream);
        case 16: return run_forward<TY, WTY, 16, 1>(a, s, stream);
        case 32: return run_forward<TY, WTY, 32, 1>(a, s, stream);
        case 64: return run_forward<TY, WTY, 64, 1>(a, s, stream);
        case 128: return run_forward<TY, WTY, 64, 2>(a, s, stream);
        case 256: return run_forward<TY, WTY, 256, 1>(a, s, stream);
        case 512: return run_forward<TY, WTY, 256, 2>(a, s, stream);
        case 1024: return run_forward<TY, WTY, 1024, 1>(a, s, stream);
        default: return run_forward<TY, WTY, 1024, 2>(a, s, stream);
    }
}
template <int TY, int WTY> void pick_backward(const Args& a, const Shape& s, hipStream_t stream) {
    switch (s.lanes * s.vectors) {
        case 8: return run_backward<TY, WTY, 8, 1>(a, s, stream);
        case 16: return run_backward<TY, WTY, 16, 1>(a, s, stream);
        case 32: return run_backward<TY, WTY, 32, 1>(a, s, stream);
        case 64: return run_backward<TY, WTY, 64, 1>(a, s, stream);
        case 128: return run_backward<TY, WTY, 64, 2>(a, s, stream);
        case 256: return run_backward<TY, WTY, 256, 1>(a, s, stream);
        case 512: return run_backward<TY, WTY, 256, 2>(a, s, stream);
        case 1024: return run_backward<TY, WTY, 1024, 1>(a, s, stream);
        default: return run_backward<TY, WTY, 1024, 2>(a, s, stream);
    }
}

template <int TY> hipError_t launch_forward(const Args& a, const Shape& s, hipStream_t stream) {
    a.in.weight_dtype == (uint32_t)TY ? pick_forward<TY, TY>(a, s, stream) : pick_forward<TY, T_F32>(a, s, stream);
    return hipGetLastError();
}
template <int WTY> void add_parts(const Args& a, const ZenoAmdNormGradients& grad, const Shape& s, hipStream_t stream) {
    norm_weights_kernel<WTY><<<dim3((a.in.dim + 31) / 32, 2), 1024, 0, stream>>>(a.parts, s.blocks, a.in.dim, grad.d_weight, grad.d_bias);
}
template <int TY> hipError_t launch_backward(const Args& a, const ZenoAmdNormGradients& grad, const Shape& s, hipStream_t stream) {
    const bool same = a.in.weight_dtype == (uint32_t)TY;
    same ? pick_backward<TY, TY>(a, s, stream) : pick_backward<TY, T_F32>(a, s, stream);
    if (a.parts) same ? add_parts<TY>(a, grad, s, stream) : add_parts<T_F32>(a, grad, s, stream);
    return hipGetLastError();
}

}  // namespace norm
}  // namespace za
