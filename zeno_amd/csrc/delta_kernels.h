// Kernels of the gated delta rule over whole sequences, and the single-token step.
//
// A chunk is C = 16 TILES tokens. With S the state before it (key_dim x value_dim), G_i the sum
// of g up to token i, D_ij = exp(G_i - G_j), gam_i = exp(G_i), B = diag(beta), the C dependent
// updates of the definition are
//     Z = strict_lower(D * K K^T);   X = V - gam K S;   (I + Z B) E = X;   U = B E
//     O = scale (gam Q S + lower(D * Q K^T) U);          S' = gam_C S + K^T (D_C U)
// Column c of E, U, O and S' depends on column c of V and S alone. A wave therefore owns 16
// value columns and keeps their state in registers as result tiles; every right operand is its
// own registers' content (mma.h), and the waves of a workgroup share only the left operands, in
// LDS: K, Q, K^T, the decayed Q K^T, Z below the diagonal tile, and the inverses of the 16x16
// diagonal tiles of I + Z B. Those come from forward substitution, 16 columns in 16 lanes: the
// cheaper product of powers (I - N)(I + N^2)... loses all digits where keys repeat, as they do
// for an environment that stands still.
//
// A chunk ends at a token of the grid of C and before every reset, so nothing is masked inside
// it and no value from before a reset is ever multiplied by a zero. Partial chunks are filled
// with zero keys, zero beta and zero g, which change nothing.
#pragma once
#include <type_traits>

#include "delta.h"
#include "mma.h"

namespace za {
namespace delta {

using namespace mma;

constexpr float kNormEps = 1e-6f;
constexpr float kClears = -104.0f;  // exp of less is 0 in fp32: a reset

// Operands along a chunk's tokens: 32 of them in `slot` order, or 16 in their own.
template <int TILES> struct Tok;
template <> struct Tok<2> {
    template <int P> using Op = Frag<P>;
    template <int P> static __device__ __forceinline__ Frag<P> make(const f4* x) { return split<P>(x[0], x[1]); }
    template <int P> static __device__ __forceinline__ Frag<P> at(const uint16_t* row, int g, int part) { return frag_at<P>(row + 8 * g, part); }
    static __device__ __forceinline__ int slot_of(int x) { return slot(x); }
    static __device__ __forceinline__ int tile_at(int g, int tile) { return 8 * g + 4 * tile; }  // one tile's four values
    static constexpr int stride = 40;
};
template <> struct Tok<1> {
    template <int P> using Op = Half<P>;
    template <int P> static __device__ __forceinline__ Half<P> make(const f4* x) { return split<P>(x[0]); }
    template <int P> static __device__ __forceinline__ Half<P> at(const uint16_t* row, int g, int part) { return half_at<P>(row + 4 * g, part); }
    static __device__ __forceinline__ int slot_of(int x) { return x; }
    static __device__ __forceinline__ int tile_at(int g, int) { return 4 * g; }
    static constexpr int stride = 24;
};

constexpr int kInvStride = 20;  // of 16x16 tiles in LDS, bf16 or float

template <int TY, int DK, int NW, int TILES> struct Geo {
    static constexpr int NP = Elem<TY>::parts;        // parts of an input value
    static constexpr int C = 16 * TILES;
    static constexpr int DV = 16 * NW;
    static constexpr int KS = DK + 8;                 // row strides, a multiple of 16 bytes off the banks' period
    static constexpr int TS = Tok<TILES>::stride;
    static constexpr int VS = DV + 8;
    static constexpr int threads = 64 * NW;
};

template <int TILES> struct Scalars {  // one float a token
    static constexpr int C = 16 * TILES;
    alignas(16) float hi[C], lo[C];    // G in two floats: differences keep their digits after a strong decay
    alignas(16) float beta[C], rk[C], rq[C], gam[C], end[C];
};

__device__ __forceinline__ f4 row4(const float* s, int tile, int g) { return *reinterpret_cast<const f4*>(s + 16 * tile + 4 * g); }

// One thread's eight values of a chunk's rows of q or k (or of rows as wide as DK).
template <int TY, int DK, int NW, int TILES> struct Rows {
    typedef Geo<TY, DK, NW, TILES> G;
    static constexpr int per = DK / 8;
    static_assert(G::C * per <= G::threads, "one piece a thread");
    Raw<TY> raw;
    static __device__ __forceinline__ bool mine() { return G::C * per == G::threads || threadIdx.x < G::C * per; }
    // The first `rows` rows (others repeat the last one). FULL: the head has DK dimensions, aligned.
    template <bool FULL> __device__ __forceinline__ void fetch(const typename Elem<TY>::type* base, int64_t stride, int rows, int dim, bool vec) {
        const int row = min((int)threadIdx.x / per, rows - 1), e = 8 * (threadIdx.x % per);
        if (mine()) raw.template load<FULL>(base + row * stride + e, dim - e, vec);
    }
    // The first `len` rows and zeros into LDS: row-major in `slot` order along the head's
    // dimension, and (cols not null) transposed. norm: 1 / sqrt(sum of squares + eps) of each row, or 1.
    __device__ __forceinline__ void store(int len, bool normalize, uint16_t* rows, uint16_t* cols, float* norm) {
        const int row = threadIdx.x / per, e = 8 * (threadIdx.x % per);
        if (!mine()) return;
        raw.keep(row < len);
        float ss = 0.0f;
        if (normalize) {
            float x[8];
            raw.get(x);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
            if (per > 8) ss += dpp<0x128>(ss);  // rotation by 8 within 16 lanes: sums of 8 in either half
            ss += dpp<0x141>(ss);               // the half's mirror image, and so on
            ss += dpp<0x1b>(ss);                // lanes 3 2 1 0 of four
            ss += dpp<0xb1>(ss);                // lanes 1 0 3 2
        }
        if (e == 0) norm[row] = normalize ? __builtin_amdgcn_rsqf(ss + kNormEps) : 1.0f;
        uint32_t w[4][G::NP];
        raw.parts(w);
        const int ts = Tok<TILES>::slot_of(row);
#pragma unroll
        for (int p = 0; p < G::NP; ++p) {
            uint16_t* to = rows + (p * G::C + row) * G::KS;
            *reinterpret_cast<u2*>(to + slot(e)) = u2{w[0][p], w[1][p]};
            *reinterpret_cast<u2*>(to + slot(e + 4)) = u2{w[2][p], w[3][p]};
            if (cols) {
                uint16_t* tc = cols + (p * DK + e) * G::TS + ts;
#pragma unroll
                for (int j = 0; j < 8; ++j) tc[j * G::TS] = (uint16_t)(w[j >> 1][p] >> (16 * (j & 1)));
            }
        }
    }
};

// g and beta of a chunk (one lane a token, wave 0): sums in 64 bits.
template <int TILES>
__device__ __forceinline__ void load_scalars(float g, float beta, int lane, bool first, Scalars<TILES>& s) {
    constexpr int C = 16 * TILES;
    double sum = (first && lane == 0) ? 0.0 : (double)g;
#pragma unroll
    for (int d = 1; d < C; d <<= 1) {
        const double up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    const double all = __shfl(sum, C - 1);
    if (lane < C) {
        const float hi = (float)sum;
        s.hi[lane] = hi;
        s.lo[lane] = (float)(sum - (double)hi);
        s.beta[lane] = beta;
        s.gam[lane] = __expf(hi);
        s.end[lane] = __expf((float)(all - sum));
    }
}

// A 16x16 tile of rows x rows products (K K^T or Q K^T), times the decay and the norms.
template <int TY, int DK, int NW, int TILES>
__device__ __forceinline__ f4 decayed(const uint16_t* rows_i, const uint16_t* rows_j, const float* ri, int ti, int tj, int n, int g,
                                      const Scalars<TILES>& s) {
    typedef Geo<TY, DK, NW, TILES> G;
    f4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < DK / 32; ++ks)
        acc = mul<2>(frag_at<G::NP>(rows_i + (16 * ti + n) * G::KS + 32 * ks + 8 * g, G::C * G::KS),
                     frag_at<G::NP>(rows_j + (16 * tj + n) * G::KS + 32 * ks + 8 * g, G::C * G::KS), acc);
    const int j = 16 * tj + n;
    const float hj = s.hi[j], lj = s.lo[j], rj = s.rk[j];
    const f4 hi = row4(s.hi, ti, g), lo = row4(s.lo, ti, g), nr = row4(ri, ti, g);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] *= __expf((hi[r] - hj) + (lo[r] - lj)) * (nr[r] * rj);
    return acc;
}

// Row r (of 16) of the inverse of I + N, N strictly lower triangular and row-major: of t (I + N) =
// e_r, from the last column to the first, each value taken out of all sums that still need it.
__device__ __forceinline__ void inverse_row(const float* N, int r, float* t) {
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = j == r ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 15; j > 0; --j) {
#pragma unroll
        for (int c = 0; c < j; c += 4) {
            const f4 w = *reinterpret_cast<const f4*>(N + j * kInvStride + c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < j) t[c + i] -= t[j] * w[i];
        }
    }
}
// Column c of the same, from N transposed.
__device__ __forceinline__ void inverse_column(const float* NT, int c, float* t) {
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = j == c ? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < 15; ++j) {
#pragma unroll
        for (int b = (j + 1) & ~3; b < 16; b += 4) {
            const f4 w = *reinterpret_cast<const f4*>(NT + j * kInvStride + b);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (b + i > j) t[b + i] -= t[j] * w[i];
        }
    }
}
__device__ __forceinline__ void put_row(uint16_t* to, const float* t) {  // 16 values in three parts
#pragma unroll
    for (int b = 0; b < 16; b += 4) put4<3>(to + b, 16 * kInvStride, f4{t[b], t[b + 1], t[b + 2], t[b + 3]});
}

template <int P> __device__ __forceinline__ void put_parts(uint16_t* to, int part, float x) {
    uint32_t w[P];
    split_pair<P>(x, 0.0f, w);
#pragma unroll
    for (int p = 0; p < P; ++p) to[p * part] = (uint16_t)w[p];
}


// The matrices inside a chunk that both directions use.
template <int TILES> struct Inner {
    static constexpr int C = 16 * TILES, TS = Tok<TILES>::stride;
    alignas(16) uint16_t P[3 * C * TS];                     // lower(D * Q K^T) scale
    alignas(16) uint16_t off[3 * 16 * kInvStride];          // Z, lower left tile
    alignas(16) uint16_t inv[TILES * 3 * 16 * kInvStride];  // of I + Z B, diagonal tiles
    alignas(16) float diag[TILES * 16 * kInvStride];        // Z B, diagonal tiles
};
template <int TILES> struct InnerBack : Inner<TILES> {
    typedef Inner<TILES> I;
    alignas(16) uint16_t PT[3 * I::C * I::TS];                // transposed
    alignas(16) uint16_t offT[3 * 16 * kInvStride];
    alignas(16) uint16_t invT[TILES * 3 * 16 * kInvStride];   // of I + B Z, transposed
    alignas(16) float diag2[TILES * 16 * kInvStride];         // B Z, diagonal tiles
};

// A result tile (rows from i0 = 16 ti + 4 g, this lane's column j) into a matrix along tokens,
// [row][slot of column], and its transpose.
template <int P, int TILES> __device__ __forceinline__ void put_rows(uint16_t* m, f4 v, int ti, int tj, int lane) {
    typedef Tok<TILES> K;
    const int n = lane & 15, g = lane >> 4;
    put4<P>(m + (16 * ti + 4 * g + (n & 3)) * K::stride + K::slot_of(16 * tj + (n & 12)), 16 * TILES * K::stride, turn(v, lane));
}
template <int P, int TILES> __device__ __forceinline__ void put_cols(uint16_t* m, f4 v, int ti, int tj, int lane) {
    typedef Tok<TILES> K;
    const int n = lane & 15, g = lane >> 4;
    put4<P>(m + (16 * tj + n) * K::stride + K::slot_of(16 * ti + 4 * g), 16 * TILES * K::stride, v);
}

// Fills Inner (and InnerBack) from the rows in LDS, the tiles spread over the waves; a wave that
// makes a diagonal tile of Z inverts it. USED tiles of 16 tokens are in use. The caller
// synchronises before and after.
enum Want { W_P = 1, W_PT = 2, W_INV = 4, W_INVT = 8 };  // the latter two with Z below the diagonal
template <int TY, int DK, int NW, int TILES, int USED, int WANT, class M>
__device__ __forceinline__ void fill_inner(const uint16_t* K, const uint16_t* Q, const Scalars<TILES>& s, float scale, M& m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    // Jobs by wave of four (of two tiles): Z00 and its inverse, Z11 and its inverse, Z10 and P00,
    // P10 and P11; eight waves take one each.
#pragma unroll
    for (int job = 0; job < 3 * TILES; ++job) {
        constexpr int order[6][3] = {{0, 0, 0}, {0, 1, 1}, {0, 1, 0}, {1, 1, 0}, {1, 0, 0}, {1, 1, 1}};  // product, tile
        const int what = TILES == 2 ? order[job][0] : job, ti = TILES == 2 ? order[job][1] : 0, tj = TILES == 2 ? order[job][2] : 0;
        const int by = NW >= 6 ? job : job < 4 ? job : job - 2;
        if ((TILES == 1 && job > 1) || ti >= USED || by != wave || (what == 1 && !(WANT & (W_P | W_PT)))) continue;
        const int j = 16 * tj + n;
        if (what == 0) {
            const f4 z = decayed<TY, DK, NW, TILES>(K, K, s.rk, ti, tj, n, g, s);
            if (ti == tj) {
                const float bj = s.beta[j];
                const f4 bi = row4(s.beta, ti, g);
                f4 zb, bz;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = n < 4 * g + r ? z[r] : 0.0f;
                    zb[r] = v * bj;
                    bz[r] = v * bi[r];
                }
                if constexpr (WANT & W_INV) *reinterpret_cast<f4*>(m.diag + (ti * 16 + 4 * g + (n & 3)) * kInvStride + (n & 12)) = turn(zb, lane);
                if constexpr (WANT & W_INVT) *reinterpret_cast<f4*>(m.diag2 + (ti * 16 + n) * kInvStride + 4 * g) = bz;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                float t[16];
                if constexpr (WANT & W_INV)
                    if (lane < 16) {
                        inverse_row(m.diag + ti * 16 * kInvStride, n, t);
                        put_row(m.inv + (ti * 3 * 16 + n) * kInvStride, t);
                    }
                if constexpr (WANT & W_INVT)
                    if (lane >= 48) {
                        inverse_column(m.diag2 + ti * 16 * kInvStride, n, t);
                        put_row(m.invT + (ti * 3 * 16 + n) * kInvStride, t);
                    }
            } else {
                if constexpr (WANT & W_INV) put4<3>(m.off + (4 * g + (n & 3)) * kInvStride + (n & 12), 16 * kInvStride, turn(z, lane));
                if constexpr (WANT & W_INVT) put4<3>(m.offT + n * kInvStride + 4 * g, 16 * kInvStride, z);
            }
        } else {
            f4 p = decayed<TY, DK, NW, TILES>(Q, K, s.rq, ti, tj, n, g, s);
#pragma unroll
            for (int r = 0; r < 4; ++r) p[r] = j <= 16 * ti + 4 * g + r ? p[r] * scale : 0.0f;
            if constexpr (WANT & W_P) put_rows<3, TILES>(m.P, p, ti, tj, lane);
            if constexpr (WANT & W_PT) put_cols<3, TILES>(m.PT, p, ti, tj, lane);
        }
    }
}

// E (and U = beta E, and its parts) from X, in place in registers.
template <int TILES, int USED, class M>
__device__ __forceinline__ void solve(const M& m, const Scalars<TILES>& s, int n, int g, f4* x, f4* u, Half<3>* up) {
    constexpr int tile = 16 * kInvStride;
    const f4 zero = {0, 0, 0, 0};
    const uint16_t* row = m.inv + n * kInvStride + 4 * g;
    x[0] = mul<2>(half_at<3>(row, tile), split<3>(x[0]), zero);
    u[0] = x[0] * row4(s.beta, 0, g);
    up[0] = split<3>(u[0]);
    if constexpr (USED == 2) {
        const f4 d = mul<2>(half_at<3>(m.off + n * kInvStride + 4 * g, tile), up[0], zero);
        x[1] = mul<2>(half_at<3>(row + 3 * tile, tile), split<3>(x[1] - d), zero);
        u[1] = x[1] * row4(s.beta, 1, g);
        up[1] = split<3>(u[1]);
    }
}

// acc += lower(D Q K^T) scale U
template <int TILES, int USED, class M>
__device__ __forceinline__ void add_PU(const M& m, int n, int g, const Half<3>* up, f4* acc) {
    constexpr int TS = Tok<TILES>::stride, part = 16 * TILES * TS;
    acc[0] = mul<2>(half_at<3>(m.P + n * TS + Tok<TILES>::tile_at(g, 0), part), up[0], acc[0]);
    if constexpr (USED == 2) acc[1] = mul<2>(frag_at<3>(m.P + (16 + n) * TS + 8 * g, part), join<3>(up[0], up[1]), acc[1]);
}

// This wave's columns of a state [rows, cols] in memory (leading dimension ld), as result tiles:
// a lane reads four columns of a row, and four lanes exchange them.
template <int DK, bool FULL> __device__ __forceinline__ void load_state(const float* at, int rows, int cols, int ld, bool vec, int col0, int lane, f4* S) {
    const int row = 4 * (lane >> 4) + (lane & 3), col = col0 + (lane & 12);
    if (at) {
        const float* from = at + row * ld + col;
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) S[i] = load4<T_F32, FULL>(from + 16 * i * ld, 16 * i + row < rows ? cols - col : 0, vec);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) S[i] = turn(S[i], lane);
    } else {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) S[i] = f4{0, 0, 0, 0};
    }
}
template <int DK, bool FULL> __device__ __forceinline__ void store_state(float* at, int rows, int cols, int ld, bool vec, int col0, int lane, const f4* S) {
    const int row = 4 * (lane >> 4) + (lane & 3), col = col0 + (lane & 12);
    float* to = at + row * ld + col;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) store4<T_F32, FULL>(to + 16 * i * ld, 16 * i + row < rows ? cols - col : 0, vec, turn(S[i], lane));
}

// ---- forward -------------------------------------------------------------------------------
template <int TY, int DK, int NW, int TILES> struct ForwardLds {
    typedef Geo<TY, DK, NW, TILES> G;
    alignas(16) uint16_t K[G::NP * G::C * G::KS], Q[G::NP * G::C * G::KS], KT[G::NP * DK * G::TS];
    Inner<TILES> m;
    Scalars<TILES> s;
};

// FULL: heads of exactly DK and 16 NW dimensions, aligned, need no masks (a fifth of the instructions).
// STATES: no outputs; of each segment but the last, N, the state after it from zeros (from the
// caller's state in the first segment), and M, the same without values from the unit matrix: with
// S the state before the segment, the state after it is M S + N.
template <int TY, int DK, int NW, int TILES, bool FULL, bool STATES>
__global__ __launch_bounds__(64 * NW) void delta_forward_kernel(const Args a) {
    typedef Geo<TY, DK, NW, TILES> G;
    typedef typename Elem<TY>::type E;
    __shared__ ForwardLds<TY, DK, NW, TILES> lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t b = blockIdx.x / in.value_heads, h = blockIdx.x % in.value_heads, hk = h / a.share;
    const int dk = in.key_dim, dv = in.value_dim, segment = blockIdx.y;
    const int begin = segment * a.segment_length, T = min((int)in.length, begin + a.segment_length);  // this segment's tokens
    const bool unit = STATES && blockIdx.z;
    if (unit && segment == 0) return;
    const int col0 = wave * 16, row0 = 4 * g + (n & 3), col = col0 + (n & 12);  // memory: four columns of a row
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2];
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2];
    const E* v = (const E*)in.v + b * in.v_stride[0] + h * in.v_stride[2] + col;
    const float* gp = in.g + b * in.g_stride[0] + h * in.g_stride[2];
    const float* bp = in.beta + b * in.beta_stride[0] + h * in.beta_stride[2];
    const uint8_t* rp = in.reset ? in.reset + b * in.reset_stride[0] : nullptr;
    E* o = (E*)a.o + b * a.o_stride[0] + h * a.o_stride[2] + col;
    const int64_t bh = b * in.value_heads + h;

    f4 S[DK / 16];
    if (segment == 0) {
        load_state<DK, FULL>(in.state ? in.state + bh * dk * dv : nullptr, dk, dv, dv, a.s_vec, col0, lane, S);
    } else if (STATES) {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = unit && 16 * i + 4 * g + r == col0 + n ? 1.0f : 0.0f;
    } else {
        load_state<DK, true>(a.starts + (bh * (a.segments - 1) + segment - 1) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, S);
    }

    // What a chunk reads from memory, fetched one chunk ahead: up to the grid, as where the chunk
    // ends is known only when its resets are here.
    Rows<TY, DK, NW, TILES> kr, qr;
    f4 vr[TILES];
    float gv, bv;
    bool cut, any_cut = false;
    auto fetch = [&](int t) {
        const int rows = min(T, (t / G::C + 1) * G::C) - t;
        const int tok = t + min(lane, rows - 1);
        gv = gp[tok * in.g_stride[1]];
        bv = bp[tok * in.beta_stride[1]];
        cut = lane < rows && ((rp && rp[tok * in.reset_stride[1]]) || gv < kClears);
        kr.template fetch<FULL>(k + t * in.k_stride[1], in.k_stride[1], rows, dk, a.k_vec);
        if (!STATES) qr.template fetch<FULL>(q + t * in.q_stride[1], in.q_stride[1], rows, dk, a.q_vec);
#pragma unroll
        for (int i = 0; i < TILES; ++i)
            vr[i] = unit ? f4{0, 0, 0, 0} : load4<TY, FULL>(v + (t + min(16 * i + row0, rows - 1)) * in.v_stride[1], dv - col, a.v_vec);
    };
    // The chunk of tokens t to t + len, in USED tiles (len <= 16 needs but one of two). No branch is
    // inside: where one lies between a matrix instruction and the use of its result, the compiler
    // has been seen to leave out the wait.
    auto chunk = [&](auto used, int t, int len, f4* x) {
        constexpr int USED = decltype(used)::value;
        fill_inner<TY, DK, NW, TILES, USED, STATES ? W_INV : W_INV | W_P>(lds.K, lds.Q, lds.s, in.scale, lds.m);
        f4 ks[USED], o4[USED], u[USED];
        Half<3> up[USED];
#pragma unroll
        for (int i = 0; i < USED; ++i) ks[i] = o4[i] = f4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) {
            const Frag<3> sb = split<3>(S[2 * c], S[2 * c + 1]);
#pragma unroll
            for (int i = 0; i < USED; ++i) {
                const int at = (16 * i + n) * G::KS + 32 * c + 8 * g;
                ks[i] = mul<2>(frag_at<G::NP>(lds.K + at, G::C * G::KS), sb, ks[i]);
                if constexpr (!STATES) o4[i] = mul<2>(frag_at<G::NP>(lds.Q + at, G::C * G::KS), sb, o4[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < USED; ++i) {
            const f4 gam = row4(lds.s.gam, i, g);
            x[i] -= gam * row4(lds.s.rk, i, g) * ks[i];
            o4[i] *= gam * row4(lds.s.rq, i, g) * in.scale;
        }
        __syncthreads();
        solve<TILES, USED>(lds.m, lds.s, n, g, x, u, up);
        if constexpr (!STATES) {
            add_PU<TILES, USED>(lds.m, n, g, up, o4);
#pragma unroll
            for (int i = 0; i < USED; ++i) {
                const f4 y = turn(o4[i], lane);
                if (16 * i + row0 < len) store4<TY, FULL>(o + (t + 16 * i + row0) * a.o_stride[1], dv - col, a.o_vec, y);
            }
        }
#pragma unroll
        for (int i = 0; i < USED; ++i) u[i] *= row4(lds.s.end, i, g) * row4(lds.s.rk, i, g);
        const float all = lds.s.gam[G::C - 1];
        if constexpr (USED == TILES) {
            const auto ub = Tok<TILES>::template make<3>(u);
#pragma unroll
            for (int i = 0; i < DK / 16; ++i)
                S[i] = mul<2>(Tok<TILES>::template at<G::NP>(lds.KT + (16 * i + n) * G::TS, g, DK * G::TS), ub, S[i] * all);
        } else {
            const Half<3> ub = split<3>(u[0]);
#pragma unroll
            for (int i = 0; i < DK / 16; ++i)
                S[i] = mul<2>(half_at<G::NP>(lds.KT + (16 * i + n) * G::TS + Tok<TILES>::tile_at(g, 0), DK * G::TS), ub, S[i] * all);
        }
    };
    fetch(begin);
    for (int t = begin; t < T;) {
        const int lim = min(T, (t / G::C + 1) * G::C);
        const uint64_t cuts = __ballot(cut);
        const bool first = cuts & 1;
        const uint64_t later = cuts & ~1ull;
        const int len = later ? __ffsll((unsigned long long)later) - 1 : lim - t;
        f4 x[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) x[i] = turn(16 * i + row0 < len ? vr[i] : f4{0, 0, 0, 0}, lane);
        if (!STATES && a.saved && t && t % G::C == 0)
            store_state<DK, true>(a.saved + (bh * (a.chunks - 1) + t / G::C - 1) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, S);
        if (first) {
            any_cut = true;
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) S[i] = f4{0, 0, 0, 0};
        }

        __syncthreads();  // the last chunk's operands are read
        if (wave == 0) load_scalars<TILES>(lane < len ? gv : 0.0f, lane < len ? bv : 0.0f, lane, first, lds.s);
        kr.store(len, in.normalize, lds.K, lds.KT, lds.s.rk);
        if (!STATES) qr.store(len, in.normalize, lds.Q, nullptr, lds.s.rq);
        if (t + len < T) fetch(t + len);
        __syncthreads();
        if (TILES == 2 && len <= 16) chunk(std::integral_constant<int, 1>{}, t, len, x);
        else chunk(std::integral_constant<int, TILES>{}, t, len, x);
        t += len;
    }
    if constexpr (STATES) {
        if (unit) {
            float* to = a.jumps + (bh * (a.segments - 1) + segment) * (DK * DK + 4);
            if (col0 < DK) store_state<DK, true>(to, DK, DK, DK, true, col0, lane, S);
            if (threadIdx.x == 0) to[DK * DK] = any_cut ? 0.0f : 1.0f;  // whether anything passes the segment
        } else {
            store_state<DK, true>(a.starts + (bh * (a.segments - 1) + segment) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, S);
        }
    } else if (segment == (int)a.segments - 1)
        store_state<DK, FULL>(a.last + bh * dk * dv, dk, dv, dv, a.last_vec, col0, lane, S);
}

// ---- joining segments ------------------------------------------------------------------------
// The states between the segments from M and N of each: S_{p+1} = M_p S_p + N_p, in place of N.
// BACK: the same for the state's gradient from the last segment to the first, with M transposed.
// A workgroup joins one head; its waves hold 16 columns each, M goes through LDS in three parts.
template <int DK, int NW, bool BACK> __global__ __launch_bounds__(64 * NW) void delta_join_kernel(float* states, const float* jumps, int segments) {
    constexpr int KS = DK + 8, DV = 16 * NW, pieces = DK * DK / 8 / (64 * NW);
    __shared__ __attribute__((aligned(16))) uint16_t lds[3 * DK * KS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4, col0 = 16 * wave;
    const int64_t bh = blockIdx.x, between = segments - 1;
    // Between segments p and p + 1 lies state p; jump p leads from state p - 1 to state p.
    const int first = BACK ? segments - 2 : 0, last = BACK ? 0 : segments - 2, step = BACK ? -1 : 1;
    float* at = states + bh * between * (DK * DV);
    const float* jump = jumps + bh * between * (DK * DK + 4);
    Raw<T_F32> raw[pieces];
    auto fetch = [&](int p) {
#pragma unroll
        for (int i = 0; i < pieces; ++i) raw[i].template load<true>(jump + (int64_t)p * (DK * DK + 4) + 8 * (threadIdx.x + 64 * NW * i), 8, true);
    };
    f4 S[DK / 16];
    load_state<DK, true>(at + (int64_t)first * (DK * DV), DK, DV, DV, true, col0, lane, S);
    for (int p = first; p != last; p += step) {
        // Forward: from state p to p + 1 by jump p + 1. Back: from state p to p - 1 by jump p.
        const int j = BACK ? p : p + 1, to = p + step;
        if (p == first) fetch(j);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            const int piece = threadIdx.x + 64 * NW * i, row = piece / (DK / 8), e = 8 * (piece % (DK / 8));
            uint32_t w[4][3];
            raw[i].parts(w);
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                if (BACK) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) lds[(q * DK + e + x) * KS + slot(row)] = (uint16_t)(w[x >> 1][q] >> (16 * (x & 1)));
                } else {
                    uint16_t* y = lds + (q * DK + row) * KS;
                    *reinterpret_cast<u2*>(y + slot(e)) = u2{w[0][q], w[1][q]};
                    *reinterpret_cast<u2*>(y + slot(e + 4)) = u2{w[2][q], w[3][q]};
                }
            }
        }
        if (to != last) fetch(j + step);
        f4 N[DK / 16];
        load_state<DK, true>(at + (int64_t)to * (DK * DV), DK, DV, DV, true, col0, lane, N);
        __syncthreads();
        if (jump[(int64_t)j * (DK * DK + 4) + DK * DK] == 0.0f)  // a reset: NaN times a zero matrix would pass it
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) S[i] = f4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) {
            const Frag<3> sb = split<3>(S[2 * c], S[2 * c + 1]);
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) N[i] = mul<2>(frag_at<3>(lds + (16 * i + n) * KS + 32 * c + 8 * g, DK * KS), sb, N[i]);
        }
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) S[i] = N[i];
        store_state<DK, true>(at + (int64_t)to * (DK * DV), DK, DV, DV, true, col0, lane, S);
    }
}

// ---- backward ------------------------------------------------------------------------------
// Chunks from the last to the first, dS' the gradient of the state after the chunk. With the
// matrices and solutions of the forward pass recomputed from the state before the chunk:
//     dU = P^T dO + D_C K dS';  (I + Z^T B) dR = dU;  dX = B dR;  dV = dX;  dbeta_i = dR_i . E_i
//     dS = gam_C dS' + scale (gam Q)^T dO - K^T (gam dX)
//     W = lower(D * dO U^T) scale;  Y = -strict_lower(D * dX U^T)
//     dQ = scale gam dO S^T + W K;  dK = D_C U dS'^T - gam dX S^T + W^T Q + (Y + Y^T) K
// O and V enter the chunk's result only through products with decays, so each decay's gradient
// follows from the others: with dG_i the gradient of G_i,
//     dG_i = dO_i . O_i - dV_i . V_i,  dG_C += <dS', S'>,  dg_t = sum over i >= t of dG_i
// (every other term cancels against its partner). The first line is column-local like the
// forward pass (phase A); dQ and dK sum over the value columns, whose operands (U, dX, dO, dS'
// transposed) go through LDS (phase B). Phase A feeds fp32 results and takes three parts; phase
// B feeds results of the element type alone and takes `NO` parts: two for 16-bit types, 2^-17 of
// each operand against the 2^-9 or 2^-12 of the results' own rounding.
template <int TY, int DK, int NW, int TILES> struct BackwardLds {
    typedef Geo<TY, DK, NW, TILES> G;
    static constexpr int NO = TY == T_F32 ? 3 : 2;
    static constexpr int slab = DK < 64 ? DK : 64;  // rows of dS' that are in LDS at once
    static constexpr int SS = G::DV + 4, OS = DK + 4;
    alignas(16) uint16_t K[G::NP * G::C * G::KS], Q[G::NP * G::C * G::KS], KT[G::NP * DK * G::TS], QT[G::NP * DK * G::TS];
    alignas(16) uint16_t DO[G::NP * G::C * G::VS];
    union {
        InnerBack<TILES> m;  // phase A
        struct {             // phase B
            alignas(16) uint16_t W[NO * G::C * G::TS], WT[NO * G::C * G::TS], Y[NO * G::C * G::TS];
            alignas(16) float dS[slab * SS];
        } b;
    };
    union {
        struct { alignas(16) uint16_t U[NO * G::C * G::VS], X[NO * G::C * G::VS]; } c;
        struct { alignas(16) float q[G::C * OS], k[G::C * OS]; } out;
    };
    Scalars<TILES> s;
    float decay[NW][G::C], beta[NW][G::C], edge[NW];  // sums over each wave's columns
};

// Eight values of a row of a state [dk, dv] in memory (zero outside).
__device__ __forceinline__ void state8(const float* at, int n, bool vec, f4& x, f4& y) {
    float v[8];
    load8<T_F32>(at, n, vec, v);
    x = f4{v[0], v[1], v[2], v[3]};
    y = f4{v[4], v[5], v[6], v[7]};
}

// dR and dX = beta dR of dU + P^T dO, dU in du.
template <int TY, int TILES, class M>
__device__ __forceinline__ void solve_back(const M& m, const Scalars<TILES>& s, int n, int g, const f4* d_o, f4* du, f4* dr, f4* dx) {
    constexpr int tile = 16 * kInvStride, NP = Elem<TY>::parts, TS = Tok<TILES>::stride, part = 16 * TILES * TS;
    const f4 zero = {0, 0, 0, 0};
    const uint16_t* invT = m.invT + n * kInvStride + 4 * g;
    du[0] = mul<2>(Tok<TILES>::template at<3>(m.PT + n * TS, g, part), Tok<TILES>::template make<NP>(d_o), du[0]);
    if constexpr (TILES == 2) {
        du[1] = mul<2>(half_at<3>(m.PT + (16 + n) * TS + Tok<TILES>::tile_at(g, 1), part), split<NP>(d_o[1]), du[1]);
        dr[1] = mul<2>(half_at<3>(invT + 3 * tile, tile), split<3>(du[1]), zero);
        dx[1] = dr[1] * row4(s.beta, 1, g);
        du[0] -= mul<2>(half_at<3>(m.offT + n * kInvStride + 4 * g, tile), split<3>(dx[1]), zero);
    }
    dr[0] = mul<2>(half_at<3>(invT, tile), split<3>(du[0]), zero);
    dx[0] = dr[0] * row4(s.beta, 0, g);
}

// dS = gam_C dS' + scale (gam Q)^T dO - K^T (gam dX)
template <int TY, int DK, int TILES>
__device__ __forceinline__ void pull_state(const uint16_t* KT, const uint16_t* QT, const Scalars<TILES>& s, float scale, int n, int g, const f4* d_o,
                                           const f4* dx, f4* dS) {
    constexpr int NP = Elem<TY>::parts, TS = Tok<TILES>::stride;
    f4 so[TILES], sx[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        const f4 gam = row4(s.gam, i, g);
        sx[i] = dx[i] * gam * row4(s.rk, i, g) * -1.0f;
        so[i] = d_o[i] * gam * row4(s.rq, i, g) * scale;
    }
    const auto xb = Tok<TILES>::template make<3>(sx);
    const auto ob = Tok<TILES>::template make<3>(so);
    const float all = s.gam[16 * TILES - 1];
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) {
        f4 y = dS[i] * all;
        y = mul<2>(Tok<TILES>::template at<NP>(KT + (16 * i + n) * TS, g, DK * TS), xb, y);
        dS[i] = mul<2>(Tok<TILES>::template at<NP>(QT + (16 * i + n) * TS, g, DK * TS), ob, y);
    }
}

// The gradient of the state alone, for the segments: of every segment but the first, what its
// outputs (and, of the last, d_last) add to the gradient of the state before it. It needs neither
// states nor values.
template <int TY, int DK, int NW, int TILES> struct PullLds {
    typedef Geo<TY, DK, NW, TILES> G;
    alignas(16) uint16_t K[G::NP * G::C * G::KS], Q[G::NP * G::C * G::KS], KT[G::NP * DK * G::TS], QT[G::NP * DK * G::TS];
    InnerBack<TILES> m;
    Scalars<TILES> s;
};

// Where the chunk that ends before token te begins: at the grid, or at the last reset since.
struct Cut {
    int t;
    bool first;
};
template <int C> __device__ __forceinline__ Cut chunk_before(int te, int lane, const float* gp, int64_t g_stride, const uint8_t* rp, int64_t r_stride) {
    const int t0 = (te - 1) / C * C;
    const bool inside = lane < C && t0 + lane < te;
    const uint64_t cuts = __ballot(inside && (gp[(t0 + lane) * g_stride] < kClears || (rp && rp[(t0 + lane) * r_stride])));
    return Cut{cuts ? t0 + 63 - __clzll((long long)cuts) : t0, cuts != 0};
}

template <int TY, int DK, int NW, int TILES, bool FULL>
__global__ __launch_bounds__(64 * NW) void delta_pull_kernel(const Args a) {
    typedef Geo<TY, DK, NW, TILES> G;
    typedef typename Elem<TY>::type E;
    __shared__ PullLds<TY, DK, NW, TILES> lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t b = blockIdx.x / in.value_heads, h = blockIdx.x % in.value_heads, hk = h / a.share;
    const int dk = in.key_dim, dv = in.value_dim, segment = blockIdx.y + 1;
    const int begin = segment * a.segment_length, T = min((int)in.length, begin + a.segment_length);
    const int col0 = wave * 16, row0 = 4 * g + (n & 3), col = col0 + (n & 12);
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2];
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2];
    const float* gp = in.g + b * in.g_stride[0] + h * in.g_stride[2];
    const float* bp = in.beta + b * in.beta_stride[0] + h * in.beta_stride[2];
    const uint8_t* rp = in.reset ? in.reset + b * in.reset_stride[0] : nullptr;
    const E* d_o = (const E*)a.d_o + b * a.d_o_stride[0] + h * a.d_o_stride[2] + col;
    const int64_t bh = b * in.value_heads + h;
    f4 dS[DK / 16];
    load_state<DK, FULL>(a.d_last && segment == (int)a.segments - 1 ? a.d_last + bh * dk * dv : nullptr, dk, dv, dv, a.d_last_vec, col0, lane, dS);
    for (int te = T; te > begin;) {
        const Cut cut = chunk_before<G::C>(te, lane, gp, in.g_stride[1], rp, in.reset_stride[1]);
        const int t = cut.t, len = te - t;
        Rows<TY, DK, NW, TILES> kr, qr;
        kr.template fetch<FULL>(k + t * in.k_stride[1], in.k_stride[1], len, dk, a.k_vec);
        qr.template fetch<FULL>(q + t * in.q_stride[1], in.q_stride[1], len, dk, a.q_vec);
        f4 d4[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const f4 x = load4<TY, FULL>(d_o + (t + min(16 * i + row0, len - 1)) * a.d_o_stride[1], dv - col, a.d_o_vec);
            d4[i] = turn(16 * i + row0 < len ? x : f4{0, 0, 0, 0}, lane);
        }
        __syncthreads();
        if (wave == 0)
            load_scalars<TILES>(lane < len ? gp[(t + lane) * in.g_stride[1]] : 0.0f, lane < len ? bp[(t + lane) * in.beta_stride[1]] : 0.0f, lane,
                                cut.first, lds.s);
        kr.store(len, in.normalize, lds.K, lds.KT, lds.s.rk);
        qr.store(len, in.normalize, lds.Q, lds.QT, lds.s.rq);
        __syncthreads();
        fill_inner<TY, DK, NW, TILES, TILES, W_PT | W_INVT>(lds.K, lds.Q, lds.s, in.scale, lds.m);
        f4 du[TILES], dr[TILES], dx[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) du[i] = f4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) {
            const Frag<3> db = split<3>(dS[2 * c], dS[2 * c + 1]);
#pragma unroll
            for (int i = 0; i < TILES; ++i)
                du[i] = mul<2>(frag_at<G::NP>(lds.K + (16 * i + n) * G::KS + 32 * c + 8 * g, G::C * G::KS), db, du[i]);
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) du[i] *= row4(lds.s.end, i, g) * row4(lds.s.rk, i, g);
        __syncthreads();
        solve_back<TY, TILES>(lds.m, lds.s, n, g, d4, du, dr, dx);
        pull_state<TY, DK, TILES>(lds.KT, lds.QT, lds.s, in.scale, n, g, d4, dx, dS);
        if (cut.first)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) dS[i] = f4{0, 0, 0, 0};
        te = t;
    }
    store_state<DK, true>(a.d_starts + (bh * (a.segments - 1) + segment - 1) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, dS);
}

template <int TY, int DK, int NW, int TILES, bool FULL>
__global__ __launch_bounds__(64 * NW, NW == 8 || sizeof(BackwardLds<TY, DK, NW, TILES>) <= 80 * 1024 ? 2 : 1) void delta_backward_kernel(const Args a) {
    typedef Geo<TY, DK, NW, TILES> G;
    typedef BackwardLds<TY, DK, NW, TILES> L;
    typedef typename Elem<TY>::type E;
    constexpr int NP = G::NP, NO = L::NO, SO = NO - 1, C = G::C;
    __shared__ L lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t b = blockIdx.x / in.value_heads, h = blockIdx.x % in.value_heads, hk = h / a.share;
    const int dk = in.key_dim, dv = in.value_dim, segment = blockIdx.y;
    const int begin = segment * a.segment_length, T = min((int)in.length, begin + a.segment_length);  // this segment's tokens
    const int col0 = wave * 16, row0 = 4 * g + (n & 3), col = col0 + (n & 12);  // memory: four columns of a row
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2];
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2];
    const E* v = (const E*)in.v + b * in.v_stride[0] + h * in.v_stride[2] + col;
    const float* gp = in.g + b * in.g_stride[0] + h * in.g_stride[2];
    const float* bp = in.beta + b * in.beta_stride[0] + h * in.beta_stride[2];
    const uint8_t* rp = in.reset ? in.reset + b * in.reset_stride[0] : nullptr;
    const E* d_o = (const E*)a.d_o + b * a.d_o_stride[0] + h * a.d_o_stride[2];
    E* d_v = (E*)a.dv + b * a.dv_stride[0] + h * a.dv_stride[2] + col;
    const int64_t bh = b * in.value_heads + h;

    f4 dS[DK / 16], Sn[DK / 16];  // the gradient of the state, and the state, after the chunk
    if (segment == (int)a.segments - 1) {
        load_state<DK, FULL>(a.d_last ? a.d_last + bh * dk * dv : nullptr, dk, dv, dv, a.d_last_vec, col0, lane, dS);
        load_state<DK, FULL>(a.last + bh * dk * dv, dk, dv, dv, a.last_vec, col0, lane, Sn);
    } else {
        load_state<DK, true>(a.d_starts + (bh * (a.segments - 1) + segment) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, dS);
        load_state<DK, true>(a.saved + (bh * (a.chunks - 1) + T / C - 1) * (DK * G::DV), DK, G::DV, G::DV, true, col0, lane, Sn);
    }

    for (int te = T; te > begin;) {
        const Cut cut = chunk_before<C>(te, lane, gp, in.g_stride[1], rp, in.reset_stride[1]);
        const int t = cut.t;
        const bool first = cut.first;
        const int len = te - t;
        // The state before the chunk: nothing, the caller's, or a saved one.
        const float* sp = nullptr;
        int s_rows = dk, s_cols = dv, s_ld = dv;
        bool s_vec = a.s_vec;
        if (!first) {
            if (t == 0) {
                if (in.state) sp = in.state + bh * dk * dv;
            } else {
                sp = a.saved + (bh * (a.chunks - 1) + t / C - 1) * (DK * G::DV);
                s_rows = DK, s_cols = s_ld = G::DV, s_vec = true;
            }
        }

        __syncthreads();
        if (wave == 0)
            load_scalars<TILES>(lane < len ? gp[(t + lane) * in.g_stride[1]] : 0.0f, lane < len ? bp[(t + lane) * in.beta_stride[1]] : 0.0f, lane,
                                first, lds.s);
        Rows<TY, DK, NW, TILES> kr, qr;
        kr.template fetch<FULL>(k + t * in.k_stride[1], in.k_stride[1], len, dk, a.k_vec);
        qr.template fetch<FULL>(q + t * in.q_stride[1], in.q_stride[1], len, dk, a.q_vec);
        kr.store(len, in.normalize, lds.K, lds.KT, lds.s.rk);
        qr.store(len, in.normalize, lds.Q, lds.QT, lds.s.rq);
#pragma unroll
        for (int it0 = 0; it0 < C * G::DV / 8; it0 += G::threads) {
            const int it = it0 + threadIdx.x, row = it / (G::DV / 8), e = 8 * (it % (G::DV / 8));
            if (C * G::DV / 8 % G::threads && it >= C * G::DV / 8) break;
            Raw<TY> x;
            x.template load<FULL>(d_o + (t + min(row, len - 1)) * a.d_o_stride[1] + e, dv - e, a.d_o_vec);
            x.keep(row < len);
            uint32_t w[4][NP];
            x.parts(w);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<u4*>(lds.DO + (p * C + row) * G::VS + e) = u4{w[0][p], w[1][p], w[2][p], w[3][p]};
        }
        f4 S[DK / 16];
        load_state<DK, FULL>(sp, s_rows, s_cols, s_ld, s_vec, col0, lane, S);
        f4 vv[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i)
            vv[i] = turn(load4<TY, FULL>(v + (t + min(16 * i + row0, len - 1)) * in.v_stride[1], dv - col, a.v_vec), lane);
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) vv[i][r] = 16 * i + 4 * g + r < len ? vv[i][r] : 0.0f;
        __syncthreads();
        fill_inner<TY, DK, NW, TILES, TILES, W_P | W_PT | W_INV | W_INVT>(lds.K, lds.Q, lds.s, in.scale, lds.m);

        // ---- phase A: this wave's columns
        f4 ks[TILES], o4[TILES], du[TILES], d4[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            ks[i] = o4[i] = du[i] = f4{0, 0, 0, 0};
            f4 x = {0, 0, 0, 0};
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) x += load4<T_BF16>(lds.DO + (p * C + 16 * i + row0) * G::VS + col, 4, true);
            d4[i] = turn(x, lane);
        }
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) {
            const Frag<3> sb = split<3>(S[2 * c], S[2 * c + 1]), db = split<3>(dS[2 * c], dS[2 * c + 1]);
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const int at = (16 * i + n) * G::KS + 32 * c + 8 * g;
                const Frag<NP> kf = frag_at<NP>(lds.K + at, C * G::KS);
                ks[i] = mul<2>(kf, sb, ks[i]);
                du[i] = mul<2>(kf, db, du[i]);
                o4[i] = mul<2>(frag_at<NP>(lds.Q + at, C * G::KS), sb, o4[i]);
            }
        }
        f4 x[TILES], u[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const f4 gam = row4(lds.s.gam, i, g), rk = row4(lds.s.rk, i, g);
            x[i] = vv[i] - gam * rk * ks[i];
            o4[i] *= gam * row4(lds.s.rq, i, g) * in.scale;
            du[i] *= row4(lds.s.end, i, g) * rk;
        }
        // <dS', S'>, the decay's gradient from all that passes the chunk's end.
        float edge = 0.0f;
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) edge += dS[i][r] * Sn[i][r];
        edge = sum64(edge);
        if (lane == 0) lds.edge[wave] = edge;
        __syncthreads();
        Half<3> up[TILES];
        solve<TILES, TILES>(lds.m, lds.s, n, g, x, u, up);
        add_PU<TILES, TILES>(lds.m, n, g, up, o4);
        const f4 zero = {0, 0, 0, 0};
        f4 dr[TILES], dx[TILES];
        solve_back<TY, TILES>(lds.m, lds.s, n, g, d4, du, dr, dx);
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * i + 4 * g + r;
                const float de = sum16(d4[i][r] * o4[i][r] - dx[i][r] * vv[i][r]), be = sum16(dr[i][r] * x[i][r]);
                if (n == 0) {
                    lds.decay[wave][row] = de;
                    lds.beta[wave][row] = be;
                }
            }
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int at = (16 * i + row0) * G::VS + col;
            const f4 y = turn(dx[i], lane);
            put4<NO>(lds.c.U + at, C * G::VS, turn(u[i], lane));
            put4<NO>(lds.c.X + at, C * G::VS, y);
            if (16 * i + row0 < len) store4<TY, FULL>(d_v + (t + 16 * i + row0) * a.dv_stride[1], dv - col, a.dv_vec, y);
        }
        __syncthreads();

        // ---- phase B: gradients of q and k
        if (wave == NW - 1) {
            double sum = 0.0;
            float bsum = 0.0f;
            if (lane < C)
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    sum += (double)lds.decay[w][lane];
                    bsum += lds.beta[w][lane];
                }
            if (lane == C - 1)
#pragma unroll
                for (int w = 0; w < NW; ++w) sum += (double)lds.edge[w];
#pragma unroll
            for (int d = 1; d < C; d <<= 1) {
                const double dn = __shfl_down(sum, d);
                if (lane + d < C) sum += dn;
            }
            if (lane < len) {
                a.dg[b * a.dg_stride[0] + (t + lane) * a.dg_stride[1] + h * a.dg_stride[2]] = first && lane == 0 ? 0.0f : (float)sum;
                a.dbeta[b * a.dbeta_stride[0] + (t + lane) * a.dbeta_stride[1] + h * a.dbeta_stride[2]] = bsum;
            }
        }
        constexpr int pairs = TILES * (TILES + 1) / 2;
        for (int job = wave; job < 2 * pairs; job += NW) {
            const int pair = job % pairs, ti = pair > 0 ? 1 : 0, tj = pair > 1 ? 1 : 0, j = 16 * tj + n;
            f4 acc = zero;
#pragma unroll
            for (int c = 0; c < G::DV / 32; ++c) {
                const int ai = (16 * ti + n) * G::VS + 32 * c + 8 * g, aj = (16 * tj + n) * G::VS + 32 * c + 8 * g;
                const Frag<NO> uf = frag_at<NO>(lds.c.U + aj, C * G::VS);
                if (job < pairs) acc = mul<SO>(frag_at<NP>(lds.DO + ai, C * G::VS), uf, acc);
                else acc = mul<SO>(frag_at<NO>(lds.c.X + ai, C * G::VS), uf, acc);
            }
            const float hj = lds.s.hi[j], lj = lds.s.lo[j], rj = lds.s.rk[j];
            f4 by_col, by_row;  // times the norm of the column's token, and of the row's
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * g + r;
                const float w = acc[r] * __expf((lds.s.hi[i] - hj) + (lds.s.lo[i] - lj));
                const float y = job < pairs ? (j <= i ? w * in.scale : 0.0f) : (j < i ? -w : 0.0f);
                by_col[r] = y * rj;
                by_row[r] = y * (job < pairs ? lds.s.rq[i] : lds.s.rk[i]);
            }
            if (job < pairs) {
                put_rows<NO, TILES>(lds.b.W, by_col, ti, tj, lane);
                put_cols<NO, TILES>(lds.b.WT, by_row, ti, tj, lane);
            } else if (ti != tj) {
                put_rows<NO, TILES>(lds.b.Y, by_col, ti, tj, lane);
                put_cols<NO, TILES>(lds.b.Y, by_row, ti, tj, lane);
            } else {
                // A diagonal tile of Y + Y^T: the mirrored values come through LDS.
                put_rows<NO, TILES>(lds.b.Y, by_col, ti, tj, lane);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (j < 16 * ti + 4 * g + r)
                        put_parts<NO>(lds.b.Y + j * G::TS + Tok<TILES>::slot_of(16 * ti + 4 * g + r), C * G::TS, by_row[r]);
            }
        }
        constexpr int blocks = L::slab / 16, slabs = DK / L::slab;
        constexpr bool spread = NW >= 2 * blocks && TILES == 2;  // one tile a wave
        constexpr int rounds = spread ? 1 : (blocks + NW - 1) / NW, per = spread ? 1 : TILES;
        f4 dq[slabs * rounds * per], dkk[slabs * rounds * per];
#pragma unroll
        for (int sl = 0; sl < slabs; ++sl) {
            if (sl) __syncthreads();
#pragma unroll
            for (int i = 0; i < L::slab / 16; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) lds.b.dS[(16 * i + 4 * g + r) * L::SS + col0 + n] = dS[sl * (L::slab / 16) + i][r];
            __syncthreads();
#pragma unroll
            for (int rd = 0; rd < rounds; ++rd) {
                const int blk = spread ? wave % blocks : wave + rd * NW;
                const int tile0 = spread ? wave / blocks : 0;
                if (blk < blocks && tile0 < TILES) {
                    const int row = sl * L::slab + 16 * blk + n;  // of the key dimension: this lane's column of the results
                    f4 aq[per], ar[per], ac[per];
#pragma unroll
                    for (int i = 0; i < per; ++i) aq[i] = ar[i] = ac[i] = zero;
#pragma unroll
                    for (int c = 0; c < G::DV / 32; ++c) {
                        const int e = 32 * c + 8 * g;
                        f4 s0 = zero, s1 = zero;
                        if (sp && row < s_rows) state8(sp + row * s_ld + e, s_cols - e, s_vec, s0, s1);
                        const Frag<NO> sf = split<NO>(s0, s1);
                        const float* ds = lds.b.dS + (16 * blk + n) * L::SS + e;
                        const Frag<NO> df = split<NO>(*reinterpret_cast<const f4*>(ds), *reinterpret_cast<const f4*>(ds + 4));
#pragma unroll
                        for (int i = 0; i < per; ++i) {
                            const int at = (16 * (tile0 + i) + n) * G::VS + e;
                            if (sp) {
                                aq[i] = mul<SO>(frag_at<NP>(lds.DO + at, C * G::VS), sf, aq[i]);
                                ar[i] = mul<SO>(frag_at<NO>(lds.c.X + at, C * G::VS), sf, ar[i]);
                            }
                            ac[i] = mul<SO>(frag_at<NO>(lds.c.U + at, C * G::VS), df, ac[i]);
                        }
                    }
                    const auto kt = Tok<TILES>::template at<NP>(lds.KT + row * G::TS, g, DK * G::TS);
                    const auto qt = Tok<TILES>::template at<NP>(lds.QT + row * G::TS, g, DK * G::TS);
#pragma unroll
                    for (int i = 0; i < per; ++i) {
                        const int ti = tile0 + i, at = (16 * ti + n) * G::TS, to = (sl * rounds + rd) * per + i;
                        const f4 gam = row4(lds.s.gam, ti, g);
                        f4 yq = aq[i] * gam * in.scale, yk = ac[i] * row4(lds.s.end, ti, g) - ar[i] * gam;
                        yk = mul<SO>(Tok<TILES>::template at<NO>(lds.b.Y + at, g, C * G::TS), kt, yk);
                        if (TILES == 2 && ti == 0) {  // the upper right tile of W is not written
                            yq = mul<SO>(half_at<NO>(lds.b.W + at + Tok<TILES>::tile_at(g, 0), C * G::TS),
                                         half_at<NP>(lds.KT + row * G::TS + Tok<TILES>::tile_at(g, 0), DK * G::TS), yq);
                            yk = mul<SO>(Tok<TILES>::template at<NO>(lds.b.WT + at, g, C * G::TS), qt, yk);
                        } else if (TILES == 2) {
                            yq = mul<SO>(Tok<TILES>::template at<NO>(lds.b.W + at, g, C * G::TS), kt, yq);
                            yk = mul<SO>(half_at<NO>(lds.b.WT + at + Tok<TILES>::tile_at(g, 1), C * G::TS),
                                         half_at<NP>(lds.QT + row * G::TS + Tok<TILES>::tile_at(g, 1), DK * G::TS), yk);
                        } else {
                            yq = mul<SO>(Tok<TILES>::template at<NO>(lds.b.W + at, g, C * G::TS), kt, yq);
                            yk = mul<SO>(Tok<TILES>::template at<NO>(lds.b.WT + at, g, C * G::TS), qt, yk);
                        }
                        dq[to] = yq;
                        dkk[to] = yk;
                    }
                }
            }
        }
        // the state's gradient, from this wave's columns
        pull_state<TY, DK, TILES>(lds.KT, lds.QT, lds.s, in.scale, n, g, d4, dx, dS);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) {
            if (first) dS[i] = zero;
            Sn[i] = S[i];
        }
        __syncthreads();  // U and dX are read
#pragma unroll
        for (int sl = 0; sl < slabs; ++sl)
#pragma unroll
            for (int rd = 0; rd < rounds; ++rd) {
                const int blk = spread ? wave % blocks : wave + rd * NW;
                const int tile0 = spread ? wave / blocks : 0;
                if (blk < blocks && tile0 < TILES)
#pragma unroll
                    for (int i = 0; i < per; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int at = (16 * (tile0 + i) + 4 * g + r) * L::OS + sl * L::slab + 16 * blk + n, from = (sl * rounds + rd) * per + i;
                            lds.out.q[at] = dq[from][r];
                            lds.out.k[at] = dkk[from][r];
                        }
            }
        __syncthreads();
        // rows out, through the norms: d(x / |x|) = (d - x^ (x^ . d)) / |x|, |x|^2 with its eps; of
        // one dimension alone that is d eps / |x|^3, which the difference would lose to rounding
        constexpr int pieces = DK / 8;
        for (int it = threadIdx.x; it < C * pieces; it += G::threads) {
            const int row = it / pieces, e = 8 * (it % pieces);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float* from = (w ? lds.out.k : lds.out.q) + row * L::OS + e;
                const f4 x0 = *reinterpret_cast<const f4*>(from), x1 = *reinterpret_cast<const f4*>(from + 4);
                float y[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
                if (in.normalize) {
                    const float nr = w ? lds.s.rk[row] : lds.s.rq[row];
                    const uint16_t* src = (w ? lds.K : lds.Q) + row * G::KS;
                    float xs[8], dot = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float z = 0.0f;
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) z += __uint_as_float((uint32_t)src[p * C * G::KS + slot(e + j)] << 16);
                        xs[j] = z * nr;
                        dot += xs[j] * y[j];
                    }
#pragma unroll
                    for (int d = 1; d < pieces; d <<= 1) dot += __shfl_xor(dot, d);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = dk == 1 ? y[j] * kNormEps * nr * nr * nr : nr * (y[j] - xs[j] * dot);
                }
                if (row < len) {
                    if (a.part_q) {
                        float* to = (w ? a.part_k : a.part_q) + ((b * T + t + row) * in.value_heads + h) * dk + e;
                        store8<T_F32>(to, dk - e, dk % 8 == 0, y);
                    } else if (w) {
                        store8<TY>((E*)a.dk + b * a.dk_stride[0] + (t + row) * a.dk_stride[1] + hk * a.dk_stride[2] + e, dk - e, a.dk_vec, y);
                    } else {
                        store8<TY>((E*)a.dq + b * a.dq_stride[0] + (t + row) * a.dq_stride[1] + hk * a.dq_stride[2] + e, dk - e, a.dq_vec, y);
                    }
                }
            }
        }
        te = t;
    }
    if (a.d_state && segment == 0) store_state<DK, FULL>(a.d_state + bh * dk * dv, dk, dv, dv, a.d_state_vec, col0, lane, dS);
}

// Sums the value heads of each key head, in their order; one thread a value.
template <int TY> __global__ __launch_bounds__(256) void delta_share_kernel(const Args a) {
    typedef typename Elem<TY>::type E;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t all = (int64_t)in.batch * in.length * in.key_heads * in.key_dim;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= all) return;
    const int64_t x = id % in.key_dim, hk = id / in.key_dim % in.key_heads, bt = id / in.key_dim / in.key_heads;
    const int64_t t = bt % in.length, b = bt / in.length;
    const int64_t from = (bt * in.value_heads + hk * a.share) * in.key_dim + x;
    float sq = 0.0f, sk = 0.0f;
    for (uint32_t s = 0; s < a.share; ++s) {
        sq += a.part_q[from + s * in.key_dim];
        sk += a.part_k[from + s * in.key_dim];
    }
    ((E*)a.dq)[b * a.dq_stride[0] + t * a.dq_stride[1] + hk * a.dq_stride[2] + x] = Elem<TY>::put(sq);
    ((E*)a.dk)[b * a.dk_stride[0] + t * a.dk_stride[1] + hk * a.dk_stride[2] + x] = Elem<TY>::put(sk);
}

// ---- one token -----------------------------------------------------------------------------
// The state is read once and written once (8 bytes a value and step: bound by memory). A wave
// holds all rows of 4 LANES columns, 16 (or 4) rows and 4 columns a lane, so both products with
// the state, S^T k and S^T q, come from one pass over registers and three or fewer exchanges:
//     o = scale (a S^T q + (k . q) u),  u = beta (v - a S^T k),  S <- a S + k u^T
// LANES lanes lie along the columns, 64 / LANES along the rows.
template <int TY, int LANES, int ROWS, bool VEC>
__global__ __launch_bounds__(256) void delta_step_kernel(const Args a, float* state) {
    typedef typename Elem<TY>::type E;
    const ZenoAmdDeltaInputs& in = a.in;
    const int lane = threadIdx.x & 63, cl = lane % LANES, rg = lane / LANES;
    const int dk = in.key_dim, dv = in.value_dim;
    const uint32_t blocks = (dv + 4 * LANES - 1) / (4 * LANES);
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t bh = id / blocks;
    const int col = ((int)(id % blocks) * LANES + cl) * 4, row0 = rg * ROWS;
    if (bh >= (int64_t)in.batch * in.value_heads) return;
    const int64_t b = bh / in.value_heads, h = bh % in.value_heads, hk = h / a.share;
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2] + row0;
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2] + row0;
    const E* v = (const E*)in.v + b * in.v_stride[0] + h * in.v_stride[2] + col;
    const float g = in.g[b * in.g_stride[0] + h * in.g_stride[2]], beta = in.beta[b * in.beta_stride[0] + h * in.beta_stride[2]];
    const bool first = g < kClears || (in.reset && in.reset[b * in.reset_stride[0]]);
    float* s = state + bh * dk * dv + (int64_t)row0 * dv + col;

    f4 S[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        S[i] = f4{0, 0, 0, 0};
        if (!first && row0 + i < dk) {
            if (VEC) {
                if (col < dv) S[i] = *reinterpret_cast<const f4*>(s + i * dv);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (col + c < dv) S[i][c] = s[i * dv + c];
            }
        }
    }
    float kv[ROWS], qv[ROWS], vv[4];
#pragma unroll
    for (int i = 0; i < ROWS; i += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kv[i + j] = row0 + i + j < dk ? Elem<TY>::get(k[i + j]) : 0.0f;
            qv[i + j] = row0 + i + j < dk ? Elem<TY>::get(q[i + j]) : 0.0f;
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = col + c < dv ? Elem<TY>::get(v[c]) : 0.0f;
    float kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        kk += kv[i] * kv[i];
        qq += qv[i] * qv[i];
        kq += kv[i] * qv[i];
    }
    f4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        sk += S[i] * kv[i];
        sq += S[i] * qv[i];
    }
#pragma unroll
    for (int d = LANES; d < 64; d <<= 1) {
        kk += __shfl_xor(kk, d);
        qq += __shfl_xor(qq, d);
        kq += __shfl_xor(kq, d);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            sk[c] += __shfl_xor(sk[c], d);
            sq[c] += __shfl_xor(sq[c], d);
        }
    }
    const float rk = in.normalize ? 1.0f / sqrtf(kk + kNormEps) : 1.0f, rq = in.normalize ? 1.0f / sqrtf(qq + kNormEps) : 1.0f;
    const float decay = first ? 0.0f : __expf(g);
    f4 u;
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = beta * (vv[c] - decay * rk * sk[c]);
    if (rg == 0) {
        E* o = (E*)a.o + b * a.o_stride[0] + h * a.o_stride[2] + col;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (col + c < dv) o[c] = Elem<TY>::put(in.scale * rq * (decay * sq[c] + kq * rk * u[c]));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (row0 + i >= dk) continue;
        const f4 y = S[i] * decay + u * (kv[i] * rk);
        if (VEC) {
            if (col < dv) *reinterpret_cast<f4*>(s + i * dv) = y;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (col + c < dv) s[i * dv + c] = y[c];
        }
    }
}

// ---- launches ------------------------------------------------------------------------------
template <int TY, int DK, int NW, int TILES, bool FULL> void forward_shape(const Args& a, hipStream_t stream) {
    const uint32_t heads = a.in.batch * a.in.value_heads;
    if (a.segments > 1) {
        delta_forward_kernel<TY, DK, NW, TILES, FULL, true><<<dim3(heads, a.segments - 1, 2), 64 * NW, 0, stream>>>(a);
        if (a.segments > 2) delta_join_kernel<DK, NW, false><<<heads, 64 * NW, 0, stream>>>(a.starts, a.jumps, a.segments);
    }
    delta_forward_kernel<TY, DK, NW, TILES, FULL, false><<<dim3(heads, a.segments), 64 * NW, 0, stream>>>(a);
}
template <int TY, int DK, int NW, int TILES, bool FULL> void backward_shape(const Args& a, hipStream_t stream) {
    const uint32_t heads = a.in.batch * a.in.value_heads;
    if (a.segments > 1) {
        delta_pull_kernel<TY, DK, NW, TILES, FULL><<<dim3(heads, a.segments - 1), 64 * NW, 0, stream>>>(a);
        if (a.segments > 2) delta_join_kernel<DK, NW, true><<<heads, 64 * NW, 0, stream>>>(a.d_starts, a.jumps, a.segments);
    }
    delta_backward_kernel<TY, DK, NW, TILES, FULL><<<dim3(heads, a.segments), 64 * NW, 0, stream>>>(a);
}
template <int TY, int DK, int NW, int TILES> void forward_shape(const Args& a, hipStream_t stream) {
    a.full ? forward_shape<TY, DK, NW, TILES, true>(a, stream) : forward_shape<TY, DK, NW, TILES, false>(a, stream);
}
template <int TY, int DK, int NW, int TILES> void backward_shape(const Args& a, hipStream_t stream) {
    a.full ? backward_shape<TY, DK, NW, TILES, true>(a, stream) : backward_shape<TY, DK, NW, TILES, false>(a, stream);
}

template <int TY> hipError_t launch_forward(const Args& a, const Shape& s, hipStream_t stream) {
    if (s.dk == 64 && s.waves == 4) forward_shape<TY, 64, 4, 2>(a, stream);
    else if (s.dk == 64 && s.tiles == 2) forward_shape<TY, 64, 8, 2>(a, stream);
    else if (s.tiles == 2) forward_shape<TY, 128, 8, 2>(a, stream);
    else if constexpr (TY == T_F32) {
        if (s.dk == 64) forward_shape<TY, 64, 8, 1>(a, stream);
        else forward_shape<TY, 128, 8, 1>(a, stream);
    } else if constexpr (TY == T_F16) {
        forward_shape<TY, 128, 8, 1>(a, stream);
    }
    return hipGetLastError();
}

template <int TY> hipError_t launch_backward(const Args& a, const Shape& s, hipStream_t stream) {
    if (s.dk == 64 && s.waves == 4) backward_shape<TY, 64, 4, 2>(a, stream);
    else if (s.dk == 64) backward_shape<TY, 64, 8, TY == T_F32 ? 1 : 2>(a, stream);
    else backward_shape<TY, 128, 8, TY == T_BF16 ? 2 : 1>(a, stream);
    if (a.part_q) {
        const int64_t all = (int64_t)a.in.batch * a.in.length * a.in.key_heads * a.in.key_dim;
        delta_share_kernel<TY><<<dim3((uint32_t)((all + 255) / 256)), 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

template <int TY> hipError_t launch_step(const Args& a, float* state, hipStream_t stream) {
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t heads = (int64_t)in.batch * in.value_heads;
    const bool vec = in.value_dim % 4 == 0 && (uintptr_t)state % 16 == 0;
    const int lanes = in.key_dim <= 32 || in.key_dim > 64 ? 8 : 16;
    const int64_t waves = heads * ((in.value_dim + 4 * lanes - 1) / (4 * lanes));
    const dim3 grid((uint32_t)((waves + 3) / 4));
    if (in.key_dim <= 32) {
        if (vec) delta_step_kernel<TY, 8, 4, true><<<grid, 256, 0, stream>>>(a, state);
        else delta_step_kernel<TY, 8, 4, false><<<grid, 256, 0, stream>>>(a, state);
    } else if (in.key_dim <= 64) {
        if (vec) delta_step_kernel<TY, 16, 16, true><<<grid, 256, 0, stream>>>(a, state);
        else delta_step_kernel<TY, 16, 16, false><<<grid, 256, 0, stream>>>(a, state);
    } else {
        if (vec) delta_step_kernel<TY, 8, 16, true><<<grid, 256, 0, stream>>>(a, state);
        else delta_step_kernel<TY, 8, 16, false><<<grid, 256, 0, stream>>>(a, state);
    }
    return hipGetLastError();
}

}  // namespace delta
}  // namespace za
