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
// diagonal tiles of I + Z B. Those come from forward substitution in registers: the cheaper
// product of powers (I - N)(I + N^2)... loses all digits where keys repeat, as they do for an
// environment that stands still.
//
// A chunk ends at a token of the grid of C and before every reset, so nothing is masked inside
// it and no value from before a reset is ever multiplied by a zero. Nor may an output meet a NaN or an
// infinity of a later token by way of the zeros above a diagonal: a chunk that holds one goes token by
// token. Partial chunks are filled with zero keys, zero beta and zero g, which change nothing.
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

constexpr int kInvStride = 20;  // of 16x16 tiles in LDS

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

// A double from other lanes: shifted up by CTRL - 0x110 lanes or down by CTRL - 0x100 within each 16
// (zeros come in), or (0x142) the last lane of the 16 before, in every second 16.
template <int CTRL> __device__ __forceinline__ double dpp64(double x) {
    constexpr int rows = CTRL == 0x142 ? 0xa : 0xf;
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, rows, 0xf, CTRL != 0x142);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, rows, 0xf, CTRL != 0x142);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double from_lane(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane));
}

// g and beta of a chunk (one lane a token, one wave): sums in 64 bits.
template <int TILES>
__device__ __forceinline__ void load_scalars(float g, float beta, int lane, bool first, Scalars<TILES>& s) {
    constexpr int C = 16 * TILES;
    double sum = (first && lane == 0) ? 0.0 : (double)g;
    sum += dpp64<0x111>(sum);
    sum += dpp64<0x112>(sum);
    sum += dpp64<0x114>(sum);
    sum += dpp64<0x118>(sum);
    if constexpr (TILES == 2) sum += dpp64<0x142>(sum);
    const double all = from_lane(sum, C - 1);
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

// A value of row group G (lanes 16 G to 16 G + 15) in all four groups.
template <int G> __device__ __forceinline__ float from_group(float x) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t pair = __builtin_amdgcn_permlane16_swap(b, b, false, false)[G & 1];
    return __uint_as_float(__builtin_amdgcn_permlane32_swap(pair, pair, false, false)[G >> 1]);
}
// Rows 4 G to 4 G + 3 of W = Z - Z B W, and what they take from the rows below; zb is -Z B. Rows
// that are final take only zeros.
template <int G> __device__ __forceinline__ void solve_rows(f4 zb, int g, f4& w) {
    constexpr int lane = 0x150 + 4 * G;  // the first of these rows' columns, from within each 16 lanes
    f4 u = w;
    u[1] += dpp<lane>(zb[1]) * u[0];
    u[2] += dpp<lane>(zb[2]) * u[0];
    u[3] += dpp<lane>(zb[3]) * u[0];
    u[2] += dpp<lane + 1>(zb[2]) * u[1];
    u[3] += dpp<lane + 1>(zb[3]) * u[1];
    u[3] += dpp<lane + 2>(zb[3]) * u[2];
    if constexpr (G == 3) {
        w = g == 3 ? u : w;
    } else {
        const f4 y = {from_group<G>(u[0]), from_group<G>(u[1]), from_group<G>(u[2]), from_group<G>(u[3])};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            w[r] += dpp<lane>(zb[r]) * y[0];
            w[r] += dpp<lane + 1>(zb[r]) * y[1];
            w[r] += dpp<lane + 2>(zb[r]) * y[2];
            w[r] += dpp<lane + 3>(zb[r]) * y[3];
        }
    }
}
// W = (I + Z B)^-1 Z of a strictly lower 16x16 tile, by forward substitution of four rows at a time,
// in registers: with Z read from LDS, one lane a column, latency was three quarters of the time.
// The inverses of I + Z B and I + B Z are I - W B and I - B W.
__device__ __forceinline__ f4 solve_tile(f4 z, float beta, int g) {
    const f4 zb = z * -beta;
    solve_rows<0>(zb, g, z);
    solve_rows<1>(zb, g, z);
    solve_rows<2>(zb, g, z);
    solve_rows<3>(zb, g, z);
    return z;
}

// The matrices inside a chunk. Of the diagonal tiles: the inverse of I + Z B, and for gradients
// behind it the transposed inverse of I + B Z.
template <int TILES> struct Inner {
    static constexpr int C = 16 * TILES, TS = Tok<TILES>::stride, sides = 1;
    static constexpr int tile = 16 * kInvStride;                // of one 16x16 tile
    alignas(16) uint16_t P[3 * C * TS];                         // lower(D * Q K^T) scale
    alignas(16) uint16_t off[3 * tile];                         // Z, lower left tile
    alignas(16) uint16_t inv[TILES * 3 * tile];
};
template <int TILES> struct InnerBack {
    static constexpr int C = 16 * TILES, TS = Tok<TILES>::stride, sides = 2;
    static constexpr int tile = 16 * kInvStride;
    alignas(16) uint16_t PT[3 * C * TS];                        // transposed
    alignas(16) uint16_t off[3 * tile], offT[3 * tile];
    alignas(16) uint16_t inv[2 * TILES * 3 * tile];
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
                constexpr int second = M::sides == 2 ? TILES : 0;  // tiles before the transposed ones
                const float bj = s.beta[j];
                const f4 bi = row4(s.beta, ti, g);
                f4 lower, t, tt;
#pragma unroll
                for (int r = 0; r < 4; ++r) lower[r] = n < 4 * g + r ? z[r] : 0.0f;
                const f4 w = solve_tile(lower, bj, g);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float one = n == 4 * g + r ? 1.0f : 0.0f;
                    t[r] = one - w[r] * bj;
                    tt[r] = one - bi[r] * w[r];
                }
                if constexpr (WANT & W_INV) put4<3>(m.inv + ti * 3 * M::tile + (4 * g + (n & 3)) * kInvStride + (n & 12), M::tile, turn(t, lane));
                if constexpr (WANT & W_INVT) put4<3>(m.inv + (second + ti) * 3 * M::tile + n * kInvStride + 4 * g, M::tile, tt);
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

// This wave's columns of a state [rows, cols] in memory (leading dimension ld; null: zeros) as
// result tiles, one value an access: 64 bytes of four rows at a time, and no exchange between lanes.
// FULL: [DK, LD].
template <int DK, int LD, bool FULL> __device__ __forceinline__ void load_state(const float* at, int rows, int cols, int ld, int col0, int lane, f4* S) {
    const int row = 4 * (lane >> 4), col = col0 + (lane & 15), stride = FULL ? LD : ld;
    const float* from = at + row * stride + col;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) S[i] = f4{0, 0, 0, 0};
    if (at)
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (FULL || (16 * i + r + row < rows && col < cols)) S[i][r] = from[(16 * i + r) * stride];
}
template <int DK, int LD, bool FULL> __device__ __forceinline__ void store_state(float* at, int rows, int cols, int ld, int col0, int lane, const f4* S) {
    const int row = 4 * (lane >> 4), col = col0 + (lane & 15), stride = FULL ? LD : ld;
    float* to = at + row * stride + col;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (FULL || (16 * i + r + row < rows && col < cols)) to[(16 * i + r) * stride] = S[i][r];
}

// The matrices over segments are kept in the parts and the order in which a lane holds them as
// left operands: [row tile][32 of the contraction][part][lane][8]; M and, behind it, M transposed.
template <int DK> struct Jump {
    static constexpr int steps = DK / 32, part = 64 * 8, row = steps * 3 * part, size = DK / 16 * row;  // in bf16
    static constexpr int floats = size + 4;  // of both, and whether anything passes the segment at all
};
// M's columns from the 16 that this wave holds as result tiles.
template <int DK> __device__ __forceinline__ void store_jump(uint16_t* to, int wave, int lane, const f4* S) {
    typedef Jump<DK> J;
    const int n = lane & 15, g = lane >> 4;
    // Row 16 i + 4 g + n % 4, columns 16 wave + 4 (n / 4) + 0..3 of M: half of a lane's eight values.
    uint16_t* m = to + (wave >> 1) * 3 * J::part + (4 * g + (n & 3) + 16 * (n >> 2)) * 8 + 4 * (wave & 1);
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) put4<3>(m + i * J::row, J::part, turn(S[i], lane));
    // Of M transposed these registers are the operand already.
    uint16_t* t = to + J::size + wave * J::row + lane * 8;
#pragma unroll
    for (int c = 0; c < J::steps; ++c) {
        const Frag<3> f = split<3>(S[2 * c], S[2 * c + 1]);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u4*>(t + (c * 3 + p) * J::part) = f.p[p];
    }
}

// ---- forward -------------------------------------------------------------------------------
template <int TY, int DK, int NW, int TILES> struct ForwardLds {
    typedef Geo<TY, DK, NW, TILES> G;
    alignas(16) uint16_t K[G::NP * G::C * G::KS], Q[G::NP * G::C * G::KS], KT[G::NP * DK * G::TS];
    Inner<TILES> m;
    Scalars<TILES> s;
    alignas(16) uint32_t odd[NW];  // whether a wave has fetched a value that is not finite
};

// What bounds it: of many short sequences memory (16384 of 16 tokens, two heads of 64 x 64, bfloat16:
// 335 us, 3.9 TB/s of inputs, outputs and states; a large copy reaches 5.1), else a chunk's chain of
// dependent products and exchanges, of which the workgroups of a CU (four of four waves) take turns (4096
// of 32 tokens, four heads, with the states for the gradients: 253 us). The look for values that are not finite takes 4%.
// FULL: heads of exactly DK and 16 NW dimensions, aligned, need no masks: a quarter of the
// instructions less (3345 and 4595 of 64 x 64, bfloat16).
// Waves a SIMD that the registers are cut down to: as many workgroups as fit the LDS, but not more
// than the registers bear (128 of four waves spill in the wide kernel with outputs: 107 us, 130 so). The
// segments' pass of 128x128 spills a few too and is faster all the same (one sequence of 16384, 8 heads: bfloat16
// 4 registers, 277 us a pass, 309 without; float16 28, 362 and 392).
constexpr int forward_waves(int waves, bool states, size_t lds) {
    const int groups = (int)(160 * 1024 / lds), fit = groups * waves / 4;
    return waves == 8 && !states ? 2 : fit >= 4 ? 4 : fit == 3 ? 3 : 2;
}

// STATES: no outputs; of each segment but the last, N, the state after it from zeros (from the
// caller's state in the first segment), and M, the same without values from the unit matrix: with
// S the state before the segment, the state after it is M S + N.
template <int TY, int DK, int NW, int TILES, bool FULL, bool STATES>
__global__ __launch_bounds__(64 * NW, forward_waves(NW, STATES, sizeof(ForwardLds<TY, DK, NW, TILES>))) void delta_forward_kernel(const Args a) {
    typedef Geo<TY, DK, NW, TILES> G;
    typedef typename Elem<TY>::type E;
    __shared__ ForwardLds<TY, DK, NW, TILES> lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t b = blockIdx.x / in.value_heads, h = blockIdx.x % in.value_heads, hk = h / a.share;
    const int dk = in.key_dim, dv = in.value_dim, segment = blockIdx.y;
    const int begin = segment * a.segment_length, T = begin + min((int)in.length - begin, (int)a.segment_length);  // this segment's tokens
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
        load_state<DK, G::DV, FULL>(in.state ? in.state + bh * dk * dv : nullptr, dk, dv, dv, col0, lane, S);
    } else if (STATES) {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = unit && 16 * i + 4 * g + r == col0 + n ? 1.0f : 0.0f;
    } else {
        load_state<DK, G::DV, true>(a.starts + (bh * (a.segments - 1) + segment - 1) * (DK * G::DV), DK, G::DV, G::DV, col0, lane, S);
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
        int len = later ? __ffsll((unsigned long long)later) - 1 : lim - t;
        if (!STATES && a.saved && t && t % G::C == 0)
            store_state<DK, G::DV, true>(a.saved + (bh * (a.chunks - 1) + t / G::C - 1) * (DK * G::DV), DK, G::DV, G::DV, col0, lane, S);
        if (first) {
            any_cut = true;
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) S[i] = f4{0, 0, 0, 0};
        }

        if constexpr (!STATES) {
            bool fine = kr.raw.finite();  // no branch here either
            fine &= qr.raw.finite();
            fine |= !kr.mine();
            fine &= gv < __builtin_inff();
            fine &= finite(bv);
#pragma unroll
            for (int i = 0; i < TILES; ++i) fine &= finite(vr[i]);
            lds.odd[wave] = __ballot(!fine) != 0;
        }
        __syncthreads();  // the last chunk's operands are read
        if constexpr (!STATES) {
            uint32_t odd = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) odd |= lds.odd[w];
            len = __builtin_amdgcn_readfirstlane(odd) ? 1 : len;
        }
        f4 x[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) x[i] = turn(16 * i + row0 < len ? vr[i] : f4{0, 0, 0, 0}, lane);
        if (wave == NW - 1) load_scalars<TILES>(lane < len ? gv : 0.0f, lane < len ? bv : 0.0f, lane, first, lds.s);
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
            float* to = a.jumps + (bh * (a.segments - 1) + segment) * Jump<DK>::floats;
            if (col0 < DK) store_jump<DK>(reinterpret_cast<uint16_t*>(to), wave, lane, S);
            if (threadIdx.x == 0) to[Jump<DK>::size] = any_cut ? 0.0f : 1.0f;
        } else {
            store_state<DK, G::DV, true>(a.starts + (bh * (a.segments - 1) + segment) * (DK * G::DV), DK, G::DV, G::DV, col0, lane, S);
        }
    } else if (segment == (int)a.segments - 1)
        store_state<DK, G::DV, FULL>(a.last + bh * dk * dv, dk, dv, dv, col0, lane, S);
}

// ---- joining segments ------------------------------------------------------------------------
// The states between the segments from M and N of each: S_{p+1} = M_p S_p + N_p, in place of N.
// BACK: the same for the state's gradient from the last segment to the first, with M transposed.
// A workgroup joins 16 value columns of a head. Its four waves share the rows of the result; each
// step's state reaches them as a right operand through LDS, the matrices come from memory a step
// ahead. A wave has DK / 64 chains of DK / 32 x 6 matrix instructions a step, each behind the one before.
// Bound by the steps in a row: of 128 x 128 one takes 1.9 us (8 heads, 32 segments: 57 us), in which a CU
// draws 106 KB in; by the counters a wave waits for memory and LDS a quarter of that, its products take a
// sixth and the rest goes to their order. Loads two steps ahead gained 3%. More workgroups would each read all
// of a head's matrices again.
template <int DK, int DV, bool BACK>
__global__ __launch_bounds__(256) void delta_join_kernel(float* states, const float* jumps, int segments) {
    typedef Jump<DK> J;
    constexpr int TR = DK / 64;  // row tiles a wave
    __shared__ __attribute__((aligned(16))) uint16_t lds[2][J::steps * 3 * J::part];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col0 = 16 * blockIdx.y;
    const int64_t bh = blockIdx.x, between = segments - 1;
    // Between segments p and p + 1 lies state p; jump p leads from state p - 1 to state p.
    const int first = BACK ? segments - 2 : 0, last = BACK ? 0 : segments - 2, step = BACK ? -1 : 1;
    float* at = states + bh * between * (DK * DV) + (int64_t)wave * TR * 16 * DV;  // this wave's rows
    const float* jump = jumps + bh * between * J::floats;
    Frag<3> m[TR][J::steps];
    f4 N[TR];
    float passes;
    auto fetch = [&](int j, int to) {  // what leads to state `to`
        const float* from = jump + (int64_t)j * J::floats;
        const uint16_t* f = reinterpret_cast<const uint16_t*>(from) + (BACK ? J::size : 0) + wave * TR * J::row + lane * 8;
#pragma unroll
        for (int i = 0; i < TR; ++i)
#pragma unroll
            for (int c = 0; c < J::steps; ++c) m[i][c] = frag_at<3>(f + i * J::row + c * 3 * J::part, J::part);
        load_state<16 * TR, DV, true>(at + (int64_t)to * (DK * DV), 16 * TR, DV, DV, col0, lane, N);
        passes = from[J::size];
    };
    f4 S[TR];
    load_state<16 * TR, DV, true>(at + (int64_t)first * (DK * DV), 16 * TR, DV, DV, col0, lane, S);
    // Forward: from state p to p + 1 by jump p + 1. Back: from state p to p - 1 by jump p.
    fetch(BACK ? first : first + 1, first + step);
    for (int p = first; p != last; p += step) {
        uint16_t* buf = lds[p & 1];
#pragma unroll
        for (int i = 0; i < TR; ++i) {
            // Over a reset nothing passes, not even NaN times a zero matrix.
            const f4 x = passes == 0.0f ? f4{0, 0, 0, 0} : S[i];
            const int tile = wave * TR + i;
            put4<3>(buf + (tile >> 1) * 3 * J::part + lane * 8 + 4 * (tile & 1), J::part, x);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TR; ++i) S[i] = N[i];
#pragma unroll
        for (int c = 0; c < J::steps; ++c) {
            const Frag<3> sb = frag_at<3>(buf + c * 3 * J::part + lane * 8, J::part);
#pragma unroll
            for (int i = 0; i < TR; ++i) S[i] = mul<2>(m[i][c], sb, S[i]);
        }
        const int to = p + step;
        if (to != last) fetch(BACK ? to : to + 1, to + step);
        store_state<16 * TR, DV, true>(at + (int64_t)to * (DK * DV), 16 * TR, DV, DV, col0, lane, S);
    }
}

// ---- backward ------------------------------------------------------------------------------
// Chunks from the last to the first, dS' the gradient of the state after the chunk. With the
// matrices and solutions of the forward pass recomputed from the state before the chunk:
//     dU = P^T dO + D_C K dS';  (I + Z^T B) dR = dU;  dX = B dR;  dV = dX;  dbeta_i = dR_i . E_i
//     dS = gam_C dS' + scale (gam Q)^T dO - K^T (gam dX)
//     W = lower(D * dO U^T) scale;  Y = -strict_lower(D * dX U^T)
//     dQ = scale gam dO S^T + W K;  dK = D_C U dS'^T - gam dX S^T + W^T Q + (Y + Y^T) K
// The decay of token t is in every term that passes it, from a token before t (or the state) to t or
// a later token (or the end): with w_ij = W_ij (q_i . k_j) + Y_ij (k_i . k_j) between two tokens,
// f_i = scale gam_i q_i S . dO_i - gam_i k_i S . dX_i, e_j = D_Cj k_j dS' . U_j,
//     dg_t = sum over j < t <= i of w_ij + sum over i >= t of f_i + sum over j < t of e_j + gam_C <dS', S>
// Nothing in it cancels but what the signs make cancel: each term carries the decay itself, so the
// gradients of heads that forget fast, which are as small as exp(g), keep their digits. (dO_i . O_i - dV_i .
// V_i summed over i >= t, the same in exact numbers, left 1e-2 of them at g = -8 and nothing at -16.)
// f, e, dU and dX are column-local like the forward pass (phase A); w, dQ and dK sum over the value
// columns, whose operands (U, dX, dO, dS' transposed) go through LDS (phase B). No digit of fp32 is lost
// before dQ and dK are rounded: behind the norms they may be a small rest of large terms.
// What bounds it: instructions, and two workgroups a CU, as LDS and registers allow (in float16 and
// float32 one). Of a wave's 54,000 cycles a chunk 35% issue its 4,700 vector instructions and 37% wait for
// LDS, barriers and memory; the matrix units are busy 18% of two such waves' time (4096 sequences of 32,
// four heads of 64 x 64, bfloat16: 950 us, about 1.1 TB/s; 2 of 4096, 8 heads of 128 x 128: 260).

// What phase B multiplies, in LDS: as three parts, or in fp32 and split as it is read, which takes two thirds
// of the room and some time more (4096 sequences of 32 with gradients, four heads of 64 x 64: float32 1210 and
// 1272 us, float16 1086 and 1156). bfloat16 has it in fp32, with which two workgroups of four waves fit a
// CU, and float16 where 32 tokens of 128 columns would not fit at all as parts; the other kernels fit a CU
// once either way.
template <int TY, int C, int DV, int TILES> struct Held {
    static constexpr bool parts = TY == T_F32 || (TY == T_F16 && C * DV <= 2048);
    typedef std::conditional_t<parts, uint16_t, float> T;
    static constexpr int RS = parts ? DV + 8 : DV + 4, rows = (parts ? 3 : 1) * C * RS;               // along the head
    static constexpr int TS = parts ? Tok<TILES>::stride : C + 4, tokens = (parts ? 3 : 1) * C * TS;  // along the tokens
    // Four consecutive values of a row, from a multiple of four on.
    static __device__ __forceinline__ void put_row(T* m, int row, int col, f4 v) {
        if constexpr (parts) put4<3>(m + row * RS + col, C * RS, v);
        else *reinterpret_cast<f4*>(m + row * RS + col) = v;
    }
    static __device__ __forceinline__ void put_tokens(T* m, int row, int col, f4 v) {
        if constexpr (parts) put4<3>(m + row * TS + Tok<TILES>::slot_of(col), C * TS, v);
        else *reinterpret_cast<f4*>(m + row * TS + col) = v;
    }
    // Operands: eight consecutive values of a row, or a lane's values along the tokens.
    static __device__ __forceinline__ Frag<3> along_row(const T* m, int row, int col) {
        if constexpr (parts) return frag_at<3>(m + row * RS + col, C * RS);
        else return frag_of(m + row * RS + col);
    }
    static __device__ __forceinline__ auto along_tokens(const T* m, int row, int g) {
        if constexpr (parts) {
            return Tok<TILES>::template at<3>(m + row * TS, g, C * TS);
        } else {
            f4 x[TILES];
#pragma unroll
            for (int i = 0; i < TILES; ++i) x[i] = *reinterpret_cast<const f4*>(m + row * TS + 16 * i + 4 * g);
            return Tok<TILES>::template make<3>(x);
        }
    }
};

template <int TY, int DK, int NW, int TILES> struct BackwardLds {
    typedef Geo<TY, DK, NW, TILES> G;
    static constexpr int slab = DK < 64 ? DK : 64;  // rows of dS' that are in LDS at once
    static constexpr int SS = G::DV + 4, OS = DK + 4;
    typedef Held<TY, G::C, G::DV, TILES> H;
    alignas(16) uint16_t K[G::NP * G::C * G::KS], Q[G::NP * G::C * G::KS], KT[G::NP * DK * G::TS], QT[G::NP * DK * G::TS];
    alignas(16) uint16_t DO[G::NP * G::C * G::VS];
    union {
        InnerBack<TILES> m;  // phase A
        struct {             // phase B
            alignas(16) typename H::T W[H::tokens], WT[H::tokens], Y[H::tokens];
            alignas(16) float dS[slab * SS];
        } b;
    };
    union {
        struct { alignas(16) typename H::T U[H::rows], X[H::rows]; } c;
        struct { alignas(16) float q[G::C * OS], k[G::C * OS]; } out;
    };
    Scalars<TILES> s;
    float from[NW][G::C], end[NW][G::C], beta[NW][G::C], past[NW];  // sums over each wave's columns: f, e, of beta, <dS', S>
    alignas(16) float cross[2][TILES][G::C];  // sums of w over j < t <= i: W's and Y's, inside the 16 tokens of t and between the two 16
};

// Of a 16x16 result tile of terms between tokens (row i, column j): the sum over all columns before
// token t of the rows from t on (ALL: of all rows), for t = n + 1 in lane n; 0 in lane 15, where t is the next tile's.
template <bool ALL> __device__ __forceinline__ float sum_over(f4 w, int n, int g) {
    float y = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float x = w[r];
        if constexpr (!ALL) {
            x += dpp<0x111>(x);  // from 1, 2, 4 and 8 lanes before, within 16
            x += dpp<0x112>(x);
            x += dpp<0x114>(x);
            x += dpp<0x118>(x);
        }
        y += ALL || 4 * g + r > n ? x : 0.0f;
    }
    uint32_t b = __float_as_uint(y);
    auto rows = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    y = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    b = __float_as_uint(y);
    rows = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    y = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    if constexpr (ALL) {
        y += dpp<0x111>(y);
        y += dpp<0x112>(y);
        y += dpp<0x114>(y);
        y += dpp<0x118>(y);
    }
    return n == 15 ? 0.0f : y;
}
// The sum of all columns over each of this lane's rows and those below it.
__device__ __forceinline__ f4 sum_below(f4 w, int g) {
#pragma unroll
    for (int r = 0; r < 4; ++r) w[r] = sum16(w[r]);
    w[2] += w[3];
    w[1] += w[2];
    w[0] += w[1];
    const float y1 = from_group<1>(w[0]), y2 = from_group<2>(w[0]), y3 = from_group<3>(w[0]);
    const float y = g == 0 ? (y3 + y2) + y1 : g == 1 ? y3 + y2 : g == 2 ? y3 : 0.0f;
    return w + y;
}

// dR and dX = beta dR of dU + P^T dO, dU in du.
template <int TY, int TILES, class M>
__device__ __forceinline__ void solve_back(const M& m, const Scalars<TILES>& s, int n, int g, const f4* d_o, f4* du, f4* dr, f4* dx) {
    constexpr int tile = 16 * kInvStride, NP = Elem<TY>::parts, TS = Tok<TILES>::stride, part = 16 * TILES * TS;
    const f4 zero = {0, 0, 0, 0};
    const uint16_t* invT = m.inv + TILES * 3 * tile + n * kInvStride + 4 * g;
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
// states nor values: 72 us where the gradients' own pass takes 262 (2 sequences of 4096, 8 heads of
// 128 x 128, bfloat16).
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
    const int begin = segment * a.segment_length, T = begin + min((int)in.length - begin, (int)a.segment_length);
    const int col0 = wave * 16, row0 = 4 * g + (n & 3), col = col0 + (n & 12);
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2];
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2];
    const float* gp = in.g + b * in.g_stride[0] + h * in.g_stride[2];
    const float* bp = in.beta + b * in.beta_stride[0] + h * in.beta_stride[2];
    const uint8_t* rp = in.reset ? in.reset + b * in.reset_stride[0] : nullptr;
    const E* d_o = (const E*)a.d_o + b * a.d_o_stride[0] + h * a.d_o_stride[2] + col;
    const int64_t bh = b * in.value_heads + h;
    f4 dS[DK / 16];
    load_state<DK, G::DV, FULL>(a.d_last && segment == (int)a.segments - 1 ? a.d_last + bh * dk * dv : nullptr, dk, dv, dv, col0, lane, dS);
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
        if (wave == NW - 1)
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
    store_state<DK, G::DV, true>(a.d_starts + (bh * (a.segments - 1) + segment - 1) * (DK * G::DV), DK, G::DV, G::DV, col0, lane, dS);
}

template <int TY, int DK, int NW, int TILES, bool FULL>
__global__ __launch_bounds__(64 * NW, NW == 8 || sizeof(BackwardLds<TY, DK, NW, TILES>) <= 80 * 1024 ? 2 : 1) void delta_backward_kernel(const Args) {
    typedef Geo<TY, DK, NW, TILES> G;
    typedef BackwardLds<TY, DK, NW, TILES> L;
    typedef typename L::H H;
    typedef typename Elem<TY>::type E;
    constexpr int NP = G::NP, C = G::C;
    __shared__ L lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    // The arguments are read where they are used: as values held over the loop they would not fit
    // the scalar registers (two hundred spills, a tenth of the instructions).
    typedef const __attribute__((address_space(4))) Args* ArgsAt;
    ArgsAt ap = (ArgsAt)__builtin_amdgcn_kernarg_segment_ptr();
    const int64_t b = blockIdx.x / ap->in.value_heads, h = blockIdx.x % ap->in.value_heads, hk = h / ap->share;
    const int dk = ap->in.key_dim, dv = ap->in.value_dim, segment = blockIdx.y;
    const int begin = segment * ap->segment_length, T = begin + min((int)ap->in.length - begin, (int)ap->segment_length);  // this segment's tokens
    const int col0 = wave * 16, row0 = 4 * g + (n & 3), col = col0 + (n & 12);  // memory: four columns of a row
    const int64_t bh = b * ap->in.value_heads + h;

    f4 dS[DK / 16];  // the gradient of the state after the chunk
    if (segment == (int)ap->segments - 1) {
        load_state<DK, G::DV, FULL>(ap->d_last ? ap->d_last + bh * dk * dv : nullptr, dk, dv, dv, col0, lane, dS);
    } else {
        load_state<DK, G::DV, true>(ap->d_starts + (bh * (ap->segments - 1) + segment) * (DK * G::DV), DK, G::DV, G::DV, col0, lane, dS);
    }

    // What a chunk reads from memory.
    Rows<TY, DK, NW, TILES> kr, qr;
    Raw<TY> dor;
    f4 vr[TILES];
    float gv, bv;
    bool cut;
    constexpr int pieces_o = G::DV / 8;
    static_assert(C * pieces_o <= G::threads, "one piece a thread");
    const int row_o = threadIdx.x / pieces_o, e_o = 8 * (threadIdx.x % pieces_o);
    auto fetch = [&](int t, int te) {
        const ZenoAmdDeltaInputs __attribute__((address_space(4)))& in = ap->in;
        const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2];
        const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2];
        const E* v = (const E*)in.v + b * in.v_stride[0] + h * in.v_stride[2] + col;
        const E* d_o = (const E*)ap->d_o + b * ap->d_o_stride[0] + h * ap->d_o_stride[2];
        const float* gp = in.g + b * in.g_stride[0] + h * in.g_stride[2];
        const float* bp = in.beta + b * in.beta_stride[0] + h * in.beta_stride[2];
        const uint8_t* rp = in.reset ? in.reset + b * in.reset_stride[0] : nullptr;
        const int rows = te - t;
        const int64_t tok = t + min(lane, rows - 1);
        gv = gp[tok * in.g_stride[1]];
        bv = bp[tok * in.beta_stride[1]];
        cut = lane < rows && ((rp && rp[tok * in.reset_stride[1]]) || gv < kClears);
        kr.template fetch<FULL>(k + t * in.k_stride[1], in.k_stride[1], rows, dk, ap->k_vec);
        qr.template fetch<FULL>(q + t * in.q_stride[1], in.q_stride[1], rows, dk, ap->q_vec);
        if (C * pieces_o == G::threads || row_o < C) dor.template load<FULL>(d_o + (t + min(row_o, rows - 1)) * ap->d_o_stride[1] + e_o, dv - e_o, ap->d_o_vec);
#pragma unroll
        for (int i = 0; i < TILES; ++i) vr[i] = load4<TY, FULL>(v + (t + min(16 * i + row0, rows - 1)) * in.v_stride[1], dv - col, ap->v_vec);
    };
    for (int te = T; te > begin;) {
        asm volatile("" : "+s"(ap));
        // From the grid, and where a reset lies inside, once more from the last one.
        int t = (te - 1) / C * C;
        uint64_t cuts;
        for (;;) {
            fetch(t, te);
            cuts = __ballot(cut);
            if (cuts <= 1) break;
            t += 63 - __clzll((long long)cuts);
        }
        const bool first = cuts != 0;
        const int len = te - t;
        // The state before the chunk: nothing, the caller's, or a saved one.
        const float* sp = nullptr;
        int s_rows = dk, s_cols = dv, s_ld = dv;
        bool s_vec = ap->s_vec;
        if (!first) {
            if (t == 0) {
                if (ap->in.state) sp = ap->in.state + bh * dk * dv;
            } else {
                sp = ap->saved + (bh * (ap->chunks - 1) + t / C - 1) * (DK * G::DV);
                s_rows = DK, s_cols = s_ld = G::DV, s_vec = true;
            }
        }
        f4 S[DK / 16];
        load_state<DK, G::DV, FULL>(sp, s_rows, s_cols, s_ld, col0, lane, S);

        __syncthreads();
        if (wave == NW - 1) load_scalars<TILES>(lane < len ? gv : 0.0f, lane < len ? bv : 0.0f, lane, first, lds.s);
        kr.store(len, ap->in.normalize, lds.K, lds.KT, lds.s.rk);
        qr.store(len, ap->in.normalize, lds.Q, lds.QT, lds.s.rq);
        if (C * pieces_o == G::threads || row_o < C) {
            dor.keep(row_o < len);
            uint32_t w[4][NP];
            dor.parts(w);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<u4*>(lds.DO + (p * C + row_o) * G::VS + e_o) = u4{w[0][p], w[1][p], w[2][p], w[3][p]};
        }
        f4 vv[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) vv[i] = turn(16 * i + row0 < len ? vr[i] : f4{0, 0, 0, 0}, lane);
        __syncthreads();
        fill_inner<TY, DK, NW, TILES, TILES, W_PT | W_INV | W_INVT>(lds.K, lds.Q, lds.s, ap->in.scale, lds.m);

        // ---- phase A: this wave's columns
        asm volatile("" : "+s"(ap));
        f4 ks[TILES], o4[TILES], du[TILES], d4[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            ks[i] = o4[i] = du[i] = f4{0, 0, 0, 0};
            f4 x = {0, 0, 0, 0};
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) x += load4<T_BF16, true>(lds.DO + (p * C + 16 * i + row0) * G::VS + col, 4, true);
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
        f4 x[TILES], u[TILES], meet = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const f4 gam = row4(lds.s.gam, i, g), rk = row4(lds.s.rk, i, g);
            ks[i] *= gam * rk;
            x[i] = vv[i] - ks[i];
            o4[i] *= gam * row4(lds.s.rq, i, g) * ap->in.scale;
            du[i] *= row4(lds.s.end, i, g) * rk;
        }
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) meet += dS[i] * S[i];
        const float met = sum64((meet[0] + meet[1]) + (meet[2] + meet[3]));
        if (lane == 0) lds.past[wave] = met;
        __syncthreads();
        Half<3> up[TILES];
        solve<TILES, TILES>(lds.m, lds.s, n, g, x, u, up);
        const f4 zero = {0, 0, 0, 0};
        f4 dr[TILES], dx[TILES], en[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) en[i] = du[i] * u[i];
        solve_back<TY, TILES>(lds.m, lds.s, n, g, d4, du, dr, dx);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            f4 fr = d4[i] * o4[i] - dx[i] * ks[i], be = dr[i] * x[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) fr[r] = sum16(fr[r]), en[i][r] = sum16(en[i][r]), be[r] = sum16(be[r]);
            if (n == 0) {
                *reinterpret_cast<f4*>(lds.from[wave] + 16 * i + 4 * g) = fr;
                *reinterpret_cast<f4*>(lds.end[wave] + 16 * i + 4 * g) = en[i];
                *reinterpret_cast<f4*>(lds.beta[wave] + 16 * i + 4 * g) = be;
            }
            const f4 y = turn(dx[i], lane);
            H::put_row(lds.c.U, 16 * i + row0, col, turn(u[i], lane));
            H::put_row(lds.c.X, 16 * i + row0, col, y);
            if (16 * i + row0 < len) store4<TY, FULL>((E*)ap->dv + b * ap->dv_stride[0] + h * ap->dv_stride[2] + col + (t + 16 * i + row0) * ap->dv_stride[1], dv - col, ap->dv_vec, y);
        }
        __syncthreads();

        // ---- phase B: gradients of q and k
        asm volatile("" : "+s"(ap));
        constexpr int blocks = L::slab / 16, slabs = DK / L::slab;
        constexpr bool spread = NW >= 2 * blocks && TILES == 2;  // one tile a wave
        constexpr int rounds = spread ? 1 : (blocks + NW - 1) / NW, per = spread ? 1 : TILES;
        static_assert(rounds == 1, "one block of the slab a wave");
        const int blk = spread ? wave % blocks : wave, tile0 = spread ? wave / blocks : 0;
        const bool busy = blk < blocks && tile0 < TILES;
        // S transposed as a right operand: this lane's row of the key dimension, from memory. Rows and
        // columns outside the head are zero.
        f4 st[G::DV / 32][2];
        auto fetch_rows = [&](int sl) {
            const int row = sl * L::slab + 16 * blk + n;
            const bool ok = busy && sp && row < s_rows;
#pragma unroll
            for (int c = 0; c < G::DV / 32; ++c) {
                const int e = 32 * c + 8 * g;
                st[c][0] = st[c][1] = zero;
                if (ok) {
                    st[c][0] = load4<T_F32, FULL>(sp + row * s_ld + e, s_cols - e, s_vec);
                    st[c][1] = load4<T_F32, FULL>(sp + row * s_ld + e + 4, s_cols - e - 4, s_vec);
                }
            }
        };
        fetch_rows(0);
        // W and Y + Y^T (times the norms of the rows that they multiply), a tile a wave; and w's sums.
        constexpr int pairs = TILES * (TILES + 1) / 2;
#pragma unroll
        for (int job = 0; job < 2 * pairs; ++job) {
            const int pair = job % pairs, ti = pair > 0 ? 1 : 0, tj = pair > 1 ? 1 : 0, j = 16 * tj + n;
            if (wave != (NW >= 2 * pairs ? job : pair)) continue;
            f4 acc = zero, mirror = zero, dot = zero;
#pragma unroll
            for (int c = 0; c < DK / 32; ++c)
                dot = mul<2>(frag_at<NP>((job < pairs ? lds.Q : lds.K) + (16 * ti + n) * G::KS + 32 * c + 8 * g, C * G::KS),
                             frag_at<NP>(lds.K + j * G::KS + 32 * c + 8 * g, C * G::KS), dot);
#pragma unroll
            for (int c = 0; c < G::DV / 32; ++c) {
                const int e = 32 * c + 8 * g;
                const Frag<3> uf = H::along_row(lds.c.U, 16 * tj + n, e);
                if (job < pairs) {
                    acc = mul<2>(frag_at<NP>(lds.DO + (16 * ti + n) * G::VS + e, C * G::VS), uf, acc);
                } else {
                    const Frag<3> xf = H::along_row(lds.c.X, 16 * ti + n, e);
                    acc = mul<2>(xf, uf, acc);
                    if (ti == tj) mirror = mul<2>(uf, xf, mirror);  // the tile's transpose
                }
            }
            const float hj = lds.s.hi[j], lj = lds.s.lo[j], rj = lds.s.rk[j];
            const f4 hi = row4(lds.s.hi, ti, g), lo = row4(lds.s.lo, ti, g), nr = row4(job < pairs ? lds.s.rq : lds.s.rk, ti, g);
            f4 by_col, by_row, w;  // times the norm of the column's token, of the row's, and times the product
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * g + r;
                const float d = (hi[r] - hj) + (lo[r] - lj);
                float y;
                if (job < pairs) y = j <= i ? acc[r] * __expf(d) * ap->in.scale : 0.0f;
                else if (ti != tj) y = -acc[r] * __expf(d);
                else y = j == i ? 0.0f : -(j < i ? acc[r] : mirror[r]) * __expf(j < i ? d : -d);
                by_col[r] = y * rj;
                by_row[r] = y * nr[r];
                w[r] = j < i ? by_col[r] * nr[r] * dot[r] : 0.0f;
            }
            if (ti == tj) {
                const float y = sum_over<false>(w, n, g);
                if (g == 0) lds.cross[job >= pairs][0][16 * ti + ((n + 1) & 15)] = y;
            } else {
                const float y = sum_over<true>(w, n, g);
                if (g == 0) lds.cross[job >= pairs][TILES - 1][(n + 1) & 15] = y;
                const f4 z = sum_below(w, g);
                if (n == 0) *reinterpret_cast<f4*>(lds.cross[job >= pairs][TILES - 1] + 16 + 4 * g) = z;
            }
            // Rows of a matrix along tokens, and of its transpose.
            auto rows_out = [&](typename H::T* m, f4 v, int ti, int tj) { H::put_tokens(m, 16 * ti + row0, 16 * tj + (n & 12), turn(v, lane)); };
            auto cols_out = [&](typename H::T* m, f4 v, int ti, int tj) { H::put_tokens(m, 16 * tj + n, 16 * ti + 4 * g, v); };
            rows_out(job < pairs ? lds.b.W : lds.b.Y, by_col, ti, tj);
            if (job < pairs) cols_out(lds.b.WT, by_row, ti, tj);
            if (job < pairs && ti != tj) {  // above the diagonal
                rows_out(lds.b.W, zero, tj, ti);
                rows_out(lds.b.WT, zero, ti, tj);
            } else if (ti != tj) cols_out(lds.b.Y, by_row, ti, tj);
        }
        f4 dq[slabs * per], dkk[slabs * per];
#pragma unroll
        for (int sl = 0; sl < slabs; ++sl) {
            if (sl) __syncthreads();
#pragma unroll
            for (int i = 0; i < L::slab / 16; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) lds.b.dS[(16 * i + 4 * g + r) * L::SS + col0 + n] = dS[sl * (L::slab / 16) + i][r];
            __syncthreads();
            // Waves without a block multiply what they hold and drop it: no branch around matrix instructions.
            const int row = sl * L::slab + 16 * (blk % blocks) + n;  // of the key dimension: this lane's column of the results
            const int t1 = tile0 % TILES;
            f4 aq[per], ar[per], ac[per];
#pragma unroll
            for (int i = 0; i < per; ++i) aq[i] = ar[i] = ac[i] = zero;
#pragma unroll
            for (int c = 0; c < G::DV / 32; ++c) {
                const int e = 32 * c + 8 * g;
                const Frag<3> sf = split<3>(st[c][0], st[c][1]), df = frag_of(lds.b.dS + (16 * (blk % blocks) + n) * L::SS + e);
#pragma unroll
                for (int i = 0; i < per; ++i) {
                    const int row = 16 * (t1 + i) + n;
                    aq[i] = mul<2>(frag_at<NP>(lds.DO + row * G::VS + e, C * G::VS), sf, aq[i]);
                    ar[i] = mul<2>(H::along_row(lds.c.X, row, e), sf, ar[i]);
                    ac[i] = mul<2>(H::along_row(lds.c.U, row, e), df, ac[i]);
                }
            }
            if (sl + 1 < slabs) fetch_rows(sl + 1);
            const auto kt = Tok<TILES>::template at<NP>(lds.KT + row * G::TS, g, DK * G::TS);
            const auto qt = Tok<TILES>::template at<NP>(lds.QT + row * G::TS, g, DK * G::TS);
#pragma unroll
            for (int i = 0; i < per; ++i) {
                const int ti = t1 + i, at = 16 * ti + n;
                const f4 gam = row4(lds.s.gam, ti, g);
                f4 yq = aq[i] * gam * ap->in.scale, yk = ac[i] * row4(lds.s.end, ti, g) - ar[i] * gam;
                yk = mul<2>(H::along_tokens(lds.b.Y, at, g), kt, yk);
                yq = mul<2>(H::along_tokens(lds.b.W, at, g), kt, yq);
                yk = mul<2>(H::along_tokens(lds.b.WT, at, g), qt, yk);
                dq[sl * per + i] = yq;
                dkk[sl * per + i] = yk;
            }
        }
        // the state's gradient, from this wave's columns
        pull_state<TY, DK, TILES>(lds.KT, lds.QT, lds.s, ap->in.scale, n, g, d4, dx, dS);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) dS[i] = first ? zero : dS[i];
        __syncthreads();  // U and dX are read
        if (wave == NW - 1) {
            // f of this token and the later ones, e of those before it, in 64 bits
            double later = 0.0, before = 0.0, past = 0.0;
            float bsum = 0.0f, w = 0.0f;
            if (lane < C) {
#pragma unroll
                for (int v = 0; v < NW; ++v) {
                    later += (double)lds.from[v][lane];
                    if (lane) before += (double)lds.end[v][lane - 1];
                    past += (double)lds.past[v];
                    bsum += lds.beta[v][lane];
                }
#pragma unroll
                for (int i = 0; i < TILES; ++i) w += lds.cross[0][i][lane] + lds.cross[1][i][lane];
            }
            later += dpp64<0x101>(later);
            later += dpp64<0x102>(later);
            later += dpp64<0x104>(later);
            later += dpp64<0x108>(later);
            before += dpp64<0x111>(before);
            before += dpp64<0x112>(before);
            before += dpp64<0x114>(before);
            before += dpp64<0x118>(before);
            if constexpr (TILES == 2) {
                const double behind = from_lane(later, 16);
                if (lane < 16) later += behind;
                before += dpp64<0x142>(before);
            }
            if (lane < len) {
                const float sum = (float)(later + before + (double)lds.s.gam[C - 1] * past + (double)w);
                ap->dg[b * ap->dg_stride[0] + (t + lane) * ap->dg_stride[1] + h * ap->dg_stride[2]] = first && lane == 0 ? 0.0f : sum;
                ap->dbeta[b * ap->dbeta_stride[0] + (t + lane) * ap->dbeta_stride[1] + h * ap->dbeta_stride[2]] = bsum;
            }
        }
        if (busy)
#pragma unroll
            for (int sl = 0; sl < slabs; ++sl)
#pragma unroll
                for (int i = 0; i < per; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = (16 * (tile0 + i) + 4 * g + r) * L::OS + sl * L::slab + 16 * blk + n;
                        lds.out.q[at] = dq[sl * per + i][r];
                        lds.out.k[at] = dkk[sl * per + i][r];
                    }
        __syncthreads();
        asm volatile("" : "+s"(ap));
        // rows out, through the norms: d(x / |x|) = (d - x^ (x^ . d)) / |x|, |x|^2 with its eps; of
        // one dimension alone that is d eps / |x|^3, which the difference would lose to rounding
        constexpr int pieces = DK / 8;
        const int row = threadIdx.x / pieces, e = 8 * (threadIdx.x % pieces);
        if (C * pieces == G::threads || row < C) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float* from = (w ? lds.out.k : lds.out.q) + row * L::OS + e;
                f4 y0 = *reinterpret_cast<const f4*>(from), y1 = *reinterpret_cast<const f4*>(from + 4);
                if (ap->in.normalize) {
                    const float nr = w ? lds.s.rk[row] : lds.s.rq[row];
                    const uint16_t* src = (w ? lds.K : lds.Q) + row * G::KS;
                    f4 x0 = zero, x1 = zero;
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) {
                        x0 += load4<T_BF16, true>(src + p * C * G::KS + slot(e), 4, true);
                        x1 += load4<T_BF16, true>(src + p * C * G::KS + slot(e + 4), 4, true);
                    }
                    x0 *= nr;
                    x1 *= nr;
                    const f4 d = x0 * y0 + x1 * y1;
                    float dot = d[0] + d[1] + d[2] + d[3];
                    if (pieces > 8) dot += dpp<0x128>(dot);
                    dot += dpp<0x141>(dot);
                    dot += dpp<0x1b>(dot);
                    dot += dpp<0xb1>(dot);
                    if (dk == 1) {
                        y0 *= kNormEps * nr * nr * nr;
                    } else {
                        y0 = (y0 - x0 * dot) * nr;
                        y1 = (y1 - x1 * dot) * nr;
                    }
                }
                if (row < len) {
                    const float y[8] = {y0[0], y0[1], y0[2], y0[3], y1[0], y1[1], y1[2], y1[3]};
                    if (ap->part_q) {
                        float* to = (w ? ap->part_k : ap->part_q) + ((b * ap->in.length + t + row) * ap->in.value_heads + h) * dk + e;
                        store8<T_F32, FULL>(to, dk - e, dk % 8 == 0, y);
                    } else if (w) {
                        store8<TY, FULL>((E*)ap->dk + b * ap->dk_stride[0] + (t + row) * ap->dk_stride[1] + hk * ap->dk_stride[2] + e, dk - e, ap->dk_vec, y);
                    } else {
                        store8<TY, FULL>((E*)ap->dq + b * ap->dq_stride[0] + (t + row) * ap->dq_stride[1] + hk * ap->dq_stride[2] + e, dk - e, ap->dq_vec, y);
                    }
                }
            }
        }
        te = t;
    }
    if (ap->d_state && segment == 0) store_state<DK, G::DV, FULL>(ap->d_state + bh * dk * dv, dk, dv, dv, col0, lane, dS);
}

// Sums the value heads of each key head, in their order; a thread a value, several where there are more
// than 2^28 (a launch takes less than 2^32 threads). Memory-bound and small: 4 us
// of 250 (19 sequences of 333 tokens, two value heads a key head, fp32).
template <int TY> __global__ __launch_bounds__(256) void delta_share_kernel(const Args a) {
    typedef typename Elem<TY>::type E;
    const ZenoAmdDeltaInputs& in = a.in;
    const int64_t all = (int64_t)in.batch * in.length * in.key_heads * in.key_dim;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += (int64_t)gridDim.x * 256) {
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
}

// ---- one token -----------------------------------------------------------------------------
// The state is read once and written once (8 bytes a value and step: bound by memory; 4096
// environments, four heads of 64 x 64, 106 us, 5.2 TB/s, the rate of a copy). A wave
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
        if (a.segments > 2) delta_join_kernel<DK, 16 * NW, false><<<dim3(heads, NW), 256, 0, stream>>>(a.starts, a.jumps, a.segments);
    }
    delta_forward_kernel<TY, DK, NW, TILES, FULL, false><<<dim3(heads, a.segments), 64 * NW, 0, stream>>>(a);
}
template <int TY, int DK, int NW, int TILES, bool FULL> void backward_shape(const Args& a, hipStream_t stream) {
    const uint32_t heads = a.in.batch * a.in.value_heads;
    if (a.segments > 1) {
        delta_pull_kernel<TY, DK, NW, TILES, FULL><<<dim3(heads, a.segments - 1), 64 * NW, 0, stream>>>(a);
        if (a.segments > 2) delta_join_kernel<DK, 16 * NW, true><<<dim3(heads, NW), 256, 0, stream>>>(a.d_starts, a.jumps, a.segments);
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
        const int64_t blocks = (all + 255) / 256, most = 1 << 20;
        delta_share_kernel<TY><<<dim3((uint32_t)(blocks < most ? blocks : most)), 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

template <int TY> hipError_t launch_step(const Args& a, float* state, hipStream_t stream) {
    const ZenoAmdDeltaInputs& in = a.in;
    const bool vec = in.value_dim % 4 == 0 && (uintptr_t)state % 16 == 0;
    const dim3 grid((uint32_t)((step_waves(in) + 3) / 4));
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
