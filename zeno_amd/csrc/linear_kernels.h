// Kernels of linear attention with a decay for each head: walks over whole sequences, and the
// single-token step.
//
// A chunk is one or two tiles of 16 tokens. With S the state before it, a walk forward is
//     P_ij = scale exp(g (i - j)) A_i . B_j  for j <= i with no reset after j up to i, else 0
//     out  = P C + scale exp(g (i + 1)) A S      (the second where no reset is before or at i)
//     S'   = exp(g L) S + sum_j exp(g (L - 1 - j)) B_j C_j^T      (L tokens; nothing across a reset)
// and a walk back the same with the tokens' order reversed. The decays of a head are one number, so
// they are a table in registers that is made once.
//
// A wave owns 32 or 64 columns of the state, all of its rows, and works alone: no LDS, no barrier. That leaves no
// wait but for memory, and the vector instructions bound it: of 16384 tokens of 8 heads of 128 x 128, float16, each of a SIMD's two
// waves issues them 40 % of its time and keeps the matrix units busy for 23 % (outputs 95 us). Many short sequences are bound by
// memory: 16384 of 16 tokens, two heads of 64 x 64, bfloat16: 1.34 GB in 269 us, 5.0 TB/s.
// Rows are read as they lie, 16 bytes a lane: lane (n, g) has row n's dimensions 8 g to 8 g + 7 of
// every 32. That is an operand of the matrix units as it is, for contractions along the dimensions.
// The other operands come from results without an exchange: a result tile has its rows in registers and
// its columns in lanes, as operands have their contraction index and their other one. So P is computed
// transposed and is then an operand along its tokens; the state's tiles are operands along its rows; and
// B and C along the tokens are their rows' product with a unit matrix. P and the state are operands in three parts, so all
// of fp32, in every type (two, 2^-17 of a term, took up to 20 % less, but where terms cancel that is no small part of the sum). To let eight contiguous dimensions
// meet the four registers of two tiles, row 4 g + r of tile h of a pair stands for dimension 8 g + 4 h + r.
// Outputs are computed transposed, so that a lane has eight contiguous columns of its token.
//
// Gradient of g: every term between tokens i and j is (i - j) times itself, so with the slope
// N <- exp(g) (N + S), the state's derivative, beside the state, it is a sum over tokens of q . (A N) and
// of products inside the chunk. No difference is taken, so heads that forget fast keep their digits.
//
// From a chunk on that holds a value that is not finite, a walk goes token by token on the vector units, so that none
// meets an output before its token, or behind a reset, by way of the zeros in P, or another column by way of those in
// the unit matrix. So do heads whose decays are so far above one that a chunk's would pass fp32's range.
// There is one body for the chunk: with others for resets and for odd values beside it the compiler needed 168 registers
// and spilled where 100 do.
#pragma once
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "linear.h"
#include "rows.h"

namespace za {
namespace linear {

using namespace mma;

// exp(g m), off by an ulp or two for large products too.
__device__ __forceinline__ float decay(float g, float m) {
    constexpr float l2e = 1.44269504f, rest = 1.92596303e-8f, ln2 = 0.693147181f;  // log2(e) in two floats
    const float x = g * m, low = __builtin_fmaf(g, m, -x), p = x * l2e;
    const float e = __builtin_fmaf(x, l2e, -p) + __builtin_fmaf(x, rest, low * l2e);
    return __builtin_amdgcn_exp2f(p) * __builtin_fmaf(e, ln2, 1.0f);
}

// x exp(g m) as part of it times a power of two: where exp(g m) passes fp32's range a zero stays zero, and a small x is no
// infinity before its time.
struct Grown {
    float part;
    int twos;
    __device__ __forceinline__ Grown(float g, float m) {
        constexpr float l2e = 1.44269504f, rest = 1.92596303e-8f, ln2 = 0.693147181f;
        const float x = g * m, low = __builtin_fmaf(g, m, -x), p = x * l2e, e = __builtin_fmaf(x, l2e, -p) + __builtin_fmaf(x, rest, low * l2e);
        const bool far = fabsf(p) > 600.0f;  // all of fp32's range and its like below zero
        const float whole = far ? copysignf(600.0f, p) : ceilf(p);
        part = far ? 0.5f : __builtin_amdgcn_exp2f(p - whole - 1.0f) * __builtin_fmaf(e, ln2, 1.0f);
        twos = (int)whole + 1;
    }
    __device__ __forceinline__ float operator()(float x) const { return __builtin_ldexpf(x * part, twos); }
};

template <int TY> __device__ __forceinline__ Frag<Elem<TY>::parts> operand(const Eight<TY>& x) {
    uint32_t w[4][Elem<TY>::parts];
    x.parts(w);
    Frag<Elem<TY>::parts> f;
#pragma unroll
    for (int p = 0; p < Elem<TY>::parts; ++p) f.p[p] = u4{w[0][p], w[1][p], w[2][p], w[3][p]};
    return f;
}

// A row's eight values as an operand for products with other rows: 16-bit types as they are, for the matrix
// instructions of their own type, float32 in three parts.
template <int TY> struct Own {
    static constexpr int parts = TY == T_F32 ? 3 : 1;
    static constexpr uint32_t one = TY == T_F16 ? 0x3c00u : 0x3f80u;  // of the parts' type
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Frag<parts> make(const Eight<TY>& x) {
        if constexpr (TY == T_F32) return operand(x);
        else return Frag<1>{{x.a[0]}};
    }
    template <int PB> static __device__ __forceinline__ f4 product(const Frag<parts>& a, const Frag<PB>& b, f4 acc) {
        if constexpr (TY == T_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a.p[0]), __builtin_bit_cast(h8, b.p[0]), acc, 0, 0, 0);
        else return mul<2>(a, b, acc);
    }
    // Four of a lane's eight, with 16 along the contraction.
    static __device__ __forceinline__ f4 product(const Half<parts>& a, const Half<1>& b, f4 acc) {
        if constexpr (TY == T_F16) return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, a.p[0]), __builtin_bit_cast(h4, b.p[0]), acc, 0, 0, 0);
        else return mul<2>(a, b, acc);
    }
};
template <int P> __device__ __forceinline__ Half<P> four_of(const Frag<P>& f, int i) {
    Half<P> h;
#pragma unroll
    for (int p = 0; p < P; ++p) h.p[p] = i ? u2{f.p[p][2], f.p[p][3]} : u2{f.p[p][0], f.p[p][1]};
    return h;
}
// acc[i] + A[i] B, the smallest part products first, those of one weight side by side as they do not wait for one another.
template <int N, class A, class B> __device__ __forceinline__ void mul_each(const A* a, const B& b, f4* acc) {
    constexpr int PA = sizeof(a->p) / sizeof(a->p[0]), PB = sizeof(b.p) / sizeof(b.p[0]);
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int x = 0; x < PA; ++x)
            if (s - x >= 0 && s - x < PB)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (sizeof(a->p[0]) == 16)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a[i].p[x]), __builtin_bit_cast(bf8, b.p[s - x]), acc[i], 0, 0, 0);
                    else
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a[i].p[x]), __builtin_bit_cast(s4, b.p[s - x]), acc[i], 0, 0, 0);
                }
}

// Four floats at any address, the first `n` of them in bounds.
template <bool FULL> __device__ __forceinline__ f4 load_floats(const float* at, int n) {
    if (FULL || n >= 4) return __builtin_bit_cast(f4, reinterpret_cast<const Loose<T_F32>::U*>(at)->v);
    f4 x = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) x[i] = at[i];
    return x;
}
template <bool FULL> __device__ __forceinline__ void store_floats(float* at, int n, f4 x) {
    if (FULL || n >= 4) {
        reinterpret_cast<Loose<T_F32>::U*>(at)->v = __builtin_bit_cast(u4, x);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) at[i] = x[i];
    }
}

// This lane's number, found anew: what depends on it is then not kept in registers from use to use. (The empty asm hides
// where the zero comes from; it holds no instruction, so the compiler's waits stay right.)
__device__ __forceinline__ int lane_anew() {
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}

// Operands along the tokens of a chunk: of two tiles or of one.
template <int TILES> struct Along;
template <> struct Along<2> {
    template <int P> using Op = Frag<P>;
    template <int P> static __device__ __forceinline__ Frag<P> make(const f4* x) { return split<P>(x[0], x[1]); }
};
template <> struct Along<1> {
    template <int P> using Op = Half<P>;
    template <int P> static __device__ __forceinline__ Half<P> make(const f4* x) { return split<P>(x[0]); }
};

// One walk of one wave in one segment of one head: of 64 or 32 columns of the state (JS 4 or 2 tiles of 16), or of
// every other four of 32 (JS 1: tile `half` of the pair).
template <int TY, int STEPS, int TILES, int JS, bool BACK, int KIND, bool FULL>
__device__ __forceinline__ void walk(const Walk& a, const uint32_t bh, const uint32_t segment, const int block, const int half, const uint32_t unit) {
    typedef typename Elem<TY>::type E;
    constexpr int NP = Elem<TY>::parts, C = 16 * TILES;
    constexpr bool OUT = KIND == OUTPUTS, SLOPE = KIND == SLOPES || KIND == STATES_SLOPE, GRAD = KIND == SLOPES, READ = OUT || GRAD;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int64_t b = bh / a.heads, h = bh % a.heads;
    const int begin = segment * a.segment_length, T = begin + min(a.length - begin, a.segment_length);
    constexpr int U = (JS + 1) / 2;  // times 32 columns
    const int col0 = block * 32 * U;
    const int da = a.da, dc = a.dc - col0;
    float gh = a.g[h];  // before anything else, as loads come back in order
    auto rows_of = [&](const Rows& x) { return (const E*)x.at + b * x.stride[0] + (h / x.share) * x.stride[2]; };
    const E* ap = READ ? rows_of(a.a) : nullptr;
    const E* bp = rows_of(a.b);
    const E* cp = rows_of(a.c) + col0;
    const E* qp = GRAD ? rows_of(a.q) + col0 : nullptr;
    const uint8_t* rp = a.reset ? a.reset + b * a.reset_stride[0] : nullptr;

    // ---- what a chunk reads: dimensions 8 g to 8 g + 7 of every 32, of token n of each tile of 16
    Eight<TY> ar[TILES][STEPS], br[TILES][STEPS], cr[TILES][U], qr[TILES];
    bool cut = false, any_cut = false;
    auto fetch = [&](int t, int rows) {
        cut = rp && lane < rows && rp[(t + lane) * a.reset_stride[1]];
#pragma unroll
        for (int k = 0; k < TILES; ++k) {
            const int row = min(16 * k + n, rows - 1);
            auto place = [&](const E* x, const Rows& r) { return x + t * r.stride[1] + (row * r.stride[1] + 8 * g); };
            const E* x = place(bp, a.b);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) br[k][s].template load<FULL>(x + 32 * s, da - 32 * s - 8 * g);
            if constexpr (READ) {
                x = place(ap, a.a);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) ar[k][s].template load<FULL>(x + 32 * s, da - 32 * s - 8 * g);
            }
            x = place(cp, a.c);
#pragma unroll
            for (int u = 0; u < U; ++u) cr[k][u].template load<FULL>(x + 32 * u, dc - 32 * u - 8 * g);
            if constexpr (GRAD) qr[k].template load<FULL>(place(qp, a.q), dc - 8 * g);
        }
    };
    auto bounds = [&](int at, int& t, int& rows) {  // the chunk of the grid that `at` is in, from it (or up to it) on
        if (BACK) {
            t = begin + (at - 1 - begin) / C * C;
            rows = at - t;
        } else {
            t = at;
            rows = min(T, begin + ((at - begin) / C + 1) * C) - t;
        }
    };
    int at = BACK ? T : begin, t, rows;
    bounds(at, t, rows);
    fetch(t, rows);

    // ---- the state, by row tiles of 16 (pairs of them make 32 rows) and column tiles
    f4 S[2 * STEPS][JS], N[SLOPE ? 2 * STEPS : 1][JS];
    // A lane takes four values that lie side by side: of one of four rows, which four lanes then exchange, or of a
    // column where columns lie side by side (`turned`). Places are found anew each time: kept from the walk's begin
    // to its end they would not fit the registers.
    auto each_four = [&](auto&& access) {
        const int m = lane_anew(), mn = m & 15, mg = m >> 4;
        const int mine = a.turned ? (8 * (mn >> 2) + (mn & 3)) * a.ld + 8 * mg : (8 * mg + (mn & 3)) * a.ld + 8 * (mn >> 2);
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int j = 0; j < JS; ++j) {
                const int row = 32 * (i >> 1) + 4 * (i & 1), col = JS == 1 ? 4 * half : 32 * (j >> 1) + 4 * (j & 1);
                const int base = a.turned ? (col0 + col) * a.ld + row : row * a.ld + col0 + col;
                int left = 4;
                if (!FULL) {
                    if (a.turned) left = 8 * (mn >> 2) + (mn & 3) + col < dc ? da - row - 8 * mg : 0;
                    else left = 8 * mg + (mn & 3) + row < da ? dc - col - 8 * (mn >> 2) : 0;
                }
                access(i, j, base, mine, left);
            }
    };
    auto load_state = [&](auto& X, const float* from) {
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int j = 0; j < JS; ++j) X[i][j] = f4{0, 0, 0, 0};
        if (from) each_four([&](int i, int j, int base, int mine, int left) { X[i][j] = load_floats<FULL>(from + base + mine, left); });
    };
    auto turn_state = [&](auto& X) {
        if (a.turned) return;
        const int m = lane_anew();
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int j = 0; j < JS; ++j) {
                X[i][j] = turn(X[i][j], m);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    auto store_state = [&](auto& X, float* to) {
        turn_state(X);
        each_four([&](int i, int j, int base, int mine, int left) { store_floats<FULL>(to + base + mine, left, X[i][j]); });
    };
    const bool at_first = BACK ? segment == a.segments - 1 : segment == 0;
    const int64_t between = (int64_t)bh * (a.segments - 1) + (BACK ? segment : segment - 1);  // the start of this walk
    load_state(S, at_first ? (a.first ? a.first + bh * a.size : nullptr) : READ ? a.starts + between * a.size : nullptr);
    if constexpr (SLOPE) load_state(N, READ && !at_first ? a.slopes + between * a.size : nullptr);

    // ---- the head's decays between the tokens of a chunk of `len` with resets in `cuts`; 0 across a reset, and where
    // a token is behind the other. `read`: of the state to a token, `write`: of a token to the next state, `all`: of
    // the state to the next. None is over more than `len` tokens: behind the last token zeros are multiplied by them, which must not be infinite.
    gh = gh < -200.0f ? -200.0f : gh;  // 0 in fp32 from one token to the next
    constexpr int tile_pairs = TILES == 2 ? 3 : 1;  // each tile with itself, and the first with the second
    float near[tile_pairs][4], read[TILES], all;
    f4 write[TILES];
    int measured;
    uint32_t measured_cuts;
    auto measure = [&](int len, uint32_t cuts) {
        measured = len;
        measured_cuts = cuts;
        const int m = lane_anew(), i0 = m & 15, j0 = 4 * (m >> 4);
        all = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(decay(gh, len))));
#pragma unroll
        for (int k = 0; k < TILES; ++k) {
            const int i = 16 * k + i0;
            read[k] = BACK ? decay(gh, max(len - 1 - i, 0)) : a.scale * decay(gh, min(i + 1, len));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * k + j0 + r;
                write[k][r] = BACK ? a.scale * decay(gh, min(j + 1, len)) : decay(gh, max(len - 1 - j, 0));
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int apart = BACK ? j0 + r - i0 : i0 - j0 - r;
            near[0][r] = apart < 0 ? 0.0f : a.scale * decay(gh, min(max(apart, 0), len));
            if constexpr (TILES == 2) {
                near[1][r] = near[0][r];
                near[2][r] = a.scale * decay(gh, min(16 + apart, len));
            }
        }
        if (cuts) {
            const int last = 31 - __builtin_clz(cuts), first = __builtin_ctz(cuts);
            auto reset_to = [&](int token) { return 31 - __clz((int)(cuts & (0xffffffffu >> (31 - token)))); };  // the last one up to it
            all = 0.0f;
#pragma unroll
            for (int k = 0; k < TILES; ++k) {
                const int i = 16 * k + i0;
                if (BACK ? i < last : reset_to(i) >= 0) read[k] = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * k + j0 + r;
                    if (BACK ? j >= first : j < last) write[k][r] = 0.0f;
                    if (BACK ? i < reset_to(j) : j < reset_to(i)) near[k][r] = 0.0f;
                }
            }
            if constexpr (TILES == 2)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (BACK ? i0 < reset_to(16 + j0 + r) : j0 + r < reset_to(16 + i0)) near[2][r] = 0.0f;
        }
    };

    // A unit matrix as an operand. With four of a lane's eight values (dimensions 8 g + 4 i + 0..3 of a row's 32) it
    // gives a tile whose column n is dimension 8 (n / 4) + 4 i + n % 4.
    Half<1> unit_matrix;
#pragma unroll
    for (int w = 0; w < 2; ++w) unit_matrix.p[0][w] = g == (n >> 2) && ((n & 3) >> 1) == w ? Own<TY>::one << (16 * (n & 1)) : 0u;
    double dg = 0.0;

    // The chunk's rows as operands, and the products of A's with B's, row j = 16 tj + 4 g + r, column i = 16 ti + n: P without
    // its decays. Returns whether all that was read is finite, which these products tell, and sums of rows where they do
    // not. (A look at every value was a third of a chunk's vector instructions.)
    Frag<Own<TY>::parts> ao[TILES][STEPS], bo[TILES][STEPS], co[TILES][U];
    f4 p[tile_pairs];
    auto products = [&](int rows, uint32_t cuts) {
        const f4 zero = {0, 0, 0, 0};
        if (rows < C)
#pragma unroll
            for (int k = 0; k < TILES; ++k) {
                const bool keep = 16 * k + n < rows;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    br[k][s].keep(keep);
                    if constexpr (READ) ar[k][s].keep(keep);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) cr[k][u].keep(keep);
                if constexpr (GRAD) qr[k].keep(keep);
            }
        Frag<1> ones;
        ones.p[0] = u4{Own<TY>::one * 0x10001u, Own<TY>::one * 0x10001u, Own<TY>::one * 0x10001u, Own<TY>::one * 0x10001u};
        bool fine = true;
#pragma unroll
        for (int k = 0; k < tile_pairs; ++k) p[k] = zero;
#pragma unroll
        for (int k = 0; k < TILES; ++k) {
            f4 sums = zero;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                bo[k][s] = Own<TY>::make(br[k][s]);
                if constexpr (READ) {
                    ao[k][s] = Own<TY>::make(ar[k][s]);
                    p[k] = Own<TY>::product(bo[k][s], ao[k][s], p[k]);
                } else {
                    sums = Own<TY>::product(bo[k][s], ones, sums);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                co[k][u] = Own<TY>::make(cr[k][u]);
                sums = Own<TY>::product(co[k][u], ones, sums);
            }
            if constexpr (GRAD) sums = Own<TY>::product(Own<TY>::make(qr[k]), ones, sums);
            fine &= finite(sums);
        }
        if constexpr (READ && TILES == 2)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) p[2] = Own<TY>::product(bo[BACK ? 1 : 0][s], ao[BACK ? 0 : 1][s], p[2]);
        if constexpr (READ)
#pragma unroll
            for (int k = 0; k < tile_pairs; ++k) fine &= finite(p[k]);
        if (cuts) {  // nothing of the state passes: it must not be multiplied by zero if it is not finite
            asm volatile("");  // a branch, not a look at every chunk
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
                for (int j = 0; j < JS; ++j) {
                    fine &= finite(S[i][j]);
                    if constexpr (SLOPE) fine &= finite(N[i][j]);
                }
        }
        return __ballot(!fine) == 0;
    };

    // The chunk of tokens t to t + len. But for the stores of 32 columns, between the products of two column tiles, no branch is
    // inside: where one lies between a matrix instruction and the use of its result, the compiler has been seen to leave out
    // the wait (tests/test_matrix_waits.py follows every path of what it made). The scheduler is kept from starting everything at
    // once, which takes more registers than there are.
    auto chunk = [&](int t, int len) {
        const f4 zero = {0, 0, 0, 0};
        // ---- B along the tokens, P
        typename Along<TILES>::template Op<NP> bt[2 * STEPS];
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i) {
            f4 x[TILES];
#pragma unroll
            for (int k = 0; k < TILES; ++k) x[k] = Own<TY>::product(four_of(bo[k][i >> 1], i & 1), unit_matrix, zero);
            bt[i] = Along<TILES>::template make<NP>(x);
            if (i & 1) __builtin_amdgcn_sched_barrier(0);
        }
        Frag<NP> af[TILES][STEPS];
        if constexpr (READ)
#pragma unroll
            for (int k = 0; k < TILES; ++k)
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if constexpr (TY == T_F16) af[k][s] = operand(ar[k][s]);
                    else af[k][s] = ao[k][s];
                }
        constexpr int one = BACK ? TILES - 1 : 0;  // the tile whose tokens see no other
        Half<3> alone;
        Frag<3> both;
        float pairs = 0.0f;
        if constexpr (READ) {
#pragma unroll
            for (int k = 0; k < tile_pairs; ++k) {
                f4 y = zero;
                const int ti = k < 2 ? k : BACK ? 0 : 1, tj = k < 2 ? k : 1 - ti;
                if constexpr (GRAD) y = Own<TY>::product(co[tj][0], Own<TY>::make(qr[ti]), zero);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[k][r] *= near[k][r];
                    if (GRAD) pairs += (float)(16 * (ti - tj) + n - 4 * g - r) * p[k][r] * y[r];
                }
            }
            alone = split<3>(p[one]);
            if constexpr (TILES == 2) both = BACK ? split<3>(p[0], p[2]) : split<3>(p[2], p[1]);
        }
        if (GRAD && JS == 1) pairs = half ? 0.0f : pairs;  // once for the two waves of these columns
        float out[TILES][U][8];
#pragma unroll
        for (int j = 0; j < JS; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            f4 ct[TILES];
#pragma unroll
            for (int k = 0; k < TILES; ++k) {
                auto cj = four_of(co[k][j >> 1], j & 1);
                if (JS == 1)
#pragma unroll
                    for (int p = 0; p < Own<TY>::parts; ++p) cj.p[p] = half ? four_of(co[k][0], 1).p[p] : cj.p[p];
                ct[k] = Own<TY>::product(cj, unit_matrix, zero);
            }
            if constexpr (READ) {
                f4 x[TILES], slope[TILES];
#pragma unroll
                for (int k = 0; k < TILES; ++k) x[k] = slope[k] = zero;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const Frag<3> sf = split<3>(S[2 * s][j], S[2 * s + 1][j]);
#pragma unroll
                    for (int k = 0; k < TILES; ++k) x[k] = mul<2>(sf, af[k][s], x[k]);
                    if constexpr (GRAD) {
                        const Frag<3> nf = split<3>(N[2 * s][j], N[2 * s + 1][j]);
#pragma unroll
                        for (int k = 0; k < TILES; ++k) slope[k] = mul<2>(nf, af[k][s], slope[k]);
                    }
                }
#pragma unroll
                for (int k = 0; k < TILES; ++k) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[k][r] = read[k] != 0.0f ? x[k][r] * read[k] : 0.0f;
                    if constexpr (GRAD) {
                        float q[8];
                        qr[k].get(q);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            pairs += ((float)(16 * k + n + 1) * x[k][r] + (read[k] != 0.0f ? slope[k][r] * read[k] : 0.0f)) * (JS == 1 ? half ? q[4 + r] : q[r] : q[4 * (j & 1) + r]);
                    }
                }
                if constexpr (OUT) {
                    x[one] = mul<2>(split<NP>(ct[one]), alone, x[one]);
                    if constexpr (TILES == 2) x[1 - one] = mul<2>(split<NP>(ct[0], ct[1]), both, x[1 - one]);
#pragma unroll
                    for (int k = 0; k < TILES; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) out[k][j >> 1][4 * (j & 1) + r] = x[k][r];
                }
            }
            // ---- the state behind the chunk
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < TILES; ++k) ct[k] *= write[k];
            const auto wf = Along<TILES>::template make<3>(ct);
            if constexpr (SLOPE) {
#pragma unroll
                for (int k = 0; k < TILES; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) ct[k][r] *= (float)max(len - 1 - 16 * k - 4 * g - r, 0);
                const auto nf = Along<TILES>::template make<3>(ct);
                f4 x[2 * STEPS];
#pragma unroll
                for (int i = 0; i < 2 * STEPS; ++i) x[i] = (N[i][j] + S[i][j] * (float)len) * all;
                mul_each<2 * STEPS>(bt, nf, x);
#pragma unroll
                for (int i = 0; i < 2 * STEPS; ++i) N[i][j] = x[i];
            }
            f4 x[2 * STEPS];
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) x[i] = S[i][j] * all;
            mul_each<2 * STEPS>(bt, wf, x);
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) S[i][j] = x[i];
            // ---- 32 columns of the outputs
            if constexpr (OUT)
                if (j & 1) {
                    const int l = lane_anew(), u = j >> 1;
#pragma unroll
                    for (int k = 0; k < TILES; ++k) {
                        const int row = 16 * k + (l & 15);
                        const int64_t to = (b * a.out_stride[0] + h * a.out_stride[2] + t * a.out_stride[1] + col0 + 32 * u) + (row * a.out_stride[1] + 8 * (l >> 4));
                        if (row < len) {
                            if (a.out_f32) {
                                Eight<T_F32> x;
                                x.set(out[k][u]);
                                x.template store<FULL>((float*)a.out + to, dc - 32 * u - 8 * g);
                            } else {
                                Eight<TY> x;
                                x.set(out[k][u]);
                                x.template store<FULL>((E*)a.out + to, dc - 32 * u - 8 * g);
                            }
                        }
                    }
                }
        }
        if (GRAD) dg += (double)pairs;
    };

    // The rest of the walk token by token, without the matrix units: of values that are not finite their zeros would
    // make NaN where the definition has none, and heads that grow fast have no table of decays. The state goes through memory and the walk does not come back from
    // here, so that this rare path takes no registers from the other (with a way back each chunk moved the whole state
    // to other registers).
    auto tokens = [&](int from, int to) {  // in order of time
        volatile float kept[SLOPE ? 2 : 1][2 * STEPS][4][JS];
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < JS; ++j) {
                    kept[0][i][r][j] = S[i][j][r];
                    if (SLOPE) kept[SLOPE][i][r][j] = N[i][j][r];
                }
        const int m = lane_anew();
        const Grown next(gh, 1.0f);
#pragma unroll 1
        for (int k = from; k < to; ++k) {
            const int64_t tok = BACK ? from + to - 1 - k : k;
            const bool cut = rp && rp[tok * a.reset_stride[1]];
            any_cut |= cut;
            float o[JS], v[JS], slope[JS];
            int c[JS];
#pragma unroll
            for (int j = 0; j < JS; ++j) {
                c[j] = 8 * (m >> 2 & 3) + (m & 3) + (JS == 1 ? 4 * half : 32 * (j >> 1) + 4 * (j & 1));
                v[j] = (c[j] < dc ? Elem<TY>::get(cp[tok * a.c.stride[1] + c[j]]) : 0.0f) * (BACK ? a.scale : 1.0f);
                o[j] = slope[j] = 0.0f;
            }
#pragma unroll 1
            for (int i = 0; i < 8 * STEPS; ++i) {
                const int d = 32 * (i >> 3) + 8 * (m >> 4) + (i & 7);
                const float B = d < da ? Elem<TY>::get(bp[tok * a.b.stride[1] + d]) : 0.0f;
                const float A = READ && d < da ? Elem<TY>::get(ap[tok * a.a.stride[1] + d]) : 0.0f;
#pragma unroll
                for (int j = 0; j < JS; ++j) {
                    float x = kept[0][i >> 2][i & 3][j];
                    if constexpr (SLOPE) {
                        const float y = cut ? 0.0f : next(kept[1][i >> 2][i & 3][j] + x);
                        kept[1][i >> 2][i & 3][j] = y;
                        slope[j] += y * A;
                    }
                    if (!BACK) x = cut ? 0.0f : next(x);
                    x += B * v[j];
                    o[j] += x * A;
                    if (BACK) x = cut ? 0.0f : next(x);
                    kept[0][i >> 2][i & 3][j] = x;
                }
            }
#pragma unroll
            for (int j = 0; j < JS; ++j) {
                o[j] += __shfl_xor(o[j], 16);
                o[j] += __shfl_xor(o[j], 32);
                if (OUT && m < 16 && c[j] < dc) {
                    const int64_t to = b * a.out_stride[0] + h * a.out_stride[2] + tok * a.out_stride[1] + col0 + c[j];
                    const float y = o[j] * (BACK ? 1.0f : a.scale);
                    if (a.out_f32) ((float*)a.out)[to] = y;
                    else ((E*)a.out)[to] = Elem<TY>::put(y);
                }
                if constexpr (GRAD)
                    if (c[j] < dc && !cut) dg += (double)(a.scale * slope[j] * Elem<TY>::get(qp[tok * a.q.stride[1] + c[j]]));
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < JS; ++j) {
                    S[i][j][r] = kept[0][i][r][j];
                    if (SLOPE) N[i][j][r] = kept[SLOPE][i][r][j];
                }
    };

    // ---- the walk. Nothing is fetched ahead: more waves a SIMD, for which that leaves no registers, hide more.
    uint32_t cuts = (uint32_t)__ballot(cut);
    measure(rows, cuts);
    turn_state(S);  // which has arrived by now
    if constexpr (SLOPE) turn_state(N);
    bool more = true;
    // A head that grows by more than exp(40) in a chunk goes token by token from the start: the chunk's decays, of which only
    // zeros meet some, must be no infinities, and leave room for the products that they are multiplied with.
    const bool steep = __ballot(gh * (float)min(C, a.length) > 40.0f) != 0;
    bool fine = products(rows, cuts) && !steep;
    while (more && fine) {  // with one way out, else the state moves to other registers in every round
        any_cut |= cuts != 0;
        chunk(t, rows);
        at = BACK ? t : t + rows;
        more = BACK ? at > begin : at < T;
        if (more) {
            bounds(at, t, rows);
            fetch(t, rows);
            cuts = (uint32_t)__ballot(cut);
            if (rows != measured || cuts != measured_cuts) measure(rows, cuts);
            fine = products(rows, cuts);
        }
    }
    if (more) tokens(BACK ? begin : t, BACK ? at : T);

    // ---- what it leaves
    if constexpr (OUT) {
        if (a.last && (BACK ? segment == 0 : segment == a.segments - 1)) store_state(S, a.last + bh * a.size);
    } else if constexpr (GRAD) {
        if (a.d_last && segment == a.segments - 1) {
            load_state(S, a.d_last + bh * a.size);
            turn_state(S);
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
                for (int j = 0; j < JS; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) dg += S[i][j][r] == 0.0f ? 0.0 : (double)(S[i][j][r] * N[i][j][r]);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) dg += __shfl_xor(dg, d);
        if (lane == 0) a.parts[unit] = dg;
    } else {
        const int64_t to = (int64_t)bh * (a.segments - 1) + (BACK ? segment - 1 : segment);
        store_state(S, a.starts + to * a.size);
        if constexpr (SLOPE) store_state(N, a.slopes + to * a.size);
        if (block == 0 && half == 0 && lane == 0) a.passes[to] = any_cut ? 0.0f : 1.0f;
    }
}

// Waves read the rows that their neighbours read, and workgroups go to the eight dies in turn: each die is given a
// range of its own. Returns the number of this wave's work.
template <int WAVES> __device__ __forceinline__ uint32_t unit_of_wave() {
    const uint32_t each = gridDim.x / 8;  // the grid is a multiple of 8
    return __builtin_amdgcn_readfirstlane(((blockIdx.x & 7) * each + (blockIdx.x >> 3)) * WAVES + (threadIdx.x >> 6));
}

// Waves a SIMD that the registers are cut down to: as many as the state, its rows and their operands bear without
// spilling, which costs more than a wave gains (27 registers spilled: 415 us, none 306; 16384 sequences of 16, two heads of 64 x 64).
constexpr int walk_waves(int type, int steps, int tiles, int js, int kind) {
    if (type == T_F32) return steps == 4 && (kind == OUTPUTS || kind == SLOPES) ? 1 : steps == 1 ? 3 : 2;
    if (js == 2 && kind == SLOPES) return 2;
    return tiles == 2 || steps == 4 || (js == 4 && steps == 2) ? 2 : kind == SLOPES || type == T_F16 ? 3 : 4;
}
constexpr int gradient_waves(int type, int steps, int tiles, int js, bool learned) {
    return learned ? std::min(walk_waves(type, steps, tiles, js, OUTPUTS), walk_waves(type, steps, 1, slope_tiles(steps, js), SLOPES)) : walk_waves(type, steps, tiles, js, OUTPUTS);
}

template <int TY, int STEPS, int TILES, int JS, bool BACK, int KIND, bool FULL>
__global__ __launch_bounds__(256, walk_waves(TY, STEPS, TILES, JS, KIND)) void linear_walk_kernel(const Walk a) {
    constexpr bool READ = KIND == OUTPUTS;
    const uint32_t walks = READ ? a.segments : a.segments - 1;  // of the segments, all but the last in the walk's direction
    const uint32_t unit = unit_of_wave<4>(), block = unit / (JS == 1 ? 2 : 1) % a.blocks, rest = unit / (JS == 1 ? 2 : 1) / a.blocks;
    const uint32_t bh = rest / walks, segment = rest % walks + (!READ && BACK ? 1 : 0);
    if (bh >= a.batch * a.heads) return;
    walk<TY, STEPS, TILES, JS, BACK, KIND, FULL>(a, bh, segment, block, JS == 1 ? unit & 1 : 0, unit);
}

// All gradients: the walks of d_v, d_k and d_q of a head and segment side by side, as they read the same rows: of 4096
// sequences of 32 tokens, four heads of 64 x 64, in bfloat16, 346 us (one after the other 490 where this took 366). Where the decays are
// learned the walk of their gradient too: 471 us (behind the others 366 and 235, this 520); 19 sequences of 333, four heads of 24 x 48,
// float32: 35 (34 and 25, this 36). A workgroup is one wave, as the walks take unlike times (of four, the first three: 400, this 366).
// Bound by neither of memory and instructions: caches hold the second and third readings (788 MB read, 462 written, what they
// cannot be without is 804 and 470), which flow at 3.6 TB/s, as a wave reads, multiplies, stores and ends, and two a SIMD overlap.
struct Walks {
    Walk v, k, q;
    uint32_t slopes;  // waves of the decays' gradient, for each head and segment
};
template <int TY, int STEPS, int TILES, int JS, bool FULL, bool LEARNED>
__global__ __launch_bounds__(64, gradient_waves(TY, STEPS, TILES, JS, LEARNED)) void linear_gradients_kernel(const Walks a) {
    const uint32_t back = a.v.blocks + a.k.blocks, outputs = back + a.q.blocks, waves = outputs + (LEARNED ? a.slopes : 0), unit = unit_of_wave<1>(), rest = unit / waves;
    const uint32_t bh = rest / a.v.segments, segment = rest % a.v.segments;
    if (bh >= a.v.batch * a.v.heads) return;
    const uint32_t at = unit % waves;
    if (at < back) {
        const bool v = at < a.v.blocks;
        walk<TY, STEPS, TILES, JS, true, OUTPUTS, FULL>(v ? a.v : a.k, bh, segment, v ? at : at - a.v.blocks, 0, 0);
    } else if (!LEARNED || at < outputs) {
        walk<TY, STEPS, TILES, JS, false, OUTPUTS, FULL>(a.q, bh, segment, at - back, 0, 0);
    } else {
        constexpr int SJ = slope_tiles(STEPS, JS);
        const uint32_t s = at - outputs;
        walk<TY, STEPS, 1, SJ, false, SLOPES, FULL>(a.q, bh, segment, SJ == 1 ? s / 2 : s, SJ == 1 ? s & 1 : 0, rest * a.slopes + s);
    }
}

// ---- joining segments ------------------------------------------------------------------------
// The states between segments from what each adds: S_{p+1} = exp(g L) S_p + U_p, in place of U, where
// the segment passes a state at all; and the slopes, N_{p+1} = exp(g L) (N_p + L S_p) + V_p. A thread a value;
// eight segments' values are read at once, as each read waits for memory. Bound by those waits: 64 segments of 8 heads of
// 128 x 128, 33 MB read and written: 14 us, 4.8 TB/s of which caches hold most; with slopes and 32 segments of 16 heads 21.
template <bool BACK, bool SLOPE> __global__ __launch_bounds__(256) void linear_join_kernel(const Walk a) {
    const int64_t between = a.segments - 1, blocks = (a.size + 255) / 256;
    const int64_t bh = blockIdx.x / blocks, at = blockIdx.x % blocks * 256 + threadIdx.x;
    if (at >= a.size) return;
    float gh = a.g[bh % a.heads];
    gh = gh < -200.0f ? -200.0f : gh;
    const Grown whole(gh, a.segment_length);
    float* starts = a.starts + bh * between * a.size + at;
    float* slopes = SLOPE ? a.slopes + bh * between * a.size + at : nullptr;
    const float* passes = a.passes + bh * between;
    float S = 0.0f, N = 0.0f;
    for (int64_t k0 = 0; k0 < between; k0 += 8) {
        float U[8], V[8], pass[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k0 + k >= between) continue;
            const int64_t p = BACK ? between - 1 - k0 - k : k0 + k;
            U[k] = starts[p * a.size];
            if (SLOPE) V[k] = slopes[p * a.size];
            pass[k] = passes[p];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k0 + k >= between) continue;
            const int64_t p = BACK ? between - 1 - k0 - k : k0 + k;
            const bool through = k0 + k > 0 && pass[k] != 0.0f;  // nothing, NaN included, passes a reset
            if (SLOPE) {
                N = through ? V[k] + whole(N + (float)a.segment_length * S) : V[k];
                slopes[p * a.size] = N;
            }
            S = through ? U[k] + whole(S) : U[k];
            starts[p * a.size] = S;
        }
    }
}

// Sums the value heads of each key head, in their order, for q and for k (blockIdx.y); a thread a value, several where there
// are more than 2^28 (a launch takes less than 2^32 threads). Bound by memory, of which the parts in fp32 are most.
struct Shared {
    const float* parts[2];
    void* out[2];
    int64_t stride[2][3], all;
    uint32_t length, heads, share, dim;
};
template <int TY> __global__ __launch_bounds__(256) void linear_share_kernel(const Shared a) {
    typedef typename Elem<TY>::type E;
    const float* parts = a.parts[blockIdx.y];
    E* out = (E*)a.out[blockIdx.y];
    const int64_t* stride = a.stride[blockIdx.y];
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < a.all; id += (int64_t)gridDim.x * 256) {
        const int64_t x = id % a.dim, h = id / a.dim % a.heads, bt = id / a.dim / a.heads;
        const float* from = parts + (bt * a.heads + h) * a.share * a.dim + x;
        float sum = 0.0f;
        for (uint32_t s = 0; s < a.share; ++s) sum += from[(int64_t)s * a.dim];
        out[bt / a.length * stride[0] + bt % a.length * stride[1] + h * stride[2] + x] = Elem<TY>::put(sum);
    }
}

// ---- one token -----------------------------------------------------------------------------
// The state is read once and written once. A wave holds all rows of 4 LANES columns, 16 (or 4) rows and 4
// columns a lane:  o = scale (a S^T q + (k . q) v),  S <- a S + k v^T.  LANES lanes lie along the
// columns, 64 / LANES along the rows. Bound by memory: 4096 sequences of four heads of 64 x 64, 0.55 GB of state in 118 us,
// 4.6 TB/s.
template <int TY, int LANES, int ROWS, bool VEC>
__global__ __launch_bounds__(256) void linear_step_kernel(const ZenoAmdLinearInputs in, void* out, int64_t o_batch, int64_t o_head, float* state) {
    typedef typename Elem<TY>::type E;
    const int lane = threadIdx.x & 63, cl = lane % LANES, rg = lane / LANES;
    const int dk = in.key_dim, dv = in.value_dim;
    const uint32_t blocks = (dv + 4 * LANES - 1) / (4 * LANES);
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t bh = id / blocks;
    const int col = ((int)(id % blocks) * LANES + cl) * 4, row0 = rg * ROWS;
    if (bh >= (int64_t)in.batch * in.value_heads) return;
    const int64_t b = bh / in.value_heads, h = bh % in.value_heads, hk = h / (in.value_heads / in.key_heads);
    const E* q = (const E*)in.q + b * in.q_stride[0] + hk * in.q_stride[2] + row0;
    const E* k = (const E*)in.k + b * in.k_stride[0] + hk * in.k_stride[2] + row0;
    const E* v = (const E*)in.v + b * in.v_stride[0] + h * in.v_stride[2] + col;
    const bool first = in.reset && in.reset[b * in.reset_stride[0]];
    const float g = in.g[h];
    float a = first ? 0.0f : expf(g);
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
    float kv[ROWS], qv[ROWS];
    f4 vv;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        kv[i] = row0 + i < dk ? Elem<TY>::get(k[i]) : 0.0f;
        qv[i] = row0 + i < dk ? Elem<TY>::get(q[i]) : 0.0f;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = col + c < dv ? Elem<TY>::get(v[c]) : 0.0f;
    if (g > 80.0f && !first) {  // exp(g) may pass fp32's range
        const Grown grown(g, 1.0f);
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) S[i][c] = grown(S[i][c]);
        a = 1.0f;
    }
    float kq = 0.0f;
    f4 sq = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        kq += kv[i] * qv[i];
        sq += S[i] * qv[i];
    }
#pragma unroll
    for (int d = LANES; d < 64; d <<= 1) {
        kq += __shfl_xor(kq, d);
#pragma unroll
        for (int c = 0; c < 4; ++c) sq[c] += __shfl_xor(sq[c], d);
    }
    if (rg == 0) {
        E* o = (E*)out + b * o_batch + h * o_head + col;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (col + c < dv) o[c] = Elem<TY>::put(in.scale * (a * sq[c] + kq * vv[c]));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (row0 + i >= dk) continue;
        const f4 y = S[i] * a + vv * kv[i];
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
inline dim3 walk_grid(uint64_t units, int waves) { return dim3((uint32_t)((units + 8 * waves - 1) / (8 * waves) * 8)); }

// Runs launch(steps, tiles, js, full) with the launch shape as constants, and sets the walks' number of blocks.
// Waves of 64 columns where the registers bear them and enough of them come of it for two a SIMD: they read and multiply
// A and B once where two of 32 do it twice (4096 sequences of 32, four heads of 64 x 64, bfloat16: 167 us, 191; with gradients, float32:
// 667, 778; but 100 of them with gradients, bfloat16: 30, 25), and where none of the 64 is idle that
// 32 would spare (gradients of 1000 sequences of 64, four heads of 32 x 64, float16: 163 us, 106). Chunks of two tiles where
// the registers bear them: what is done to the state, its parts as operands and its decay, is done for 32 tokens at once
// (the same 4096 sequences with gradients, bfloat16: 517, 588). With 128 rows those of the states between segments do, those of the outputs
// do not (2 of 4096 tokens, 8 heads of 128 x 128, bfloat16: outputs 43 us and gradients 159; two tiles, 63 and 261 registers spilled: 53 and 191).
template <int TY, class F> void by_shape(int steps, std::initializer_list<Walk*> walks, bool outputs, F&& launch) {
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    int blocks = 0, halves = 0;  // of 64 columns and of 32
    for (const Walk* w : walks) {
        blocks += (w->dc + 63) / 64;
        halves += (w->dc + 31) / 32;
    }
    const Walk& w0 = **walks.begin();
    const bool four_tiles = wide((uint64_t)w0.batch * w0.heads * w0.segments, blocks, halves), tall = w0.length > 16;
    auto by_steps = [&](auto s) {
        constexpr int STEPS = decltype(s)::value;
        auto by_full = [&](auto tiles, auto js) {
            constexpr int width = 16 * decltype(js)::value;
            bool full = true;
            for (Walk* w : walks) {
                w->blocks = (w->dc + width - 1) / width;
                full = full && w->da == 32 * STEPS && w->dc % width == 0;
            }
            full ? launch(s, tiles, js, std::true_type{}) : launch(s, tiles, js, std::false_type{});
        };
        auto by_tiles = [&](auto js) {
            if constexpr (TY == T_BF16 || (TY == T_F16 && STEPS == 1)) {
                if (tall && !(STEPS == 4 && outputs)) return by_full(two, js);
            }
            by_full(one, js);
        };
        if constexpr (STEPS < 4) {
            if (four_tiles) return by_tiles(four);
        }
        by_tiles(two);
    };
    if (steps == 1) by_steps(one);
    else if (steps == 2) by_steps(two);
    else by_steps(four);
}

template <int TY> hipError_t launch_walk(Walk w, Kind kind, bool back, hipStream_t stream) {
    const bool read = kind == OUTPUTS;
    hipError_t shape = hipErrorInvalidValue;  // of no kernel
    by_shape<TY>(steps_of(w.da), {&w}, read, [&](auto steps, auto tiles, auto js, auto is_full) {
        constexpr int STEPS = decltype(steps)::value, TILES = decltype(tiles)::value, JS = decltype(js)::value;
        constexpr bool FULL = decltype(is_full)::value;
        const uint64_t walks = (uint64_t)w.batch * w.heads * (read ? w.segments : w.segments - 1);
        auto run = [&](auto kernel, uint64_t waves) {
            kernel<<<walk_grid(waves, 4), 256, 0, stream>>>(w);
            shape = hipSuccess;
        };
        if (kind == STATES_SLOPE) {
            w.blocks = (w.dc + 31) / 32;
            run(linear_walk_kernel<TY, STEPS, TILES, 1, false, STATES_SLOPE, FULL>, walks * w.blocks * 2);
        } else if (kind == OUTPUTS) {
            if constexpr (STEPS < 4 || TILES == 1) run(linear_walk_kernel<TY, STEPS, TILES, JS, false, OUTPUTS, FULL>, walks * w.blocks);
        } else if constexpr (JS == 2) {
            if (back) run(linear_walk_kernel<TY, STEPS, TILES, 2, true, STATES, FULL>, walks * w.blocks);
            else run(linear_walk_kernel<TY, STEPS, TILES, 2, false, STATES, FULL>, walks * w.blocks);
        }
    });
    if (shape != hipSuccess) return shape;
    if (!read && w.segments > 2) {
        const dim3 join(w.batch * w.heads * (uint32_t)((w.size + 255) / 256));
        if (back) linear_join_kernel<true, false><<<join, 256, 0, stream>>>(w);
        else if (kind == STATES) linear_join_kernel<false, false><<<join, 256, 0, stream>>>(w);
        else linear_join_kernel<false, true><<<join, 256, 0, stream>>>(w);
    }
    return hipGetLastError();
}

// Sets `slopes` to the waves of each head and segment that leave a part of the decays' gradient.
template <int TY> hipError_t launch_gradients(Walk v, Walk k, Walk q, uint32_t* slopes, hipStream_t stream) {
    hipError_t shape = hipErrorInvalidValue;  // of no kernel
    by_shape<TY>(std::max(steps_of(v.da), steps_of(k.da)), {&v, &k, &q}, true, [&](auto steps, auto tiles, auto js, auto full) {
        constexpr int STEPS = decltype(steps)::value, TILES = decltype(tiles)::value, JS = decltype(js)::value;
        constexpr bool FULL = decltype(full)::value;
        if constexpr ((STEPS > 1 || JS == 2) && (STEPS < 4 || TILES == 1)) {  // with 32 rows at most there are 32 columns at most
            *slopes = q.parts ? (q.dc + 31) / 32 * (2 / slope_tiles(STEPS, JS)) : 0;
            const Walks all{v, k, q, *slopes};
            const dim3 grid = walk_grid((uint64_t)v.batch * v.heads * v.segments * (v.blocks + k.blocks + q.blocks + *slopes), 1);
            if (q.parts) linear_gradients_kernel<TY, STEPS, TILES, JS, FULL, true><<<grid, 64, 0, stream>>>(all);
            else linear_gradients_kernel<TY, STEPS, TILES, JS, FULL, false><<<grid, 64, 0, stream>>>(all);
            shape = hipSuccess;
        }
    });
    return shape != hipSuccess ? shape : hipGetLastError();
}

template <int TY> hipError_t launch_share(const ZenoAmdLinearInputs& in, const float* part_q, const float* part_k, const ZenoAmdLinearGradients& grad, hipStream_t stream) {
    Shared a{{part_q, part_k}, {grad.d_q, grad.d_k}, {}, (int64_t)in.batch * in.length * in.key_heads * in.key_dim, in.length, in.key_heads, in.value_heads / in.key_heads, in.key_dim};
    for (int i = 0; i < 3; ++i) {
        a.stride[0][i] = grad.d_q_stride[i];
        a.stride[1][i] = grad.d_k_stride[i];
    }
    linear_share_kernel<TY><<<dim3((uint32_t)std::min<int64_t>((a.all + 255) / 256, 1 << 20), 2), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <int TY> hipError_t launch_step(const ZenoAmdLinearInputs& in, void* o, const int64_t* o_stride, float* state, hipStream_t stream) {
    const bool vec = in.value_dim % 4 == 0 && (uintptr_t)state % 16 == 0;
    const dim3 grid((uint32_t)((step_waves(in) + 3) / 4));
    auto by_shape = [&](auto lanes, auto rows) {
        constexpr int LANES = decltype(lanes)::value, ROWS = decltype(rows)::value;
        if (vec) linear_step_kernel<TY, LANES, ROWS, true><<<grid, 256, 0, stream>>>(in, o, o_stride[0], o_stride[2], state);
        else linear_step_kernel<TY, LANES, ROWS, false><<<grid, 256, 0, stream>>>(in, o, o_stride[0], o_stride[2], state);
    };
    constexpr std::integral_constant<int, 4> four{};
    constexpr std::integral_constant<int, 8> eight{};
    constexpr std::integral_constant<int, 16> sixteen{};
    if (in.key_dim <= 32) by_shape(eight, four);
    else if (in.key_dim <= 64) by_shape(sixteen, sixteen);
    else by_shape(eight, sixteen);
    return hipGetLastError();
}

}  // namespace linear
}  // namespace za
