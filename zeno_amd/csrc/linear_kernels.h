// Kernels of linear attention with a decay for each head: walks over whole sequences, and the
// single-token step.
//
// A chunk is 32 tokens (16 where registers are short). With S the state before it, a walk forward is
//     P_ij = scale exp(g (i - j)) A_i . B_j  for j <= i with no reset after j up to i, else 0
//     out  = P C + scale exp(g (i + 1)) A S      (the second where no reset is before or at i)
//     S'   = exp(g L) S + sum_j exp(g (L - 1 - j)) B_j C_j^T      (L tokens; nothing across a reset)
// and a walk back the same with the tokens' order reversed. The decays of a head are one number, so
// they are a table in registers that is made once.
//
// A wave owns 32 columns of the state, all of its rows, and works alone: no LDS, no barrier.
// Rows are read as they lie, 16 bytes a lane: lane (n, g) has row n's dimensions 8 g to 8 g + 7 of
// every 32. That is an operand of the matrix units as it is, for contractions along the dimensions.
// The other operands come from results without an exchange: a result tile has its rows in registers and
// its columns in lanes, as operands have their contraction index and their other one. So P is computed
// transposed and is then an operand along its tokens; the state's tiles are operands along its rows; and
// B and C along the tokens are their rows' product with a unit matrix. To let eight contiguous dimensions
// meet the four registers of two tiles, row 4 g + r of tile h of a pair stands for dimension 8 g + 4 h + r.
// Outputs are computed transposed, so that a lane has eight contiguous columns of its token.
//
// Gradient of g: every term between tokens i and j is (i - j) times itself, so with the slope
// N <- exp(g) (N + S), the state's derivative, beside the state, it is a sum over tokens of q . (A N) and
// of products inside the chunk. No difference is taken, so heads that forget fast keep their digits.
//
// A chunk that holds a value that is not finite goes token by token, so that none meets an output before
// its token, or behind a reset, by way of the zeros in P.
#pragma once
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

template <int TY> __device__ __forceinline__ Frag<Elem<TY>::parts> operand(const Eight<TY>& x) {
    uint32_t w[4][Elem<TY>::parts];
    x.parts(w);
    Frag<Elem<TY>::parts> f;
#pragma unroll
    for (int p = 0; p < Elem<TY>::parts; ++p) f.p[p] = u4{w[0][p], w[1][p], w[2][p], w[3][p]};
    return f;
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

template <int TY, int STEPS, int TILES, bool AHEAD, bool BACK, int KIND, bool FULL>
__global__ __launch_bounds__(256, 2) void linear_walk_kernel(const Walk a) {
    typedef typename Elem<TY>::type E;
    constexpr int NP = Elem<TY>::parts, C = 16 * TILES;
    constexpr bool OUT = KIND == OUTPUTS || KIND == OUTPUTS_SLOPE, SLOPE = KIND == OUTPUTS_SLOPE || KIND == STATES_SLOPE;
    constexpr bool GRAD = KIND == OUTPUTS_SLOPE;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t walks = OUT ? a.segments : a.segments - 1;  // of the segments, all but the last in the walk's direction
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const uint32_t block = unit % a.blocks, walk = unit / a.blocks % walks, bh = unit / a.blocks / walks;
    if (bh >= a.batch * a.heads) return;
    const int64_t b = bh / a.heads, h = bh % a.heads;
    const uint32_t segment = !OUT && BACK ? walk + 1 : walk;
    const int begin = segment * a.segment_length, T = begin + min(a.length - begin, a.segment_length);
    const int col0 = block * 32;
    const int da = a.da, dc = a.dc - col0;
    auto row_of = [&](const Rows& x, int e) { return (const E*)x.at + b * x.stride[0] + (h / x.share) * x.stride[2] + e + 8 * g; };
    const E* ap = OUT ? row_of(a.a, 0) : nullptr;
    const E* bp = row_of(a.b, 0);
    const E* cp = row_of(a.c, col0);
    const E* qp = GRAD ? row_of(a.q, col0) : nullptr;
    const uint8_t* rp = a.reset ? a.reset + b * a.reset_stride[0] : nullptr;

    // ---- what a chunk reads
    Eight<TY> ar[OUT ? TILES : 1][STEPS], br[TILES][STEPS], cr[TILES], qr[GRAD ? TILES : 1];
    bool cut = false, any_cut = false;
    auto fetch = [&](int t, int rows) {
        cut = rp && lane < rows && rp[(t + lane) * a.reset_stride[1]];
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            const int64_t tok = t + min(16 * i + n, rows - 1);
            const E* x = bp + tok * a.b.stride[1];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) br[i][s].template load<FULL>(x + 32 * s, da - 32 * s - 8 * g);
            if constexpr (OUT) {
                x = ap + tok * a.a.stride[1];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) ar[i][s].template load<FULL>(x + 32 * s, da - 32 * s - 8 * g);
            }
            cr[i].template load<FULL>(cp + tok * a.c.stride[1], dc - 8 * g);
            if constexpr (GRAD) qr[i].template load<FULL>(qp + tok * a.q.stride[1], dc - 8 * g);
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

    // ---- the state, by row tiles of 16 (pairs of them make 32 rows) and two column tiles
    f4 S[2 * STEPS][2], N[SLOPE ? 2 * STEPS : 1][2];
    // A lane takes four values that lie side by side: of one of four rows, which four lanes then exchange, or
    // of a column, where columns lie side by side.
    auto place = [&](int i, int j, int& left) {
        const int row = 32 * (i >> 1) + 8 * g + 4 * (i & 1), col = 8 * (n >> 2) + 4 * j;
        if (a.row == 1) {
            left = FULL ? 4 : col + (n & 3) < dc ? da - row : 0;
            return row + (int64_t)(col0 + col + (n & 3)) * a.col;
        }
        left = FULL ? 4 : row + (n & 3) < da ? dc - col : 0;
        return (int64_t)(row + (n & 3)) * a.row + col0 + col;
    };
    auto load_state = [&](auto& X, const float* from) {
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                int left;
                const int64_t at = place(i, j, left);
                X[i][j] = f4{0, 0, 0, 0};
                if (from) X[i][j] = load_floats<FULL>(from + at, left);
            }
        if (from && a.row != 1)
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) X[i][j] = turn(X[i][j], lane);
    };
    auto store_state = [&](const auto& X, float* to) {
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                int left;
                const int64_t at = place(i, j, left);
                store_floats<FULL>(to + at, left, a.row == 1 ? X[i][j] : turn(X[i][j], lane));
            }
    };
    const bool at_first = BACK ? segment == a.segments - 1 : segment == 0;
    const int64_t between = (int64_t)bh * (a.segments - 1) + (BACK ? segment : segment - 1);  // the start of this walk
    load_state(S, at_first ? (a.first ? a.first + bh * a.size : nullptr) : OUT ? a.starts + between * a.size : nullptr);
    if constexpr (SLOPE) load_state(N, OUT && !at_first ? a.slopes + between * a.size : nullptr);

    // ---- the head's decays. `read`: of the state to a token, `write`: of a token to the next state.
    float gh = a.g[h];
    gh = gh < -200.0f ? -200.0f : gh;  // 0 in fp32 from one token to the next
    float near[4], far[4];  // inside a tile of 16, and between the two
    float read[TILES], all = 0.0f;
    f4 write[TILES];
    int measured = -1;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int m = BACK ? 4 * g + r - n : n - 4 * g - r;
        near[r] = m < 0 ? 0.0f : a.scale * decay(gh, m);
        far[r] = a.scale * decay(gh, 16 + m);
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        if (!BACK) read[i] = a.scale * decay(gh, 16 * i + n + 1);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (BACK) write[i][r] = a.scale * decay(gh, 16 * i + 4 * g + r + 1);
    }
    auto measure = [&](int len) {  // those that depend on the chunk's length
        measured = len;
        all = decay(gh, len);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            if (BACK) read[i] = decay(gh, max(len - 1 - 16 * i - n, 0));
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (!BACK) write[i][r] = decay(gh, max(len - 1 - 16 * i - 4 * g - r, 0));
        }
    };

    // ---- unit matrices as operands: they pick dimension 8 (n / 4) + 4 i + n % 4 of a row's 32
    Frag<1> unit_of[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int e = 4 * i + (n & 3);
            unit_of[i].p[0][w] = g == (n >> 2) && (e >> 1) == w ? 0x3f80u << (16 * (e & 1)) : 0u;
        }
    double dg = 0.0;

    // The chunk of tokens t to t + len, in USED tiles. CUTS: there may be resets inside, in `cuts`. ODD: one token,
    // with values that are not finite: its operands along the tokens are read one by one. No branch is inside: where
    // one lies between a matrix instruction and the use of its result, the compiler has been seen to leave out the
    // wait. The scheduler is kept from starting everything at once, which takes more registers than there are.
    auto chunk = [&](auto used, auto with_cuts, auto is_odd, int t, int len, uint32_t cuts, auto&& next) {
        constexpr int USED = decltype(used)::value;
        constexpr bool CUTS = decltype(with_cuts)::value, ODD = decltype(is_odd)::value;
        const f4 zero = {0, 0, 0, 0};
        Frag<NP> af[OUT ? USED : 1][STEPS], bf[USED][STEPS], cf[USED];
        Eight<TY> qe[GRAD ? USED : 1];
#pragma unroll
        for (int i = 0; i < USED; ++i) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                bf[i][s] = operand(br[i][s]);
                if constexpr (OUT) af[i][s] = operand(ar[i][s]);
            }
            cf[i] = operand(cr[i]);
            if constexpr (GRAD) qe[i] = qr[i];
        }
        f4 odd_b[ODD ? 2 * STEPS : 1], odd_c[2];
        if constexpr (ODD) {
            const int e = 8 * (n >> 2) + (n & 3) - 8 * g;  // from this lane's place in its rows to the dimension that it stands for
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) {
                const int x = 32 * (i >> 1) + 4 * (i & 1);
                odd_b[i] = f4{g == 0 && x + e < da ? Elem<TY>::get(bp[t * a.b.stride[1] + x + e]) : 0.0f, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) odd_c[j] = f4{g == 0 && 4 * j + e < dc ? Elem<TY>::get(cp[t * a.c.stride[1] + 4 * j + e]) : 0.0f, 0, 0, 0};
        }
        if (AHEAD) next();

        // Resets: the last one up to a token (this lane's, and those of its registers), and of the chunk.
        int mine[USED], theirs[USED][4], last_cut = -1, first_cut = 64;
        if constexpr (CUTS) {
            last_cut = cuts ? 31 - __builtin_clz(cuts) : -1;
            first_cut = cuts ? __builtin_ctz(cuts) : 64;
#pragma unroll
            for (int i = 0; i < USED; ++i) {
                mine[i] = 31 - __clz((int)(cuts & (0xffffffffu >> (31 - 16 * i - n))));
#pragma unroll
                for (int r = 0; r < 4; ++r) theirs[i][r] = 31 - __clz((int)(cuts & (0xffffffffu >> (31 - 16 * i - 4 * g - r))));
            }
        }

        // ---- P transposed (row j = 16 tj + 4 g + r, column i = 16 ti + n), as operands along j
        Half<3> alone;  // of the tokens that see one tile
        Frag<3> both;   // of those that see two
        float pairs = 0.0f;
        if constexpr (OUT) {
            f4 pt[USED][USED];
#pragma unroll
            for (int tj = 0; tj < USED; ++tj)
#pragma unroll
                for (int ti = 0; ti < USED; ++ti) {
                    if (BACK ? tj < ti : tj > ti) continue;
                    f4 x = zero, y = zero;
#pragma unroll
                    for (int s = 0; s < STEPS; ++s) x = mul<2>(bf[tj][s], af[ti][s], x);
                    if constexpr (GRAD) y = mul<2>(cf[tj], operand(qe[ti]), y);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 16 * ti + n, j = 16 * tj + 4 * g + r;
                        x[r] *= tj == ti ? near[r] : far[r];
                        // A product that is not finite does not pass the zeros either.
                        if (tj == ti) x[r] = (BACK ? j >= i : j <= i) ? x[r] : 0.0f;
                        if (CUTS) x[r] = (BACK ? i >= theirs[tj][r] : j >= mine[ti]) ? x[r] : 0.0f;
                        if (GRAD) pairs += (float)(i - j) * x[r] * y[r];
                    }
                    pt[tj][ti] = x;
                }
            constexpr int one = BACK ? USED - 1 : 0;
            alone = split<3>(pt[one][one]);
            if constexpr (USED == 2) both = split<3>(pt[0][1 - one], pt[1][1 - one]);
        }
        typename Along<USED>::template Op<NP> bt[2 * STEPS];
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i) {
            f4 x[USED];
#pragma unroll
            for (int k = 0; k < USED; ++k) x[k] = ODD ? odd_b[ODD ? i : 0] : mul<2>(bf[k][i >> 1], unit_of[i & 1], zero);
            bt[i] = Along<USED>::template make<NP>(x);
        }
        f4 out[USED][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            f4 ct[USED], wc[USED];
#pragma unroll
            for (int k = 0; k < USED; ++k) ct[k] = ODD ? odd_c[j] : mul<2>(cf[k], unit_of[j], zero);
            if constexpr (OUT) {
                f4 slope[USED];
#pragma unroll
                for (int k = 0; k < USED; ++k) out[k][j] = slope[k] = zero;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const Frag<3> sf = split<3>(S[2 * s][j], S[2 * s + 1][j]);
#pragma unroll
                    for (int k = 0; k < USED; ++k) out[k][j] = mul<2>(sf, af[k][s], out[k][j]);
                    if constexpr (GRAD) {
                        const Frag<3> nf = split<3>(N[2 * s][j], N[2 * s + 1][j]);
#pragma unroll
                        for (int k = 0; k < USED; ++k) slope[k] = mul<2>(nf, af[k][s], slope[k]);
                    }
                }
#pragma unroll
                for (int k = 0; k < USED; ++k) {
                    const bool reach = !CUTS || (BACK ? 16 * k + n >= last_cut : mine[k] < 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[k][j][r] = reach ? out[k][j][r] * read[k] : 0.0f;
                    if constexpr (GRAD) {
                        float q[8];
                        qe[k].get(q);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = (float)(16 * k + n + 1) * out[k][j][r] + (reach ? slope[k][r] * read[k] : 0.0f);
                            pairs += x * q[4 * j + r];
                        }
                    }
                }
                constexpr int one = BACK ? USED - 1 : 0;
                out[one][j] = mul<2>(split<NP>(ct[one]), alone, out[one][j]);
                if constexpr (USED == 2) out[1 - one][j] = mul<2>(split<NP>(ct[0], ct[1]), both, out[1 - one][j]);
            }
            // ---- the state behind the chunk
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < USED; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = 16 * k + 4 * g + r;
                    wc[k][r] = !CUTS || (BACK ? at < first_cut : at >= last_cut) ? ct[k][r] * write[k][r] : 0.0f;
                }
            const auto wf = Along<USED>::template make<3>(wc);
            if constexpr (SLOPE) {
#pragma unroll
                for (int k = 0; k < USED; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) wc[k][r] *= (float)max(len - 1 - 16 * k - 4 * g - r, 0);
                const auto nf = Along<USED>::template make<3>(wc);
#pragma unroll
                for (int i = 0; i < 2 * STEPS; ++i) {
                    f4 x = (N[i][j] + S[i][j] * (float)len) * all;
                    if (CUTS) x = cuts ? zero : x;
                    N[i][j] = mul<2>(bt[i], nf, x);
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) {
                f4 x = S[i][j] * all;
                if (CUTS) x = cuts ? zero : x;
                S[i][j] = mul<2>(bt[i], wf, x);
            }
        }
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < USED; ++k) {
                const int row = 16 * k + n, e = 8 * g;
                const float y[8] = {out[k][0][0], out[k][0][1], out[k][0][2], out[k][0][3], out[k][1][0], out[k][1][1], out[k][1][2], out[k][1][3]};
                const int64_t to = b * a.out_stride[0] + (t + row) * a.out_stride[1] + (h / a.out_share) * a.out_stride[2] + col0 + e;
                if (row < len) {
                    if (a.out_f32) {
                        Eight<T_F32> x;
                        x.set(y);
                        x.template store<FULL>((float*)a.out + to, dc - e);
                    } else {
                        Eight<TY> x;
                        x.set(y);
                        x.template store<FULL>((E*)a.out + to, dc - e);
                    }
                }
            }
        }
        if (GRAD) dg += (double)pairs;
        if (!AHEAD) next();
    };

    // ---- the walk
    while (BACK ? at > begin : at < T) {
        int len = rows, first = t;
        bool fine = true;
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                fine &= br[i][s].finite();
                if (OUT) fine &= ar[OUT ? i : 0][s].finite();
            }
            fine &= cr[i].finite();
            if (GRAD) fine &= qr[GRAD ? i : 0].finite();
        }
        uint32_t cuts = (uint32_t)__ballot(cut);
        const bool odd = __ballot(!fine) != 0;
        if (odd) {
            if (BACK && rows > 1) {  // the last token of the chunk first
                first = at - 1;
                fetch(first, 1);
                cuts = (uint32_t)__ballot(cut);
            }
            cuts &= 1;
            len = 1;
        }
        any_cut |= cuts != 0;
        if (len < C) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const bool keep = 16 * i + n < len;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    br[i][s].keep(keep);
                    if (OUT) ar[OUT ? i : 0][s].keep(keep);
                }
                cr[i].keep(keep);
                if (GRAD) qr[GRAD ? i : 0].keep(keep);
            }
        }
        if (len != measured) measure(len);
        const int now = first;
        at = BACK ? first : first + len;
        const bool more = BACK ? at > begin : at < T;
        auto next = [&] {
            if (more) {
                bounds(at, t, rows);
                fetch(t, rows);
            }
        };
        constexpr std::integral_constant<int, 1> one{};
        constexpr std::integral_constant<int, TILES> whole{};
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        if (odd) {
            chunk(one, yes, yes, now, len, cuts, next);
        } else if (TILES == 2 && len <= 16) {
            if (cuts) chunk(one, yes, no, now, len, cuts, next);
            else chunk(one, no, no, now, len, cuts, next);
        } else {
            if (cuts) chunk(whole, yes, no, now, len, cuts, next);
            else chunk(whole, no, no, now, len, cuts, next);
        }
    }

    // ---- what it leaves
    if constexpr (OUT) {
        if (BACK ? segment == 0 : segment == a.segments - 1) {
            if (a.last) store_state(S, a.last + bh * a.size);
            if constexpr (GRAD) {
                if (a.d_last) {
                    load_state(S, a.d_last + bh * a.size);
#pragma unroll
                    for (int i = 0; i < 2 * STEPS; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) dg += S[i][j][r] == 0.0f ? 0.0 : (double)(S[i][j][r] * N[i][j][r]);
                }
            }
        }
        if constexpr (GRAD) {
#pragma unroll
            for (int d = 32; d; d >>= 1) dg += __shfl_xor(dg, d);
            if (lane == 0) a.parts[unit] = dg;
        }
    } else {
        const int64_t to = (int64_t)bh * (a.segments - 1) + walk;
        store_state(S, a.starts + to * a.size);
        if constexpr (SLOPE) store_state(N, a.slopes + to * a.size);
        if (block == 0 && lane == 0) a.passes[to] = any_cut ? 0.0f : 1.0f;
    }
}

// ---- joining segments ------------------------------------------------------------------------
// The states between segments from what each adds: S_{p+1} = exp(g L) S_p + U_p, in place of U, where
// the segment passes a state at all; and the slopes, N_{p+1} = exp(g L) (N_p + L S_p) + V_p. A thread a value.
template <bool BACK, bool SLOPE> __global__ __launch_bounds__(256) void linear_join_kernel(const Walk a) {
    const int64_t between = a.segments - 1, blocks = (a.size + 255) / 256;
    const int64_t bh = blockIdx.x / blocks, at = blockIdx.x % blocks * 256 + threadIdx.x;
    if (at >= a.size) return;
    float gh = a.g[bh % a.heads];
    gh = gh < -200.0f ? -200.0f : gh;
    const float whole = decay(gh, a.segment_length), rest = decay(gh, a.length - between * a.segment_length);
    float* starts = a.starts + bh * between * a.size + at;
    float* slopes = SLOPE ? a.slopes + bh * between * a.size + at : nullptr;
    const float* passes = a.passes + bh * between;
    float S = 0.0f, N = 0.0f;
    for (int64_t k = 0; k < between; ++k) {
        const int64_t p = BACK ? between - 1 - k : k;
        const bool pass = k > 0 && passes[p] != 0.0f;  // nothing, NaN included, passes a reset
        const float length = BACK && k == 0 ? a.length - between * a.segment_length : a.segment_length;
        const float d = BACK && k == 0 ? rest : whole, before = S;
        S = starts[p * a.size];
        if (pass) S += d * before;
        starts[p * a.size] = S;
        if (SLOPE) {
            const float n = N;
            N = slopes[p * a.size];
            if (pass) N += d * (n + length * before);
            slopes[p * a.size] = N;
        }
    }
}

// Sums the value heads of each key head, in their order; a thread a value, several where there are more
// than 2^28 (a launch takes less than 2^32 threads).
template <int TY>
__global__ __launch_bounds__(256) void linear_share_kernel(const float* parts, void* out, int64_t s0, int64_t s1, int64_t s2, int64_t all, uint32_t length, uint32_t heads,
                                                           uint32_t share, uint32_t dim) {
    typedef typename Elem<TY>::type E;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += (int64_t)gridDim.x * 256) {
        const int64_t x = id % dim, h = id / dim % heads, bt = id / dim / heads;
        const float* from = parts + (bt * heads + h) * share * dim + x;
        float sum = 0.0f;
        for (uint32_t s = 0; s < share; ++s) sum += from[(int64_t)s * dim];
        ((E*)out)[bt / length * s0 + bt % length * s1 + h * s2 + x] = Elem<TY>::put(sum);
    }
}

// ---- one token -----------------------------------------------------------------------------
// The state is read once and written once. A wave holds all rows of 4 LANES columns, 16 (or 4) rows and 4
// columns a lane:  o = scale (a S^T q + (k . q) v),  S <- a S + k v^T.  LANES lanes lie along the
// columns, 64 / LANES along the rows.
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
    const float a = first ? 0.0f : expf(in.g[h]);
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
#ifndef TILES_OF
#define TILES_OF(TY, STEPS) ((TY) == T_F32 ? 1 : 2)
#endif
#ifndef AHEAD_OF
#define AHEAD_OF(TY, STEPS, KIND) ((STEPS) < 4 && (KIND) != OUTPUTS_SLOPE)
#endif
template <int TY, int STEPS, bool FULL> void walk_shape(const Walk& w, Kind kind, bool back, hipStream_t stream) {
    constexpr int TILES = TILES_OF(TY, STEPS);
    const bool out = kind == OUTPUTS || kind == OUTPUTS_SLOPE;
    const uint32_t units = w.batch * w.heads * w.blocks * (out ? w.segments : w.segments - 1);
    const dim3 grid((units + 3) / 4);
    if (back) {
        if (out) linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, OUTPUTS), true, OUTPUTS, FULL><<<grid, 256, 0, stream>>>(w);
        else linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, STATES), true, STATES, FULL><<<grid, 256, 0, stream>>>(w);
    } else if (kind == OUTPUTS) {
        linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, OUTPUTS), false, OUTPUTS, FULL><<<grid, 256, 0, stream>>>(w);
    } else if (kind == STATES) {
        linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, STATES), false, STATES, FULL><<<grid, 256, 0, stream>>>(w);
    } else if (out) {
        linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, OUTPUTS_SLOPE), false, OUTPUTS_SLOPE, FULL><<<grid, 256, 0, stream>>>(w);
    } else {
        linear_walk_kernel<TY, STEPS, TILES, AHEAD_OF(TY, STEPS, STATES_SLOPE), false, STATES_SLOPE, FULL><<<grid, 256, 0, stream>>>(w);
    }
    if (!out && w.segments > 2) {
        const dim3 join(w.batch * w.heads * (uint32_t)((w.size + 255) / 256));
        if (back) linear_join_kernel<true, false><<<join, 256, 0, stream>>>(w);
        else if (kind == STATES) linear_join_kernel<false, false><<<join, 256, 0, stream>>>(w);
        else linear_join_kernel<false, true><<<join, 256, 0, stream>>>(w);
    }
}

template <int TY> hipError_t launch_walk(const Walk& w, const Shape& s, Kind kind, bool back, hipStream_t stream) {
    if (s.steps == 1) s.full ? walk_shape<TY, 1, true>(w, kind, back, stream) : walk_shape<TY, 1, false>(w, kind, back, stream);
    else if (s.steps == 2) s.full ? walk_shape<TY, 2, true>(w, kind, back, stream) : walk_shape<TY, 2, false>(w, kind, back, stream);
    else s.full ? walk_shape<TY, 4, true>(w, kind, back, stream) : walk_shape<TY, 4, false>(w, kind, back, stream);
    return hipGetLastError();
}

template <int TY> hipError_t launch_share(const float* parts, void* out, const int64_t* stride, uint32_t batch, uint32_t length, uint32_t key_heads, uint32_t share,
                                          uint32_t dim, hipStream_t stream) {
    const int64_t all = (int64_t)batch * length * key_heads * dim, blocks = (all + 255) / 256, most = 1 << 20;
    linear_share_kernel<TY><<<dim3((uint32_t)(blocks < most ? blocks : most)), 256, 0, stream>>>(parts, out, stride[0], stride[1], stride[2], all, length, key_heads, share, dim);
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
