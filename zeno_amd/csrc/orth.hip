// Newton-Schulz orthogonalisation: X = G / (|G| + eps), then `steps` times
//     A = X X^T,  B = b A + c A A,  X <- a X + B X          (rows <= columns, else G^T)
// which drives every singular value towards 1.
//
// Everything is a matrix product, (m m n + m m m + 2 m m n) operations a step with the symmetric
// ones done by half, on the fp16 matrix units. Their operands are bounded: no singular value of X
// exceeds about 1.2 (the host checks the coefficients), so X, A and B are held in fp16 at fixed
// scales far from either end of its range, in two parts that carry 22 bits: three of the four part
// products give fp32's accuracy at a third of the units' rate, five times the fp32 units'. X itself
// stays in fp32 and is what a X adds: a small singular value grows 3.4-fold a step by that term, and
// with it every rounding of X that the term would carry (momenta with strong directions 4.3e-3 off with 11
// bits there; emulated, the operand's 22 bits would do as well as 32). bfloat16 takes two parts as well: with one of 11 bits a result of 256 x 512 with 37 rows
// that are not zero is off by 3.3e-3 of its norm and one of 1024 x 1024 Gaussian values by 1.3e-3,
// where its own rounding is 1.7e-3; with two, 4e-6. Sums are fp32, the norm's fp64.
//
// Layout. X and X^T are both kept as operands (every product then reads two operands along their
// rows); rows and columns are padded with zeros to the tile. The two parts alternate every 32 columns,
// so 128 bytes of a row are 32 columns.
#include <algorithm>
#include <cmath>
#include <utility>

#include "mma.h"
#include "orth.h"
#include "overlap.h"

namespace za {
namespace orth {
namespace {

using namespace mma;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr float kScale = 1024.0f;   // of X, A and B in fp16
constexpr float kLargest = 32.0f;   // entries that the scale leaves room for, twice over
constexpr int kNormBlocks = 256;

struct Args {
    ZenoAmdOrthogonalize in;
    int m, n;             // of X
    int mp, np;           // padded
    bool flip;            // X = G^T
    double* partial;      // [count][kNormBlocks]
    float* master;        // X^T in fp32, each value read and written by one thread
    float* sums;          // of the slices of a product
    int slices;
    bool x_vec;           // eight values along x's dense dimension are 16 bytes aligned (32 of fp32)
    bool out_vec;         // four values along out's dense dimension are aligned
    _Float16 *x, *xt, *gram, *poly;  // [count][...]
    _Float16* xt2;        // the next X^T (X is no operand of the product that makes the next one)
};

constexpr int kParts = 2;           // fp16 numbers that hold a value

__device__ __forceinline__ int64_t place(int64_t row, int col, int ld) { return row * ld * kParts + (col >> 5) * 64 + (col & 31); }
__device__ __forceinline__ void put(_Float16* at, float x) {
    const _Float16 h = (_Float16)x;
    at[0] = h;
    at[32] = (_Float16)(x - (float)h);
}

template <int TY> __device__ __forceinline__ float input(const Args& a, int64_t k, int row, int col) {  // of G
    typedef typename Elem<TY>::type E;
    return Elem<TY>::get(((const E*)a.in.x)[k * a.in.x_stride[0] + row * a.in.x_stride[1] + col * a.in.x_stride[2]]);
}

// Sums of squares: pieces of eight values along the dense dimension, spread over the blocks. One read
// of G (4096 x 4096 bfloat16 22 us, the first touch of 34 MB).
template <int TY> __global__ __launch_bounds__(256) void norm_kernel(const Args a) {
    typedef typename Elem<TY>::type E;
    __shared__ double part[4];
    const int64_t k = blockIdx.y;
    const bool by_col = a.in.x_stride[2] <= a.in.x_stride[1];
    const uint32_t inner = by_col ? a.in.cols : a.in.rows, pieces = (inner + 7) / 8;
    const int64_t step = a.in.x_stride[by_col ? 2 : 1], ld = a.in.x_stride[by_col ? 1 : 2];
    const uint32_t all = pieces * (by_col ? a.in.rows : a.in.cols);
    const E* x = (const E*)a.in.x + k * a.in.x_stride[0];
    double sum = 0.0;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
        const uint32_t row = i / pieces, e = 8 * (i % pieces);
        const E* at = x + row * ld + e * step;
        float v[8];
        if (a.x_vec && e + 8 <= inner) {
            Raw<TY> raw;
            raw.template load<true>(at, 8, true);
            raw.get(v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = e + j < inner ? Elem<TY>::get(at[j * step]) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += (double)v[j] * (double)v[j];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.partial[k * kNormBlocks + blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// X and X^T in fp16 from G, a 64x64 tile a block. Bound by memory: 4096 x 4096 bfloat16 60 us, 3.9 TB/s.
template <int TY> __global__ __launch_bounds__(256) void load_kernel(const Args a) {
    __shared__ float tile[64][65];
    const int64_t k = blockIdx.z;
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of X
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kNormBlocks; i += 64) s += a.partial[k * kNormBlocks + i + (threadIdx.x & 63)];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    const double f = (double)kScale / (sqrt(s) + (double)a.in.eps);  // beyond fp32's range where both are small
    const bool dense_cols = a.flip ? a.in.x_stride[1] <= a.in.x_stride[2] : a.in.x_stride[2] <= a.in.x_stride[1];
    const int w = threadIdx.x & 63, u = threadIdx.x >> 6;
#pragma unroll
    for (int i = u, t = 0; t < 16; ++t, i += 4) {
        const int r = dense_cols ? i : w, c = dense_cols ? w : i;
        float v = 0.0f;
        if (r0 + r < a.m && c0 + c < a.n) v = a.flip ? input<TY>(a, k, c0 + c, r0 + r) : input<TY>(a, k, r0 + r, c0 + c);
        tile[r][c] = (float)((double)v * f);
    }
    __syncthreads();
    _Float16* x = a.x + k * a.mp * a.np * kParts;
    _Float16* xt = a.xt + k * a.mp * a.np * kParts;
#pragma unroll
    for (int i = u, t = 0; t < 16; ++t, i += 4) {
        a.master[(k * a.np + c0 + i) * a.mp + r0 + w] = tile[w][i];
        put(x + place(r0 + i, c0 + w, a.np), tile[i][w]);
        put(xt + place(c0 + i, r0 + w, a.mp), tile[w][i]);
    }
}

// Four values of a row-major operand row that start at a multiple of four.
__device__ __forceinline__ void put4(_Float16* at, f4 x) {
    h4 h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        h[r] = (_Float16)x[r];
        l[r] = (_Float16)(x[r] - (float)h[r]);
    }
    *reinterpret_cast<h4*>(at) = h;
    *reinterpret_cast<h4*>(at + 32) = l;
}
__device__ __forceinline__ f4 get4(const _Float16* at) {
    const h4 h = *reinterpret_cast<const h4*>(at), l = *reinterpret_cast<const h4*>(at + 32);
    f4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = (float)h[r] + (float)l[r];
    return x;
}

// Consecutive blocks go to the eight dies in turn; each die gets a run of the work.
__device__ __forceinline__ int run_at(int block, int blocks) {
    const int per = blocks / 8, rest = blocks % 8, die = block % 8;
    return die * per + min(die, rest) + block / 8;
}
// Which tile that is: in bands of eight rows and column by column within a band, so that the tiles
// which run at once on a die share as many operand rows as they can in its L2. cols 0: the tiles on
// and below the diagonal.
__device__ __forceinline__ void tile_at(int id, int cols, int rows, int& ti, int& tj) {
    constexpr int band = 8;
    for (int r0 = 0;; r0 += band) {
        const int high = min(band, rows - r0);
        const int left = cols ? cols : r0, count = left * high + (cols ? 0 : high * (high + 1) / 2);
        if (id >= count) {
            id -= count;
            continue;
        }
        if (id < left * high) {
            ti = r0 + id % high;
            tj = id / high;
        } else {  // the band's own triangle
            id -= left * high;
            int i = 0;
            while (id > i) id -= ++i;
            ti = r0 + i;
            tj = r0 + id;
        }
        return;
    }
}

enum Kind { GRAM, POLY, NEXT, LAST };
enum Share { WHOLE, SLICE, JOIN };  // of the contraction: all of it; a slice, sums kept; the sum of the slices

// C = L R^T of rows along the contraction, and what follows from it. A block computes BM x BN; its
// WR x WC waves hold their part in registers. 128 bytes of every row of both operands are a step;
// steps come into LDS by loads that write it themselves, their 16-byte pieces permuted by half the
// row number, which leaves the operand reads without bank conflicts. Few tiles with a long
// contraction are cut into slices along it (SLICE), whose sums another launch adds in their order (JOIN).
// Bound by the matrix units and the operands' way from L2 together, and at its end by memory: X, X^T and
// the fp32 X are written at once by all blocks. Rates of part products: 4096 x 4096 B X 387 us (1.07
// PFLOP/s; a large library product of fp16 1.18), the symmetric products 247 and 259 (half the operations;
// 0.8); 1000 x 4000 B X 37 us (0.65, of which 14 are the end), X X^T 18 and 7 for the join.
template <int TY, int BM, int BN, int WR, int WC, int STAGES, int KIND, int SHARE>
__global__ __launch_bounds__(64 * WR * WC) void product_kernel(const Args a) {
    constexpr int threads = 64 * WR * WC, waves = WR * WC;
    constexpr int rows = BM / WR / 16, TM = SHARE == JOIN ? 1 : rows, TN = BN / WC / 16;  // a join: one row of result tiles a wave
    const int i0 = SHARE == JOIN ? blockIdx.z : 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int64_t k = blockIdx.y;
    constexpr bool half = KIND == GRAM || KIND == POLY;  // symmetric: tiles on and below the diagonal
    // Slices are the outer order: a die then reads little more than a slice of the operands.
    const int tiles = SHARE == SLICE ? gridDim.x / a.slices : gridDim.x, run = run_at(blockIdx.x, gridDim.x);
    const int slice = SHARE == SLICE ? run / tiles : 0, tile = run - slice * tiles;
    int ti, tj;
    tile_at(tile, half ? 0 : a.np / BN, a.mp / BM, ti, tj);
    f4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f4{0, 0, 0, 0};
    // The sums of slice s of this tile: [matrix][slice][tile][value][thread].
    auto sums = [&](int s) { return (f4*)a.sums + (((k * a.slices + s) * tiles + tile) * (rows * TN) + i0 * TN) * threads + threadIdx.x; };

    if constexpr (SHARE == JOIN) {
#pragma unroll 4
        for (int s = 0; s < a.slices; ++s) {
            const f4* from = sums(s);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] += from[(i * TN + j) * threads];
        }
    } else {
        constexpr int stages = STAGES;
        __shared__ __attribute__((aligned(128))) char lds[stages][(BM + BN) * 128];
        const int ld = KIND == GRAM ? a.np : a.mp;  // of the contraction
        const _Float16* left = (KIND == GRAM ? a.x + k * a.mp * a.np * kParts : KIND == POLY ? a.gram + k * a.mp * a.mp * kParts : a.poly + k * a.mp * a.mp * kParts);
        const _Float16* right = KIND == NEXT || KIND == LAST ? a.xt + k * a.mp * a.np * kParts : left;
        left += (int64_t)ti * BM * ld * kParts;
        right += (int64_t)tj * BN * ld * kParts;
        int b0 = 0, blocks = ld * kParts / 64;
        if constexpr (SHARE == SLICE) {
            const int all = blocks;
            b0 = (int)((int64_t)all * slice / a.slices);
            blocks = (int)((int64_t)all * (slice + 1) / a.slices);
        }
        // A load instruction of a wave brings eight rows of 128 bytes.
        constexpr int loads = (BM + BN) / 8 / waves;
        static_assert(BM / 8 % waves == 0 && BN / 8 % waves == 0, "whole loads of either operand a wave");
        uint32_t from[loads];
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int row = 8 * (wave + i * waves) + (lane >> 3), piece = (lane & 7) ^ ((row >> 1) & 7);
            from[i] = (uint32_t)(row < BM ? row : row - BM) * (uint32_t)(ld * kParts * 2) + 16 * piece;  // in bytes
        }
        auto fetch = [&](int block, int buf) {
#pragma unroll
            for (int i = 0; i < loads; ++i)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)((i * waves * 8 < BM ? left : right) + 64 * (int64_t)block) + from[i]),
                                                 (__attribute__((address_space(3))) void*)(lds[buf] + 1024 * (wave + i * waves)), 16, 0, 0);
        };
        const int row_l = (wave / WC) * (BM / WR) + n, row_r = BM + (wave % WC) * (BN / WC) + n;
        // A step is 32 of the contraction. Its operands are read while the step before is multiplied, and
        // `stages` more steps are in LDS or on their way. Every step fetches, past the end the last one
        // again, so that the number of loads under way is the same at every wait. The products are spread between the LDS reads, then between the loads (1000 x 4000
        // 438 us with the reads of a step before its products, 361 so).
        constexpr int products = 3 * TM * TN, reads = 2 * (TM + TN);
        struct Operands {
            h8 l[2][TM], r[2][TN];
        } now, next;
        auto read = [&](int buf, Operands& o) {
            const char* at = lds[buf];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int c = 4 * p + g;
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const int row = row_l + 16 * i;
                    o.l[p][i] = *reinterpret_cast<const h8*>(at + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const int row = row_r + 16 * j;
                    o.r[p][j] = *reinterpret_cast<const h8*>(at + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
                }
            }
        };
        int buf = 0;  // of this step
        auto step = [&](int b, Operands& x, Operands& y) {
            // The next step's operands are here, and this step's are read: all waves' after the barrier.
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((stages - 2) * loads) : "memory");
            const int other = buf + 1 == stages ? 0 : buf + 1;
            read(other, y);  // past the end: read and not used
            fetch(min(b + stages, blocks - 1), buf);
            buf = other;
#pragma unroll
            for (int p = 2; p >= 0; --p)  // second part by first, first by second, first by first
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.l[p >> 1][i], x.r[p & 1][j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < reads; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product,
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
            }
#pragma unroll
            for (int i = 0; i < loads; ++i) {
                if constexpr (products - reads >= loads) __builtin_amdgcn_sched_group_barrier(0x008, (products - reads) / loads, 0);  // some products,
                __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);                                                                   // a load
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int i = 0; i < stages; ++i) fetch(min(b0 + i, blocks - 1), i);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((stages - 1) * loads) : "memory");
        read(0, now);
        int b = b0;
        if ((blocks - b0) & 1) {
            step(b++, now, next);
            now = next;
        }
        for (; b < blocks; b += 2) {
            step(b, now, next);
            step(b + 1, next, now);
        }
        // No load may still write the LDS when the workgroup's share of it is handed on.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    if constexpr (SHARE == SLICE) {
        f4* to = sums(slice);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) to[(i * TN + j) * threads] = acc[i][j];
        return;
    }
    // Products of two numbers at kScale: once too much.
    const float down = 1.0f / kScale;
    const int q = n & 3, qc = n & 12;
    // What the results are added to is read for `batch` rows of tiles before any of them is stored: a
    // read behind a store waits for memory each time (B X of 4096 x 4096: 165 us so, 147 in batches).
    constexpr int batch = TM < 4 ? TM : 4;
#pragma unroll
    for (int i1 = 0; i1 < TM; i1 += batch) {
        f4 old[batch][TN];
        auto row_of = [&](int i) { return ti * BM + (wave / WC) * (BM / WR) + 16 * (i0 + i1 + i) + 4 * g; };
        auto col_of = [&](int j) { return tj * BN + (wave % WC) * (BN / WC) + 16 * j; };
        auto master = [&](int i, int j) { return reinterpret_cast<f4*>(a.master + (k * a.np + col_of(j) + n) * a.mp + row_of(i)); };
#pragma unroll
        for (int i = 0; i < batch; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if constexpr (KIND == POLY) old[i][j] = get4(a.gram + k * a.mp * a.mp * kParts + place(col_of(j) + n, row_of(i), a.mp));
                if constexpr (!half) old[i][j] = *master(i, j);
            }
#pragma unroll
        for (int i = 0; i < batch; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int row0 = row_of(i), col0 = col_of(j);
                f4 v = acc[i1 + i][j] * down;
                if constexpr (half) {
                    _Float16* to = (KIND == GRAM ? a.gram : a.poly) + k * a.mp * a.mp * kParts;
                    if constexpr (KIND == POLY) v = a.in.b * old[i][j] + a.in.c * v;
                    put4(to + place(col0 + n, row0, a.mp), v);  // the mirrored tile (of a diagonal tile, the same)
                    if (ti != tj) put4(to + place(row0 + q, col0 + qc, a.mp), turn(v, lane));
                } else {
                    v += a.in.a * old[i][j];
                    if constexpr (KIND == NEXT) {
                        *master(i, j) = v;
                        put4(a.xt2 + k * a.mp * a.np * kParts + place(col0 + n, row0, a.mp), v);
                        put4(a.x + k * a.mp * a.np * kParts + place(row0 + q, col0 + qc, a.np), turn(v, lane));
                    } else {
                        typedef typename Elem<TY>::type E;
                        // Four consecutive values along the dimension of out that is dense.
                        const bool along_rows = a.flip ? a.in.out_stride[2] == 1 : a.in.out_stride[1] == 1;
                        const f4 w = (along_rows ? v : turn(v, lane)) * down;
                        const int row = along_rows ? row0 : row0 + q, col = along_rows ? col0 + n : col0 + qc;
                        const int64_t sr = a.in.out_stride[a.flip ? 2 : 1], sc = a.in.out_stride[a.flip ? 1 : 2];
                        E* to = (E*)a.in.out + k * a.in.out_stride[0] + row * sr + col * sc;
                        const int64_t step = along_rows ? sr : sc;
                        const int left = along_rows ? (col < a.n ? a.m - row : 0) : (row < a.m ? a.n - col : 0);
                        if (a.out_vec && left >= 4) {
                            if constexpr (TY == T_F32) *reinterpret_cast<f4*>(to) = w;
                            else {
                                u2 e;
#pragma unroll
                                for (int r = 0; r < 2; ++r)
                                    e[r] = (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(w[2 * r])) |
                                           (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(w[2 * r + 1])) << 16;
                                *reinterpret_cast<u2*>(to) = e;
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (r < left) to[r * step] = Elem<TY>::put(w[r]);
                        }
                    }
                }
            }
    }
}

struct Plan {
    int m, n, mp, np;
    int gram, slices;  // X X^T: tile, slices
    uint64_t norm, master, x, square, sums;  // bytes: partial norms, X in fp32, X as an operand, m x m as an operand, slices' sums
};

// Tiles of 64 or 128 squared, 128 where they make a block for half the CUs (2048 x 2048 715 us, 773 with 64).
int64_t tiles_of(const Plan& p, uint32_t count, bool half, int t) {
    const int64_t r = p.mp / t, c = p.np / t;
    return (half ? r * (r + 1) / 2 : r * c) * count;
}
int tile_of(const Plan& p, uint32_t count, bool half) {
    if (p.mp % 128 || (!half && p.np % 128)) return 64;  // sizes are multiples of 64
    return tiles_of(p, count, half, 128) >= 128 ? 128 : 64;
}
// Of X X^T, whose contraction is the longer dimension, also the slices. With tiles of 128 as many as
// fill the CUs once, of at least 16 steps (1000 x 4000 361 us, 382 without; 640 x 4000, which would
// come to 105 blocks, 275 so and 251 with 64). With tiles of 64 up to one block a CU, where that spares a
// block 24 steps, more than the join costs (512 x 2048 162 us, 193 without; four of 512 x 512, 8 of 16
// steps spared, 170 and 153).
void slice(Plan& p, uint32_t count) {
    const int64_t steps = (int64_t)p.np * kParts / 64;
    p.slices = 1;
    if (p.mp % 128 == 0) {
        const int64_t tiles = tiles_of(p, count, true, 128);
        p.gram = 128;
        p.slices = (int)std::max<int64_t>(1, std::min(256 / tiles, steps / 16));
        if (tiles * p.slices >= 128) return;
    }
    p.gram = tile_of(p, count, true);
    const int64_t tiles = tiles_of(p, count, true, p.gram);
    p.slices = 1;
    while (p.slices < 16 && tiles * p.slices * 2 <= 256 && steps / (p.slices * 2) >= 8) p.slices *= 2;
    if (steps - steps / p.slices < 24) p.slices = 1;
}

Plan plan_of(const ZenoAmdOrthogonalize& a) {
    Plan p;
    p.m = (int)(a.rows < a.cols ? a.rows : a.cols);
    p.n = (int)(a.rows < a.cols ? a.cols : a.rows);
    const int pad = p.m <= 512 ? 64 : 128;
    p.mp = (p.m + pad - 1) / pad * pad;
    p.np = (p.n + pad - 1) / pad * pad;
    p.norm = (uint64_t)a.count * kNormBlocks * sizeof(double);
    p.master = (uint64_t)a.count * p.mp * p.np * 4;
    p.x = (uint64_t)a.count * p.mp * p.np * kParts * 2;
    p.square = (uint64_t)a.count * p.mp * p.mp * kParts * 2;
    slice(p, a.count);
    p.sums = p.slices > 1 ? (uint64_t)tiles_of(p, a.count, true, p.gram) * p.slices * p.gram * p.gram * 4 : 0;
    return p;
}

template <int TY, int KIND, int SHARE> void product(const Args& a, int tile, hipStream_t stream) {
    const int rows = a.mp / tile, cols = a.np / tile, tiles = KIND == GRAM || KIND == POLY ? rows * (rows + 1) / 2 : rows * cols;
    const dim3 grid(SHARE == SLICE ? tiles * a.slices : tiles, a.in.count, SHARE == JOIN ? tile / 32 : 1);  // a join: a block for each row of result tiles of a wave
    if (tile == 64) product_kernel<TY, 64, 64, 2, 2, 4, KIND, SHARE><<<grid, 256, 0, stream>>>(a);
    else product_kernel<TY, 128, 128, 2, 2, 3, KIND, SHARE><<<grid, 256, 0, stream>>>(a);
}

template <int TY> hipError_t launch(Args a, const Plan& p, hipStream_t stream) {
    const int square = tile_of(p, a.in.count, true), whole = tile_of(p, a.in.count, false);
    norm_kernel<TY><<<dim3(kNormBlocks, a.in.count), 256, 0, stream>>>(a);
    load_kernel<TY><<<dim3(a.np / 64, a.mp / 64, a.in.count), 256, 0, stream>>>(a);
    for (uint32_t s = 0; s < a.in.steps; ++s) {
        if (p.slices == 1) {
            product<TY, GRAM, WHOLE>(a, p.gram, stream);
        } else {
            product<TY, GRAM, SLICE>(a, p.gram, stream);
            product<TY, GRAM, JOIN>(a, p.gram, stream);
        }
        product<TY, POLY, WHOLE>(a, square, stream);
        if (s + 1 < a.in.steps) product<TY, NEXT, WHOLE>(a, whole, stream);
        else product<TY, LAST, WHOLE>(a, whole, stream);
        std::swap(a.xt, a.xt2);
    }
    return hipGetLastError();
}

}  // namespace

std::string check(const ZenoAmdOrthogonalize* p) {
    if (!p) return "null arguments";
    const ZenoAmdOrthogonalize& a = *p;
    if (a.dtype > T_BF16) return "dtype is none of float32, float16, bfloat16";
    if (!a.count || !a.rows || !a.cols) return "count, rows and cols must be positive";
    if (a.count > 65535) return "more than 65535 matrices";
    if (a.rows > 65536 || a.cols > 65536) return "more than 65536 rows or columns";
    if (!a.steps || a.steps > 100) return "steps must be 1 to 100";
    if (!(a.eps > 0.0f) || !std::isfinite(a.eps)) return "eps must be positive";
    if (!std::isfinite(a.a) || !std::isfinite(a.b) || !std::isfinite(a.c)) return "coefficients must be finite";
    if (!a.x || !a.out) return "null matrix";
    // What the coefficients make of singular values up to 1, on a grid of them.
    double top = 1.0;
    for (uint32_t s = 0; s < a.steps; ++s) {
        double next = 0.0, poly = 0.0;
        for (int i = 0; i <= 2048; ++i) {
            const double v = top * i / 2048, w = v * v, f = a.b * w + a.c * w * w;
            poly = std::fmax(poly, std::fabs(f));
            next = std::fmax(next, std::fabs(v * (a.a + f)));
        }
        if (top * top > kLargest || poly > kLargest || next > kLargest) return "coefficients let singular values grow out of the range of 16-bit operands";
        top = next;
    }
    return "";
}

bool out_overlaps(const ZenoAmdOrthogonalize& a) {
    const int64_t sizes[3] = {a.count, a.rows, a.cols};
    return !Memory(a.out, a.out_stride, sizes, 3, 1, a.dtype == T_F32 ? 4 : 2).apart_from_itself();
}

uint64_t workspace_bytes(const ZenoAmdOrthogonalize& a) {
    const Plan p = plan_of(a);
    return p.norm + p.master + 3 * p.x + 2 * p.square + p.sums;
}

hipError_t run(const ZenoAmdOrthogonalize& in, void* workspace, hipStream_t stream) {
    const Plan p = plan_of(in);
    Args a{};
    a.in = in;
    a.m = p.m;
    a.n = p.n;
    a.mp = p.mp;
    a.np = p.np;
    a.flip = in.rows > in.cols;
    char* at = (char*)workspace;
    a.partial = (double*)at;
    at += p.norm;
    a.master = (float*)at;
    at += p.master;
    a.x = (_Float16*)at;
    a.xt = (_Float16*)(at + p.x);
    a.xt2 = (_Float16*)(at + 2 * p.x);
    a.slices = p.slices;
    a.gram = (_Float16*)(at + 3 * p.x);
    a.poly = (_Float16*)(at + 3 * p.x + p.square);
    a.sums = (float*)(at + 3 * p.x + 2 * p.square);
    const uint64_t four = in.dtype == T_F32 ? 16 : 8;
    const int64_t* s = in.out_stride;
    const int other = (a.flip ? s[2] : s[1]) == 1 ? (a.flip ? 1 : 2) : (a.flip ? 2 : 1);  // the dimension that the stores do not run along
    const int64_t* xs = in.x_stride;
    const int dense = xs[2] <= xs[1] ? 2 : 1;
    const uint64_t eb = in.dtype == T_F32 ? 4 : 2;
    a.x_vec = xs[dense] == 1 && (uintptr_t)in.x % 16 == 0 && xs[3 - dense] * eb % 16 == 0 && (in.count == 1 || xs[0] * eb % 16 == 0);
    a.out_vec = s[3 - other] == 1 && (uintptr_t)in.out % four == 0 && s[other] % 4 == 0 && (in.count == 1 || s[0] % 4 == 0);
    return in.dtype == T_F32   ? launch<T_F32>(a, p, stream)
           : in.dtype == T_F16 ? launch<T_F16>(a, p, stream)
                               : launch<T_BF16>(a, p, stream);
}

}  // namespace orth
}  // namespace za
