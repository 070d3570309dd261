// Matrix products of 32-bit numbers on the bf16 matrix units of gfx950.
//
// A float has 24 significant bits, a bf16 eight: x = x0 + x1 + x2 exactly, with x0 the float cut
// after its first 16 bits, x1 the rest cut the same way, x2 what is left. A product of two split
// operands sums the part products of weight 2^-16 and above (six of nine for two full floats,
// three where one operand is bf16 already) in the units' 32-bit accumulators, so it is as exact
// as an fp32 product at 2.7 to 5.3 times the rate of the fp32 matrix instructions (bf16
// 16x16x32: 16 cycles; the same work in fp32 16x16x4: 256).
//
// Layouts (lane l, n = l % 16, g = l / 16). A result tile of 16x16: register r of lane l is row
// 4 g + r, column n. An operand of 32 along the contraction: eight values a lane, an operand of
// 16: four, contraction index 4 g + j. The order of the contraction index is free as long as
// both operands agree, so a result tile serves as the next product's right operand from its
// registers: of two tiles that are 32 rows, position 8 g + 4 h + j of the contraction is row
// 16 h + 4 g + j. Left operands in LDS are stored in that order (`slot`), which makes each
// lane's eight values 16 consecutive bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace za {
namespace mma {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

// Where index x of a contraction of 32 is kept among its 32 (see above).
__device__ __host__ constexpr int slot(int x) { return (x & ~31) | (((x >> 2) & 3) << 3) | (((x >> 4) & 1) << 2) | (x & 3); }

template <int P> struct Frag { u4 p[P]; };  // 8 values a lane in P bf16 parts
template <int P> struct Half { u2 p[P]; };  // 4 values a lane

__device__ __forceinline__ uint32_t hi_pair(float a, float b) {  // the upper halves of a (low word) and b
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b) {  // nearest, ties to even
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    b2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float cut(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }

// The P parts of a pair of floats. The last of one or two parts is rounded to nearest (2^-9 and
// 2^-17 of the value); three are exact.
template <int P> __device__ __forceinline__ void split_pair(float a, float b, uint32_t* out) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (p == P - 1) {
            out[p] = P == 3 ? hi_pair(a, b) : round_pair(a, b);
        } else {
            out[p] = hi_pair(a, b);
            a -= cut(a);
            b -= cut(b);
        }
    }
}

template <int P> __device__ __forceinline__ Half<P> split(f4 x) {
    Half<P> h;
    uint32_t lo[P], hi[P];
    split_pair<P>(x[0], x[1], lo);
    split_pair<P>(x[2], x[3], hi);
#pragma unroll
    for (int p = 0; p < P; ++p) h.p[p] = u2{lo[p], hi[p]};
    return h;
}

template <int P> __device__ __forceinline__ Frag<P> join(const Half<P>& a, const Half<P>& b) {
    Frag<P> f;
#pragma unroll
    for (int p = 0; p < P; ++p) f.p[p] = u4{a.p[p][0], a.p[p][1], b.p[p][0], b.p[p][1]};
    return f;
}
template <int P> __device__ __forceinline__ Frag<P> split(f4 x, f4 y) { return join<P>(split<P>(x), split<P>(y)); }

// acc + A B, the smallest part products first. SUM: the largest sum of part numbers that counts.
template <int SUM, int PA, int PB> __device__ __forceinline__ f4 mul(const Frag<PA>& a, const Frag<PB>& b, f4 acc) {
#pragma unroll
    for (int s = SUM; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < PA; ++i)
            if (s - i >= 0 && s - i < PB)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a.p[i]), __builtin_bit_cast(bf8, b.p[s - i]), acc, 0, 0, 0);
    return acc;
}
template <int SUM, int PA, int PB> __device__ __forceinline__ f4 mul(const Half<PA>& a, const Half<PB>& b, f4 acc) {
#pragma unroll
    for (int s = SUM; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < PA; ++i)
            if (s - i >= 0 && s - i < PB)
                acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a.p[i]), __builtin_bit_cast(s4, b.p[s - i]), acc, 0, 0, 0);
    return acc;
}

// Left (or right) operands from LDS: `part` elements between the parts of a tile.
template <int P> __device__ __forceinline__ Frag<P> frag_at(const uint16_t* at, int part) {
    Frag<P> f;
#pragma unroll
    for (int p = 0; p < P; ++p) f.p[p] = *reinterpret_cast<const u4*>(at + p * part);
    return f;
}
template <int P> __device__ __forceinline__ Half<P> half_at(const uint16_t* at, int part) {
    Half<P> f;
#pragma unroll
    for (int p = 0; p < P; ++p) f.p[p] = *reinterpret_cast<const u2*>(at + p * part);
    return f;
}

__device__ __forceinline__ Frag<3> frag_of(const float* at) { return split<3>(*reinterpret_cast<const f4*>(at), *reinterpret_cast<const f4*>(at + 4)); }

// ---- element types ------------------------------------------------------------------------
enum Type : uint32_t { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };
template <int TY> struct Elem;
// `parts`: bf16 parts that hold a value exactly.
template <> struct Elem<T_F32> {
    typedef float type;
    static constexpr int parts = 3;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Elem<T_F16> {
    typedef _Float16 type;
    static constexpr int parts = 2;
    static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};
template <> struct Elem<T_BF16> {
    typedef uint16_t type;
    static constexpr int parts = 1;
    static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ uint16_t put(float x) { return (uint16_t)round_pair(x, x); }
};

// Eight consecutive elements as they are in memory, the first `n` of them in bounds (the rest are
// zero). `vec`: the address is a multiple of 16 bytes whenever n is 8. FULL: n is 8, and so it is.
template <int TY> struct Raw {
    static constexpr int words = TY == T_F32 ? 8 : 4;
    u4 a[words / 4];
    template <bool FULL> __device__ __forceinline__ void load(const typename Elem<TY>::type* at, int n, bool vec) {
        typedef typename Elem<TY>::type E;
        if (FULL || (vec && n >= 8)) {
#pragma unroll
            for (int i = 0; i < words / 4; ++i) a[i] = reinterpret_cast<const u4*>(at)[i];
        } else if constexpr (TY == T_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j / 4][j % 4] = j < n ? __float_as_uint(at[j]) : 0u;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t lo = 2 * j < n ? __builtin_bit_cast(uint16_t, at[2 * j]) : 0u;
                const uint32_t hi = 2 * j + 1 < n ? __builtin_bit_cast(uint16_t, (E)at[2 * j + 1]) : 0u;
                a[0][j] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ void keep(bool yes) {
#pragma unroll
        for (int i = 0; i < words; ++i) a[i / 4][i % 4] = yes ? a[i / 4][i % 4] : 0u;
    }
    __device__ __forceinline__ bool finite() const {
        if constexpr (TY == T_F32) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < words; ++i) top = max(top, a[i / 4][i % 4] & 0x7fffffffu);
            return top < 0x7f800000u;
        } else {
            typedef uint16_t h2 __attribute__((ext_vector_type(2)));
            constexpr uint32_t inf = TY == T_BF16 ? 0x7f80u : 0x7c00u;
            h2 top = {0, 0};
#pragma unroll
            for (int i = 0; i < words; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, a[0][i] & 0x7fff7fffu));
            return top[0] < inf && top[1] < inf;
        }
    }
    __device__ __forceinline__ void get(float* x) const {
        typedef typename Elem<TY>::type E;
        if constexpr (TY == T_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(a[j / 4][j % 4]);
        } else if constexpr (TY == T_BF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = __uint_as_float(a[0][j] << 16);
                x[2 * j + 1] = __uint_as_float(a[0][j] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = Elem<TY>::get(__builtin_bit_cast(E, (uint16_t)(a[0][j] & 0xffffu)));
                x[2 * j + 1] = Elem<TY>::get(__builtin_bit_cast(E, (uint16_t)(a[0][j] >> 16)));
            }
        }
    }
    // The bf16 parts, pairs of values by pair.
    __device__ __forceinline__ void parts(uint32_t w[4][Elem<TY>::parts]) const {
        if constexpr (TY == T_BF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j][0] = a[0][j];
        } else {
            float x[8];
            get(x);
#pragma unroll
            for (int j = 0; j < 4; ++j) split_pair<Elem<TY>::parts>(x[2 * j], x[2 * j + 1], w[j]);
        }
    }
};

// The same, out.
template <int TY, bool FULL = false> __device__ __forceinline__ void store8(typename Elem<TY>::type* at, int n, bool vec, const float* x) {
    if (FULL || (vec && n >= 8)) {
        if constexpr (TY == T_F32) {
            reinterpret_cast<f4*>(at)[0] = f4{x[0], x[1], x[2], x[3]};
            reinterpret_cast<f4*>(at)[1] = f4{x[4], x[5], x[6], x[7]};
        } else {
            u4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                a[j] = (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j])) |
                       (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j + 1])) << 16;
            *reinterpret_cast<u4*>(at) = a;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) at[j] = Elem<TY>::put(x[j]);
    }
}

// Four consecutive elements, the first `n` of them in bounds. `vec`: the address is a multiple of
// the four elements' bytes whenever n is 4. FULL: n is 4, and so it is.
template <int TY, bool FULL = false> __device__ __forceinline__ f4 load4(const typename Elem<TY>::type* at, int n, bool vec) {
    typedef typename Elem<TY>::type E;
    f4 x = {0, 0, 0, 0};
    if (FULL || (vec && n >= 4)) {
        if constexpr (TY == T_F32) {
            x = *reinterpret_cast<const f4*>(at);
        } else {
            const u2 a = *reinterpret_cast<const u2*>(at);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = Elem<TY>::get(__builtin_bit_cast(E, (uint16_t)(a[j >> 1] >> (16 * (j & 1)))));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) x[j] = Elem<TY>::get(at[j]);
    }
    return x;
}
template <int TY, bool FULL = false> __device__ __forceinline__ void store4(typename Elem<TY>::type* at, int n, bool vec, f4 x) {
    if (FULL || (vec && n >= 4)) {
        if constexpr (TY == T_F32) {
            *reinterpret_cast<f4*>(at) = x;
        } else {
            u2 a;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                a[j] = TY == T_BF16 ? round_pair(x[2 * j], x[2 * j + 1])
                                    : (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j])) |
                                          (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j + 1])) << 16;
            *reinterpret_cast<u2*>(at) = a;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) at[j] = Elem<TY>::put(x[j]);
    }
}

__device__ __forceinline__ uint32_t bits_of_size(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ bool finite(float x) { return bits_of_size(x) < 0x7f800000u; }
__device__ __forceinline__ bool finite(f4 x) {
    return max(max(bits_of_size(x[0]), bits_of_size(x[1])), max(bits_of_size(x[2]), bits_of_size(x[3]))) < 0x7f800000u;
}

// A value from another lane of the same 16 (or of the same four).
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// Sum over the 16 lanes that hold one row of a result tile; every lane gets it.
__device__ __forceinline__ float sum16(float x) {
    x += dpp<0x128>(x);  // rotations within 16 lanes by 8, 4, 2 and 1
    x += dpp<0x124>(x);
    x += dpp<0x122>(x);
    return x + dpp<0x121>(x);
}
// Transposes 4x4 values across four lanes: register r of lane q becomes register q of lane r. Of a
// result tile, lane n then holds row 4 g + n % 4, columns 4 (n / 4) + 0..3.
__device__ __forceinline__ f4 turn(f4 x, int lane) {
    const bool a = lane & 1, b = lane & 2;
    const float s0 = dpp<0xb1>(a ? x[0] : x[1]), s1 = dpp<0xb1>(a ? x[2] : x[3]);  // lanes 1 0 3 2
    const f4 y = a ? f4{s0, x[1], s1, x[3]} : f4{x[0], s0, x[2], s1};
    const float t0 = dpp<0x4e>(b ? y[0] : y[2]), t1 = dpp<0x4e>(b ? y[1] : y[3]);  // lanes 2 3 0 1
    return b ? f4{t0, t1, y[2], y[3]} : f4{y[0], y[1], t0, t1};
}
// The parts of four values that are consecutive in LDS.
template <int P> __device__ __forceinline__ void put4(uint16_t* at, int part, f4 x) {
    const Half<P> h = split<P>(x);
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<u2*>(at + p * part) = h.p[p];
}
// Sum over the wave; every lane gets it.
__device__ __forceinline__ float sum64(float x) {
    x = sum16(x);
    uint32_t b = __float_as_uint(x);
    auto rows = __builtin_amdgcn_permlane16_swap(b, b, false, false);  // the 16 lanes before and after, in pairs
    x = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    b = __float_as_uint(x);
    rows = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
}

}  // namespace mma
}  // namespace za
