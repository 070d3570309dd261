// Rows of elements at any address: eight consecutive ones a lane.
//
// The operators that include this read rows of every stride, so a row begins at a multiple of its
// element's size and no more. Vector accesses need no more either (the compiler makes the same
// 16-byte instructions of them), so there is one path for aligned rows and others.
#pragma once
#include "mma.h"

namespace za {
namespace mma {

template <int TY> struct Loose {  // 16 bytes at an element's address
    struct __attribute__((packed, aligned(sizeof(typename Elem<TY>::type)))) U {
        u4 v;
    };
};

// The first `n` of eight elements (n <= 0: none; the rest are zero). FULL: all.
template <int TY> struct Eight : Raw<TY> {
    template <bool FULL> __device__ __forceinline__ void load(const typename Elem<TY>::type* at, int n) {
        typedef typename Elem<TY>::type E;
        constexpr int vectors = Raw<TY>::words / 4;
        if (FULL || n >= 8) {
#pragma unroll
            for (int i = 0; i < vectors; ++i) this->a[i] = reinterpret_cast<const typename Loose<TY>::U*>(at)[i].v;
        } else {
#pragma unroll
            for (int i = 0; i < vectors; ++i) this->a[i] = u4{0, 0, 0, 0};
            if (n > 0) {
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (j < n) {
                        if constexpr (TY == T_F32) this->a[j / 4][j % 4] = __float_as_uint(at[j]);
                        else this->a[0][j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, (E)at[j]) << (16 * (j & 1));
                    }
            }
        }
    }
    __device__ __forceinline__ void set(const float* x) {  // rounded to the type
        if constexpr (TY == T_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) this->a[j / 4][j % 4] = __float_as_uint(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                this->a[0][j] = TY == T_BF16 ? round_pair(x[2 * j], x[2 * j + 1])
                                             : (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j])) |
                                                   (uint32_t)__builtin_bit_cast(uint16_t, Elem<TY>::put(x[2 * j + 1])) << 16;
        }
    }
    template <bool FULL> __device__ __forceinline__ void store(typename Elem<TY>::type* at, int n) const {
        typedef typename Elem<TY>::type E;
        constexpr int vectors = Raw<TY>::words / 4;
        if (FULL || n >= 8) {
#pragma unroll
            for (int i = 0; i < vectors; ++i) reinterpret_cast<typename Loose<TY>::U*>(at)[i].v = this->a[i];
        } else if (n > 0) {
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (j < n) {
                    if constexpr (TY == T_F32) at[j] = __uint_as_float(this->a[j / 4][j % 4]);
                    else at[j] = __builtin_bit_cast(E, (uint16_t)(this->a[0][j / 2] >> (16 * (j & 1))));
                }
        }
    }
};

}  // namespace mma
}  // namespace za
