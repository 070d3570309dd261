// Whether arrays of strides share memory: host checks of the policy operators' outputs.
#pragma once
#include <stdint.h>

#include <utility>

namespace za {

// What an array covers: rows of `unit` bytes from `base` on, along up to three dimensions of positive
// strides in bytes, the largest first. Dimensions that repeat memory (stride 0) are left out.
struct Memory {
    int64_t base = 0, unit = 0;
    int dims = 0;
    int64_t stride[3], n[3];
    bool repeats = false;  // a stride of 0 along more than one element

    Memory(const void* p, const int64_t* strides, const int64_t* sizes, int count, int64_t row, int64_t bytes) : base((int64_t)(uintptr_t)p), unit(row * bytes) {
        for (int i = 0; i < count; ++i) {
            if (sizes[i] < 2) continue;
            int64_t s = strides[i] * bytes;
            if (s == 0) {
                repeats = true;
                continue;
            }
            if (s < 0) {
                base += s * (sizes[i] - 1);
                s = -s;
            }
            int at = dims++;
            for (; at > 0 && stride[at - 1] < s; --at) stride[at] = stride[at - 1], n[at] = n[at - 1];
            stride[at] = s;
            n[at] = sizes[i];
        }
    }
    int64_t span(int from) const {  // bytes from the first to behind the last, of the dimensions from `from` on
        int64_t x = unit;
        for (int i = from; i < dims; ++i) x += stride[i] * (n[i] - 1);
        return x;
    }
    // Every element at a place of its own: each dimension steps over all that lies inside it. (Some
    // arrays whose dimensions interleave would pass a finer test.)
    bool apart_from_itself() const {
        for (int i = 0; i < dims; ++i)
            if (stride[i] < span(i + 1)) return false;
        return !repeats;
    }
};

// Whether two arrays surely share no byte: their ranges are apart, or they step alike and what they
// hold of each step is (views of one buffer).
inline bool apart(const Memory& a, const Memory& b, int ia, int ib, int64_t offset) {  // offset: of a's base from b's
    if (offset >= b.span(ib) || -offset >= a.span(ia)) return true;
    if (ia == a.dims || ib == b.dims || a.stride[ia] != b.stride[ib]) return false;
    const int64_t s = a.stride[ia];
    if (a.span(ia + 1) > s || b.span(ib + 1) > s) return false;
    const int64_t o = ((offset % s) + s) % s;
    return apart(a, b, ia + 1, ib + 1, o) && apart(a, b, ia + 1, ib + 1, o - s);
}
inline bool apart(const Memory& a, const Memory& b) { return apart(a, b, 0, 0, a.base - b.base); }

}  // namespace za
