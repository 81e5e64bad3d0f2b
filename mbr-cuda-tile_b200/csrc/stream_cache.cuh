// stream_cache.cuh — device view of the rolling key/value cache: slot of a
// position, the values of a 4-bit row, and which keys a query sees.
#pragma once

#include "common.cuh"
#include "stream_ops.h"

namespace mbr {
namespace streamops {

// Division of 31-bit numbers by a divisor fixed for a launch: with l = ceil(log2
// d) and mul = ceil(2^(31 + l) / d), n mul / 2^(31 + l) exceeds n / d by less
// than 1 / d for n < 2^31.
struct FastDiv {
    unsigned d = 1, mul = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(unsigned n) : d(n) {
        if (n < 2) return;
        unsigned l = 1;
        while ((1ull << l) < n) ++l;
        mul = (unsigned)(((1ull << (31 + l)) + n - 1) / n);
        shift = l - 1;
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

constexpr int kGroup = 32;  // channels that share a step and an offset in a 4-bit cache

// Slot of position p >= 0.
__device__ __forceinline__ int64_t slot_of(int p, int sinks, int ring) {
    return p < sinks ? p : sinks + (int64_t)((unsigned)(p - sinks) % (unsigned)ring);
}

// The value that code c of a group with step s and offset m stands for, m + s (c
// - 8): one rounding, to the cache's type (an fp32 sum would be a second one).
template <typename T>
__device__ __forceinline__ T code_value(int c, T s, T m) {
    return __hfma(s, from_f32<T>((float)(c - 8)), m);
}

// Keys of a query at position p over `len` keys: [lo, hi) and [0, first).
// left / right < 0: no limit.  No sum here leaves 32 bits: p >= 0 or right <
// 2^30 (the host turns larger limits into "none").
struct Window {
    int lo, hi, first;
};
__device__ __forceinline__ Window window_of(int p, int len, int left, int right, int sinks) {
    Window w;
    w.hi = right < 0 || (p >= 0 && right >= len - p) ? len : min(len, p + right + 1);
    w.hi = max(w.hi, 0);
    w.lo = left < 0 ? 0 : max(0, p - left);
    w.lo = min(w.lo, w.hi);
    w.first = min(min(sinks, w.hi), w.lo);
    return w;
}

}  // namespace streamops
}  // namespace mbr
