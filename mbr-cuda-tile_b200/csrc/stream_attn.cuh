// stream_attn.cuh — what the streaming-attention kernels share: where keys and
// values live, and the attention of one row by one warp.
#pragma once

#include "stream_cache.cuh"

namespace mbr {
namespace streamops {

// One call's problem.  Keys are a strided view (cached = false) or the rolling
// cache; `len` / `q_len` give the keys and queries of each sequence.
struct AttnArgs {
    const void* q;
    void* out;
    int64_t q_seq, q_tok, q_head, o_seq, o_tok, o_head;
    const void *k, *v;
    int64_t k_seq, k_tok, k_head, v_seq, v_tok, v_head;  // view
    const void *k_scale, *v_scale;                       // cache, 4 bits
    int ring, cache_sinks;                               // cache
    int64_t slots;
    int64_t seqs;
    int Nq, Nk, Hq, Hkv, D, G;  // G = Hq / Hkv
    FastDiv by_G, by_Hkv;
    const int32_t *q_len, *kv_len;
    int left, right, sinks;
    float scale;
    const float* gates;
};

// Keys and queries of sequence s.  A cache's length may be anything; a view's
// are clamped to its extent.
template <bool CACHED>
__device__ __forceinline__ void lengths(const AttnArgs& a, int64_t s, int& n, int& m) {
    if constexpr (CACHED) {
        n = a.Nq;
        m = max(__ldg(a.kv_len + s), 0);
    } else {
        n = a.q_len ? min(max(__ldg(a.q_len + s), 0), a.Nq) : a.Nq;
        m = a.kv_len ? min(max(__ldg(a.kv_len + s), 0), a.Nk) : a.Nk;
    }
}

// Keys that query i of a sequence with n queries and m keys sees.  A cache has
// dropped the positions in [sinks, m - ring); a negative position of it sees none.
template <bool CACHED>
__device__ __forceinline__ Window row_window(const AttnArgs& a, int i, int n, int m) {
    const int p = m - n + i;
    Window w = window_of(p, m, a.left, a.right, a.sinks);
    if constexpr (CACHED) {
        if (p < 0) w.hi = 0;
        w.lo = min(max(w.lo, m - a.ring), w.hi);
        w.first = min(min(a.sinks, w.hi), w.lo);
    }
    return w;
}

// Element d of key / value row of position p.
template <typename T, bool CACHED, bool Q4>
__device__ __forceinline__ float kv_elem(const AttnArgs& a, bool val, int64_t s, int hk, int p, int d) {
    if constexpr (!CACHED) {
        const T* b = val ? (const T*)a.v + s * a.v_seq + p * a.v_tok + hk * a.v_head
                         : (const T*)a.k + s * a.k_seq + p * a.k_tok + hk * a.k_head;
        return to_f32<T>(b[d]);
    } else {
        const int64_t row = (s * a.Hkv + hk) * a.slots + slot_of(p, a.cache_sinks, a.ring);
        if constexpr (!Q4) {
            return to_f32<T>(((const T*)(val ? a.v : a.k))[row * a.D + d]);
        } else {
            const int byte = ((const uint8_t*)(val ? a.v : a.k))[row * (a.D / 2) + (d >> 1)];
            const T* sm = (const T*)(val ? a.v_scale : a.k_scale) + (row * (a.D / kGroup) + d / kGroup) * 2;
            return to_f32<T>(code_value<T>((byte >> ((d & 1) * 4)) & 15, sm[0], sm[1]));
        }
    }
}

// The attention of one row (sequence s, query i, head h) by one warp, four keys at
// a time with the running maximum and sum of the softmax in fp32; lane l holds
// channels l, l + 32, ...  Keys outside the row's window are not read, so
// nothing they hold can reach the result.  NaN scores make the row NaN.
template <typename T, bool CACHED, bool Q4>
__device__ __noinline__ void attend_row(const AttnArgs& a, int64_t s, int i, int h, int n, int m) {
    const int lane = threadIdx.x & 31, hk = h / a.G;
    T* o = (T*)a.out + s * a.o_seq + (int64_t)i * a.o_tok + (int64_t)h * a.o_head;
    const T* q = (const T*)a.q + s * a.q_seq + (int64_t)i * a.q_tok + (int64_t)h * a.q_head;
    Window w = row_window<CACHED>(a, i, n, m);
    if (i >= n) w.first = w.lo = w.hi = 0;
    float qv[4], acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int d = lane + 32 * c;
        qv[c] = d < a.D ? to_f32<T>(q[d]) : 0.f;
        acc[c] = 0.f;
    }
    float top = -INFINITY, sum = 0.f;
    constexpr int U = 4;  // keys at a time: their loads and shuffles overlap
    for (int pass = 0; pass < 2; ++pass) {
        const int j0 = pass ? w.lo : 0, j1 = pass ? w.hi : w.first;
        for (int j = j0; j < j1; j += U) {
            float x[U], v[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                x[u] = 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int d = lane + 32 * c;
                    v[u][c] = 0.f;
                    if (d < a.D && j + u < j1) {
                        x[u] = fmaf(qv[c], kv_elem<T, CACHED, Q4>(a, false, s, hk, j + u, d), x[u]);
                        v[u][c] = kv_elem<T, CACHED, Q4>(a, true, s, hk, j + u, d);
                    }
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] += __shfl_xor_sync(0xffffffffu, x[u], o);
            float now = top;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                x[u] *= a.scale;
                if (j + u < j1) now = fmaxf(now, x[u]);
            }
            // a maximum of -inf (every score so far -inf) leaves exp(-inf - -inf): such keys weigh nothing
            const float old = now == -INFINITY ? 1.f : expf(top - now);
            top = now;
            sum *= old;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= old;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j + u >= j1) break;
                const float e = now == -INFINITY && x[u] == x[u] ? 0.f : expf(x[u] - now);
                sum += e;
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] = fmaf(e, v[u][c], acc[c]);
            }
        }
    }
    const float g = a.gates ? __ldg(a.gates + (s * a.Nq + i) * a.Hq + h) : 1.f;
    const float inv = 1.f / sum;  // 0 only if every score seen is -inf: NaN, as the formula
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int d = lane + 32 * c;
        if (d < a.D) o[d] = from_f32<T>(w.hi == w.lo && w.first == 0 ? 0.f : acc[c] * inv * g);  // nothing seen: 0
    }
}

}  // namespace streamops
}  // namespace mbr
