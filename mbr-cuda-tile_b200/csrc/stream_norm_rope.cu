// stream_norm_rope.cu — norms of queries and keys per head with the rotary
// positions of several axes, in one pass.
//
// y = x * rsqrt(mean_d x^2 + eps) * gamma over one head of one token, then the
// pair (2i, 2i+1) turned by the angle of its axis' position: every element is
// read once and written once, so memory bounds it.  A group of lanes holds one
// head in registers (16 bytes a lane); the group's sum of squares is a shuffle
// butterfly, in fp32 like everything up to the final rounding.
#include <algorithm>

#include "common.cuh"
#include "stream_ops.h"

namespace mbr {
namespace streamops {

namespace {

struct NormRopeArgs {
    const void *q, *k;
    void *qo, *ko;
    int64_t q_seq, q_tok, q_head, k_seq, k_tok, k_head;
    int64_t qo_seq, qo_tok, qo_head, ko_seq, ko_tok, ko_head;
    int64_t ntok;  // seqs * tokens
    int64_t tokens;
    int Hq, Hkv, D;
    const float *gq, *gk, *cs, *sn;
    float eps;
    int64_t rows;
    const int32_t* pos;
    int axes;
    int end[4];  // pair index at which axis a's section ends (INT_MAX past the last)
    int used;    // pairs turned
};

// Axis of pair i (i < used).
__device__ __forceinline__ int axis_of(const NormRopeArgs& a, int i) {
    return (i >= a.end[0]) + (i >= a.end[1]) + (i >= a.end[2]);
}

// (cos, sin) of pair i at token `tok` (row-major [seqs][tokens]); identity for
// pairs that are not turned, NaN for a position outside the tables.
__device__ __forceinline__ float2 turn_of(const NormRopeArgs& a, int64_t tok, int i) {
    if (i >= a.used) return make_float2(1.f, 0.f);
    const int p = __ldg(a.pos + tok * a.axes + axis_of(a, i));
    if (p < 0 || p >= a.rows) return make_float2(NAN, NAN);
    const int64_t at = (int64_t)p * (a.D >> 1) + i;
    return make_float2(__ldg(a.cs + at), __ldg(a.sn + at));
}

// One warp per (token, head); lane l holds pairs l, l + 32, ... (D <= 256).
// Any even head size, any strides and alignment.
template <typename T>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(const NormRopeArgs a) {
    const int lane = threadIdx.x & 31;
    const int HT = a.Hq + a.Hkv;
    const int64_t n = a.ntok * HT, step = (int64_t)gridDim.x * 8;
    for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n; w += step) {
        const int64_t tok = w / HT;
        const int hh = (int)(w - tok * HT);
        const int64_t s = tok / a.tokens, t = tok - s * a.tokens;
        const bool isq = hh < a.Hq;
        const int h = isq ? hh : hh - a.Hq;
        const T* x = isq ? (const T*)a.q + s * a.q_seq + t * a.q_tok + h * a.q_head
                         : (const T*)a.k + s * a.k_seq + t * a.k_tok + h * a.k_head;
        T* y = isq ? (T*)a.qo + s * a.qo_seq + t * a.qo_tok + h * a.qo_head
                   : (T*)a.ko + s * a.ko_seq + t * a.ko_tok + h * a.ko_head;
        const float* g = isq ? a.gq : a.gk;
        float v[4][2];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = lane + 32 * c;
            v[c][0] = v[c][1] = 0.f;
            if (i < a.D / 2) {
                v[c][0] = to_f32<T>(x[2 * i]);
                v[c][1] = to_f32<T>(x[2 * i + 1]);
                ss += v[c][0] * v[c][0] + v[c][1] * v[c][1];
            }
        }
        ss = warp_sum(ss);
        const float r = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = lane + 32 * c;
            if (i < a.D / 2) {
                const float y0 = v[c][0] * r * (g ? __ldg(g + 2 * i) : 1.f);
                const float y1 = v[c][1] * r * (g ? __ldg(g + 2 * i + 1) : 1.f);
                const float2 cs = turn_of(a, tok, i);
                const bool turned = i < a.used;
                y[2 * i] = from_f32<T>(turned ? y0 * cs.x - y1 * cs.y : y0);
                y[2 * i + 1] = from_f32<T>(turned ? y0 * cs.y + y1 * cs.x : y1);
            }
        }
    }
}

// Vector form: a head is LANES lanes x 16 bytes (dim_head a multiple of a lane's
// elements, rows on 16-byte boundaries, every section a multiple of a lane's
// pairs).  A warp takes one token: its lanes hold the token's (cos, sin) and
// gains once and walk its heads 32 / LANES x UNROLL at a time, all loads of a
// step in flight before the first is used.
template <typename T, int LANES, int UNROLL>
__global__ void __launch_bounds__(256) norm_rope_vec_kernel(const NormRopeArgs a) {
    constexpr int E = 16 / sizeof(T);  // elements a lane
    const int lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
    constexpr int GROUPS = 32 / LANES;
    const bool in = sub * E < a.D;  // lanes past the head size hold zeros
    const int64_t tok = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (tok >= a.ntok) return;
    const int64_t s = tok / a.tokens, t = tok - s * a.tokens;
    const T* q0 = (const T*)a.q + s * a.q_seq + t * a.q_tok + sub * E;
    const T* k0 = (const T*)a.k + s * a.k_seq + t * a.k_tok + sub * E;
    T* qo0 = (T*)a.qo + s * a.qo_seq + t * a.qo_tok + sub * E;
    T* ko0 = (T*)a.ko + s * a.ko_seq + t * a.ko_tok + sub * E;
    float cs[E / 2], sn[E / 2];
    const int i0 = sub * E / 2;
    const bool turned = in && i0 < a.used;
    {
        bool ok = false;
        int64_t at = 0;
        if (turned) {
            const int p = __ldg(a.pos + tok * a.axes + axis_of(a, i0));
            ok = p >= 0 && p < a.rows;
            at = (int64_t)p * (a.D >> 1) + i0;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            cs[i] = ok ? __ldg(a.cs + at + i) : NAN;
            sn[i] = ok ? __ldg(a.sn + at + i) : NAN;
        }
    }
    const int HT = a.Hq + a.Hkv;
    const float inv_d = 1.f / (float)a.D;
    for (int h0 = grp; h0 < HT; h0 += GROUPS * UNROLL) {
        uint4 raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = h0 + u * GROUPS;
            raw[u] = make_uint4(0u, 0u, 0u, 0u);
            if (h < HT && in)
                raw[u] = *reinterpret_cast<const uint4*>(h < a.Hq ? q0 + h * a.q_head : k0 + (h - a.Hq) * a.k_head);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = h0 + u * GROUPS;
            if (u > 0 && h - grp >= HT) break;  // no group has a head left (warp-uniform)
            const T* x = reinterpret_cast<const T*>(&raw[u]);
            float v[E], ss = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = to_f32<T>(x[i]), ss += v[i] * v[i];
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * inv_d + a.eps);
            const float* g = h < a.Hq ? a.gq : a.gk;
            union {
                T e[E];
                uint4 w;
            } y;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const float y0 = v[i] * r * (g && in ? __ldg(g + sub * E + i) : 1.f);
                const float y1 = v[i + 1] * r * (g && in ? __ldg(g + sub * E + i + 1) : 1.f);
                y.e[i] = from_f32<T>(turned ? y0 * cs[i / 2] - y1 * sn[i / 2] : y0);
                y.e[i + 1] = from_f32<T>(turned ? y0 * sn[i / 2] + y1 * cs[i / 2] : y1);
            }
            if (h < HT && in)
                *reinterpret_cast<uint4*>(h < a.Hq ? qo0 + h * a.qo_head : ko0 + (h - a.Hq) * a.ko_head) = y.w;
        }
    }
}

// Launches the vector form if the call fits it.
template <typename T>
bool launch_vec(const NormRopeArgs& a, bool aligned, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    bool sections = a.used % (E / 2) == 0;
    for (int i = 0; i < 3; ++i) sections = sections && (a.end[i] == INT32_MAX || a.end[i] % (E / 2) == 0);
    const int lanes = a.D / E;
    const int64_t grid = ceil_div(a.ntok, 8);
    if (!aligned || a.D % E != 0 || !sections || lanes > 32 || grid > INT32_MAX) return false;
    const unsigned n = (unsigned)grid;
    if (lanes <= 4) norm_rope_vec_kernel<T, 4, 2><<<n, 256, 0, st>>>(a);
    else if (lanes <= 8) norm_rope_vec_kernel<T, 8, 4><<<n, 256, 0, st>>>(a);
    else if (lanes <= 16) norm_rope_vec_kernel<T, 16, 4><<<n, 256, 0, st>>>(a);
    else norm_rope_vec_kernel<T, 32, 4><<<n, 256, 0, st>>>(a);
    return true;
}

}  // namespace

void qk_norm_rope(const mbr_view& q, const mbr_view& k, const mbr_view& qo, const mbr_view& ko, int64_t seqs,
                  int64_t tokens, int Hq, int Hkv, int D, const float* gamma_q, const float* gamma_k, float eps,
                  const float* cs, const float* sn, int64_t table_rows, const int32_t* pos, int axes,
                  const int* pairs, int dtype, cudaStream_t st) {
    MBR_CHECK(seqs >= 0 && tokens >= 0 && Hq >= 0 && Hkv >= 0, "qk_norm_rope: negative size");
    MBR_CHECK(D >= 2 && D <= 256 && D % 2 == 0, "qk_norm_rope: dim_head must be even, 2..256");
    MBR_CHECK(axes >= 0 && axes <= 4, "qk_norm_rope: axes must be 0..4");
    MBR_CHECK(eps >= 0.f, "qk_norm_rope: eps must not be negative");
    MBR_CHECK(dtype == DT_F32 || dtype == DT_F16 || dtype == DT_BF16, "qk_norm_rope: dtype must be fp32, fp16 or bf16");
    NormRopeArgs a{};
    a.used = 0;
    for (int i = 0; i < 4; ++i) a.end[i] = INT32_MAX;
    if (axes > 0) {
        MBR_CHECK(pairs && cs && sn && table_rows >= 0, "qk_norm_rope: tables and sections are needed");
        for (int i = 0; i < axes; ++i) {
            MBR_CHECK(pairs[i] >= 0 && pairs[i] <= D / 2 - a.used, "qk_norm_rope: sections exceed dim_head / 2 pairs");
            a.used += pairs[i];
            if (i + 1 < axes) a.end[i] = a.used;
        }
    }
    if (seqs == 0 || tokens == 0 || Hq + Hkv == 0) return;
    MBR_CHECK(axes == 0 || pos, "qk_norm_rope: positions are needed");
    MBR_CHECK((Hq == 0 || (q.data && qo.data)) && (Hkv == 0 || (k.data && ko.data)), "qk_norm_rope: null buffer");
    MBR_CHECK(tokens <= INT64_MAX / 4096 / seqs && Hq < (1 << 20) && Hkv < (1 << 20), "qk_norm_rope: too large");
    a.q = q.data, a.k = k.data, a.qo = qo.data, a.ko = ko.data;
    a.q_seq = q.seq, a.q_tok = q.token, a.q_head = q.head;
    a.k_seq = k.seq, a.k_tok = k.token, a.k_head = k.head;
    a.qo_seq = qo.seq, a.qo_tok = qo.token, a.qo_head = qo.head;
    a.ko_seq = ko.seq, a.ko_tok = ko.token, a.ko_head = ko.head;
    a.ntok = seqs * tokens, a.tokens = tokens, a.Hq = Hq, a.Hkv = Hkv, a.D = D;
    a.gq = gamma_q, a.gk = gamma_k, a.cs = cs, a.sn = sn, a.eps = eps;
    a.rows = table_rows, a.pos = pos, a.axes = axes;
    const int64_t warps = a.ntok * (Hq + Hkv);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(warps, 8), 148 * 64);
    const int es = (int)dtype_bytes(dtype);
    const bool aligned = (Hq == 0 || (rows_aligned16(q, es) && rows_aligned16(qo, es))) &&
                         (Hkv == 0 || (rows_aligned16(k, es) && rows_aligned16(ko, es)));
    MBR_DISPATCH_DTYPE(dtype, T, {
        if (!launch_vec<T>(a, aligned, st)) norm_rope_any_kernel<T><<<grid, 256, 0, st>>>(a);
    });
    MBR_CUDA(cudaGetLastError());
}

}  // namespace streamops
}  // namespace mbr
