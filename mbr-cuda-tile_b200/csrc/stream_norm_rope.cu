// stream_norm_rope.cu — norms of queries and keys per head with the rotary
// positions of several axes, in one pass.
//
// y = x * rsqrt(mean_d x^2 + eps) * gamma over one head of one token, then the
// pair (2i, 2i+1) turned by the angle of its axis' position: every element is
// read once and written once, so memory is its floor.  A group of lanes holds one
// head in registers (16 bytes a lane); the group's sum of squares is a shuffle
// butterfly, in fp32 like everything up to the final rounding.  60 x 801 tokens
// of 8 + 8 heads of 64 in fp16, two axes, read in place from a packed q|k|v
// (197 MB): 41.6 us, 4.7 TB/s (DRAM 41 % and issue slots 60 % busy: latency; the
// form for any layout: 253 us); 60 tokens 2.2 us.
// At fp32, heads of 32 and three axes the angles' loads and the instructions of
// the turn weigh more: 51 MB in 14.7 us, 3.5 TB/s.
#include <algorithm>

#include "common.cuh"
#include "stream_cache.cuh"

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
    FastDiv by_tokens, by_chunks;  // vector form: tokens of a sequence, steps of a token
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
// pairs).  A step is 32 / LANES x UNROLL heads of one token; a warp walks steps
// with the next step's loads (heads, then angles) in flight while it works on
// one.  The gains lie in shared memory: in registers they would halve the warps.
// WHOLE: every pair is turned.
template <typename T, int LANES, int UNROLL, bool WHOLE>
__global__ void __launch_bounds__(256, 3) norm_rope_vec_kernel(const NormRopeArgs a) {
    constexpr int E = 16 / sizeof(T);  // elements a lane
    constexpr int GROUPS = 32 / LANES;
    const int lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
    const bool in = sub * E < a.D;  // lanes past the head size hold zeros
    const int i0 = sub * E / 2;
    const bool turned = in && (WHOLE || i0 < a.used);
    const int axis = turned ? axis_of(a, i0) : 0, HT = a.Hq + a.Hkv;
    const float inv_d = 1.f / (float)a.D;
    __shared__ float gain[2][LANES * E];
    struct Step {
        uint4 raw[UNROLL];
        float cs[E / 2], sn[E / 2];
    };
    auto place = [&](unsigned step, unsigned& s, unsigned& t, int& h0) {
        const unsigned tok = a.by_chunks.div(step);
        s = a.by_tokens.div(tok);
        t = tok - s * a.by_tokens.d;
        h0 = (int)(step - tok * a.by_chunks.d) * GROUPS * UNROLL + grp;
        return tok;
    };
    auto load = [&](Step& x, unsigned step) {
        unsigned s, t;
        int h0;
        const unsigned tok = place(step, s, t, h0);
        const int p = turned ? __ldg(a.pos + (int64_t)tok * a.axes + axis) : -1;
        const T* q0 = (const T*)a.q + (int64_t)s * a.q_seq + t * a.q_tok + sub * E;
        const T* k0 = (const T*)a.k + (int64_t)s * a.k_seq + t * a.k_tok + sub * E;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = h0 + u * GROUPS;
            x.raw[u] = make_uint4(0u, 0u, 0u, 0u);
            if (h < HT && in)
                x.raw[u] = *reinterpret_cast<const uint4*>(h < a.Hq ? q0 + h * a.q_head : k0 + (h - a.Hq) * a.k_head);
        }
        const bool ok = p >= 0 && p < a.rows;
        const int64_t at = ok ? (int64_t)p * (a.D >> 1) + i0 : 0;
        // sections are multiples of a lane's pairs: its angles are one (or, in 32 bits, half a) 16-byte piece
        if constexpr (E == 8) {
            const float4 c = ok ? __ldg(reinterpret_cast<const float4*>(a.cs + at)) : make_float4(NAN, NAN, NAN, NAN);
            const float4 n = ok ? __ldg(reinterpret_cast<const float4*>(a.sn + at)) : make_float4(NAN, NAN, NAN, NAN);
            x.cs[0] = c.x, x.cs[1] = c.y, x.cs[2] = c.z, x.cs[3] = c.w;
            x.sn[0] = n.x, x.sn[1] = n.y, x.sn[2] = n.z, x.sn[3] = n.w;
        } else {
            const float2 c = ok ? __ldg(reinterpret_cast<const float2*>(a.cs + at)) : make_float2(NAN, NAN);
            const float2 n = ok ? __ldg(reinterpret_cast<const float2*>(a.sn + at)) : make_float2(NAN, NAN);
            x.cs[0] = c.x, x.cs[1] = c.y;
            x.sn[0] = n.x, x.sn[1] = n.y;
        }
    };
    const unsigned steps = (unsigned)a.ntok * a.by_chunks.d, stride = gridDim.x * 8;
    unsigned step = blockIdx.x * 8 + (threadIdx.x >> 5);
    Step x;
    if (step < steps) load(x, step);
    for (int i = threadIdx.x; i < 2 * LANES * E; i += 256) {
        const int d = i % (LANES * E);
        const float* g = i < LANES * E ? a.gq : a.gk;
        gain[i / (LANES * E)][d] = g && d < a.D ? __ldg(g + d) : 1.f;
    }
    __syncthreads();
    if (step >= steps) return;
    for (;;) {
        const bool more = step + stride < steps;
        Step y;
        if (more) load(y, step + stride);
        unsigned s, t;
        int h0;
        place(step, s, t, h0);
        T* qo0 = (T*)a.qo + (int64_t)s * a.qo_seq + t * a.qo_tok + sub * E;
        T* ko0 = (T*)a.ko + (int64_t)s * a.ko_seq + t * a.ko_tok + sub * E;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = h0 + u * GROUPS;
            // pairs (2i, 2i + 1) throughout, two fp32 operations an instruction
            const typename PairOf<T>::type* e = reinterpret_cast<const typename PairOf<T>::type*>(&x.raw[u]);
            float2 v[E / 2], sq = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < E / 2; ++i) v[i] = pair_to_f32<T>(e[i]), sq = __ffma2_rn(v[i], v[i], sq);
            float ss = sq.x + sq.y;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * inv_d + a.eps);
            const bool isq = h < a.Hq;
            const float2* g = reinterpret_cast<const float2*>(&gain[isq ? 0 : 1][sub * E]);
            union {
                T e[E];
                uint4 w;
            } z;
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                const float2 y = __fmul2_rn(__fmul2_rn(v[i], make_float2(r, r)), g[i]);
                const float2 n = __ffma2_rn(y, make_float2(x.cs[i], x.cs[i]),
                                            __fmul2_rn(make_float2(y.y, y.x), make_float2(-x.sn[i], x.sn[i])));
                store_pair<T>(&z.e[2 * i], WHOLE || turned ? n : y);
            }
            if (h < HT && in)
                *reinterpret_cast<uint4*>(isq ? qo0 + h * a.qo_head : ko0 + (h - a.Hq) * a.ko_head) = z.w;
        }
        if (!more) break;
        x = y;
        step += stride;
    }
}

template <typename T, int LANES, int UNROLL, bool WHOLE>
void launch_steps(NormRopeArgs a, cudaStream_t st) {
    constexpr int heads = 32 / LANES * UNROLL;
    const int64_t chunks = ceil_div(a.Hq + a.Hkv, heads);
    a.by_tokens = FastDiv((unsigned)a.tokens), a.by_chunks = FastDiv((unsigned)chunks);
    auto kern = norm_rope_vec_kernel<T, LANES, UNROLL, WHOLE>;
    static int wave[kMaxStreamDevices] = {};  // CTAs that fit the device at once
    const int dev = stream_device();
    if (!wave[dev]) {
        int per = 0, sms = 0;
        MBR_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, 256, 0));
        MBR_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        wave[dev] = std::max(1, per * sms);
    }
    kern<<<(unsigned)std::min<int64_t>(ceil_div(a.ntok * chunks, 8), wave[dev]), 256, 0, st>>>(a);
}

// With few tokens a step is one head a lane group (more warps share the latency),
// otherwise four (more loads in flight a warp).  16 heads of 64 in fp16 (us, one /
// four): 480 tokens 2.6 / 3.3, 960 tokens 3.0 / 3.4, 3840 tokens 5.8 / 5.4, 48060
// tokens 55 / 41.  Three where four would leave more lanes without a head (us, three /
// four, 48060 tokens, one axis): 8 + 2 heads of 32 in fp32 29 / 32, of 64 in fp16 33 / 37, 16 + 4 of 64 in
// fp16 62 / 72; where they leave as many or more, four: 8 + 8 heads of 64 in fp16 61 / 41, 12 +
// 4 of 32 in fp32 51 / 39, 16 + 4 of 64 in fp32 105 / 98.
template <typename T, int LANES, bool WHOLE>
void launch_unrolled(const NormRopeArgs& a, cudaStream_t st) {
    constexpr int GROUPS = 32 / LANES;
    const int heads = a.Hq + a.Hkv;
    if (a.ntok * (a.Hq + a.Hkv) <= 148 * 64 * 32 / LANES) launch_steps<T, LANES, 1, WHOLE>(a, st);
    else if (ceil_div(heads, 3 * GROUPS) * 3 < ceil_div(heads, 4 * GROUPS) * 4) launch_steps<T, LANES, 3, WHOLE>(a, st);
    else launch_steps<T, LANES, 4, WHOLE>(a, st);
}
template <typename T, int LANES>
void launch_lanes(const NormRopeArgs& a, cudaStream_t st) {
    if (2 * a.used == a.D) launch_unrolled<T, LANES, true>(a, st);
    else launch_unrolled<T, LANES, false>(a, st);
}
// Launches the vector form if the call fits it.
template <typename T>
bool launch_vec(const NormRopeArgs& a, bool aligned, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    bool sections = a.used % (E / 2) == 0;
    for (int i = 0; i < 3; ++i) sections = sections && (a.end[i] == INT32_MAX || a.end[i] % (E / 2) == 0);
    const int lanes = a.D / E;
    if (!aligned || a.D % E != 0 || !sections || lanes > 32 || a.ntok * (a.Hq + a.Hkv) >= (1ll << 30)) return false;
    if (lanes <= 4) launch_lanes<T, 4>(a, st);
    else if (lanes <= 8) launch_lanes<T, 8>(a, st);
    else if (lanes <= 16) launch_lanes<T, 16>(a, st);
    else launch_lanes<T, 32>(a, st);
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
                         (Hkv == 0 || (rows_aligned16(k, es) && rows_aligned16(ko, es))) &&
                         (((uintptr_t)cs | (uintptr_t)sn) & 15) == 0;
    MBR_DISPATCH_DTYPE(dtype, T, {
        if (!launch_vec<T>(a, aligned, st)) norm_rope_any_kernel<T><<<grid, 256, 0, st>>>(a);
    });
    MBR_CUDA(cudaGetLastError());
}

}  // namespace streamops
}  // namespace mbr
