// stream_attn.cu — entry points of the streaming attention (prompt form and
// few-token form over the rolling cache) and the few-token form's fp32 kernel.
#include <algorithm>
#include <cmath>

#include "stream_attn.cuh"
#include "stream_attn_simt.h"
#include "stream_attn_step.h"
#include "stream_attn_tc.h"

namespace mbr {
namespace streamops {

int stream_device() {
    int dev = 0;
    MBR_CUDA(cudaGetDevice(&dev));
    MBR_CHECK(dev >= 0 && dev < kMaxStreamDevices, "device index out of range");
    return dev;
}

namespace {

// Attention over an fp32 cache, a CTA a row: LANES lanes (four channels each) hold a
// key, a CTA's groups of lanes take every so many keys, four at a time with their
// values' loads in flight too, each with a running maximum and sum; the groups
// are joined through shared memory in a fixed order.  Only what the row sees is
// read, and rows of a shared key head read it once each, so memory (or L2) bounds it:
// 60 x 8 rows over 1004 keys of 64 (247 MB) 42.4 us, 5.8 TB/s (a warp a row, four keys at a
// time: 1605 us).
template <int LANES>
__global__ void __launch_bounds__(256) attend_rows_kernel(const AttnArgs a) {
    constexpr int NG = 256 / LANES, U = 4;
    __shared__ float2 state[NG];  // offset, sum
    __shared__ float4 part[NG][LANES];
    const int sub = threadIdx.x % LANES, grp = threadIdx.x / LANES, D = a.D;
    const bool in = 4 * sub < D;
    const int64_t rows = a.seqs * a.Nq * a.Hq;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t si = r / a.Hq, s = si / a.Nq;
        const int i = (int)(si - s * a.Nq), h = (int)(r - si * a.Hq), hk = h / a.G;
        int n, m;
        lengths<true>(a, s, n, m);
        const Window w = row_window<true>(a, i, n, m);
        const unsigned total = w.first + (w.hi - w.lo), first = w.first;
        // slot of the u-th key: the first tokens, then the window, whose ring starts over at most once
        const int slot0 = w.lo < a.cache_sinks ? w.lo : (int)slot_of(w.lo, a.cache_sinks, a.ring);
        const float4* k = (const float4*)((const float*)a.k + (s * a.Hkv + hk) * a.slots * D) + sub;
        const float4* v = (const float4*)((const float*)a.v + (s * a.Hkv + hk) * a.slots * D) + sub;
        const int row4 = D / 4;
        const float* q = (const float*)a.q + s * a.q_seq + (int64_t)i * a.q_tok + (int64_t)h * a.q_head + 4 * sub;
        float4 qv = make_float4(0.f, 0.f, 0.f, 0.f), acc = qv;
        if (in) qv = make_float4(q[0], q[1], q[2], q[3]);
        float top = -INFINITY, sum = 0.f;
        for (unsigned u0 = grp; u0 - grp < total; u0 += NG * U) {  // the same rounds for all lanes of a warp
            float4 kx[U], vx[U];
            float x[U];
#pragma unroll
            for (int c = 0; c < U; ++c) {
                const unsigned u = u0 + c * NG;
                kx[c] = vx[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (in && u < total) {
                    int64_t at = u < first ? (int64_t)u : (int64_t)slot0 + (u - first);
                    if (at >= a.slots) at -= a.ring;
                    kx[c] = k[at * row4], vx[c] = v[at * row4];
                }
            }
#pragma unroll
            for (int c = 0; c < U; ++c)
                x[c] = fmaf(qv.x, kx[c].x, fmaf(qv.y, kx[c].y, fmaf(qv.z, kx[c].z, qv.w * kx[c].w)));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
                for (int c = 0; c < U; ++c) x[c] += __shfl_xor_sync(0xffffffffu, x[c], o);
            float now = top;
#pragma unroll
            for (int c = 0; c < U; ++c) {
                x[c] *= a.scale;
                if (u0 + c * NG < total) now = fmaxf(now, x[c]);
            }
            // a maximum of -inf (every score so far -inf) leaves exp(-inf - -inf): such keys weigh nothing
            const float old = now == -INFINITY ? 1.f : expf(top - now);
            top = now;
            sum *= old;
            acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
#pragma unroll
            for (int c = 0; c < U; ++c) {
                const bool on = u0 + c * NG < total;
                const float e = !on || (now == -INFINITY && x[c] == x[c]) ? 0.f : expf(x[c] - now);
                sum += e;
                if (on) {
                    acc.x = fmaf(e, vx[c].x, acc.x), acc.y = fmaf(e, vx[c].y, acc.y);
                    acc.z = fmaf(e, vx[c].z, acc.z), acc.w = fmaf(e, vx[c].w, acc.w);
                }
            }
        }
        if (sub == 0) state[grp] = make_float2(top, sum);
        part[grp][sub] = acc;
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += 256) {
            float most = -INFINITY, l = 0.f, o = 0.f;
            for (int b = 0; b < NG; ++b) most = fmaxf(most, state[b].x);
            for (int b = 0; b < NG; ++b) {
                // a group without a score above -inf holds zeros (or NaN, which stay)
                const float f = state[b].x == -INFINITY ? 1.f : expf(state[b].x - most);
                l = fmaf(f, state[b].y, l);
                o = fmaf(f, reinterpret_cast<const float*>(part[b])[d], o);
            }
            const float g = a.gates ? __ldg(a.gates + (s * a.Nq + i) * a.Hq + h) : 1.f;
            float* out = (float*)a.out + s * a.o_seq + (int64_t)i * a.o_tok + (int64_t)h * a.o_head;
            out[d] = total == 0 ? 0.f : o / l * g;  // a sum of 0 (every score -inf): NaN, as the formula
        }
        __syncthreads();
    }
}

void launch_rows(const AttnArgs& a, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.seqs * a.Nq * a.Hq, 148 * 64);
    if (a.D <= 32) attend_rows_kernel<8><<<grid, 256, 0, st>>>(a);
    else if (a.D <= 64) attend_rows_kernel<16><<<grid, 256, 0, st>>>(a);
    else attend_rows_kernel<32><<<grid, 256, 0, st>>>(a);
    MBR_CUDA(cudaGetLastError());
}

// A limit of 2^30 or more is none (keys number fewer).
int limit(int v) { return v >= (1 << 30) ? -1 : v; }

// The most keys that the rows of one call can see together.
int64_t most_keys(const AttnArgs& a, int64_t held) {
    if (a.left < 0 || a.right < 0) return held;
    return std::min<int64_t>(held, (int64_t)a.left + a.right + a.Nq + a.sinks);
}

AttnArgs common_args(const mbr_view& q, const mbr_view& out, int64_t seqs, int64_t Nq, int Hq, int Hkv, int D,
                     int left, int right, int sinks, float scale, const float* gates) {
    MBR_CHECK(seqs >= 0 && Nq >= 0 && Hq >= 0 && Hkv >= 0, "attention: negative size");
    MBR_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "attention: dim_head must be a multiple of 8 up to 128");
    MBR_CHECK(Hkv == 0 ? Hq == 0 : Hq % Hkv == 0, "attention: q_heads must be a multiple of kv_heads");
    MBR_CHECK(Nq < (1 << 30) && Hq < (1 << 20), "attention: too many queries or heads");
    MBR_CHECK(seqs <= ((int64_t)1 << 40) / std::max<int64_t>(1, Nq * Hq), "attention: too many rows");
    MBR_CHECK(std::isfinite(scale), "attention: scale must be finite");
    AttnArgs a{};
    a.q = q.data, a.out = out.data;
    a.q_seq = q.seq, a.q_tok = q.token, a.q_head = q.head;
    a.o_seq = out.seq, a.o_tok = out.token, a.o_head = out.head;
    a.seqs = seqs, a.Nq = (int)Nq, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.G = Hkv ? Hq / Hkv : 1;
    a.by_G = FastDiv((unsigned)std::max(1, a.G)), a.by_Hkv = FastDiv((unsigned)std::max(1, Hkv));
    a.left = limit(left), a.right = limit(right), a.sinks = sinks;
    a.scale = scale == 0.f ? 1.f / std::sqrt((float)D) : scale;
    a.gates = gates;
    return a;
}

}  // namespace

namespace {

AttnArgs window_args(const mbr_view& q, const mbr_view& k, const mbr_view& v, const mbr_view& out, int64_t seqs,
                     int64_t Nq, int64_t Nk, int Hq, int Hkv, int D, int left, int right, int sinks, float scale,
                     const float* gates, int dtype) {
    AttnArgs a = common_args(q, out, seqs, Nq, Hq, Hkv, D, left, right, sinks, scale, gates);
    MBR_CHECK(Nk >= 0 && Nk < (1 << 30) && sinks >= 0, "window_attention: bad key count or sinks");
    MBR_CHECK(dtype == DT_F32 || dtype == DT_F16 || dtype == DT_BF16,
              "window_attention: dtype must be fp32, fp16 or bf16");
    a.Nk = (int)Nk;
    a.k = k.data, a.v = v.data;
    a.k_seq = k.seq, a.k_tok = k.token, a.k_head = k.head;
    a.v_seq = v.seq, a.v_tok = v.token, a.v_head = v.head;
    return a;
}

// The form for few queries: it takes 16 rows at a time, a CTA or more each, and splits
// their keys over its warps; the tile form takes 128 rows and all their keys.
bool takes_few(const AttnArgs& a) { return (int64_t)a.Nq * a.G <= 16; }
// Where it is the faster one: up to 16 rows of heads up to 64; otherwise (it reads the keys once for
// each 16 rows, and has half the keys in flight past heads of 64) up to 32 rows if they make fewer CTAs than
// there are SMs.  us, few-token form / tiles, for 1, 16 and 32 rows a key head, fp16:
//   heads of 32, 480 key heads (sequences x heads) of 1301 keys 27/46  31/46  56/47
//   heads of 64, 480 of 1301 42/49  49/49  84/49;   240 of 1301 26/27  29/26  48/26
//                 64 of 1301 16/23  18/23  18/23;    24 of 8001 20/109 21/109 30/109
//                 64 of 300   8/9   10/9   11/9  (it loses where keys are few)
//   heads of 128, 240 of 1301 47/43 53/43  -;       160 of 4001 122/102 131/102  -
//                128 of 1301 28/31  33/31 52/28;     64 of 4001 65/94 72/94 72/94
//                  8 of 1301 27/27  30/27 30/27;     24 of 8001 32/166 39/173 57/174
bool few_rows(const AttnArgs& a) {
    const int64_t rows = (int64_t)a.Nq * a.G;
    return (rows <= 16 && a.D <= 64) || (rows <= 32 && a.seqs * a.Hkv * ceil_div(rows, 16) < 148);
}

StepPlan plan_of(const AttnArgs& a, bool q4, int64_t held) {
    return step_plan(a.seqs, a.Nq, a.Hq, a.Hkv, a.D, q4, most_keys(a, held));
}

}  // namespace

int64_t window_attention_workspace(int64_t seqs, int64_t Nq, int64_t Nk, int Hq, int Hkv, int D, int left, int right,
                                   int sinks, int dtype) {
    const mbr_view none{};
    const AttnArgs a =
        window_args(none, none, none, none, seqs, Nq, Nk, Hq, Hkv, D, left, right, sinks, 0.f, nullptr, dtype);
    if (seqs == 0 || Nq == 0 || Hq == 0 || dtype == DT_F32 || !(few_rows(a) || takes_few(a))) return 0;
    return plan_of(a, false, Nk).bytes;
}

void window_attention(const mbr_view& q, const mbr_view& k, const mbr_view& v, const mbr_view& out, int64_t seqs,
                      int64_t Nq, int64_t Nk, int Hq, int Hkv, int D, const int32_t* q_len, const int32_t* kv_len,
                      int left, int right, int sinks, float scale, const float* gates, int dtype, void* workspace,
                      int64_t workspace_bytes, cudaStream_t st) {
    AttnArgs a = window_args(q, k, v, out, seqs, Nq, Nk, Hq, Hkv, D, left, right, sinks, scale, gates, dtype);
    if (seqs == 0 || Nq == 0 || Hq == 0) return;
    MBR_CHECK(q.data && out.data && (Nk == 0 || (k.data && v.data)), "window_attention: null buffer");
    a.q_len = q_len, a.kv_len = kv_len;
    const bool tiles = tile_supported(a, dtype);
    if (step_supported(a, dtype, false) && (few_rows(a) || (takes_few(a) && !tiles))) {
        const StepPlan pl = plan_of(a, false, Nk);
        MBR_CHECK(pl.bytes == 0 || (workspace && workspace_bytes >= pl.bytes), "window_attention: workspace too small");
        raise_stream_error(st);
        attend_step(a, dtype, false, false, pl, workspace, st);
        return;
    }
    raise_stream_error(st);
    if (tiles) {
        attend_tiles(a, dtype, st);
        return;
    }
    attend_simt(a, dtype, st);
}

int64_t cache_attention_workspace(const mbr_kv_cache& c, int64_t tokens, int Hq, int left, int right) {
    check_cache_fields(c);
    const mbr_view none{};
    AttnArgs a = common_args(none, none, c.seqs, tokens, Hq, c.kv_heads, c.dim_head, left, right, c.sinks, 0.f, nullptr);
    if (c.seqs == 0 || tokens == 0 || Hq == 0 || c.dtype == DT_F32) return 0;
    return plan_of(a, c.bits == 4, (int64_t)c.sinks + c.ring).bytes;
}

void cache_attention(const mbr_view& q, const mbr_kv_cache& c, const mbr_view& out, const int32_t* length,
                     int64_t tokens, int Hq, int left, int right, float scale, const float* gates, void* workspace,
                     int64_t workspace_bytes, cudaStream_t st) {
    const bool q4 = check_cache(c);
    AttnArgs a = common_args(q, out, c.seqs, tokens, Hq, c.kv_heads, c.dim_head, left, right, c.sinks, scale, gates);
    if (c.seqs == 0 || tokens == 0 || Hq == 0) return;
    MBR_CHECK(q.data && out.data && length, "cache_attention: null buffer");
    a.k = c.k, a.v = c.v, a.k_scale = c.k_scale, a.v_scale = c.v_scale;
    a.ring = c.ring, a.cache_sinks = c.sinks, a.slots = (int64_t)c.sinks + c.ring;
    a.kv_len = length;
    if (step_supported(a, c.dtype, true)) {
        const StepPlan pl = plan_of(a, q4, a.slots);
        MBR_CHECK(pl.bytes == 0 || (workspace && workspace_bytes >= pl.bytes), "cache_attention: workspace too small");
        raise_stream_error(st);
        attend_step(a, c.dtype, true, q4, pl, workspace, st);
        return;
    }
    raise_stream_error(st);
    launch_rows(a, st);
}

}  // namespace streamops
}  // namespace mbr
