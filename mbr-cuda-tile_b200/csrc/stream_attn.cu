// stream_attn.cu — entry points of the streaming attention (prompt form and
// few-token form over the rolling cache) and the warp-per-row kernel.
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

int* stream_error_word() {
    // one word for all devices, visible to each (portable); never freed
    static int* const host = [] {
        int* p = nullptr;
        MBR_CUDA(cudaHostAlloc((void**)&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        *p = 0;
        return p;
    }();
    if (__atomic_load_n(host, __ATOMIC_RELAXED) != 0) {
        __atomic_store_n(host, 0, __ATOMIC_RELAXED);
        throw Error(ERR_TIMEOUT, "an earlier streaming attention call ran out of a kernel-side wait");
    }
    return host;  // unified addressing: the device uses the same address
}

namespace {

// One warp per row over an fp32 cache, whose rows no other kernel takes.
__global__ void __launch_bounds__(256) attend_rows_kernel(const AttnArgs a) {
    const int64_t rows = a.seqs * a.Nq * a.Hq, step = (int64_t)gridDim.x * 8;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += step) {
        const int64_t si = r / a.Hq, s = si / a.Nq;
        int n, m;
        lengths<true>(a, s, n, m);
        attend_row<float, true, false>(a, s, (int)(si - s * a.Nq), (int)(r - si * a.Hq), n, m);
    }
}

void launch_rows(const AttnArgs& a, cudaStream_t st) {
    const int64_t rows = a.seqs * a.Nq * a.Hq;
    attend_rows_kernel<<<(unsigned)std::min<int64_t>(ceil_div(rows, 8), 148 * 64), 256, 0, st>>>(a);
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

// The form for few queries: it splits the keys of 16 rows at a time, where the tile
// form takes 128 rows and all their keys.  16 rows (us, few-token form / tiles; heads
// of 64): 60 sequences of 801 keys and 8 key heads 35 / 33, of 2 key heads 14.5 / 16,
// 8 sequences of 4001 keys 36 / 57.  32 rows read the keys twice: 58 / 33, 21 / 16, and
// 37 / 57 where the tiles would leave most SMs idle; 64 rows 114 / 34, 33 / 16, 64 / 57.
bool few_rows(const AttnArgs& a) {
    const int64_t rows = (int64_t)a.Nq * a.G;
    return rows <= 16 || (rows <= 32 && a.seqs * a.Hkv < 148);
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
    if (seqs == 0 || Nq == 0 || Hq == 0 || dtype == DT_F32 || !few_rows(a)) return 0;
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
    if (few_rows(a) && step_supported(a, dtype, false)) {
        const StepPlan pl = plan_of(a, false, Nk);
        MBR_CHECK(pl.bytes == 0 || (workspace && workspace_bytes >= pl.bytes), "window_attention: workspace too small");
        attend_step(a, dtype, false, false, pl, workspace, st);
        return;
    }
    if (tile_supported(a, dtype)) {
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
        attend_step(a, c.dtype, true, q4, pl, workspace, st);
        return;
    }
    launch_rows(a, st);
}

}  // namespace streamops
}  // namespace mbr
