// stream_attn_simt.cu — windowed attention of many queries on the CUDA cores: fp32,
// and 16-bit layouts that the tensor-core kernels do not take.
//
// A tile is 64 rows (tokens of one key head's query heads, token-major) against
// 64 keys at a time, staged in shared memory as fp32: 256 threads hold 4 x 4
// scores each and 4 rows x DP / 16 channels of the output, so a multiply-add
// needs an eighth of a 16-byte shared-memory load.  Rows are padded by four floats
// (neighbouring rows on different banks).  The running maximum and sum of a row are
// shared by the 16 threads that own it, in registers.  fp32 multiply-adds and their
// operands' loads from shared memory bound it: 25 TFLOP/s at heads of 64 (fp32, 60 x 8
// heads, 801 tokens, all keys), 19.5 at 32; 4 x 8 heads of 50 tokens take 9.5 us, the time
// of one block's chain.
//
// Rows that do not come out finite are computed again by attend_row, which reads
// only what the row sees (a value that another row of the tile sees enters with
// weight 0, which is NaN for one that is not finite).
#include <algorithm>

#include "stream_attn_simt.h"

namespace mbr {
namespace streamops {

namespace {

constexpr int BM = 64, BN = 64;

template <int DP>
constexpr int smem_bytes() {
    return (BM * (DP + 4) + 2 * BN * (DP + 4) + BM * (BN + 4)) * 4;
}

struct SimtArgs {
    AttnArgs a;
    int tiles, vec;  // row tiles of a (sequence, key head); 16-byte loads
    FastDiv by_tiles;
};

// Rows of a tile into shared memory as fp32, channels past the head size and rows past `n` as zeros.
template <typename T, int DP, typename Row>
__device__ __forceinline__ void stage(float* dst, int D, int n, int vec, Row row) {
    constexpr int E = 16 / sizeof(T);
    if (vec) {
        for (int i = threadIdx.x; i < 64 * (DP / E); i += 256) {
            const int r = i / (DP / E), d = i % (DP / E) * E;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < n && d < D) x = __ldg(reinterpret_cast<const uint4*>(row(r) + d));
            const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
            for (int c = 0; c < E; c += 4)
                *reinterpret_cast<float4*>(dst + r * (DP + 4) + d + c) =
                    make_float4(to_f32<T>(e[c]), to_f32<T>(e[c + 1]), to_f32<T>(e[c + 2]), to_f32<T>(e[c + 3]));
        }
    } else {
        for (int i = threadIdx.x; i < 64 * DP; i += 256) {
            const int r = i / DP, d = i % DP;
            dst[r * (DP + 4) + d] = r < n && d < D ? to_f32<T>(row(r)[d]) : 0.f;
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(256) attend_simt_kernel(const SimtArgs p) {
    extern __shared__ __align__(16) float sm_f[];
    float* const Qs = sm_f;
    float* const Ks = Qs + BM * (DP + 4);
    float* const Vs = Ks + BN * (DP + 4);
    float* const Ps = Vs + BN * (DP + 4);
    constexpr int LD = DP + 4, LP = BN + 4, ND = DP / 16;
    const AttnArgs& a = p.a;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const unsigned sg = p.by_tiles.div(blockIdx.x);
    const int r0 = (int)(blockIdx.x - sg * p.by_tiles.d) * BM;
    const unsigned sq = a.by_Hkv.div(sg);
    const int64_t s = sq;
    const int hk = (int)(sg - sq * a.Hkv);
    const int rows = min(BM, a.Nq * a.G - r0);
    int n, m;
    lengths<false>(a, s, n, m);
    auto token_of = [&](int r) { return (int)a.by_G.div(r0 + r); };
    auto q_row = [&](int r) {
        const int i = token_of(r);
        return (const T*)a.q + s * a.q_seq + (int64_t)i * a.q_tok + (int64_t)(hk * a.G + r0 + r - i * a.G) * a.q_head;
    };
    // keys: the first tokens before the window, then the window from the first row's lower end on
    int LO = 0, HI = 0, ns = 0;
    const int t0 = token_of(0), t1 = min(token_of(rows - 1), n - 1);
    if (t0 <= t1) {
        const Window w0 = row_window<false>(a, t0, n, m), w1 = row_window<false>(a, t1, n, m);
        HI = w1.hi, LO = min(w0.lo, HI), ns = min(a.sinks, LO);
    }
    const int nsb = (ns + BN - 1) / BN, blocks = nsb + (HI - LO + BN - 1) / BN;
    Window w[4];
    float o[4][ND], mx[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i, tok = token_of(r);
        w[i] = r < rows && tok < n ? row_window<false>(a, tok, n, m) : Window{0, 0, 0};
        mx[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < ND; ++c) o[i][c] = 0.f;
    }
    if (blocks) stage<T, DP>(Qs, a.D, rows, p.vec, q_row);
    const float scale = a.scale * 1.4426950408889634f;
    for (int b = 0; b < blocks; ++b) {
        const bool first = b < nsb;  // a block of first tokens
        const int key = first ? b * BN : LO + (b - nsb) * BN, cnt = min(BN, (first ? ns : HI) - key);
        __syncthreads();  // the block before is read
        stage<T, DP>(Ks, a.D, cnt, p.vec, [&](int r) {
            return (const T*)a.k + s * a.k_seq + (int64_t)(key + r) * a.k_tok + (int64_t)hk * a.k_head;
        });
        stage<T, DP>(Vs, a.D, cnt, p.vec, [&](int r) {
            return (const T*)a.v + s * a.v_seq + (int64_t)(key + r) * a.v_tok + (int64_t)hk * a.v_head;
        });
        __syncthreads();
        // ---- scores of rows 4 ty + i and keys tx + 16 j ----
        float sc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sc[i][j] = fmaf(qv[i].x, kv[j].x, sc[i][j]);
                    sc[i][j] = fmaf(qv[i].y, kv[j].y, sc[i][j]);
                    sc[i][j] = fmaf(qv[i].z, kv[j].z, sc[i][j]);
                    sc[i][j] = fmaf(qv[i].w, kv[j].w, sc[i][j]);
                }
        }
        // ---- weights; a row's 16 threads are one half of a warp ----
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = key + tx + 16 * j;
                const bool see = first ? k < min(w[i].first, ns) : (k >= w[i].lo && k < w[i].hi) || k < w[i].first;
                sc[i][j] = see ? sc[i][j] * scale : -INFINITY;
                top = fmaxf(top, sc[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(mx[i], top), off = now == -INFINITY ? 0.f : now;
            const float f = mx[i] == now ? 1.f : ex2_approx(mx[i] - now);
            mx[i] = now;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = ex2_approx(sc[i][j] - off);
                sum += e;
                Ps[(ty * 4 + i) * LP + tx + 16 * j] = e;
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            l[i] = l[i] * f + sum;
#pragma unroll
            for (int c = 0; c < ND; ++c) o[i][c] *= f;
        }
        __syncwarp();  // a warp's rows of P are read by that warp only
        // ---- O += P V: channels tx * ND' + .. in pieces of at most four ----
#pragma unroll 2
        for (int k = 0; k < BN; k += 4) {
            float4 pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(Ps + (ty * 4 + i) * LP + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float* vr = Vs + (k + e) * LD;
                float v[ND];
                if constexpr (ND == 2) {
                    const float2 x = *reinterpret_cast<const float2*>(vr + tx * 2);
                    v[0] = x.x, v[1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < ND; c += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(vr + c * 16 + tx * 4);
                        v[c] = x.x, v[c + 1] = x.y, v[c + 2] = x.z, v[c + 3] = x.w;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float pe = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
#pragma unroll
                    for (int c = 0; c < ND; ++c) o[i][c] = fmaf(pe, v[c], o[i][c]);
                }
            }
        }
        __syncwarp();  // before the next block's weights
    }
    // ---- output; rows that are not finite once more, each by its warp ----
    unsigned again = 0;  // of this thread's four rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i, tok = token_of(r), h = hk * a.G + r0 + r - tok * a.G;
        const bool sees = w[i].hi > w[i].lo || w[i].first > 0;
        if (r < rows) {
            const float gate = a.gates ? __ldg(a.gates + (s * a.Nq + tok) * a.Hq + h) : 1.f;
            const float f = sees ? gate / l[i] : 0.f;
            T* out = (T*)a.out + s * a.o_seq + (int64_t)tok * a.o_tok + (int64_t)h * a.o_head;
#pragma unroll
            for (int c = 0; c < ND; ++c) {
                const int d = ND == 2 ? tx * 2 + c : (c & ~3) * 16 + tx * 4 + (c & 3);
                const float v = sees ? o[i][c] * f : 0.f;
                if (d < a.D) {
                    out[d] = from_f32<T>(v);
                    if (!isfinite(v)) again |= 1u << i;
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned bad = __ballot_sync(0xffffffffu, again >> i & 1);  // lanes 0-15: row of the even ty, 16-31: odd
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half)
            if (bad >> (16 * half) & 0xffffu) {
                const int r = ((threadIdx.x >> 5) * 2 + half) * 4 + i, tok = token_of(r);
                attend_row<T, false, false>(a, s, tok, hk * a.G + r0 + r - tok * a.G, n, m);
            }
    }
}

template <typename T, int DP>
void launch(const SimtArgs& p, unsigned grid, cudaStream_t st) {
    auto kern = attend_simt_kernel<T, DP>;
    static bool attr[kMaxStreamDevices] = {};
    const int dev = stream_device();
    if (!attr[dev]) {
        MBR_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<DP>()));
        attr[dev] = true;
    }
    kern<<<grid, 256, smem_bytes<DP>(), st>>>(p);
    MBR_CUDA(cudaGetLastError());
}

}  // namespace

void attend_simt(const AttnArgs& a, int dtype, cudaStream_t st) {
    SimtArgs p{};
    p.a = a;
    p.tiles = (int)ceil_div((int64_t)a.Nq * a.G, BM);
    p.by_tiles = FastDiv((unsigned)p.tiles);
    const int64_t grid = a.seqs * a.Hkv * p.tiles, es = dtype == DT_F32 ? 4 : 2, e16 = 16 / es;
    MBR_CHECK((int64_t)a.Nq * a.G < (1ll << 30) && grid < (1ll << 30), "attention: too many row tiles");
    const int64_t all = a.q_seq | a.q_tok | a.q_head | a.k_seq | a.k_tok | a.k_head | a.v_seq | a.v_tok | a.v_head;
    p.vec = ((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 && all % e16 == 0) ? 1 : 0;
    MBR_DISPATCH_DTYPE(dtype, T, {
        if (a.D <= 32) launch<T, 32>(p, (unsigned)grid, st);
        else if (a.D <= 64) launch<T, 64>(p, (unsigned)grid, st);
        else launch<T, 128>(p, (unsigned)grid, st);
    });
}

}  // namespace streamops
}  // namespace mbr
