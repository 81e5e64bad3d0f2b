// stream_attn_tc.cu — windowed attention of many queries, fp16/bf16, on tcgen05.
//
// A tile is 128 rows: 128 / G tokens of the G query heads that share a key head
// (128 tokens of one head where G does not divide 128).  Its keys are walked in
// blocks of 64: those of the first tokens that lie before the window, then the
// window from its first row's lower end on, so a tile reads no more than its rows
// see together.  Per block:
//   S = Q K^T        128 x 64, fp32, tensor memory
//   P = 2^(S c - m)  16 bits, over the first half of S, the A operand of
//   O += P V         128 x D, fp32, tensor memory
// Warps 0-3 run the softmax (thread r owns row r), warp 4 issues loads (TMA) and
// products.  The exponential unit (16 a clock and SM) bounds heads of 64: 256
// operations of the tensor core an exponential.  A row's 64 exponentials take a
// warp 512 clocks of that unit, the way from P through both products to the next S
// some 850, so CTAs that interleave have to fill it: three an SM with one S each
// (128 columns of tensor memory; two past 64 channels), each of which then takes
// some 2250 clocks a block, 68 % of the unit's rate (53 % by its counter over a whole call of 6001 frames).  Column chunks of 32 that no row of
// a warp sees take no exponentials (the window's two ends).
//
// 6001 frames of 4 sequences x 8 heads of 64, a window of 1024 + 16 keys, bf16: 91 us,
// 510 TFLOP/s of what is seen; 801 frames of 60 x 8 heads, 271 + 4 keys, fp16: 94 us,
// of 30 for the bytes (a tile's start and end, and blocks that its rows see in
// part, are much of its 7 blocks).  Measured on the first, when this took 99 us: two CTAs
// with two S each, a load warp and a product warp 128, two CTAs with blocks of
// 128 keys 121; four CTAs spill registers, twice the time; two Q and two stages
// instead of three 94 where this takes 91.
//
// The offset m is a row's maximum of the block in which it first sees a key, and
// is raised (O and the sum scaled, the block taken again) only when a block's
// weights sum past 2^14: no maximum is taken otherwise, and weights stay in the
// 16-bit range.  The row sums hold the weights before their rounding to 16 bits.
//
// Values that a row does not see enter with weight 0; were one NaN or infinite,
// the row would be NaN.  Rows that do not come out finite are computed again by
// attend_row, which reads only what the row sees; values past a sequence's length
// are cleared in shared memory before they are used.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "sm100.cuh"
#include "stream_attn_tc.h"

namespace mbr {
namespace streamops {

namespace {

using namespace sm100;

constexpr int QROWS = 128, KB = 64;
constexpr float kRescaleSum = 16384.0f;

// Shared memory of a CTA: Q, NS stages of K and of V (64-channel halves of 128-byte rows, 128-byte swizzle), barriers.
template <int DH>
struct TileCfg {
    static constexpr int NS = DH == 1 ? 3 : 2;
    static constexpr int Q = 0;
    static constexpr int K = DH * 16384;
    static constexpr int V = K + NS * DH * 8192;
    static constexpr int BAR = V + NS * DH * 8192;
    static constexpr int TOTAL = BAR + 128;
    static constexpr int CTAS = DH == 1 ? 3 : 2;  // an SM
    static constexpr uint32_t TMEM = DH == 1 ? 128 : 256;
    static constexpr uint32_t O = 64;  // S at column 0, O behind it
    static_assert(CTAS * (TOTAL + 1024) <= 233472, "CTAs an SM");
};

struct TileArgs {
    AttnArgs a;
    int pack, tokens;        // query heads in a tile, tokens in a tile
    int qtiles, groups;      // tiles of a sequence's queries, head groups
    int last_first;          // order: later queries first (their rows see more)
    unsigned ntiles;
    FastDiv by_pack, by_inner, by_groups;
    float scale_log2;
    int* err;
};

// What a tile covers and which key blocks it walks.
struct Tile {
    int s, h0, hk, tok0;  // sequence, first query head, key head, first token
    int n, m;             // queries and keys of the sequence
    int LO, ns, nsb, nkv; // window start, first tokens before it, their blocks, all blocks
};

__device__ __forceinline__ Tile tile_at(const TileArgs& p, unsigned t) {
    Tile x;
    const unsigned hi = p.by_inner.div(t), lo = t - hi * p.by_inner.d;
    const unsigned sg = p.last_first ? lo : hi;
    const int qi = p.last_first ? p.qtiles - 1 - (int)hi : (int)lo;
    x.s = (int)p.by_groups.div(sg);
    x.h0 = ((int)sg - x.s * p.groups) * p.pack;
    x.hk = (int)p.a.by_G.div(x.h0);
    x.tok0 = qi * p.tokens;
    lengths<false>(p.a, x.s, x.n, x.m);
    x.LO = x.ns = x.nsb = x.nkv = 0;
    const int last = min(x.tok0 + p.tokens, x.n) - 1;
    if (last >= x.tok0) {
        const Window w0 = row_window<false>(p.a, x.tok0, x.n, x.m), w1 = row_window<false>(p.a, last, x.n, x.m);
        x.LO = min(w0.lo, w1.hi);
        x.ns = min(p.a.sinks, x.LO);
        x.nsb = (x.ns + KB - 1) / KB;
        x.nkv = x.nsb + (w1.hi - x.LO + KB - 1) / KB;
    }
    return x;
}
// First key of block j.
__device__ __forceinline__ int block_key(const Tile& x, int j) {
    return j < x.nsb ? j * KB : x.LO + (j - x.nsb) * KB;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Bits [lo, hi) of 64, bounds anywhere.
__device__ __forceinline__ uint64_t bits_between(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 64);
    if (hi <= lo) return 0;
    return (~0ull >> (64 - (hi - lo))) << lo;
}

// True in one lane of a converged warp, the same one each time.  The compiler knows that one lane runs what depends on
// it, and issues from uniform registers without a loop over lanes.
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_u32(dst)),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}

template <typename T, int DH>
__global__ void __launch_bounds__(160, TileCfg<DH>::CTAS)
    attend_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TileArgs p) {
    using Cfg = TileCfg<DH>;
    extern __shared__ __align__(1024) uint8_t sm[];
    if (!smem_aligned_or_flag(sm, p.err)) return;  // uniform over the CTA
    uint64_t* bar = (uint64_t*)(sm + Cfg::BAR);
    constexpr int NS = Cfg::NS;
    uint64_t* bar_q = bar;           // Q landed
    uint64_t* bar_s = bar + 1;       // S of the next block computed (and every product issued before it)
    uint64_t* bar_o = bar + 2;       // a tile's last product done
    uint64_t* bar_p = bar + 3;       // P written, S read (4 warps)
    uint64_t* bar_k = bar + 4;       // [NS] K stage landed
    uint64_t* bar_v = bar_k + NS;    // [NS] V stage landed
    uint64_t* bar_end = bar_v + NS;  // after a wait that ran out: every product done
    uint32_t* tmem_slot = (uint32_t*)(bar_end + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 5 + 2 * NS; ++i) mbar_init(&bar[i], i == 3 ? 4 : 1);
        fence_barrier_init();
    }
    if (warp == 4) {
        tmem_alloc(tmem_slot, Cfg::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 4) {
        // ---- loads and products; one lane issues, all wait ----
        // The blocks of all of this CTA's tiles form one stream g; K(g) and V(g) go through stage g % NS.
        struct Block {
            int key, hk, s;  // coordinates
            int left;        // keys of the sequence from here on
            bool first;      // of its tile
            bool any;        // exists
            int h0, tok0;    // its tile's Q
        };
        unsigned t = blockIdx.x;
        Tile x;
        x.nkv = 0;
        int j = 0;
        auto next_block = [&]() {
            Block b{};
            while (j >= x.nkv) {
                if (t >= p.ntiles) return b;
                x = tile_at(p, t);
                t += gridDim.x;
                j = 0;
            }
            b.key = block_key(x, j);
            b.hk = x.hk, b.s = x.s, b.h0 = x.h0, b.tok0 = x.tok0;
            b.left = x.m - b.key;
            b.first = j == 0;
            b.any = true;
            ++j;
            return b;
        };
        auto load_q = [&](const Block& b) {
            mbar_arrive_expect_tx(bar_q, DH * 16384);
#pragma unroll
            for (int h = 0; h < DH; ++h) tma_load_4d(sm + Cfg::Q + h * 16384, &tmQ, 64 * h, b.h0, b.tok0, b.s, bar_q);
        };
        auto load_k = [&](const Block& b, int st) {
            mbar_arrive_expect_tx(&bar_k[st], DH * 8192);
#pragma unroll
            for (int h = 0; h < DH; ++h)
                tma_load_4d(sm + Cfg::K + (st * DH + h) * 8192, &tmK, 64 * h, b.hk, b.key, b.s, &bar_k[st]);
        };
        auto load_v = [&](const Block& b, int st) {
            mbar_arrive_expect_tx(&bar_v[st], DH * 8192);
#pragma unroll
            for (int h = 0; h < DH; ++h)
                tma_load_4d(sm + Cfg::V + (st * DH + h) * 8192, &tmV, 64 * h, b.hk, b.key, b.s, &bar_v[st]);
        };
        auto wait_all = [&](uint64_t* b, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(b, parity, p.err));
        };
        constexpr uint32_t idS = idesc_f16(QROWS, KB, std::is_same_v<T, __nv_bfloat16>);
        constexpr uint32_t idO = idesc_f16(QROWS, 64, std::is_same_v<T, __nv_bfloat16>, /*b_mn_major=*/true);
        const uint64_t dQ = sdesc_sw128(smem_u32(sm + Cfg::Q));
        const uint64_t dK = sdesc_sw128(smem_u32(sm + Cfg::K));
        const uint64_t dV = sdesc_sw128_mn(smem_u32(sm + Cfg::V));
        const int ksteps = (p.a.D + 15) / 16;  // whole steps of channels past the head size (zeros) are left out
        auto issue_s = [&](int st) {  // 32 bytes a step, 16 KB (Q) or 8 KB (K) a half
            const uint64_t k0 = dK + (uint64_t)(512 * DH * st);
            if (ksteps == 4 * DH) {
#pragma unroll
                for (int k = 0; k < 4 * DH; ++k)
                    mma_f16(tmem, dQ + 1024 * (k >> 2) + 2 * (k & 3), k0 + 512 * (k >> 2) + 2 * (k & 3), idS, k > 0);
            } else {
                for (int k = 0; k < ksteps; ++k)
                    mma_f16(tmem, dQ + 1024 * (k >> 2) + 2 * (k & 3), k0 + 512 * (k >> 2) + 2 * (k & 3), idS, k > 0);
            }
            mma_commit(bar_s);
        };
        auto issue_pv = [&](int st, bool first) {
            const uint64_t v0 = dV + (uint64_t)(512 * DH * st);
#pragma unroll
            for (int h = 0; h < DH; ++h)
#pragma unroll
                for (int k = 0; k < KB / 16; ++k)  // 16 keys: 8 columns of P, 2 KB of V
                    mma_f16_ts(tmem + Cfg::O + 64 * h, tmem + 8 * k, v0 + 512 * h + 128 * k, idO, !first || k > 0);
        };

        Block b[NS];  // blocks g .. g + NS - 1
#pragma unroll
        for (int i = 0; i < NS; ++i) b[i] = next_block();
        if (elect_one()) {
            prefetch_tensormap(&tmQ);
            prefetch_tensormap(&tmK);
            prefetch_tensormap(&tmV);
            if (b[0].any) load_q(b[0]);
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (b[i].any) load_k(b[i], i), load_v(b[i], i);
        }
        __syncwarp();
        bool ok = true;
        uint32_t qphase = 1;  // of the next tile's Q
        bool behind = false;  // there is a block g - 1
        if (b[0].any) {
            ok = wait_all(bar_q, 0) && wait_all(&bar_k[0], 0);
            if (ok) {
                tc_fence_after();
                if (elect_one()) issue_s(0);
                __syncwarp();
            }
        }
        // stage and parity of block g and of block g + 1
        int st = 0, st1 = 1 % NS;
        uint32_t par = 0, par1 = NS == 1 ? 1 : 0;
        for (uint32_t gp = 0; b[0].any && ok; gp ^= 1) {  // gp: parity of g
            const bool more = b[1].any, fresh = b[1].first;  // a next block; it starts another tile
            ok = wait_all(&bar_v[st], par) && (!more || wait_all(&bar_k[st1], par1));
            if (!ok) break;
            if (b[0].left < KB) {  // rows past the sequence's length hold anything: zeros
                const int r0 = max(b[0].left, 0);
                for (int i = lane; i < (KB - r0) * 8 * DH; i += 32) {
                    const int row = i >> 3, h = row / (KB - r0), r = r0 + row - h * (KB - r0);
                    *reinterpret_cast<uint4*>(sm + Cfg::V + (st * DH + h) * 8192 + r * 128 + (i & 7) * 16) =
                        make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_smem();
                __syncwarp();
            }
            ok = wait_all(bar_p, gp);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                issue_pv(st, b[0].first);
                if (more && !fresh) {
                    issue_s(st1);
                } else {  // the tile's output is ready with this product; S(g) is done: the next Q may take Q's place
                    mma_commit(bar_o);
                    if (more) load_q(b[1]);
                }
            }
            __syncwarp();
            const Block fresh_block = next_block();  // block g + NS
            if (elect_one()) {
                // S(g) done: K(g)'s stage is free.  P.V(g - 1) was issued before S(g): V(g - 1)'s stage is free, for
                // block g - 1 + NS.
                if (fresh_block.any) load_k(fresh_block, st);
                if (behind && b[NS - 1].any) load_v(b[NS - 1], st == 0 ? NS - 1 : st - 1);
            }
            behind = true;
            __syncwarp();
            if (more && fresh) {
                ok = wait_all(bar_q, qphase & 1);
                if (!ok) break;
                ++qphase;
                tc_fence_after();
                if (elect_one()) issue_s(st1);
                __syncwarp();
            }
#pragma unroll
            for (int i = 0; i + 1 < NS; ++i) b[i] = b[i + 1];
            b[NS - 1] = fresh_block;
            st = st1, par = par1;
            st1 = st1 + 1 == NS ? 0 : st1 + 1;
            if (st1 == 0) par1 ^= 1;
        }
        if (!ok) {  // a wait ran out: what is in flight ends before the CTA does (waits with a limit, too)
            if (elect_one()) mma_commit(bar_end);
            __syncwarp();
            mbar_drain(bar_end, 0);
            for (uint32_t parity = 0; parity < 2; ++parity)  // a pending copy's phase is one of the two
                for (int i = 0; i < 1 + 2 * NS; ++i) mbar_drain(i == 0 ? bar_q : bar_k + i - 1, parity);
            __syncwarp();
        }
    } else {
        // ---- softmax: thread r owns row r of the tile (tensor-memory lane r) ----
        const AttnArgs& a = p.a;
        const int r = threadIdx.x;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const uint32_t tS = tmem + lanes, tO = tmem + lanes + Cfg::O;
        const int rt = (int)p.by_pack.div(r), rh = r - rt * p.pack;  // token and head within the tile
        const float c = p.scale_log2;
        int g = 0;           // blocks so far
        uint32_t tiles = 0;  // tiles with blocks so far
        bool ok = true;      // warp-uniform: tensor-memory loads and stores are warp-collective
        Tile next = tile_at(p, blockIdx.x);
        for (unsigned t = blockIdx.x; t < p.ntiles && ok; t += gridDim.x) {
            const Tile x = next;
            const int token = x.tok0 + rt;
            const bool valid = rt < p.tokens && token < a.Nq;
            Window w{0, 0, 0};
            if (valid && token < x.n) w = row_window<false>(a, token, x.n, x.m);
            const bool sees = w.hi > w.lo || w.first > 0;
            const int h = x.h0 + rh;
            const float gate = valid && a.gates ? __ldg(a.gates + ((int64_t)x.s * a.Nq + token) * a.Hq + h) : 1.f;
            // keys that every row of this warp (that sees any) sees
            const int all_lo = __reduce_max_sync(0xffffffffu, sees ? w.lo : 0);
            const int all_hi = __reduce_min_sync(0xffffffffu, sees ? w.hi : INT32_MAX);
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < x.nkv; ++j, ++g) {
                const int key = block_key(x, j);
                // columns this row sees (a first-token block holds only those before the window); chunks that some
                // row sees; chunks that every row (that sees any key) sees whole
                uint64_t see = sees ? ~0ull : 0ull;
                uint32_t need = 3, whole = 3;
                if (j < x.nsb || key < all_lo || key + KB > all_hi) {
                    see = j < x.nsb ? bits_between(0, min(w.first, x.ns) - key)
                                    : bits_between(w.lo - key, w.hi - key) | bits_between(0, w.first - key);
                    if (!sees) see = 0;
                    need = whole = 0;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t part = (uint32_t)(see >> (32 * q));
                        if (__any_sync(0xffffffffu, part != 0u)) need |= 1u << q;
                        if (__all_sync(0xffffffffu, part == 0xffffffffu || !sees)) whole |= 1u << q;
                    }
                    whole &= need;
                }
                const uint32_t half[2] = {(uint32_t)see, (uint32_t)(see >> 32)};
                ok = __all_sync(0xffffffffu, mbar_wait(bar_s, g & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                uint32_t pk[32];
                // weights with offset mo as 16-bit pairs; returns this row's sum.  A chunk's scores are loaded
                // when it comes to them: two at once would not leave registers for three CTAs.
                auto weights = [&](float mo) {
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    uint32_t sv[32];
                    auto chunk = [&](int q, auto all) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 z = __ffma2_rn(make_float2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])),
                                                        make_float2(c, c), make_float2(-mo, -mo));
                            float2 e = make_float2(ex2_approx(z.x), ex2_approx(z.y));
                            if constexpr (!decltype(all)::value) {
                                e.x = half[q] >> i & 1 ? e.x : 0.f;
                                e.y = half[q] >> (i + 1) & 1 ? e.y : 0.f;
                            }
                            sum[i / 2 & 1] = __fadd2_rn(sum[i / 2 & 1], e);
                            pk[16 * q + i / 2] = pack2(e.x, e.y, (T*)nullptr);
                        }
                    };
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (need >> q & 1) {
                            tmem_ld32(tS + 32 * q, sv);
                            tmem_ld_wait(sv);
                            if (whole >> q & 1) chunk(q, std::true_type{});
                            else chunk(q, std::false_type{});
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) pk[16 * q + i] = 0u;
                        }
                    }
                    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                };
                float rs = 0.f;
                bool low = see != 0 && m == -INFINITY, settled = false;
                // The ordinary block, every row seeing all of it with an offset: straight through (a minute of audio:
                // 104 us against 111 with such blocks in the loop below, which all others take).
                if (whole == 3 && !__any_sync(0xffffffffu, low)) {
                    const float mo = m == -INFINITY ? 0.f : m;
                    const float2 mm = make_float2(-mo, -mo), cc = make_float2(c, c);
                    float2 sum[4] = {};
                    uint32_t s0[32], s1[32];
                    tmem_ld32(tS, s0);
                    tmem_ld32(tS + 32, s1);
                    tmem_ld_wait(s0);
                    tmem_ld_wait(s1);
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        const uint32_t* sv = i < 32 ? s0 + i : s1 + i - 32;
                        const float2 x2 = make_float2(__uint_as_float(sv[0]), __uint_as_float(sv[1]));
                        const float2 z = __ffma2_rn(x2, cc, mm);
                        const float2 e = make_float2(ex2_approx(z.x), ex2_approx(z.y));
                        sum[i / 2 & 3] = __fadd2_rn(sum[i / 2 & 3], e);
                        pk[i / 2] = pack2(e.x, e.y, (T*)nullptr);
                    }
                    const float2 all = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
                    rs = all.x + all.y;
                    low = sees && !(rs <= kRescaleSum);
                    settled = !__any_sync(0xffffffffu, low);
                }
                if (!settled)
#pragma unroll 1
                for (int pass = 0; pass < 3; ++pass) {
                    if (__any_sync(0xffffffffu, low)) {
                        float top = -INFINITY;
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            if (!(need >> (q >> 1) & 1)) continue;
                            uint32_t sv[16];
                            tmem_ld16(tS + 16 * q, sv);
                            tmem_ld_wait();
                            const uint32_t bits = half[q >> 1] >> (16 * (q & 1));
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (bits >> i & 1) top = fmaxf(top, __uint_as_float(sv[i]) * c);
                        }
                        const float now = low ? fmaxf(m, top) : m;
                        const float f = now == m ? 1.f : ex2_approx(m - now);
                        m = now;
                        const bool scaled = j > 0 && f != 1.f && l != 0.f;
                        l *= f;
                        if (__any_sync(0xffffffffu, scaled)) {
#pragma unroll 1
                            for (int q = 0; q < 4 * DH; ++q) {
                                uint32_t ov[16];
                                tmem_ld16(tO + 16 * q, ov);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                                tmem_st16(tO + 16 * q, ov);
                            }
                            tmem_st_wait();
                        }
                    } else if (pass > 0) {
                        break;
                    }
                    rs = weights(m == -INFINITY ? 0.f : m);
                    low = pass < 1 && sees && !(rs <= kRescaleSum);
                }
                l += rs;
                tmem_st32(tS, pk);  // over the first half of S, which this warp has read
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p);
            }
            if (!ok) break;
            if (t + gridDim.x < p.ntiles) next = tile_at(p, t + gridDim.x);  // while the last product runs
            if (x.nkv > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar_o, tiles & 1, p.err));
                if (!ok) break;
                ++tiles;
                tc_fence_after();
            }
            const float f = sees ? gate / l : 0.f;
            T* out = (T*)a.out + (int64_t)x.s * a.o_seq + (int64_t)token * a.o_tok + (int64_t)h * a.o_head;
            float odd = 0.f;  // NaN once a value of this row is not finite
#pragma unroll
            for (int q = 0; q < 2 * DH; ++q) {
                if (32 * q >= a.D) break;
                uint32_t ov[32];
                if (x.nkv > 0) {
                    tmem_ld32(tO + 32 * q, ov);
                    tmem_ld_wait(ov);
                }
                if (valid) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        if (32 * q + i >= a.D) break;
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            v[e] = sees ? __uint_as_float(ov[i + e]) * f : 0.f;
                            odd = fmaf(v[e], 0.f, odd);
                        }
                        *reinterpret_cast<uint4*>(out + 32 * q + i) =
                            make_uint4(pack2(v[0], v[1], (T*)nullptr), pack2(v[2], v[3], (T*)nullptr),
                                       pack2(v[4], v[5], (T*)nullptr), pack2(v[6], v[7], (T*)nullptr));
                    }
                }
                __syncwarp();
            }
            tc_fence_before();  // O read before the next tile's first product overwrites it (behind this warp's next P)
            for (uint32_t rows = __ballot_sync(0xffffffffu, odd != 0.f); rows; rows &= rows - 1) {
                const int q = 32 * warp + __ffs(rows) - 1, qt = (int)p.by_pack.div(q);
                attend_row<T, false, false>(a, x.s, x.tok0 + qt, x.h0 + q - qt * p.pack, x.n, x.m);
            }
        }
        // a wait ran out: the tile's last product, if it was issued, ends before the CTA does
        if (!ok) mbar_drain(bar_o, tiles & 1);
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::TMEM);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)q;
    });
    if (!fn) throw Error(ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    return fn;
}

// (channel, head, token, sequence) view of q, k or v; the box is 64 channels of `heads` heads of `tokens` tokens.
// Channels past the head size and tokens past the end read as zeros.
void make_map(CUtensorMap* m, const void* base, int64_t seq, int64_t tok, int64_t head, int D, int H, int64_t N,
              int64_t S, int heads, int tokens, int dtype) {
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)N, (cuuint64_t)S};
    // the stride of an axis of one is never used: any value that a map takes
    cuuint64_t strides[3] = {(cuuint64_t)(H > 1 ? head * 2 : 16), (cuuint64_t)(N > 1 ? tok * 2 : 16),
                             (cuuint64_t)(S > 1 ? seq * 2 : 16)};
    cuuint32_t box[4] = {64, (cuuint32_t)heads, (cuuint32_t)tokens, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = encode_fn()(
        m, dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
}

template <typename T, int DH>
void launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileArgs& p, cudaStream_t st) {
    using Cfg = TileCfg<DH>;
    auto kern = attend_tiles_kernel<T, DH>;
    static int sms[kMaxStreamDevices] = {};
    const int dev = stream_device();
    if (!sms[dev]) {
        MBR_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::TOTAL));
        MBR_CUDA(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
    }
    // Persistent CTAs take tiles in turn and load the next one's Q behind the last product (60 x 8 heads of 801 frames:
    // 94 us against 116 with a CTA a tile; 4 x 8 heads of 6001: 91 against 93).  With lengths given, what a tile holds
    // is not known here: a CTA a tile, so that the hardware evens it out (ragged pieces, heads of 128: 50 us against 55).
    const unsigned grid =
        p.a.q_len || p.a.kv_len ? p.ntiles : std::min<unsigned>(p.ntiles, (unsigned)(sms[dev] * Cfg::CTAS));
    kern<<<grid, 160, Cfg::TOTAL, st>>>(q, k, v, p);
    MBR_CUDA(cudaGetLastError());
}

}  // namespace

bool tile_supported(const AttnArgs& a, int dtype) {
    if (dtype == DT_F32 || a.Nk == 0) return false;
    const int64_t all = a.q_seq | a.q_tok | a.q_head | a.k_seq | a.k_tok | a.k_head | a.v_seq | a.v_tok | a.v_head |
                        a.o_seq | a.o_tok | a.o_head;
    const uintptr_t ptr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out;
    // a map's strides are positive and below 2^40 bytes
    auto fits = [](int64_t s, int64_t n) { return n <= 1 || (s > 0 && s < (1ll << 39)); };
    return all % 8 == 0 && (ptr & 15) == 0 && a.seqs < (1ll << 31) && fits(a.q_seq, a.seqs) && fits(a.q_tok, a.Nq) &&
           fits(a.q_head, a.Hq) && fits(a.k_seq, a.seqs) && fits(a.k_tok, a.Nk) && fits(a.k_head, a.Hkv) &&
           fits(a.v_seq, a.seqs) && fits(a.v_tok, a.Nk) && fits(a.v_head, a.Hkv);
}

void attend_tiles(const AttnArgs& a, int dtype, cudaStream_t st) {
    TileArgs p{};
    p.a = a;
    p.pack = a.G <= QROWS && QROWS % a.G == 0 ? a.G : 1;
    p.tokens = QROWS / p.pack;
    p.qtiles = (int)ceil_div(a.Nq, p.tokens);
    p.groups = a.Hq / p.pack;
    const int64_t sg = a.seqs * p.groups;
    MBR_CHECK(sg * p.qtiles < (1ll << 30), "attention: too many tiles");
    p.ntiles = (unsigned)(sg * p.qtiles);
    // With a limit on the right the earliest queries see fewest keys.  Later ones go first, so that what is left at the
    // end is small, where there is no limit on the left (all differ) or the tiles make few rounds.  Otherwise a
    // sequence-head's tiles go together and find its keys in L2; six rounds of windows mostly fit there in any order.
    // us, later first / together, at 2, 4, 6, 8 and 20 rounds: heads of 64, 250 + 20 keys 30/34 53/56 77/78 99/100 248/237;
    // heads of 128, 4 query heads a key head, 400 + 7 keys 28/29 53/54 76/78 97/99 250/226; heads of 128, 100 keys 27/30
    // 47/47 74/70 91/83 236/201.
    const bool wide = a.D > 64;
    const unsigned round = 148 * (wide ? TileCfg<2>::CTAS : TileCfg<1>::CTAS);
    p.last_first = a.right >= 0 && (a.left < 0 || p.ntiles <= 6 * round);
    p.by_inner = FastDiv(p.last_first ? (unsigned)sg : (unsigned)p.qtiles);
    p.by_groups = FastDiv((unsigned)p.groups);
    p.by_pack = FastDiv((unsigned)p.pack);
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.err = stream_error_word(st);
    CUtensorMap q, k, v;
    make_map(&q, a.q, a.q_seq, a.q_tok, a.q_head, a.D, a.Hq, a.Nq, a.seqs, p.pack, p.tokens, dtype);
    make_map(&k, a.k, a.k_seq, a.k_tok, a.k_head, a.D, a.Hkv, a.Nk, a.seqs, 1, KB, dtype);
    make_map(&v, a.v, a.v_seq, a.v_tok, a.v_head, a.D, a.Hkv, a.Nk, a.seqs, 1, KB, dtype);
    if (dtype == DT_BF16) {
        if (wide) launch<__nv_bfloat16, 2>(q, k, v, p, st);
        else launch<__nv_bfloat16, 1>(q, k, v, p, st);
    } else {
        if (wide) launch<__half, 2>(q, k, v, p, st);
        else launch<__half, 1>(q, k, v, p, st);
    }
}

}  // namespace streamops
}  // namespace mbr
