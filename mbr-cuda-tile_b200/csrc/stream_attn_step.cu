// stream_attn_step.cu — attention of a few queries over many keys (the newest
// tokens of a stream over its cache, or a short piece over a long context),
// fp16/bf16, keys and values in 16 bits or as 4-bit codes.
//
// Every key and value is read once and used for few rows, so memory bounds it;
// the matrix products only have to keep out of the way.  One CTA per SM; each of
// its warps works alone: it walks part of the keys of one (sequence, key head, row
// tile), with a ring of its own in shared memory that it refills by bulk copies
// (the rows of a cache are contiguous: two copies a unit of 16 or 32 keys), so
// all the SM's shared memory is loads in flight and no warp waits for another.
// The parts' results (fp32, with their running maximum and sum) go to a
// workspace and a second kernel, launched to overlap this one's end, joins them
// in a fixed order.
// The products are 16 x 8 x 16 warp products whose operands come from the rows as
// they lie, by free choice of the orders:
//  - S = Q K^T contracts over channels, and the order of a contraction is
//    free: the lane (key g, quarter t) takes the 16-byte pieces 8t + 32c of its
//    key's row (4 bits: its quarter of the row), and Q is laid out the same way.
//  - O += P V has output channels in an order that is free too: lane group g
//    owns DP / 8 neighbouring channels; the pairs of keys that the product wants
//    in one register are put together by byte permutes (4 bits: before the codes
//    are widened, so the pairing costs 2 permutes for 16 codes).
//  - the accumulator of S is the A operand of P V as it lies.
// Rows are the tokens of one key head's query heads (token-major), 16 a tile (8
// rows or fewer skip the upper half's exponentials).
//
// A value that some row of the tile does not see enters that row with weight
// 0; were it NaN or infinite, the product would be NaN.  So a row that does
// not come out finite is computed again by attend_row, which reads only what the
// row sees.
#include <algorithm>

#include "sm100.cuh"
#include "stream_attn_step.h"

namespace mbr {
namespace streamops {

namespace {

using namespace sm100;

// A warp's ring: SLOTS units of UNIT keys' rows (and, 4 bits, steps and offsets).
template <int DP, bool Q4>
struct StepCfg {
    static constexpr int WARPS = DP == 128 ? 8 : 16;
    static constexpr int UNIT = Q4 || DP == 32 ? 32 : 16;
    static constexpr int ROW = Q4 ? DP / 2 : DP * 2;  // most bytes of a row
    static constexpr int SROW = Q4 ? DP / kGroup * 4 : 0;
    static constexpr int SLOT = 2 * UNIT * (ROW + SROW);
    static constexpr int BUDGET = 200 * 1024 / WARPS;
    static constexpr int SLOTS = BUDGET / SLOT < 4 ? BUDGET / SLOT : 4;
    static_assert(SLOTS >= 3, "two units in flight while one is read");
    static constexpr int TOTAL = WARPS * SLOTS * (SLOT + 8);
};

// Untiled bulk copy of `bytes` (a multiple of 16, both addresses 16-byte
// aligned), completion counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         __nv_bfloat16*) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The two values that the codes at bits 4i and 16 + 4i of x stand for: code -
// 8 (exact in 16 bits), times the step plus the offset in one rounding.
// sm: (step, offset) of the lower value in s.x / m.x, of the upper in s.y / m.y.
__device__ __forceinline__ uint32_t widen(uint32_t x, int i, uint32_t s, uint32_t m, __half*) {
    const uint32_t b = ((x >> (4 * i)) & 0x000f000fu) | 0x64006400u;  // 1024 + code
    const __half2 u = __hadd2(*reinterpret_cast<const __half2*>(&b), __floats2half2_rn(-1032.f, -1032.f));
    const __half2 v = __hfma2(u, *reinterpret_cast<const __half2*>(&s), *reinterpret_cast<const __half2*>(&m));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t widen(uint32_t x, int i, uint32_t s, uint32_t m, __nv_bfloat16*) {
    const uint32_t b = ((x >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // 128 + code
    const __nv_bfloat162 u =
        __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&b), __floats2bfloat162_rn(-136.f, -136.f));
    const __nv_bfloat162 v =
        __hfma2(u, *reinterpret_cast<const __nv_bfloat162*>(&s), *reinterpret_cast<const __nv_bfloat162*>(&m));
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* dst, const uint8_t* p) {
    if constexpr (BYTES == 2) {
        dst[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (BYTES == 4) {
        dst[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (BYTES == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        dst[0] = v.x, dst[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = *(reinterpret_cast<const uint4*>(p) + i);
            dst[4 * i] = v.x, dst[4 * i + 1] = v.y, dst[4 * i + 2] = v.z, dst[4 * i + 3] = v.w;
        }
    }
}

// What a tile's rows see, in the order the keys are walked: index u < ns is
// position u (the first tokens), u >= ns position LO + u - ns.
struct TileKeys {
    int n, m;    // queries and keys of the sequence
    int ns, LO;  // first tokens; position of index ns
    int total;   // keys
};
// Row r sees u < f or a <= u < b.
struct RowKeys {
    int f, a, b;
};

template <bool CACHED>
__device__ __forceinline__ TileKeys tile_keys(const AttnArgs& a, int64_t s, int r0, int rows) {
    TileKeys k;
    lengths<CACHED>(a, s, k.n, k.m);
    k.ns = k.LO = k.total = 0;
    // from the first token's lower end to the last one's upper end
    const int i0 = r0 / a.G, i1 = min((r0 + rows - 1) / a.G, k.n - 1);
    if (i0 <= i1) {
        const Window w0 = row_window<CACHED>(a, i0, k.n, k.m), w1 = row_window<CACHED>(a, i1, k.n, k.m);
        k.ns = min(a.sinks, w1.hi);
        k.LO = max(CACHED ? max(w0.lo, k.m - a.ring) : w0.lo, k.ns);
        k.total = k.ns + max(w1.hi - k.LO, 0);
    }
    return k;
}
template <bool CACHED>
__device__ __forceinline__ RowKeys row_keys(const AttnArgs& a, const TileKeys& k, int r0, int r, int rows) {
    RowKeys w{0, 0, 0};
    const int i = (r0 + r) / a.G;
    if (r < rows && i < k.n) {
        const Window x = row_window<CACHED>(a, i, k.n, k.m);
        if (x.hi > x.lo || x.first > 0) {
            w.f = min(k.ns, x.hi);
            w.a = k.ns + max(x.lo, k.LO) - k.LO;
            w.b = k.ns + max(x.hi, k.LO) - k.LO;
        }
    }
    return w;
}

// HALF: at most 8 rows; EX: the head size is DP itself.
template <typename T, int DP, bool Q4, bool CACHED, bool HALF, bool EX>
__global__ void __launch_bounds__(StepCfg<DP, Q4>::WARPS * 32, 1) attend_step_kernel(const StepArgs p) {
    constexpr int KS = DP / 16;  // contraction steps of S
    constexpr int NT = DP / 8;   // channel tiles of O
    using Cfg = StepCfg<DP, Q4>;
    constexpr int ROWS = HALF ? 8 : 16, UNIT = Cfg::UNIT, SLOTS = Cfg::SLOTS, JT = UNIT / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const AttnArgs& a = p.a;
    const int D = EX ? DP : a.D;
    const int rb = Q4 ? D / 2 : D * 2, sb = Q4 ? D / kGroup * 4 : 0;  // bytes of a row, of its steps and offsets
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const ring = smem + warp * (SLOTS * Cfg::SLOT);
    uint64_t* const bar = reinterpret_cast<uint64_t*>(smem + Cfg::WARPS * SLOTS * Cfg::SLOT) + warp * SLOTS;
    if (lane < SLOTS) {
        mbar_init(&bar[lane], 1);
        fence_barrier_init();
    }
    __syncwarp();
    // the join kernel may be scheduled as this grid's CTAs end (it waits for all of them)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t use = 0;  // units fetched so far by this warp: slot and parity
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale turns Q's signs
    const float scale = fabsf(p.scale_log2);

    const int64_t segs = p.items * p.parts;
    // neighbouring parts go to different SMs: what lies unevenly is spread
    for (int64_t seg = (int64_t)warp * gridDim.x + blockIdx.x; seg < segs; seg += (int64_t)gridDim.x * Cfg::WARPS) {
        const int64_t item = seg / p.parts;
        const int part = (int)(seg - item * p.parts);
        const int64_t hs = item / p.tiles;
        const int r0 = (int)(item - hs * p.tiles) * ROWS;
        const int64_t s = hs / a.Hkv;
        const int hk = (int)(hs - s * a.Hkv);
        const int rows = min(ROWS, a.Nq * a.G - r0);
        const TileKeys tk = tile_keys<CACHED>(a, s, r0, rows);
        const int total = tk.total, ns = tk.ns;
        const int units = (total + UNIT - 1) / UNIT;
        const int c0 = (int)((int64_t)units * part / p.parts), c1 = (int)((int64_t)units * (part + 1) / p.parts);

        // slot of key index u; a ring starts over at most once (total - ns <= ring), at index `wrap`
        const unsigned ring0 =
            CACHED ? (unsigned)(tk.LO < a.sinks ? tk.LO : (int)slot_of(tk.LO, a.sinks, a.ring)) : (unsigned)tk.LO;
        const int wrap = CACHED ? (int)min((int64_t)total, (int64_t)ns + a.slots - ring0) : total;
        auto slot = [&](int u) -> int64_t { return u < ns ? u : (int64_t)ring0 + (u - ns) - (u >= wrap ? a.ring : 0); };
        const uint8_t* kb0 = (const uint8_t*)a.k + s * p.k_seq + hk * p.k_head;
        const uint8_t* vb0 = (const uint8_t*)a.v + s * p.v_seq + hk * p.v_head;
        auto fetch = [&](int c, uint32_t n) {  // unit c (none past the end) into the n-th use of the ring
            if (c < c1) {
                uint8_t* dk = ring + (n % SLOTS) * Cfg::SLOT;
                uint8_t* dv = dk + UNIT * Cfg::ROW;
                const int u0 = c * UNIT, u1 = min(u0 + UNIT, total);
                if (p.packed) {
                    if (lane == 0) {  // whole runs of rows: the first tokens, up to the ring's end, from its start
                        uint64_t* b = &bar[n % SLOTS];
                        mbar_arrive_expect_tx(b, (uint32_t)(2 * (u1 - u0) * rb));
                        for (int u = u0; u < u1;) {
                            const int to = min(u1, u < ns ? ns : u < wrap ? wrap : total);
                            const int64_t src = slot(u) * rb;
                            const uint32_t at = (uint32_t)((u - u0) * rb), bytes = (uint32_t)((to - u) * rb);
                            bulk_load(dk + at, kb0 + src, bytes, b);
                            bulk_load(dv + at, vb0 + src, bytes, b);
                            u = to;
                        }
                    }
                } else {  // rows apart: 16-byte copies, neighbouring lanes on one row
                    const int per = rb >> 4;
                    for (int j = lane; j < (u1 - u0) * per; j += 32) {
                        const int r = j / per, o = (j - r * per) * 16;
                        const int64_t sl = slot(u0 + r);
                        cp_async<16>(dk + r * rb + o, kb0 + sl * p.k_tok + o);
                        cp_async<16>(dv + r * rb + o, vb0 + sl * p.v_tok + o);
                    }
                }
                if constexpr (Q4) {
                    constexpr int SC = EX ? Cfg::SROW : 4;  // bytes a copy
                    if (u0 + lane < u1) {
                        uint8_t* dst = dk + 2 * UNIT * Cfg::ROW + lane * sb;
                        const int64_t src = s * p.s_seq + hk * p.s_head + slot(u0 + lane) * sb;
#pragma unroll
                        for (int e = 0; e < Cfg::SROW / SC; ++e)
                            if (SC * e < sb) {
                                cp_async<SC>(dst + SC * e, (const uint8_t*)a.k_scale + src + SC * e);
                                cp_async<SC>(dst + UNIT * Cfg::SROW + SC * e, (const uint8_t*)a.v_scale + src + SC * e);
                            }
                    }
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int n = 0; n < SLOTS - 1; ++n) fetch(c0 + n, use + n);

        const RowKeys ka = row_keys<CACHED>(a, tk, r0, g, rows), kb = HALF ? ka : row_keys<CACHED>(a, tk, r0, g + 8, rows);
        // [full_lo, full_hi): every row of the tile sees these
        const bool in_a = g < rows, in_b = !HALF && g + 8 < rows;
        const int full_lo = __reduce_max_sync(0xffffffffu, max(in_a ? ka.a : 0, in_b ? kb.a : 0));
        const int full_hi = __reduce_min_sync(0xffffffffu, min(in_a ? ka.b : INT32_MAX, in_b ? kb.b : INT32_MAX));

        uint32_t q[KS][4];
        auto load_q = [&](int r, int hi) {
            const bool on = r < rows;
            const int i = on ? (r0 + r) / a.G : 0, h = hk * a.G + (on ? (r0 + r) - i * a.G : 0);
            const T* x = (const T*)a.q + s * a.q_seq + (int64_t)i * a.q_tok + (int64_t)h * a.q_head;
#pragma unroll
            for (int c = 0; c < KS / 2; ++c) {  // 8 channels: two contraction steps
                const int d0 = Q4 ? DP / 4 * t + 8 * c : 32 * c + 8 * t;
                uint32_t w[4] = {0u, 0u, 0u, 0u};
                if (on && d0 < D) {
                    uint16_t e[8];
                    const uint16_t* xe = reinterpret_cast<const uint16_t*>(x) + d0;
                    if (p.q_vec) {
                        *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(xe));
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = __ldg(xe + j);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // 4 bits: the pairs that widen() makes, (j, j + 4)
                        w[j] = (Q4 ? e[j] | ((uint32_t)e[j + 4] << 16) : e[2 * j] | ((uint32_t)e[2 * j + 1] << 16)) ^ flip;
                }
                q[2 * c][hi] = w[0], q[2 * c][hi + 2] = w[1];
                q[2 * c + 1][hi] = w[2], q[2 * c + 1][hi + 2] = w[3];
            }
        };
        load_q(g, 0);
        if constexpr (HALF) {
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k][1] = q[k][3] = 0u;
        } else {
            load_q(g + 8, 1);
        }

        float o[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
        float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;  // rows g and g + 8: offset (log2 units), sum

        for (int c = c0; c < c1; ++c, ++use) {
            fetch(c + SLOTS - 1, use + SLOTS - 1);  // into the slot read last, while this unit is worked on
            if (p.packed && !__all_sync(0xffffffffu, mbar_wait(&bar[use % SLOTS], use / SLOTS & 1, p.err))) return;
            cp_async_wait<SLOTS - 1>();
            __syncwarp();
            const uint8_t* kp = ring + (use % SLOTS) * Cfg::SLOT;
            const uint8_t* vp = kp + UNIT * Cfg::ROW;
            const uint8_t* ksp = vp + UNIT * Cfg::ROW;
            const uint8_t* vsp = ksp + UNIT * Cfg::SROW;
            const int u0 = c * UNIT;
            const bool full = u0 >= full_lo && u0 + UNIT <= full_hi;  // every row sees every key
            // ---- S = Q K^T: key tile j holds keys 8j + g ----
            float sc[JT][4];
            uint32_t kx[JT][Q4 ? DP / 32 : DP / 8], sm[JT];
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
                const uint8_t* row = kp + (8 * j + g) * rb;
                sm[j] = 0u;
                if constexpr (Q4) {
#pragma unroll
                    for (int w = 0; w < DP / 32; ++w) kx[j][w] = 0u;
                    if (EX || DP / 4 * t < D) {
                        load_words<DP / 8>(kx[j], row + DP / 8 * t);
                        sm[j] = *reinterpret_cast<const uint32_t*>(ksp + (8 * j + g) * sb + DP / 4 * t / kGroup * 4);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < KS / 2; ++w) {
                        kx[j][4 * w] = kx[j][4 * w + 1] = kx[j][4 * w + 2] = kx[j][4 * w + 3] = 0u;
                        if (EX || 32 * w + 8 * t < D) load_words<16>(kx[j] + 4 * w, row + 64 * w + 16 * t);
                    }
                }
            }
            // the key tiles' sums advance together: a product waits for the one before it on its tile only
#pragma unroll
            for (int w = 0; w < KS / 2; ++w)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int j = 0; j < JT; ++j) {
                        if constexpr (Q4) {
                            const uint32_t step = __byte_perm(sm[j], 0, 0x1010), off = __byte_perm(sm[j], 0, 0x3232);
                            mma16816(sc[j], q[2 * w + half], widen(kx[j][w], 2 * half, step, off, (T*)nullptr),
                                     widen(kx[j][w], 2 * half + 1, step, off, (T*)nullptr), (T*)nullptr);
                        } else {
                            mma16816(sc[j], q[2 * w + half], kx[j][4 * w + 2 * half], kx[j][4 * w + 2 * half + 1],
                                     (T*)nullptr);
                        }
                    }
            if (!full) {  // unseen keys get -inf
#pragma unroll
                for (int j = 0; j < JT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int u = u0 + 8 * j + 2 * t + e;
                        if (!(u < ka.f || (u >= ka.a && u < ka.b))) sc[j][e] = -INFINITY;
                        if (!HALF && !(u < kb.f || (u >= kb.a && u < kb.b))) sc[j][2 + e] = -INFINITY;
                    }
            }
            // ---- weights 2^(s - m) with the offset m so far; the sum tells (inf and
            // NaN too) when the offset has become too low: then m becomes the
            // maximum, what was summed is scaled, and the weights are taken again.
            // The sum holds the weights before their rounding to the values' type.
            uint32_t pr[JT][2];  // [key tile][row half]
            auto weights = [&](float& ra, float& rb_) {
                const float oa = ma == -INFINITY ? 0.f : ma, ob = mb == -INFINITY ? 0.f : mb;
                ra = rb_ = 0.f;
#pragma unroll
                for (int j = 0; j < JT; ++j) {
                    const float e0 = ex2_approx(fmaf(sc[j][0], scale, -oa)), e1 = ex2_approx(fmaf(sc[j][1], scale, -oa));
                    ra += e0 + e1;
                    pr[j][0] = pack2(e0, e1, (T*)nullptr);
                    if constexpr (HALF) {
                        pr[j][1] = 0u;
                    } else {
                        const float e2 = ex2_approx(fmaf(sc[j][2], scale, -ob)),
                                    e3 = ex2_approx(fmaf(sc[j][3], scale, -ob));
                        rb_ += e2 + e3;
                        pr[j][1] = pack2(e2, e3, (T*)nullptr);
                    }
                }
            };
            float ra, rbs;
            weights(ra, rbs);
            constexpr float kMost = 256.f;
            bool low = !(ra <= kMost) || ma == -INFINITY;
            if constexpr (!HALF) low |= !(rbs <= kMost) || mb == -INFINITY;
            if (__any_sync(0xffffffffu, low)) {
                auto row_max = [&](int e) {
                    float r = -INFINITY;
#pragma unroll
                    for (int j = 0; j < JT; ++j) r = fmaxf(r, fmaxf(sc[j][e], sc[j][e + 1]));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 1));
                    return fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 2)) * scale;
                };
                auto raise = [&](float& mx, float& l, int e) {
                    const float now = fmaxf(mx, row_max(e));
                    const float f = now == mx ? 1.f : ex2_approx(mx - now);
                    mx = now;
                    l *= f;
#pragma unroll
                    for (int i = 0; i < NT; ++i) o[i][e] *= f, o[i][e + 1] *= f;
                };
                raise(ma, la, 0);
                if constexpr (!HALF) raise(mb, lb, 2);
                weights(ra, rbs);
            }
            la += ra;
            lb += rbs;
            // ---- O += P V, 16 keys at a time: values 2t, 2t + 1, 8 + 2t, 9 + 2t ----
#pragma unroll
            for (int h = 0; h < UNIT / 16; ++h) {
                const uint32_t pa[4] = {pr[2 * h][0], pr[2 * h][1], pr[2 * h + 1][0], pr[2 * h + 1][1]};
                constexpr int W = Q4 ? (DP + 63) / 64 : DP / 16;
                uint32_t v[4][W], vs[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int kr = 16 * h + 2 * t + 8 * (j >> 1) + (j & 1);
                    const uint8_t* row = vp + kr * rb;
                    const bool on = full || u0 + kr < total;  // rows past the last key hold anything
#pragma unroll
                    for (int w = 0; w < W; ++w) v[j][w] = 0u;
                    vs[j] = 0u;
                    if constexpr (Q4) {
                        if (on && (EX || DP / 8 * g < D)) {
                            load_words<DP / 16>(v[j], row + DP / 16 * g);
                            vs[j] = *reinterpret_cast<const uint32_t*>(vsp + kr * sb + DP / 8 * g / kGroup * 4);
                        }
                    } else if constexpr (DP == 32) {
                        if (on && (EX || 4 * g < D)) load_words<8>(v[j], row + 8 * g);
                    } else {
#pragma unroll
                        for (int w = 0; w < DP / 64; ++w)
                            if (on && (EX || DP / 8 * g + 8 * w < D)) load_words<16>(v[j] + 4 * w, row + DP / 4 * g + 16 * w);
                    }
                }
                if constexpr (Q4) {
                    uint32_t step[2], off[2];  // (key 2t, key 2t + 1) of each half
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        step[j] = __byte_perm(vs[2 * j], vs[2 * j + 1], 0x5410);
                        off[j] = __byte_perm(vs[2 * j], vs[2 * j + 1], 0x7632);
                    }
#pragma unroll
                    for (int w = 0; w < NT / 4; ++w) {  // four channels at a time
                        const uint32_t sel = (w & 1) ? 0x7632 : 0x5410;
                        const uint32_t lo = __byte_perm(v[0][w >> 1], v[1][w >> 1], sel);
                        const uint32_t hi = __byte_perm(v[2][w >> 1], v[3][w >> 1], sel);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mma16816(o[4 * w + i], pa, widen(lo, i, step[0], off[0], (T*)nullptr),
                                     widen(hi, i, step[1], off[1], (T*)nullptr), (T*)nullptr);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < NT / 2; ++w) {
                        mma16816(o[2 * w], pa, __byte_perm(v[0][w], v[1][w], 0x5410),
                                 __byte_perm(v[2][w], v[3][w], 0x5410), (T*)nullptr);
                        mma16816(o[2 * w + 1], pa, __byte_perm(v[0][w], v[1][w], 0x7632),
                                 __byte_perm(v[2][w], v[3][w], 0x7632), (T*)nullptr);
                    }
                }
            }
            __syncwarp();  // the slot is read
        }

        // ---- this part's result; accumulator column 2t, 2t + 1 of tile i is channel NT * 2t + i, NT * (2t + 1) + i ----
        la += __shfl_xor_sync(0xffffffffu, la, 1);
        la += __shfl_xor_sync(0xffffffffu, la, 2);
        lb += __shfl_xor_sync(0xffffffffu, lb, 1);
        lb += __shfl_xor_sync(0xffffffffu, lb, 2);
        auto put = [&](int r, int e, float m, float l) {
            if (r >= rows) return;
            const int64_t row = seg * p.rows + r;
            if (t == 0) p.part_ml[row] = make_float2(m, l);
            float4* dst = reinterpret_cast<float4*>(p.part_o + row * DP + 2 * NT * t);
#pragma unroll
            for (int i = 0; i < NT / 4; ++i) {
                dst[i] = make_float4(o[4 * i][e], o[4 * i + 1][e], o[4 * i + 2][e], o[4 * i + 3][e]);
                dst[NT / 4 + i] =
                    make_float4(o[4 * i][e + 1], o[4 * i + 1][e + 1], o[4 * i + 2][e + 1], o[4 * i + 3][e + 1]);
            }
        };
        put(g, 0, ma, la);
        if constexpr (!HALF) put(g + 8, 2, mb, lb);
    }
}

// Joins the parts of each row: wpr warps a row (1, 2, 4 or 8), 8 / wpr rows a CTA.
template <typename T, int DP, bool Q4, bool CACHED>
__global__ void __launch_bounds__(256) join_step_kernel(const StepArgs p, int wpr, int tile_rows) {
    __shared__ float s_o[8][DP];
    __shared__ float s_l[8];
    const AttnArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % wpr;
    const int64_t n = p.items * p.rows, at = (int64_t)blockIdx.x * (8 / wpr) + warp / wpr;
    const int64_t item = at / p.rows;
    const int r = (int)(at - item * p.rows);
    const int64_t hs = item / p.tiles;
    const int r0 = (int)(item - hs * p.tiles) * tile_rows;
    const int64_t s = hs / a.Hkv;
    const int hk = (int)(hs - s * a.Hkv), rows = min(tile_rows, a.Nq * a.G - r0);
    const bool on = at < n && r < rows;
    const int i = on ? (r0 + r) / a.G : 0, h = hk * a.G + (on ? (r0 + r) - i * a.G : 0);
    TileKeys tk{};
    RowKeys k{0, 0, 0};
    float gate = 1.f;
    if (on) {
        tk = tile_keys<CACHED>(a, s, r0, rows);
        k = row_keys<CACHED>(a, tk, r0, r, rows);
        if (a.gates) gate = __ldg(a.gates + (s * a.Nq + i) * a.Hq + h);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are written
    float l = 0.f, v[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) v[e] = 0.f;
    if (on) {
        const int64_t row0 = item * p.parts * p.rows + r;
        float top = -INFINITY;
        for (int b = lane; b < p.parts; b += 32) top = fmaxf(top, p.part_ml[row0 + (int64_t)b * p.rows].x);
        top = warp_max(top);
#pragma unroll 4
        for (int b = sub; b < p.parts; b += wpr) {
            const int64_t row = row0 + (int64_t)b * p.rows;
            const float2 ml = p.part_ml[row];
            const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
            l += f * ml.y;
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) v[e] += f * p.part_o[row * DP + lane + 32 * e];
        }
    }
    if (wpr > 1) {
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) s_o[warp][lane + 32 * e] = v[e];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        if (sub == 0)
            for (int w = 1; w < wpr; ++w) {
                l += s_l[warp + w];
#pragma unroll
                for (int e = 0; e < DP / 32; ++e) v[e] += s_o[warp + w][lane + 32 * e];
            }
    }
    if (!on || sub != 0) return;
    const bool sees = k.f > 0 || k.b > k.a;
    const float inv = sees ? gate / l : 0.f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
        v[e] = sees ? v[e] * inv : 0.f;
        bad |= lane + 32 * e < a.D && !isfinite(v[e]);
    }
    if (__any_sync(0xffffffffu, bad)) {
        attend_row<T, CACHED, Q4>(a, s, i, h, tk.n, tk.m);
    } else {
        T* out = (T*)a.out + s * a.o_seq + (int64_t)i * a.o_tok + (int64_t)h * a.o_head;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
            if (lane + 32 * e < a.D) out[lane + 32 * e] = from_f32<T>(v[e]);
    }
}

int sm_count() {
    static int sms[kMaxStreamDevices] = {};
    const int dev = stream_device();
    if (!sms[dev]) MBR_CUDA(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
    return sms[dev];
}

template <typename T, int DP, bool Q4, bool CACHED, bool HALF, bool EX>
void launch(const StepArgs& p, cudaStream_t st) {
    auto kern = attend_step_kernel<T, DP, Q4, CACHED, HALF, EX>;
    using Cfg = StepCfg<DP, Q4>;
    static bool attr[kMaxStreamDevices] = {};
    const int dev = stream_device();
    if (!attr[dev]) {
        MBR_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::TOTAL));
        attr[dev] = true;
    }
    const int64_t segs = p.items * p.parts;
    const unsigned grid = (unsigned)std::min<int64_t>(segs, sm_count());
    kern<<<grid, Cfg::WARPS * 32, Cfg::TOTAL, st>>>(p);
    MBR_CUDA(cudaGetLastError());
    const int wpr = p.parts <= 8 ? 1 : p.parts <= 16 ? 2 : p.parts <= 32 ? 4 : 8;  // at most about eight parts a warp
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ceil_div(p.items * p.rows, 8 / wpr));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    MBR_CUDA(cudaLaunchKernelEx(&cfg, join_step_kernel<T, DP, Q4, CACHED>, p, wpr, HALF ? 8 : 16));
}

template <typename T, bool Q4, bool CACHED, bool HALF>
void dispatch_size(const StepArgs& p, cudaStream_t st) {
    if (p.a.D == 32) launch<T, 32, Q4, CACHED, HALF, true>(p, st);
    else if (p.a.D == 64) launch<T, 64, Q4, CACHED, HALF, true>(p, st);
    else if (p.a.D == 128) launch<T, 128, Q4, CACHED, HALF, true>(p, st);
    else launch<T, 128, Q4, CACHED, HALF, false>(p, st);
}
template <typename T, bool Q4, bool CACHED>
void dispatch(const StepArgs& p, cudaStream_t st) {
    if (p.half) dispatch_size<T, Q4, CACHED, true>(p, st);
    else dispatch_size<T, Q4, CACHED, false>(p, st);
}

}  // namespace

bool step_supported(const AttnArgs& a, int dtype, bool cached) {
    if (dtype == DT_F32) return false;
    if (cached) return true;  // a cache's rows are aligned
    const int64_t all = a.k_seq | a.k_tok | a.k_head | a.v_seq | a.v_tok | a.v_head;
    return (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 && all % 8 == 0;
}

StepPlan step_plan(int64_t seqs, int64_t tokens, int Hq, int Hkv, int D, int64_t keys) {
    StepPlan pl{};
    const int64_t rows = tokens * (Hq / Hkv);
    pl.half = rows <= 8;
    pl.rows = (int)std::min<int64_t>(rows, 16);
    pl.tiles = ceil_div(rows, 16);
    pl.items = seqs * Hkv * pl.tiles;
    const int dp = D == 32 ? 32 : D == 64 ? 64 : 128;
    const int64_t warps = 148 * (dp == 128 ? 8 : 16);
    // Parts: the time of a warp is rounds x (its part's keys + a start worth about
    // 64 keys); the join reads every part, so it has a price too.
    double best = 0.;
    pl.parts = 1;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(512, keys / 32));
    for (int64_t n = 1; n <= most && pl.items * n <= (1 << 24); ++n) {
        const double cost = (double)ceil_div(pl.items * n, warps) * ((double)keys / n + 64.) + 0.5 * n;
        if (n == 1 || cost < best) best = cost, pl.parts = (int)n;
    }
    pl.bytes = pl.items * pl.parts * pl.rows * (int64_t)(dp + 2) * 4;
    return pl;
}

void attend_step(const AttnArgs& a, int dtype, bool cached, bool q4, const StepPlan& pl, void* workspace,
                 cudaStream_t st) {
    MBR_CHECK(((uintptr_t)workspace & 15) == 0, "attention: workspace must be 16-byte aligned");
    StepArgs p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.items = pl.items, p.tiles = pl.tiles, p.parts = pl.parts, p.rows = pl.rows, p.half = pl.half;
    const int dp = a.D == 32 ? 32 : a.D == 64 ? 64 : 128;
    p.part_o = (float*)workspace;
    p.part_ml = (float2*)(p.part_o + pl.items * pl.parts * pl.rows * dp);
    p.q_vec = (((uintptr_t)a.q & 15) == 0 && (a.q_seq | a.q_tok | a.q_head) % 8 == 0) ? 1 : 0;
    const int64_t es = 2;
    if (cached) {
        const int64_t row = q4 ? a.D / 2 : a.D * es, srow = a.D / kGroup * 2 * es;
        p.k_tok = p.v_tok = row;
        p.k_head = p.v_head = a.slots * row;
        p.k_seq = p.v_seq = a.Hkv * a.slots * row;
        p.s_head = a.slots * srow, p.s_seq = a.Hkv * a.slots * srow;
    } else {
        p.k_tok = a.k_tok * es, p.k_head = a.k_head * es, p.k_seq = a.k_seq * es;
        p.v_tok = a.v_tok * es, p.v_head = a.v_head * es, p.v_seq = a.v_seq * es;
    }
    p.packed = p.k_tok == (q4 ? a.D / 2 : a.D * es) && p.v_tok == p.k_tok;
    p.err = stream_error_word();
    if (dtype == DT_BF16) {
        if (!cached) dispatch<__nv_bfloat16, false, false>(p, st);
        else if (q4) dispatch<__nv_bfloat16, true, true>(p, st);
        else dispatch<__nv_bfloat16, false, true>(p, st);
    } else {
        if (!cached) dispatch<__half, false, false>(p, st);
        else if (q4) dispatch<__half, true, true>(p, st);
        else dispatch<__half, false, true>(p, st);
    }
}

}  // namespace streamops
}  // namespace mbr
