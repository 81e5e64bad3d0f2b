// stream_attn_step.cu — attention of a few queries over many keys (the newest
// tokens of a stream over its cache, or a short piece over a long context),
// fp16/bf16, keys and values in 16 bits or as 4-bit codes.
//
// Every key and value is read once and used for few rows, so memory bounds it (in 16
// bits; in 4 bits the widening of the codes does);
// the matrix products only have to keep out of the way.  One CTA per SM; each of
// its warps works alone: it walks part of the keys of one (sequence, key head, row
// tile), with a ring of its own in shared memory that it refills by bulk copies
// (the rows of a cache are contiguous: one copy for 32 keys, one for their
// values), so all the SM's shared memory is loads in flight and no warp waits
// for another.  The parts' results (fp32, with their offset and sum) are joined
// in a fixed order: up to a CTA's warps through shared memory, more (few
// sequences, many keys) through a workspace by a second kernel.
// One frame of 60 sequences x 8 heads of 64 over 1004 keys in fp16 (124 MB): 29.7 us,
// 4.2 TB/s; 3 frames of 2 sequences, 4 key heads, over 66001 keys in bf16 (135 MB): 35.1 us,
// 3.9 TB/s, of which the join is some 4; one frame of 960 sequences over 4-bit caches of
// up to 1504 keys (615 MB): 237 us, 2.6 TB/s, the issue slots near full.
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

constexpr int UNIT = 32;  // keys a warp works on at a time

// A warp's ring: SLOTS times the rows of KEYS keys or values (and, 4 bits, their
// steps and offsets): one unit of 16-bit rows, two of codes, whose copies are
// short.
template <int DP, bool Q4>
struct StepCfg {
    static constexpr int WARPS = step_warps(DP, Q4);
    static constexpr int ROW = Q4 ? DP / 2 : DP * 2;  // most bytes of a row
    static constexpr int SROW = Q4 ? DP / kGroup * 4 : 0;
    static constexpr int SUBS = Q4 ? 2 : 1, KEYS = UNIT * SUBS;
    static constexpr int SLOT = KEYS * (ROW + SROW);
    static constexpr int BUDGET = 200 * 1024 / WARPS;
    static constexpr int SLOTS = BUDGET / SLOT < 8 ? BUDGET / SLOT : 8;
    static_assert(SLOTS >= 3, "two copies in flight while one is read");
    static constexpr int RING = SLOTS * SLOT > 16 * (DP + 2) * 4 ? SLOTS * SLOT : 16 * (DP + 2) * 4;  // holds a result
    static constexpr int TOTAL = WARPS * (RING + SLOTS * 8);
};

// Shared memory is addressed by its 32-bit addresses throughout: a unit's loads
// are one register plus constants.
// Untiled bulk copy of `bytes` (a multiple of 16, both addresses 16-byte
// aligned), completion counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits (with a limit) for the phase of the given parity.  False if it ran out (*err is set then: the host
// sees it, the results are void).
__device__ __forceinline__ bool wait_bytes(uint32_t bar, uint32_t parity, int* err) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok || mbar_wait((uint64_t*)__cvta_shared_to_generic(bar), parity, err);
}
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
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

// A constant the compiler keeps in a register instead of writing it out at each use.
__device__ __forceinline__ uint32_t held(uint32_t c) {
    uint32_t r;
    asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(c));
    return r;
}
// What widening codes takes: the mask of two codes, 1024 (fp16) or 128 (bf16)
// in both halves, whose last bits a code fits into, and minus that and eight.
template <typename T>
struct Widen;
template <>
struct Widen<__half> {
    uint32_t mask = held(0x000f000fu), base = held(0x64006400u), less = held(0xe408e408u);  // -1032
};
template <>
struct Widen<__nv_bfloat16> {
    uint32_t mask = held(0x000f000fu), base = held(0x43004300u), less = held(0xc308c308u);  // -136
};
// The two values that the codes at bits 4i and 16 + 4i of x stand for: code -
// 8 (exact in 16 bits), times the step plus the offset in one rounding.  The code
// becomes a number by the well-known way of setting it into the last bits of a
// power of two's mantissa and subtracting that.
// s, m: step and offset of both.
__device__ __forceinline__ uint32_t masked(uint32_t x, uint32_t mask, uint32_t base) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(base));  // (x & mask) | base
    return r;
}
__device__ __forceinline__ uint32_t widen(uint32_t x, int i, uint32_t s, uint32_t m, const Widen<__half>& w) {
    uint32_t u = masked(x >> (4 * i), w.mask, w.base), v;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(u) : "r"(u), "r"(w.less));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(u), "r"(s), "r"(m));
    return v;
}
__device__ __forceinline__ uint32_t widen(uint32_t x, int i, uint32_t s, uint32_t m, const Widen<__nv_bfloat16>& w) {
    uint32_t u = masked(x >> (4 * i), w.mask, w.base), v;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(u) : "r"(u), "r"(w.less));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(u), "r"(s), "r"(m));
    return v;
}

// BYTES bytes of shared memory at p (volatile: in order with the waits and copies).
template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* dst, uint32_t p) {
    if constexpr (BYTES == 2) {
        uint16_t h;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(p));
        dst[0] = h;
    } else if constexpr (BYTES == 4) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(dst[0]) : "r"(p));
    } else if constexpr (BYTES == 8) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(dst[0]), "=r"(dst[1]) : "r"(p));
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(dst[4 * i]), "=r"(dst[4 * i + 1]), "=r"(dst[4 * i + 2]), "=r"(dst[4 * i + 3])
                         : "r"(p + 16 * i));
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
    const int i0 = (int)a.by_G.div(r0), i1 = min((int)a.by_G.div(r0 + rows - 1), k.n - 1);
    if (i0 <= i1) {
        const Window w0 = row_window<CACHED>(a, i0, k.n, k.m), w1 = i1 == i0 ? w0 : row_window<CACHED>(a, i1, k.n, k.m);
        k.ns = min(a.sinks, w1.hi);
        k.LO = max(CACHED ? max(w0.lo, k.m - a.ring) : w0.lo, k.ns);
        k.total = k.ns + max(w1.hi - k.LO, 0);
    }
    return k;
}
template <bool CACHED>
__device__ __forceinline__ RowKeys row_keys(const AttnArgs& a, const TileKeys& k, int r0, int r, int rows) {
    if (a.Nq == 1) return RowKeys{r < rows ? k.ns : 0, r < rows ? k.ns : 0, r < rows ? k.total : 0};
    RowKeys w{0, 0, 0};
    const int i = (int)a.by_G.div(r0 + r);
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

// Row r of a tile from its sums v (channels lane, lane + 32, ...) and l: divided,
// gated, rounded and written, by one warp.
template <typename T, int DP, bool Q4, bool CACHED>
__device__ __forceinline__ void finish_row(const AttnArgs& a, const TileKeys& tk, const RowKeys& k, int64_t s, int hk,
                                           int rr, float (&v)[DP / 32], float l) {
    const int lane = threadIdx.x & 31, i = (int)a.by_G.div(rr), h = hk * a.G + rr - i * a.G;
    const float gate = a.gates ? __ldg(a.gates + (s * a.Nq + i) * a.Hq + h) : 1.f;
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
// Factor that brings sums with offset m to offset top.
__device__ __forceinline__ float to_offset(float m, float top) { return m == -INFINITY ? 0.f : ex2_approx(m - top); }

// HALF: at most 8 rows; EX: the head size is DP itself.
template <typename T, int DP, bool Q4, bool CACHED, bool HALF, bool EX>
__global__ void __launch_bounds__(StepCfg<DP, Q4>::WARPS * 32, 1) attend_step_kernel(const StepArgs p) {
    constexpr int KS = DP / 16;  // contraction steps of S
    constexpr int NT = DP / 8;   // channel tiles of O
    using Cfg = StepCfg<DP, Q4>;
    constexpr int ROWS = HALF ? 8 : 16, SLOTS = Cfg::SLOTS, KEYS = Cfg::KEYS, JT = UNIT / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const AttnArgs& a = p.a;
    const int D = EX ? DP : a.D;
    const int rb = Q4 ? D / 2 : D * 2, sb = Q4 ? D / kGroup * 4 : 0;  // bytes of a row, of its steps and offsets
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * Cfg::RING;
    const uint32_t bar = smem_u32(smem) + Cfg::WARPS * Cfg::RING + warp * (SLOTS * 8);
    if (lane < SLOTS) {
        mbar_init(reinterpret_cast<uint64_t*>(smem + Cfg::WARPS * Cfg::RING) + warp * SLOTS + lane, 1);
        fence_barrier_init();
    }
    __syncwarp();
    // the join kernel may be scheduled as this grid's CTAs end (it waits for all of them)
    if (p.outer > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int st = 0;           // slot to be read next
    uint32_t parity = 0;  // and the parity of its use
    bool alive = true;    // false once a wait of this warp ran out: it copies and writes nothing from then on
    auto after = [](int x, int n) { return x + n >= SLOTS ? x + n - SLOTS : x + n; };
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale turns Q's signs
    const float scale = fabsf(p.scale_log2);
    const Widen<T> wd;

    // Neighbouring shares go to different SMs: what lies unevenly is spread.
    const int inner = 1 << p.inner_log2, group = warp >> p.inner_log2, part = warp & (inner - 1);
    const unsigned todo = p.items * p.outer, stride = gridDim.x * (Cfg::WARPS >> p.inner_log2);
    for (unsigned seg = group * gridDim.x + blockIdx.x; seg < todo; seg += stride) {
        const unsigned item = p.by_outer.div(seg), share = seg - item * p.outer;
        const unsigned hs = p.by_tiles.div(item);
        const int r0 = (int)(item - hs * p.tiles) * ROWS;
        const unsigned sq = a.by_Hkv.div(hs);
        const int64_t s = sq;
        const int hk = (int)(hs - sq * a.Hkv);
        const int rows = min(ROWS, a.Nq * a.G - r0);
        const TileKeys tk = tile_keys<CACHED>(a, s, r0, rows);
        const int total = tk.total, ns = tk.ns;
        const int units = (total + KEYS - 1) / KEYS;  // of copies
        // this CTA's units (units / outer, the first units % outer shares one more), of which the group's warps
        // take every inner-th: they read neighbouring rows at about the same time
        const int each = (int)p.by_outer.div(units), more = units - each * p.outer;
        const int c0 = each * (int)share + min((int)share, more) + part,
                  c1 = each * (int)(share + 1) + min((int)share + 1, more);
        const int mine = alive && c1 > c0 ? (c1 - c0 + inner - 1) >> p.inner_log2 : 0;

        // slot of key index u; a ring starts over at most once (total - ns <= ring), at index `wrap`
        const unsigned ring0 =
            CACHED ? (unsigned)(tk.LO < a.sinks ? tk.LO : (int)slot_of(tk.LO, a.sinks, a.ring)) : (unsigned)tk.LO;
        const int wrap = CACHED ? (int)min((int64_t)total, (int64_t)ns + a.slots - ring0) : total;
        auto slot = [&](int u) -> int64_t { return u < ns ? u : (int64_t)ring0 + (u - ns) - (u >= wrap ? a.ring : 0); };
        const uint8_t* kb0 = (const uint8_t*)a.k + s * p.k_seq + hk * p.k_head;
        const uint8_t* vb0 = (const uint8_t*)a.v + s * p.v_seq + hk * p.v_head;
        // the n-th copy of this part (unit n / 2: keys, then values; none past the end) into a slot of the ring
        const int copies = 2 * mine;
        const int64_t s0 = s * p.s_seq + hk * p.s_head;
        // units [run_lo, run_hi) lie whole in one run of cache rows; unit c's keys start at run_k + c * KEYS * rb
        int run_lo = 0, run_hi = 0;
        const uint8_t *run_k = nullptr, *run_v = nullptr;
        auto fetch = [&](int n, int to_slot) {
            if (n < copies) {
                const uint32_t dst = ring + to_slot * Cfg::SLOT;
                const int c = c0 + ((n >> 1) << p.inner_log2);
                if constexpr (CACHED) {
                    if (lane == 0) {
                        const uint32_t b = bar + to_slot * 8;
                        if (c >= run_lo && c < run_hi) {
                            expect_bytes(b, KEYS * rb);
                            bulk_load(dst, (n & 1 ? run_v : run_k) + (int64_t)c * (KEYS * rb), KEYS * rb, b);
                        } else {  // the first tokens, the ring's end, its start, the last unit: run by run
                            const int u0 = c * KEYS, u1 = min(u0 + KEYS, total);
                            expect_bytes(b, (uint32_t)((u1 - u0) * rb));
                            int to = 0;
                            for (int u = u0; u < u1; u = to) {
                                const int end = u < ns ? ns : u < wrap ? wrap : total;
                                to = min(u1, end);
                                const int64_t at = slot(u);
                                bulk_load(dst + (u - u0) * rb, (n & 1 ? vb0 : kb0) + at * rb, (uint32_t)((to - u) * rb), b);
                                // the run that this unit ends in
                                run_lo = c + 1, run_hi = end / KEYS;
                                run_k = kb0 + (at - u) * rb, run_v = vb0 + (at - u) * rb;
                            }
                        }
                    }
                } else {  // rows apart: 16-byte copies, neighbouring lanes on one row
                    const int per = rb >> 4, u0 = c * KEYS, u1 = min(u0 + KEYS, total);
                    const int64_t tok = n & 1 ? p.v_tok : p.k_tok;
                    const uint8_t* src = n & 1 ? vb0 : kb0;
                    for (int j = lane; j < (u1 - u0) * per; j += 32) {
                        const int r = j / per, o = (j - r * per) * 16;
                        copy_async<16>(dst + r * rb + o, src + slot(u0 + r) * tok + o);
                    }
                }
                if constexpr (Q4) {
                    constexpr int SC = EX ? Cfg::SROW : 4;  // bytes a copy
                    const uint8_t* scales = (const uint8_t*)(n & 1 ? a.v_scale : a.k_scale) + s0;
#pragma unroll
                    for (int k = lane; k < KEYS; k += 32) {
                        const int u = c * KEYS + k;
                        if (u < total) {
                            const uint32_t d = dst + KEYS * Cfg::ROW + k * sb;
                            const uint8_t* x = scales + slot(u) * sb;
#pragma unroll
                            for (int e = 0; e < Cfg::SROW / SC; ++e)
                                if (SC * e < sb) copy_async<SC>(d + SC * e, x + SC * e);
                        }
                    }
                }
            }
            if (Q4 || !CACHED) cp_async_commit();
        };
        // The slot to be read next (copy n) has landed, and so has the one before it if `so_far` (this lane's); false (in
        // every lane) if a wait ran out.  Then what else this warp has in flight (up to the `sent`-th copy, one a slot)
        // is waited for too: nothing may land in shared memory that the warp has left.
        auto arrived = [&] { return !CACHED || wait_bytes(bar + st * 8, parity, p.err); };
        auto landed = [&](int n, int sent, bool so_far = true) {
            if constexpr (CACHED) {
                so_far &= arrived();
                if (!__all_sync(0xffffffffu, so_far)) {
                    for (int i = n - Q4; i < min(sent, copies); ++i) {
                        const int x = st + i - n, at = x < 0 ? x + SLOTS : x >= SLOTS ? x - SLOTS : x;
                        mbar_drain((uint64_t*)__cvta_shared_to_generic(bar + at * 8), parity ^ (at != x));
                    }
                    if (Q4) cp_async_wait<0>();
                    __syncwarp();
                    return alive = false;
                }
            } else {
                cp_async_wait<SLOTS - 1>();
                __syncwarp();
            }
            return true;
        };
        auto next = [&] {
            __syncwarp();  // every lane has read the slot
            st = after(st, 1);
            parity ^= st == 0;
        };
#pragma unroll
        for (int n = 0; n < SLOTS - 1; ++n) fetch(n, after(st, n));

        const RowKeys ka = row_keys<CACHED>(a, tk, r0, g, rows), kb = HALF ? ka : row_keys<CACHED>(a, tk, r0, g + 8, rows);
        // [full_lo, full_hi): every row of the tile sees these
        const bool in_a = g < rows, in_b = !HALF && g + 8 < rows;
        const int full_lo = __reduce_max_sync(0xffffffffu, max(in_a ? ka.a : 0, in_b ? kb.a : 0));
        const int full_hi = __reduce_min_sync(0xffffffffu, min(in_a ? ka.b : INT32_MAX, in_b ? kb.b : INT32_MAX));

        uint32_t q[KS][4];
        auto load_q = [&](int r, int hi) {
            const bool on = r < rows;
            const int i = on ? (int)a.by_G.div(r0 + r) : 0, h = hk * a.G + (on ? (r0 + r) - i * a.G : 0);
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

        for (int n = 0; n < copies; n += 2) {
            // 16-bit rows: the keys' slot is refilled as soon as S is computed.  Codes: both slots serve two units.
            fetch(n + SLOTS - 1, after(st, SLOTS - 1));  // into the slot read last, while this one is worked on
            bool keys = true;
            if constexpr (Q4) keys = arrived();
            else if (!landed(n, n + SLOTS)) break;
            const uint32_t k_slot = ring + st * Cfg::SLOT;
            uint32_t v_slot = 0;
            if constexpr (Q4) {
                next();
                if (!landed(n + 1, n + SLOTS, keys)) break;
                cp_async_wait<SLOTS - 2>();  // both slots' steps and offsets
                __syncwarp();
                v_slot = ring + st * Cfg::SLOT;
            }
#pragma unroll 1
            for (int sub = 0; sub < Cfg::SUBS; ++sub) {
                const int u0 = (c0 + ((n >> 1) << p.inner_log2)) * KEYS + sub * UNIT;
                if (Q4 && u0 >= total) break;
                const uint32_t kp = k_slot + (sub * UNIT + g) * rb + (Q4 ? DP / 8 * t : 16 * t);
                const uint32_t ksp = k_slot + KEYS * Cfg::ROW + (sub * UNIT + g) * sb + DP / 4 * t / kGroup * 4;
                const bool full = u0 >= full_lo && u0 + UNIT <= full_hi;  // every row sees every key
                // ---- S = Q K^T: key tile j holds keys 8j + g ----
                float sc[JT][4];
                uint32_t kx[JT][Q4 ? DP / 32 : DP / 8], sm[JT];
    #pragma unroll
                for (int j = 0; j < JT; ++j) {
                    sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
                    const uint32_t row = kp + 8 * j * rb;
                    sm[j] = 0u;
                    if constexpr (Q4) {
    #pragma unroll
                        for (int w = 0; w < DP / 32; ++w) kx[j][w] = 0u;
                        if (EX || DP / 4 * t < D) {
                            load_words<DP / 8>(kx[j], row);
                            load_words<4>(&sm[j], ksp + 8 * j * sb);
                        }
                    } else {
    #pragma unroll
                        for (int w = 0; w < KS / 2; ++w) {
                            kx[j][4 * w] = kx[j][4 * w + 1] = kx[j][4 * w + 2] = kx[j][4 * w + 3] = 0u;
                            if (EX || 32 * w + 8 * t < D) load_words<16>(kx[j] + 4 * w, row + 64 * w);
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
                                const uint32_t step = __byte_perm(sm[j], 0, 0x1010),
                                               off = __byte_perm(sm[j], 0, 0x3232);
                                mma16816(sc[j], q[2 * w + half], widen(kx[j][w], 2 * half, step, off, wd),
                                         widen(kx[j][w], 2 * half + 1, step, off, wd), (T*)nullptr);
                            } else {
                                mma16816(sc[j], q[2 * w + half], kx[j][4 * w + 2 * half], kx[j][4 * w + 2 * half + 1],
                                         (T*)nullptr);
                            }
                        }
                if constexpr (!Q4) {
                    next();
                    fetch(n + SLOTS, after(st, SLOTS - 1));
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
                        const float e0 = ex2_approx(fmaf(sc[j][0], scale, -oa)),
                                    e1 = ex2_approx(fmaf(sc[j][1], scale, -oa));
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
                if constexpr (!Q4) {
                    if (!landed(n + 1, n + SLOTS + 1)) break;
                    v_slot = ring + st * Cfg::SLOT;
                }
                const uint32_t vp = v_slot + (sub * UNIT + 2 * t) * rb + (Q4 ? DP / 16 : DP / 4) * g;
                const uint32_t vsp = v_slot + KEYS * Cfg::ROW + (sub * UNIT + 2 * t) * sb + DP / 8 * g / kGroup * 4;
                // ---- O += P V, 16 keys at a time: values 2t, 2t + 1, 8 + 2t, 9 + 2t ----
    #pragma unroll
                for (int h = 0; h < UNIT / 16; ++h) {
                    const uint32_t pa[4] = {pr[2 * h][0], pr[2 * h][1], pr[2 * h + 1][0], pr[2 * h + 1][1]};
                    constexpr int W = Q4 ? (DP + 63) / 64 : DP / 16;
                    uint32_t v[4][W], vs[4];
    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int kr = 16 * h + 8 * (j >> 1) + (j & 1);
                        const uint32_t row = vp + kr * rb;
                        if constexpr (!EX) {
    #pragma unroll
                            for (int w = 0; w < W; ++w) v[j][w] = 0u;
                            vs[j] = 0u;
                        }
                        if constexpr (Q4) {
                            if (EX || DP / 8 * g < D) {
                                load_words<DP / 16>(v[j], row);
                                load_words<4>(&vs[j], vsp + kr * sb);
                            }
                        } else if constexpr (DP == 32) {
                            if (EX || 4 * g < D) load_words<8>(v[j], row);
                        } else {
    #pragma unroll
                            for (int w = 0; w < DP / 64; ++w)
                                if (EX || DP / 8 * g + 8 * w < D) load_words<16>(v[j] + 4 * w, row + 16 * w);
                        }
                    }
                    if (!full) {  // rows past the last key hold anything: zeros instead (4 bits: by step and offset)
    #pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool on = u0 + 16 * h + 2 * t + 8 * (j >> 1) + (j & 1) < total;
                            if constexpr (Q4) {
                                vs[j] = on ? vs[j] : 0u;
                            } else {
    #pragma unroll
                                for (int w = 0; w < W; ++w) v[j][w] = on ? v[j][w] : 0u;
                            }
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
                                mma16816(o[4 * w + i], pa, widen(lo, i, step[0], off[0], wd),
                                         widen(hi, i, step[1], off[1], wd), (T*)nullptr);
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
            }
            if (!alive) break;
            next();
            if constexpr (Q4) fetch(n + SLOTS, after(st, SLOTS - 2));  // the keys' slot, read with the values'
        }

        // ---- this part's result; accumulator column 2t, 2t + 1 of tile i is channel NT * 2t + i, NT * (2t + 1) + i ----
        la += __shfl_xor_sync(0xffffffffu, la, 1);
        la += __shfl_xor_sync(0xffffffffu, la, 2);
        lb += __shfl_xor_sync(0xffffffffu, lb, 1);
        lb += __shfl_xor_sync(0xffffffffu, lb, 2);
        // The group's results are joined through its warps' rings, whose copies have all landed and are read.  (A warp
        // whose wait ran out writes nothing there and keeps to the group's barriers: the rows are void, the error
        // word says so.)
        constexpr int LD = DP + 2;  // a row's sums, its offset and sum
        auto put = [&](int r, int e, float m, float l) {
            float* dst = reinterpret_cast<float*>(smem + warp * Cfg::RING) + r * LD;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                dst[2 * NT * t + i] = o[i][e];
                dst[2 * NT * t + NT + i] = o[i][e + 1];
            }
            if (t == 0) dst[DP] = m, dst[DP + 1] = l;
        };
        if (alive && g < rows) put(g, 0, ma, la);
        if constexpr (!HALF) {
            if (alive && g + 8 < rows) put(g + 8, 2, mb, lb);
        }
        auto group_sync = [&] {
            if (inner > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(inner * 32) : "memory");
            else __syncwarp();
        };
        group_sync();
        const float* first = reinterpret_cast<const float*>(smem + (warp - part) * Cfg::RING);
        for (int r = part; r < rows; r += inner) {
            float top = -INFINITY, l = 0.f, v[DP / 32];
            for (int b = 0; b < inner; ++b) top = fmaxf(top, first[b * (Cfg::RING / 4) + r * LD + DP]);
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) v[e] = 0.f;
            for (int b = 0; b < inner; ++b) {
                const float* x = first + b * (Cfg::RING / 4) + r * LD;
                const float f = to_offset(x[DP], top);
                l += f * x[DP + 1];
#pragma unroll
                for (int e = 0; e < DP / 32; ++e) v[e] += f * x[lane + 32 * e];
            }
            if (p.outer == 1) {
                finish_row<T, DP, Q4, CACHED>(a, tk, row_keys<CACHED>(a, tk, r0, r, rows), s, hk, r0 + r, v, l);
            } else {
                const int64_t row = (int64_t)seg * p.rows + r;
#pragma unroll
                for (int e = 0; e < DP / 32; ++e) p.part_o[row * DP + lane + 32 * e] = v[e];
                if (lane == 0) p.part_ml[row] = make_float2(top, l);
            }
        }
        fence_async_smem();  // before the next item's copies overwrite what was written and read here
        group_sync();
    }
}

// Joins the shares of each row, one warp a row.
template <typename T, int DP, bool Q4, bool CACHED>
__global__ void __launch_bounds__(128) join_step_kernel(const StepArgs p, int tile_rows) {
    const AttnArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    const unsigned at = blockIdx.x * 4 + (threadIdx.x >> 5), item = at / (unsigned)p.rows;
    const int r = (int)(at - item * p.rows);
    const unsigned hs = p.by_tiles.div(item), sq = a.by_Hkv.div(hs);
    const int r0 = (int)(item - hs * p.tiles) * tile_rows, rows = min(tile_rows, a.Nq * a.G - r0);
    const bool on = item < p.items && r < rows;
    TileKeys tk{};
    RowKeys k{0, 0, 0};
    if (on) {
        tk = tile_keys<CACHED>(a, sq, r0, rows);
        k = row_keys<CACHED>(a, tk, r0, r, rows);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the shares are written
    if (!on) return;
    const int64_t row0 = (int64_t)item * p.outer * p.rows + r;
    float top = -INFINITY, l = 0.f, v[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) v[e] = 0.f;
    for (int b = lane; b < p.outer; b += 32) top = fmaxf(top, p.part_ml[row0 + (int64_t)b * p.rows].x);
    top = warp_max(top);
#pragma unroll 8
    for (int b = 0; b < p.outer; ++b) {
        const int64_t row = row0 + (int64_t)b * p.rows;
        const float2 ml = p.part_ml[row];
        const float f = to_offset(ml.x, top);
        l += f * ml.y;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) v[e] += f * p.part_o[row * DP + lane + 32 * e];
    }
    finish_row<T, DP, Q4, CACHED>(a, tk, k, sq, (int)(hs - sq * a.Hkv), r0 + r, v, l);
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
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)p.items * p.outer, sm_count());
    kern<<<grid, Cfg::WARPS * 32, Cfg::TOTAL, st>>>(p);
    MBR_CUDA(cudaGetLastError());
    if (p.outer == 1) return;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ceil_div((int64_t)p.items * p.rows, 4));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    MBR_CUDA(cudaLaunchKernelEx(&cfg, join_step_kernel<T, DP, Q4, CACHED>, p, HALF ? 8 : 16));
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

StepPlan step_plan(int64_t seqs, int64_t tokens, int Hq, int Hkv, int D, bool q4, int64_t keys) {
    StepPlan pl{};
    const int64_t rows = tokens * (Hq / Hkv);
    pl.half = rows <= 8;
    pl.rows = (int)std::min<int64_t>(rows, 16);
    pl.tiles = ceil_div(rows, 16);
    pl.items = seqs * Hkv * pl.tiles;
    const int dp = D == 32 ? 32 : D == 64 ? 64 : 128, warps = step_warps(dp, q4);
    const int64_t copy = UNIT * (q4 ? 2 : 1);  // keys a warp fetches at a time
    // A warp's time is its rounds x (its keys + a start and a join worth some 100
    // keys).  One CTA an item joins inside; more CTAs cost a second kernel (some
    // 500 keys) and the reading of each share.  960 x 8 items over 4-bit caches with
    // 1, 2, 4 or 8 warps an item: 284, 314, 263, 263 us where this takes 4.
    double best = 1e300;
    auto consider = [&](int inner, int outer) {
        const double rounds = (double)ceil_div(pl.items * outer, (int64_t)148 * (warps / inner));
        const double cost = rounds * ((double)keys / inner / outer + 100.) + (outer > 1 ? 500. + 10. * outer : 0.);
        if (cost < best) best = cost, pl.inner = inner, pl.outer = outer;
    };
    for (int n = 1; n <= warps; n *= 2) consider(n, 1);
    for (int n = 2; n <= std::min<int64_t>(148, keys / copy / warps); ++n)
        if (pl.items * n <= 148 * 4) consider(warps, n);
    pl.bytes = pl.outer == 1 ? 0 : pl.items * pl.outer * pl.rows * (int64_t)(dp + 2) * 4;
    return pl;
}

void attend_step(const AttnArgs& a, int dtype, bool cached, bool q4, const StepPlan& pl, void* workspace,
                 cudaStream_t st) {
    MBR_CHECK(((uintptr_t)workspace & 15) == 0, "attention: workspace must be 16-byte aligned");
    MBR_CHECK(pl.items < (1ll << 27), "attention: too many row tiles");
    StepArgs p{};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.items = (unsigned)pl.items, p.tiles = (int)pl.tiles, p.rows = pl.rows, p.half = pl.half;
    p.outer = pl.outer;
    while ((1 << p.inner_log2) < pl.inner) ++p.inner_log2;
    p.by_tiles = FastDiv((unsigned)pl.tiles), p.by_outer = FastDiv((unsigned)pl.outer);
    const int dp = a.D == 32 ? 32 : a.D == 64 ? 64 : 128;
    p.part_o = (float*)workspace;
    p.part_ml = (float2*)(p.part_o + pl.items * pl.outer * pl.rows * dp);
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
    p.err = stream_error_word(st);
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
