// stream_cache.cu — writing tokens to the rolling key/value cache and reading
// them back, 16/32-bit rows or 4-bit codes with a step and an offset per 32
// channels.  Both move each byte once; memory (or, for a single frame, the
// launch: 2.1 us each) bounds the 16-bit forms, the arithmetic of the codes (80 % of
// the issue slots) those of 4 bits.  801 tokens of 60 sequences and 8 heads of 64
// into a cache of 504 slots and back, bf16: append 18.9 us (6.6 TB/s), read 27.1 us
// (5.9 TB/s); 4 bits 27.8 us (3.0 TB/s) and 22.3 us (5.2 TB/s).
#include <algorithm>
#include <type_traits>

#include "stream_cache.cuh"

namespace mbr {
namespace streamops {

void check_cache_fields(const mbr_kv_cache& c) {
    MBR_CHECK(c.seqs >= 0 && c.kv_heads >= 0 && c.sinks >= 0, "kv cache: negative size");
    MBR_CHECK(c.ring >= 1, "kv cache: ring must be at least 1");
    // a query's keys are counted in 32 bits, rounded up to whole copies
    MBR_CHECK((int64_t)c.sinks + c.ring <= (1 << 30), "kv cache: sinks and ring must not exceed 2^30 together");
    MBR_CHECK(c.dtype == DT_F32 || c.dtype == DT_F16 || c.dtype == DT_BF16, "kv cache: dtype must be fp32, fp16 or bf16");
    MBR_CHECK(c.bits == 0 || c.bits == 4, "kv cache: bits must be 0 or 4");
    MBR_CHECK(c.dim_head >= 8 && c.dim_head <= 128 && c.dim_head % 8 == 0,
              "kv cache: dim_head must be a multiple of 8 up to 128");
    MBR_CHECK(c.bits == 0 || (c.dtype != DT_F32 && c.dim_head % kGroup == 0),
              "kv cache: 4 bits need fp16 or bf16 and dim_head a multiple of 32");
    MBR_CHECK(c.seqs == 0 || c.kv_heads == 0 ||
                  c.seqs <= ((int64_t)1 << 40) / c.kv_heads / ((int64_t)c.sinks + c.ring),
              "kv cache: too large");
}

bool check_cache(const mbr_kv_cache& c) {
    check_cache_fields(c);
    const bool some = c.seqs > 0 && c.kv_heads > 0;
    MBR_CHECK(!some || (c.k && c.v), "kv cache: null buffer");
    MBR_CHECK((((uintptr_t)c.k | (uintptr_t)c.v) & 15) == 0, "kv cache: buffers must be 16-byte aligned");
    if (c.bits == 4) {
        MBR_CHECK(!some || (c.k_scale && c.v_scale), "kv cache: 4 bits need the steps and offsets");
        MBR_CHECK((((uintptr_t)c.k_scale | (uintptr_t)c.v_scale) & 15) == 0, "kv cache: buffers must be 16-byte aligned");
    }
    return c.bits == 4;
}

namespace {

// What x - m and the step are multiplied by before the one goes by the other's
// reciprocal: a power of two for a bf16 step below fp32's normal range, whose
// reciprocal would be infinite (2^-133 is the least).
template <typename T>
__device__ __forceinline__ float step_scale(float step) {
    return std::is_same_v<T, __nv_bfloat16> && step < 0x1p-126f ? 0x1p24f : 1.f;
}

struct RowArgs {
    mbr_kv_cache c;
    mbr_view k, v;
    const int32_t *pos, *count;
    int64_t tokens, rows;  // rows: seqs * tokens * kv_heads
    FastDiv by_heads, by_quads;  // vector form
};

// The row (sequence, token, head) of index r, its position and cache row; held:
// it is (append: will be) in the cache.
struct Row {
    int64_t s, t, slot_row;
    int h;
    bool held;
};
__device__ __forceinline__ Row row_of(const RowArgs& a, int64_t r) {
    Row w;
    const int64_t st = r / a.c.kv_heads;
    w.h = (int)(r - st * a.c.kv_heads);
    w.s = st / a.tokens;
    w.t = st - w.s * a.tokens;
    const int64_t n = a.count ? min((int64_t)max(a.count[w.s], 0), a.tokens) : a.tokens;
    const int64_t p0 = a.pos[w.s], p = p0 + w.t, last = p0 + n - 1;
    w.held = w.t < n && p >= 0 && p <= INT32_MAX && (p < a.c.sinks || p > last - a.c.ring);
    const int64_t slots = (int64_t)a.c.sinks + a.c.ring;
    w.slot_row = (w.s * a.c.kv_heads + w.h) * slots + (w.held ? slot_of((int)p, a.c.sinks, a.c.ring) : 0);
    return w;
}

template <typename T>
__device__ __forceinline__ const T* at(const mbr_view& v, const Row& w) {
    return (const T*)v.data + w.s * v.seq + w.t * v.token + w.h * v.head;
}

// One warp per (token, head): lane l holds channels l, l + 32, ...
template <typename T, bool Q4, bool READ>
__global__ void __launch_bounds__(256) cache_rows_kernel(const RowArgs a) {
    const int lane = threadIdx.x & 31, D = a.c.dim_head;
    const int64_t step = (int64_t)gridDim.x * 8;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows; r += step) {
        const Row w = row_of(a, r);
        if (!READ && !w.held) continue;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            T* x = const_cast<T*>(at<T>(kv ? a.v : a.k, w));
            void* data = kv ? a.c.v : a.c.k;
            T* scale = (T*)(kv ? a.c.v_scale : a.c.k_scale);
            for (int c = 0; c * 32 < D; ++c) {
                const int d = c * 32 + lane;
                if constexpr (!Q4) {
                    T* row = (T*)data + w.slot_row * D;
                    if (d < D) {
                        if (READ) x[d] = w.held ? row[d] : from_f32<T>(0.f);
                        else row[d] = x[d];
                    }
                } else {  // D % 32 == 0: one group
                    uint8_t* row = (uint8_t*)data + w.slot_row * (D / 2);
                    T* sm = scale + (w.slot_row * (D / kGroup) + c) * 2;
                    if (READ) {
                        const int code = (row[d >> 1] >> ((d & 1) * 4)) & 15;
                        x[d] = w.held ? code_value<T>(code, sm[0], sm[1]) : from_f32<T>(0.f);
                    } else {
                        const float v = to_f32<T>(x[d]);
                        float lo = v, hi = v;
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) {
                            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                        }
                        const bool ok = __all_sync(0xffffffffu, isfinite(v)) && isfinite(hi - lo);
                        const T sT = from_f32<T>(__fmul_rn(hi - lo, 1.f / 15.f));
                        const float s = to_f32<T>(sT);
                        const T mT = from_f32<T>(__fadd_rn(lo, 8.f * s));
                        const float up = step_scale<T>(s);
                        const float m = to_f32<T>(mT), inv = s > 0.f ? __frcp_rn(s * up) : 0.f;
                        const float q = rintf(__fmul_rn(__fadd_rn(v, -m) * up, inv)) + 8.f;
                        int code = (int)fminf(fmaxf(q, 0.f), 15.f);
                        const int other = __shfl_down_sync(0xffffffffu, code, 1);
                        if ((lane & 1) == 0) row[d >> 1] = (uint8_t)(code | (other << 4));
                        if (lane == 0) {
                            sm[0] = ok ? sT : from_f32<T>(NAN);
                            sm[1] = ok ? mT : from_f32<T>(NAN);
                        }
                    }
                }
            }
        }
    }
}

// Least and greatest of the 32 values that 4 lanes hold, 8 each in w; NaN where one is NaN.
template <typename T>
__device__ __forceinline__ float2 low_high(const uint32_t (&w)[4]) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const T2*>(&w[i]);
    const T2 lo = __hmin2_nan(__hmin2_nan(x[0], x[1]), __hmin2_nan(x[2], x[3]));
    const T2 hi = __hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3]));
    // (least, -greatest): one minimum for both from here on
    T2 m;
    m.x = __hmin_nan(lo.x, lo.y);
    m.y = __hneg(__hmax_nan(hi.x, hi.y));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&m), o);
        m = __hmin2_nan(m, *reinterpret_cast<const T2*>(&other));
    }
    return make_float2(to_f32<T>(m.x), -to_f32<T>(m.y));
}

// Vector form: 8 channels a lane (rows on 16-byte boundaries).  A lane group takes
// four neighbouring tokens of one head, whose cache rows lie next to each other:
// their place is worked out once, and all eight loads are in flight before the
// first is used.  A 4-bit group's minimum and maximum are two shuffle steps
// (4 lanes a group), in 16 bits.
template <typename T, bool Q4, bool READ>
__global__ void __launch_bounds__(256) cache_vec_kernel(const RowArgs a, int lanes_log2) {
    const int D = a.c.dim_head, lanes = 1 << lanes_log2, sub = threadIdx.x & (lanes - 1);
    // group: head, then four tokens, then sequence (threads past the end stay for the shuffles)
    const unsigned grp = (blockIdx.x * 256 + threadIdx.x) >> lanes_log2;
    const unsigned hq = a.by_heads.div(grp), sq = a.by_quads.div(hq);
    const int h = (int)(grp - hq * a.c.kv_heads), t0 = (int)(hq - sq * a.by_quads.d) * 4;
    const bool real = sq < a.c.seqs;
    const int64_t s = real ? sq : 0;
    const int d0 = sub * 8;
    const bool in = real && d0 < D;
    const int tokens = (int)a.tokens;
    const int cnt = a.count ? min(max(__ldg(a.count + s), 0), tokens) : tokens;
    const int64_t p0 = __ldg(a.pos + s), last = p0 + cnt - 1;
    const int64_t base = (s * a.c.kv_heads + h) * ((int64_t)a.c.sinks + a.c.ring);
    int64_t row[4];  // cache row of each token, -1: not in the cache
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t p = p0 + t0 + u;
        const bool held = in && t0 + u < cnt && p >= 0 && p <= INT32_MAX && (p < a.c.sinks || p > last - a.c.ring);
        row[u] = -1;
        if (held) {
            // the token after a held one follows it in the ring, but for the ring's end
            if (u > 0 && row[u - 1] >= 0 && p > a.c.sinks)
                row[u] = row[u - 1] + 1 < base + a.c.sinks + a.c.ring ? row[u - 1] + 1 : base + a.c.sinks;
            else
                row[u] = base + slot_of((int)p, a.c.sinks, a.c.ring);
        }
    }
    // none of the warp's tokens stays in the cache
    if (!READ && !__any_sync(0xffffffffu, row[0] >= 0 || row[1] >= 0 || row[2] >= 0 || row[3] >= 0)) return;
    constexpr int W = sizeof(T) / 2;  // 16-byte pieces of 8 elements
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const mbr_view& view = kv ? a.v : a.k;
        T* const x0 = (T*)view.data + s * view.seq + t0 * view.token + h * view.head + d0;
        uint8_t* const data = (uint8_t*)(kv ? a.c.v : a.c.k);
        T* const scale = (T*)(kv ? a.c.v_scale : a.c.k_scale);
        uint4 raw[4][W];
        if constexpr (READ && Q4) {
            uint32_t codes[4], sm[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                codes[u] = sm[u] = 0;
                if (row[u] >= 0) {
                    codes[u] = *reinterpret_cast<const uint32_t*>(data + row[u] * (D / 2) + sub * 4);
                    sm[u] = *reinterpret_cast<const uint32_t*>(scale + (row[u] * (D / kGroup) + sub / 4) * 2);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {  // a token that is not held has step and offset 0: zeros
                using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
                const T* f = reinterpret_cast<const T*>(&sm[u]);
                T2* e = reinterpret_cast<T2*>(raw[u]);
                const T2 st = {f[0], f[0]}, m = {f[1], f[1]};
                // codes as the last bits of 1024 (fp16) or 128 (bf16) + code: no conversion
                constexpr uint32_t base = std::is_same_v<T, __half> ? 0x64006400u : 0x43004300u,
                                   less = std::is_same_v<T, __half> ? 0xe408e408u : 0xc308c308u;  // -1032, -136
                const uint32_t even = codes[u] & 0x0f0f0f0fu, odd = (codes[u] >> 4) & 0x0f0f0f0fu;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t x = (__byte_perm(even, odd, 0x0400 + 0x0101 * c) & 0x00ff00ffu) | base;
                    const T2 q = __hadd2(*reinterpret_cast<const T2*>(&x), *reinterpret_cast<const T2*>(&less));
                    e[c] = __hfma2(st, q, m);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint4* src = reinterpret_cast<const uint4*>(READ ? (const T*)data + row[u] * D + d0 : x0 + u * view.token);
#pragma unroll
                for (int c = 0; c < W; ++c) raw[u][c] = row[u] >= 0 ? src[c] : make_uint4(0u, 0u, 0u, 0u);
            }
        }
        if constexpr (!READ && Q4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t w[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
                const float2 range = low_high<T>(w);
                const float lo = range.x, hi = range.y;
                const bool ok = isfinite(hi - lo);  // a value that is not finite makes one of them so
                const T sT = from_f32<T>(__fmul_rn(hi - lo, 1.f / 15.f));
                const float st = to_f32<T>(sT);
                const T mT = from_f32<T>(__fadd_rn(lo, 8.f * st));
                const float up = step_scale<T>(st);
                const float m = to_f32<T>(mT), inv = st > 0.f ? __frcp_rn(st * up) : 0.f;
                // rint((v - m) / st) + 8 within 0..15: adding 1.5 2^23 rounds to an integer; four codes are put
                // together as one (their sum is below 2^16) in floating point
                float part[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float q[4];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const T* e = reinterpret_cast<const T*>(w + 2 * half + c);
                        const float2 d = __ffma2_rn(make_float2(to_f32<T>(e[0]), to_f32<T>(e[1])), make_float2(up, up),
                                                    make_float2(-m * up, -m * up));
                        float2 x = __fmul2_rn(d, make_float2(inv, inv));
                        x.x = fminf(fmaxf(x.x, -8.f), 7.f), x.y = fminf(fmaxf(x.y, -8.f), 7.f);
                        x = __fadd2_rn(x, make_float2(12582920.f, 12582920.f));
                        x = __fadd2_rn(x, make_float2(-12582912.f, -12582912.f));
                        q[2 * c] = x.x, q[2 * c + 1] = x.y;
                    }
                    part[half] = fmaf(4096.f, q[3], fmaf(256.f, q[2], fmaf(16.f, q[1], q[0]))) + 8388608.f;
                }
                const uint32_t codes = __byte_perm(__float_as_uint(part[0]), __float_as_uint(part[1]), 0x5410);
                if (row[u] >= 0) {
                    *reinterpret_cast<uint32_t*>(data + row[u] * (D / 2) + sub * 4) = codes;
                    if ((sub & 3) == 0) {
                        union {
                            T f[2];
                            uint32_t w;
                        } sm;
                        sm.f[0] = ok ? sT : from_f32<T>(NAN);
                        sm.f[1] = ok ? mT : from_f32<T>(NAN);
                        *reinterpret_cast<uint32_t*>(scale + (row[u] * (D / kGroup) + sub / 4) * 2) = sm.w;
                    }
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (READ ? !(in && t0 + u < tokens) : row[u] < 0) continue;
                uint4* dst = reinterpret_cast<uint4*>(READ ? x0 + u * view.token : (T*)data + row[u] * D + d0);
#pragma unroll
                for (int c = 0; c < W; ++c) dst[c] = raw[u][c];
            }
        }
    }
}

template <bool READ>
void run(const mbr_kv_cache& c, const mbr_view& k, const mbr_view& v, const int32_t* pos, const int32_t* count,
         int64_t tokens, cudaStream_t st) {
    const bool q4 = check_cache(c);
    MBR_CHECK(tokens >= 0, "kv cache: negative token count");
    if (c.seqs == 0 || c.kv_heads == 0 || tokens == 0) return;
    MBR_CHECK(k.data && v.data && pos, "kv cache: null buffer");
    MBR_CHECK(tokens < (1 << 30) && c.seqs <= ((int64_t)1 << 50) / tokens / c.kv_heads, "kv cache: too many rows");
    RowArgs a{c, k, v, pos, count, tokens, c.seqs * tokens * c.kv_heads, {}, {}};
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(a.rows, 8), 148 * 64);
    const int es = (int)dtype_bytes(c.dtype);
    int lanes_log2 = 0;
    while ((8 << lanes_log2) < c.dim_head) ++lanes_log2;
    const int64_t quads = (tokens + 3) >> 2, threads = (c.seqs * quads * c.kv_heads) << lanes_log2;
    if (rows_aligned16(k, es) && rows_aligned16(v, es) && threads < (1ll << 31) - 256) {
        a.by_heads = FastDiv((unsigned)c.kv_heads), a.by_quads = FastDiv((unsigned)quads);
        const int64_t blocks = ceil_div(threads, 256);
        MBR_DISPATCH_DTYPE(c.dtype, T, {
            if constexpr (std::is_same_v<T, float>) {
                cache_vec_kernel<T, false, READ><<<(unsigned)blocks, 256, 0, st>>>(a, lanes_log2);
            } else {
                if (q4) cache_vec_kernel<T, true, READ><<<(unsigned)blocks, 256, 0, st>>>(a, lanes_log2);
                else cache_vec_kernel<T, false, READ><<<(unsigned)blocks, 256, 0, st>>>(a, lanes_log2);
            }
        });
        MBR_CUDA(cudaGetLastError());
        return;
    }
    MBR_DISPATCH_DTYPE(c.dtype, T, {
        if constexpr (std::is_same_v<T, float>) {
            cache_rows_kernel<T, false, READ><<<grid, 256, 0, st>>>(a);
        } else {
            if (q4) cache_rows_kernel<T, true, READ><<<grid, 256, 0, st>>>(a);
            else cache_rows_kernel<T, false, READ><<<grid, 256, 0, st>>>(a);
        }
    });
    MBR_CUDA(cudaGetLastError());
}

}  // namespace

void cache_append(const mbr_kv_cache& c, const mbr_view& k, const mbr_view& v, const int32_t* pos,
                  const int32_t* count, int64_t tokens, cudaStream_t st) {
    run<false>(c, k, v, pos, count, tokens, st);
}
void cache_read(const mbr_kv_cache& c, const int32_t* pos, const int32_t* count, int64_t tokens, const mbr_view& k,
                const mbr_view& v, cudaStream_t st) {
    run<true>(c, k, v, pos, count, tokens, st);
}

}  // namespace streamops
}  // namespace mbr
