// A cache of keys and values in 4 bits, in pages of 64 positions (see include/sal_decode_ops.h for the format): rows are rotated,
// quantised and stored, read back, attended to, and pages copied.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <new>
#include <type_traits>

#include "sal_decode_ops.h"
#include "sal_launch.h"
#include "sal_lutgemm.h"

namespace {

constexpr int PAGE = 64;          // positions of a page
constexpr int GROUP = 64;         // numbers that share a scale
constexpr int POS_LIMIT = 1 << 30;
constexpr int MAX_PAGES = 1 << 20;   // of a sequence

__device__ __forceinline__ void pdl_prologue() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Bytes of the parts of a record (one page and kv head): codes of K, codes of V, parameters of K, parameters of V.
template <int HD>
struct Record {
    static constexpr int G = HD / GROUP;
    static constexpr int ROW = HD / 2;               // bytes of codes of a position
    static constexpr int CODES = PAGE * ROW;
    static constexpr int PARAMS = PAGE * G * 4;      // (scale, low) as two halves per position and group
    static constexpr int BYTES = 2 * (CODES + PARAMS);
    // Where group g of a position lies in its row, in blocks of 32 bytes.  The order depends on the position so that the lanes
    // of a matrix fragment, which read the same group of several positions at once, find them in different banks.
    __host__ __device__ static constexpr int place(int g, int p) {
        const int f = (p & 3) ^ ((p >> 1) & 2);
        return G == 4 ? g ^ f : G == 2 ? g ^ (f >> 1) : 0;
    }
    static constexpr int FOUR_ON = G / 2;            // place(g, p + 4) = place(g ^ FOUR_ON, p), place(g, p + 8) = place(g, p)
};

// a * c - b * s to the nearest 32-bit number of the exact sum (products split into value and error), then to 16 bits: the same
// bits as 64-bit arithmetic gives, at a fraction of its price.
__device__ __noinline__ __half turned_exactly(float a, float c, float b, float s) {
    const float p = __fmul_rn(a, c), pe = __fmaf_rn(a, c, -p);
    const float q = __fmul_rn(b, s), qe = __fmaf_rn(b, s, -q);
    const float d = __fsub_rn(p, q), bb = __fsub_rn(d, p);
    const float de = __fsub_rn(__fsub_rn(p, __fsub_rn(d, bb)), __fadd_rn(q, bb));
    const float r = __fadd_rn(d, __fadd_rn(de, __fsub_rn(pe, qe)));
    return __float2half_rn(isfinite(r) ? r : d);   // an infinite product has no error term
}
// The sum with the second product's error taken off is within two units of the exact one in its last place.  That decides the 16-bit number unless
// it lies so near to the middle between two of them (`unsure`), is subnormal there, or overflows: one number in a thousand.
__device__ __forceinline__ float nearly_turned(float a, float c, float b, float s, bool &unsure) {
    const float q = __fmul_rn(b, s);
    const float r = __fsub_rn(__fmaf_rn(a, c, -q), __fmaf_rn(b, s, -q));
    const uint32_t u = __float_as_uint(r);
    unsure = (u - 0x0ffcu & 0x1fffu) <= 8u || (u & 0x7fffffffu) - 0x38800000u >= 0x47700000u - 0x38800000u;
    return r;
}

// The position of row i of a sequence, clamped so that the sum cannot overflow; the caller compares it with the positions that exist.
__device__ __forceinline__ int row_position(int64_t first, int i) {
    const int64_t p = first > POS_LIMIT ? POS_LIMIT : first < -POS_LIMIT ? -POS_LIMIT : first;
    return (int)p + i;
}
__device__ __forceinline__ int rows_of(const int32_t *rows, int b, int m) {
    if (!rows) return m;
    const int r = rows[b];
    return r < 0 ? 0 : r > m ? m : r;
}

struct CacheArgs {
    uint8_t *pool;
    const int32_t *table;   // [batch][max_pages]
    int kv_heads, max_pages, pages;
};
// The record of a position, or null where its page does not exist.
template <int HD>
__device__ __forceinline__ uint8_t *record_of(const CacheArgs &c, int b, int p, int kvh) {
    if (p < 0 || p >= c.max_pages * PAGE) return nullptr;
    const int page = c.table[(size_t)b * c.max_pages + p / PAGE];
    if (page < 0 || page >= c.pages) return nullptr;
    return c.pool + ((size_t)page * c.kv_heads + kvh) * Record<HD>::BYTES;
}

// Writing and reading: a thread has eight neighbouring numbers of a head, 16 bytes of 16-bit numbers or 4 bytes of codes, HD / 8 threads a head.  The
// other numbers of its rotary pairs are HD / 16 threads on, a group is eight threads.  Writing takes 27 us for 1537 rows of 64 + 8 heads of 128, 57 MB, a
// third of the copy rate: 17 million warp instructions (conversions, the checks of the rounding, shuffles) in 62 % of the issue slots, the rest
// latency of loads and of dependent steps at 23 warps an SM.  Reading them back takes 5.7 us; one row of 16 sequences 3.1 and 1.9 us, a launch's
// latency.  Blocks go over a sequence's rows with a stride, threads of a block over the heads of a row.
constexpr int ROW_THREADS = 256;

template <int HD>
__global__ void __launch_bounds__(ROW_THREADS, 4) rope_kv4_write_kernel(const __half *q, const __half *k, const __half *v, const float *cos_t, const float *sin_t,
                                                                     const int64_t *pos, const int32_t *rows, CacheArgs c, __half *q_out, int m, int heads,
                                                                     int max_len) {
    using R = Record<HD>;
    constexpr int T = HD / 8;
    pdl_prologue();
    const int unit = blockIdx.y * (ROW_THREADS / T) + threadIdx.x / T, t = threadIdx.x % T, d = 8 * t;
    const bool is_q = unit < heads, is_v = unit >= heads + c.kv_heads, real = unit < heads + 2 * c.kv_heads;
    const int h = is_q ? unit : is_v ? unit - heads - c.kv_heads : unit - heads;
    const int stride = (is_q ? heads : c.kv_heads) * HD;
    const __half *src = (is_q ? q : is_v ? v : k) + (size_t)h * HD + d;
    const bool any_turned = __any_sync(0xffffffffu, !is_v);      // of the warp
    // this sequence's rows that are there and have a position: first .. last - 1 of its m
    const int b = blockIdx.z, start = row_position(pos[b], 0);
    const int last = real ? min(rows_of(rows, b, m), min(max_len, c.max_pages * PAGE) - start) : 0;      // start may be negative, or far behind
    const size_t base = (size_t)b * m;
    // the next row's numbers are asked for in front of this row's work
    uint4 next = make_uint4(0, 0, 0, 0);
    auto there = [&](int i) { return i < last && start + i >= 0; };
    auto ask = [&](int i) {
        if (there(i)) next = *reinterpret_cast<const uint4 *>(src + (base + i) * stride);
    };
    ask(blockIdx.x);
    for (int i = blockIdx.x; i < m; i += gridDim.x) {
        const bool on = there(i);
        const int p = start + i;
        const size_t row = base + i;
        uint4 x = next;
        ask(i + gridDim.x);
        uint8_t *record = nullptr;
        if (on && !is_q) record = record_of<HD>(c, b, p, h);
        __half2 *xh = reinterpret_cast<__half2 *>(&x);
        if (any_turned) {
            const uint32_t flip = d < HD / 2 ? 0u : 0x80008000u;      // b * c + a * s = b * c - (-a) * s
            uint4 y;
            y.x = __shfl_xor_sync(0xffffffffu, x.x, T / 2) ^ flip, y.y = __shfl_xor_sync(0xffffffffu, x.y, T / 2) ^ flip;
            y.z = __shfl_xor_sync(0xffffffffu, x.z, T / 2) ^ flip, y.w = __shfl_xor_sync(0xffffffffu, x.w, T / 2) ^ flip;
            if (on && !is_v) {
                const float4 *cs = reinterpret_cast<const float4 *>(cos_t + (size_t)p * (HD / 2) + d % (HD / 2));
                const float4 *sn = reinterpret_cast<const float4 *>(sin_t + (size_t)p * (HD / 2) + d % (HD / 2));
                const float4 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
                const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                const __half2 *yh = reinterpret_cast<const __half2 *>(&y);
                uint4 z;
                __half2 *zh = reinterpret_cast<__half2 *>(&z);
                unsigned unsure = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 u = __half22float2(xh[e]), w = __half22float2(yh[e]);
                    bool f0, f1;
                    zh[e] = __floats2half2_rn(nearly_turned(u.x, cc[2 * e], w.x, ss[2 * e], f0), nearly_turned(u.y, cc[2 * e + 1], w.y, ss[2 * e + 1], f1));
                    unsure |= (f0 ? 1u << (2 * e) : 0u) | (f1 ? 2u << (2 * e) : 0u);
                }
                if (unsure) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = __half22float2(xh[e]), w = __half22float2(yh[e]);
                        if (unsure >> (2 * e) & 1u) zh[e] = __half2(turned_exactly(u.x, cc[2 * e], w.x, ss[2 * e]), zh[e].y);
                        if (unsure >> (2 * e) & 2u) zh[e] = __half2(zh[e].x, turned_exactly(u.y, cc[2 * e + 1], w.y, ss[2 * e + 1]));
                    }
                }
                x = z;
            }
        }
        if (on && is_q) *reinterpret_cast<uint4 *>(q_out + row * stride + (size_t)h * HD + d) = x;
        if (!__any_sync(0xffffffffu, record != nullptr)) continue;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 u = __half22float2(xh[e]);
            f[2 * e] = u.x, f[2 * e + 1] = u.y;
        }
        float lo = f[0], hi = f[0];
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) lo = fminf(lo, f[e]), hi = fmaxf(hi, f[e]), odd |= !(fabsf(f[e]) <= 65504.f);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const bool bad = __ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 24) & 0xffu;
        const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
        const float s = __half2float(scale);
        const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
        uint32_t codes = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) codes |= (uint32_t)fminf(rintf(__fmul_rn(__fsub_rn(f[e], lo), inv)), 15.f) << (4 * e);
        if (record) {
            const int at = p % PAGE, g = t / 8;
            *reinterpret_cast<uint32_t *>(record + (is_v ? R::CODES : 0) + at * R::ROW + R::place(g, at) * 32 + 4 * (t % 8)) = bad ? 0u : codes;
            if (t % 8 == 0)
                reinterpret_cast<__half2 *>(record + 2 * R::CODES + (is_v ? R::PARAMS : 0))[at * R::G + g] =
                    bad ? __half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff)) : __half2(scale, __float2half_rn(lo));
        }
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(ROW_THREADS) read_kv4_kernel(CacheArgs c, const int64_t *pos, T *k_out, T *v_out, int m) {
    using R = Record<HD>;
    constexpr int N = HD / 8;
    pdl_prologue();
    const int unit = blockIdx.y * (ROW_THREADS / N) + threadIdx.x / N, t = threadIdx.x % N;
    if (unit >= 2 * c.kv_heads) return;
    const bool is_v = unit >= c.kv_heads;
    const int h = is_v ? unit - c.kv_heads : unit, g = t / 8;
    T *dst = (is_v ? v_out : k_out) + (size_t)h * HD + 8 * t;
    const int b = blockIdx.z, start = row_position(pos[b], 0);
    for (int i = blockIdx.x; i < m; i += gridDim.x) {
        const int p = start + i, at = p & (PAGE - 1);
        const uint8_t *record = record_of<HD>(c, b, p, h);
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (record) {
            const uint32_t codes = *reinterpret_cast<const uint32_t *>(record + (is_v ? R::CODES : 0) + at * R::ROW + R::place(g, at) * 32 + 4 * (t % 8));
            const float2 sl = __half22float2(reinterpret_cast<const __half2 *>(record + 2 * R::CODES + (is_v ? R::PARAMS : 0))[at * R::G + g]);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = fmaf(sl.x, (float)(codes >> (4 * e) & 15u), sl.y);
        }
        T *to = dst + ((size_t)b * m + i) * c.kv_heads * HD;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(to)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4 *>(to)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            uint4 o;
            __half2 *oh = reinterpret_cast<__half2 *>(&o);
#pragma unroll
            for (int e = 0; e < 4; ++e) oh[e] = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
            *reinterpret_cast<uint4 *>(to) = o;
        }
    }
}

// ---- attention on the tensor cores -----------------------------------------------------------------------------------------------
//
// A score is scale * sum_g (s_g * D_g + low_g * Q_g) with D_g = sum over the group of q * code and Q_g = sum of q; an output is
// E_g * A_g + sum_t p_t * (low_t + 8 s_t) with A_g = sum over positions of (p * s_g / E_g) * (code - 8).  The codes are 16-bit floats without any error, so D_g and A_g are matrix products of 16-bit operands (m16n8k16, 32-bit sums) in which only the
// weight p * s is rounded; it goes in as the sum of two 16-bit numbers.  E_g, a power of two not below the scales at hand, keeps the weights in
// their range.  Neither keys nor values are ever formed.
//
// Matrix fragments hold keys (or, for the second product, dimensions) as rows and query columns as columns: a lane's part of a row are
// 16 neighbouring codes of one group, fetched with one 8-byte load of shared memory, two codes per logic operation and one 16-bit fused
// multiply-add or addition.  The weights pass from the first product's result to the second's operand by an 8x8 transpose in registers.
//
// The work of a launch is a list of (sequence and column tile, kv head, page), dealt to the thread blocks in equal contiguous runs by the blocks
// themselves, from the positions on the device: texts of any lengths keep all SMs equally busy, and a captured launch follows the texts.  A
// page of a head is one contiguous record, so its fetch is one bulk copy into a ring of shared memory.  Blocks that share an item leave
// their part (maximum, sum, unnormalised output) in scratch; the last one to arrive adds them up in the order of the positions.
//
// Bound by the latency of dependent steps at 12 warps an SM, neither by bytes nor by issue (35 % of HBM, 52 % of the issue slots; the 390 instructions a
// warp for 16 positions would take half the time at full issue): 54 us for 159 MB of records (16 sequences of 300 to 4000 positions, 32 heads
// of 128; 2.9 TB/s), 97 us for 294 MB (three of 70 to 100 thousand, 64 query and 8 kv heads).

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait: false after about a second.
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity) {
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t - t0 > 1000000000ull) return false;
    }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || mbar_wait_slow(bar, parity); }
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t selector) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(selector));
    return d;
}
template <int G>
__device__ __forceinline__ void load_params(uint32_t (&p)[G], const uint8_t *a) {
    if constexpr (G == 1) {
        p[0] = *reinterpret_cast<const uint32_t *>(a);
    } else if constexpr (G == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(a);
        p[0] = v.x, p[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(a);
        p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
    }
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two codes of a word, in bits 4..7 and 20..23 (mid) or 0..3 and 16..19 (low), as two 16-bit floats of code * 2**-20.  The middle ones are that as
// they stand: subnormal floats, exact, and exact in the products.  The low ones go over 1024 + code: as they stand (code * 2**-24) they would
// cost the tensor core's sums four bits more, since it aligns a subnormal's product by its exponent and not by its first bit.
__device__ __forceinline__ uint32_t codes_mid(uint32_t x) { return x & 0x00f000f0u; }
__device__ __forceinline__ uint32_t codes_low(uint32_t x) {
    uint32_t h;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(h) : "r"(x));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(h) : "r"(0x00100010u), "r"(0x94009400u));   // * 2**-20 - 2**-10
    return h;
}
constexpr float UNIT = 1048576.f;
// The same less 8.  Sums over the positions of a long text are made of these: an output is the mean of many values and small beside each, so the
// sums should be no larger than it either (with codes from 0 on, 100 thousand positions lost two digits to the tensor core's rounding).
__device__ __forceinline__ uint32_t codes_mid_8(uint32_t x) {
    uint32_t h = x & 0x00f000f0u;
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(h) : "r"(0x80808080u));      // - 2**-17
    return h;
}
__device__ __forceinline__ uint32_t codes_low_8(uint32_t x) {
    uint32_t h;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(h) : "r"(x));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(h) : "r"(0x00100010u), "r"(0x94089408u));   // * 2**-20 - 2**-10 - 2**-17
    return h;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t h) { return *reinterpret_cast<__half2 *>(&h); }
__device__ __forceinline__ float2 as_float2(uint32_t h) { return __half22float2(*reinterpret_cast<__half2 *>(&h)); }

// Scratch: status word, a counter of arrivals per item that can be shared, then two parts per thread block.  The counters have a place of their own
// whatever the call's size: they have to be zero between calls, and the parts of a call of another size must not lie there.
constexpr int WS_HEADER = 256;
constexpr int MAX_KV_HEADS = 256;
constexpr int CHUNK = 128;             // units of a block's run that are looked up at once
constexpr int MAX_LIST = 256;                // (sequence, column tile) pairs whose work is dealt out; with more, a block takes an item
constexpr int SET_ASIDE = 16;         // pages of a warp
constexpr size_t WS_COUNTERS = (size_t)MAX_LIST * MAX_KV_HEADS * 4;
constexpr float MOVE_AT = 256.f;      // weights stay below 2**8 ..
constexpr float W_ONE = 64.f;         // .. and, times this, inside 16 bits; the second parts' last bit is then 2**-30 of a weight of 1

struct AttnArgs {
    const __half *q;
    CacheArgs c;
    const int64_t *pos;
    const int32_t *rows;
    __half *out;
    int *status;
    unsigned *counters;
    float *parts;
    int batch, m, heads, rep;
    int col_tiles;      // column tiles of a sequence
    int whole;          // a block takes an item
    int splits;         // of an item's pages, at most (many columns)
    float scale_log2;   // scale * log2(e) * UNIT
};

// NT column tiles of 8 per warp, WK warps that share a page's keys, PG pages that are worked on side by side, WC warps side by side in
// columns.  DUP: at most four columns; the other four of the tile are the same queries again and carry the second parts of the weights.
template <int HD, int NT, bool DUP, int WK, int PG, int WC>
struct AttnShape {
    static constexpr int COLS = DUP ? 4 : 8 * NT * WC;
    static constexpr int WARPS = WK * PG * WC;
    static constexpr int THREADS = WARPS * 32;
    static constexpr int PARTS = WK * PG;                              // warps that share a column
    static constexpr int REC = Record<HD>::BYTES;
    static constexpr int PART = COLS * (HD + 2);                       // floats of a part: outputs, maxima, sums
    static constexpr int SUMS = NT * (HD / 16) * 4;                    // a lane's running sums
    static constexpr int SLOT = PARTS > 1 && PART > SUMS * 32 ? PART : SUMS * 32;      // floats of a warp's own memory: its sums, at last its part
    static constexpr int MERGE = WARPS * SLOT * 4;
    static constexpr bool QUERIES = WC == 1;                           // an item's queries travel with its first page
    static constexpr int STAGE = REC + (QUERIES ? COLS * HD * 2 : 0);
    // What an item costs by itself (its first page's wait, the sum over the warps, the output or the part) in pages: 2.8 us against 1.2 us a page
    // with one column and heads of 128.  Counted as 1, 2, 3, 4 pages: 63, 55, 54, 54 us for 16 sequences of 300 to 4000 positions with 32 heads; as
    // 1 and 3 with 32 columns and heads of 256: 111 and 94 (four sequences, 33 rows behind 1000 to 5000 positions), 154 and 158 (512 rows of one).
    static constexpr int ITEM_UNITS = 3;
    static constexpr int MIN_UNITS = ITEM_UNITS + 2;
    static constexpr int STAGES = 4;      // a power of two; so many pages on lie within 32 units, ITEM_UNITS at most being in front of each
    static constexpr int SMEM = STAGES * STAGE + MERGE + 2 * CHUNK * 8 + MAX_LIST * 4 + 16;
    static constexpr int MIN_BLOCKS = HD < 256 && NT == 1 ? 3 : 2;
};

struct Item {
    int b, ct, h;       // sequence, column tile, kv head
    int pages;          // pages that some column sees
    int last;           // last position that some column sees
    int rows;           // rows of the sequence
    int first;          // position of its first row
};

// Rows of sequence b, and the last position that a column of tile ct sees (-1: none); false if the tile has no row.
template <int COLS>
__device__ __forceinline__ bool item_of(const AttnArgs &a, int b, int ct, Item &it) {
    it.b = b, it.ct = ct, it.rows = rows_of(a.rows, b, a.m);
    const int i0 = ct * COLS / a.rep;
    if (i0 >= it.rows) return false;
    const int i1 = min((ct * COLS + COLS - 1) / a.rep, it.rows - 1);
    it.first = row_position(a.pos[b], 0);
    it.last = min(it.first + i1, a.c.max_pages * PAGE - 1);
    it.pages = it.last < 0 ? 1 : it.last / PAGE + 1;
    return true;
}

__device__ __forceinline__ void store_output(__half *dst, float4 o, float total) {
    const float inv = 1.f / total;
    if (total == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);      // no position: zeros
    else o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(as_u32(__floats2half2_rn(o.x, o.y)), as_u32(__floats2half2_rn(o.z, o.w)));
}

template <int HD, int NT, bool DUP, int WK, int PG, int WC>
__global__ void __launch_bounds__(AttnShape<HD, NT, DUP, WK, PG, WC>::THREADS, AttnShape<HD, NT, DUP, WK, PG, WC>::MIN_BLOCKS) attention_tiles_kernel(AttnArgs a) {
    using S = AttnShape<HD, NT, DUP, WK, PG, WC>;
    using R = Record<HD>;
    constexpr int G = R::G, COLS = S::COLS, ITEM_UNITS = S::ITEM_UNITS;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    float *merge = reinterpret_cast<float *>(smem + S::STAGES * S::STAGE);      // a slot for every warp
    int2 *sched = reinterpret_cast<int2 *>(smem + S::STAGES * S::STAGE + S::MERGE);      // of two chunks of units: (record or none, item if its first page)
    int *list = reinterpret_cast<int *>(sched + 2 * CHUNK);                              // units in front of a pair, per kv head
    __shared__ uint64_t bars[S::STAGES];
    __shared__ unsigned s_done[S::STAGES];     // warps that are through with a stage, counted on
    __shared__ int s_scan[33];
    __shared__ int s_flag;
    __shared__ long long s_out[S::COLS];       // where a column's output lies
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t full = smem_u32(bars);
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) mbar_init(full + 8 * i, 1), s_done[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_prologue();
    const int kvh = a.c.kv_heads, pairs = a.batch * a.col_tiles;
    Item it = {};
    // The list counts an item as ITEM_UNITS and its pages.  This block's run: `left` units from unit `at` of the item on.
    int at, pair;
    long long left, per = 0;
    if (a.whole) {
        pair = blockIdx.x / kvh;
        it.h = blockIdx.x % kvh;
        if (!item_of<COLS>(a, pair / a.col_tiles, pair % a.col_tiles, it)) return;
        at = 0, left = it.pages + ITEM_UNITS;
    } else {
        int total = 0;         // units of all pairs, and in front of each
        for (int i0 = 0; i0 < pairs; i0 += S::THREADS) {
            const int i = i0 + tid;
            Item x = {};
            const int n = i < pairs && item_of<COLS>(a, i / a.col_tiles, i % a.col_tiles, x) ? x.pages + ITEM_UNITS : 0;
            int run = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += t;
            }
            if (lane == 31) s_scan[warp] = run;
            __syncthreads();
            int front = total;
            for (int w = 0; w < S::WARPS; ++w) {
                if (w < warp) front += s_scan[w];
                total += s_scan[w];
            }
            if (i < pairs) list[i] = front + run - n;
            __syncthreads();
        }
        if (tid == 0) list[pairs] = total;
        __syncthreads();
        const long long all = (long long)total * kvh;
        per = (all + gridDim.x - 1) / gridDim.x;
        if (per < S::MIN_UNITS) per = S::MIN_UNITS;
        const long long begin = per * blockIdx.x;
        if (begin >= all) return;
        left = begin + per < all ? per : all - begin;
        // the last pair whose units (of all heads) begin at or in front of `begin`: one that has some
        int lo = 0, hi = pairs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((long long)list[mid] * kvh <= begin) lo = mid;
            else hi = mid;
        }
        pair = lo;
        const int in_pair = (int)(begin - (long long)list[pair] * kvh);
        item_of<COLS>(a, pair / a.col_tiles, pair % a.col_tiles, it);
        it.h = in_pair / (it.pages + ITEM_UNITS);
        at = in_pair % (it.pages + ITEM_UNITS);
    }
    const int cols = a.m * a.rep;

    // ---- what the run fetches: unit by unit, a chunk at a time, one unit per thread ----------------------------------------------------
    const long long units = left, begin = per * blockIdx.x;
    constexpr int NOTHING = -2, NO_PAGE = -1;       // an item's own units, or behind the run; a page that does not exist
    const int pair0 = pair, h0 = it.h, at0 = at;
    auto look_up = [&](int chunk) {
        static_assert(CHUNK == S::THREADS, "a thread looks up one unit");
        const long long u = (long long)chunk * CHUNK + tid;
        int2 e = make_int2(NOTHING, -1);
        if (u < units) {
            int p = pair0, h = h0, t = at0 + (int)u;      // pair, kv head, unit of the item
            if (!a.whole) {
                int lo = pair0, hi = pairs;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if ((long long)list[mid] * kvh <= begin + u) lo = mid;
                    else hi = mid;
                }
                p = lo;
                const int in_pair = (int)(begin + u - (long long)list[p] * kvh), n = list[p + 1] - list[p];
                h = in_pair / n, t = in_pair % n;
            }
            if (t >= ITEM_UNITS) {
                const int page = a.c.table[(size_t)(p / a.col_tiles) * a.c.max_pages + t - ITEM_UNITS];
                e.x = page >= 0 && page < a.c.pages ? page * kvh + h : NO_PAGE;
                if (t == ITEM_UNITS || u == 0) e.y = p * kvh + h;
            }
        }
        sched[(chunk & 1) * CHUNK + tid] = e;
    };
    // one lane asks for a page, and for the item's queries if it is the first
    auto fetch = [&](int2 e, int st) {
        const uint32_t dst = smem_u32(ring + st * S::STAGE), bar = full + 8 * st;
        if (S::QUERIES && e.y >= 0) {
            const int p = e.y / kvh, h = e.y % kvh, b = p / a.col_tiles, j0 = p % a.col_tiles * COLS;
            const int j1 = min(min(j0 + COLS, cols), rows_of(a.rows, b, a.m) * a.rep);      // columns that are there
            mbar_expect_tx(bar, (e.x >= 0 ? S::REC : 0) + (j1 - j0) * HD * 2);
            for (int j = j0; j < j1;) {      // heads of a row that share this kv head lie side by side
                const int i = j / a.rep, upto = min((i + 1) * a.rep, j1);
                bulk_copy(dst + S::REC + (j - j0) * HD * 2, a.q + (((size_t)b * a.m + i) * a.heads + h * a.rep + (j - i * a.rep)) * HD, (upto - j) * HD * 2, bar);
                j = upto;
            }
        } else {
            mbar_expect_tx(bar, e.x >= 0 ? S::REC : 0);
        }
        if (e.x >= 0) bulk_copy(dst, a.c.pool + (size_t)e.x * S::REC, S::REC, bar);
    };
    look_up(0);
    look_up(1);
    __syncthreads();
    if (warp == 0) {      // all stages are filled at once
        const int2 e = sched[lane];
        const unsigned pages = __ballot_sync(0xffffffffu, e.x != NOTHING);
        const int rank = __popc(pages & ((1u << lane) - 1));
        if (e.x != NOTHING && rank < S::STAGES) fetch(e, rank);
        __syncwarp();
    }
    // moves on to the next item: the next kv head, or the next pair that has rows
    auto next_item = [&] {
        left -= it.pages + ITEM_UNITS - at;
        at = 0;
        if (left <= 0 || ++it.h < kvh) return;
        do ++pair;
        while (!item_of<COLS>(a, pair / a.col_tiles, pair % a.col_tiles, it));
        it.h = 0;
    };

    // ---- a run's items ------------------------------------------------------------------------------------------------------------------
    const int r = lane >> 2, c = lane & 3;
    const int wk = warp % WK, pg = warp / WK % PG, wc = warp / (WK * PG);
    const int krow = (r >> 1) + 4 * (r & 1);       // the key (of 8) that row r of a fragment stands for
    // where this lane's codes and parameters lie in a record; group g of a key's or value's row: that address ^ 32 g, rows being aligned
    const uint32_t k_lane = (32 * wk + krow) * R::ROW + R::place(0, krow) * 32 + 8 * c, p_lane = 2 * R::CODES + (32 * wk + krow) * G * 4;
    const uint32_t v_lane = R::CODES + (32 * wk + c) * R::ROW + R::place(0, c) * 32 + 4 * r;
    int seq = 0, next_chunk = CHUNK;               // pages of the run in front of the item
    bool alive = true;
    for (; left > 0; next_item()) {
        const int base = max(at - ITEM_UNITS, 0), n = (int)min((long long)at + left, (long long)it.pages + ITEM_UNITS) - ITEM_UNITS - base;
        if (n <= 0) continue;       // units of the item itself only
        const int there = min(min(COLS, cols - it.ct * COLS), it.rows * a.rep - it.ct * COLS);      // columns of the item
        if (tid < there) {
            const int j = it.ct * COLS + tid;
            s_out[tid] = (((long long)it.b * a.m + j / a.rep) * a.heads + it.h * a.rep + j % a.rep) * HD;
        }
        const int st0 = seq & (S::STAGES - 1);
        if (S::QUERIES && alive) alive = mbar_wait(full + 8 * st0, seq / S::STAGES & 1);
        // columns of this warp: column j of the item is head j % rep of row j / rep
        uint32_t qf[NT][HD / 16][2];
        uint32_t qm[NT][(G + 1) / 2];      // sums of q over the groups, times 2**-6: first, second and third 16-bit parts in lanes c = 0, 1, 2
        int lim[NT][2];
        int low_lim = 0x7fffffff, top_lim = -1;     // positions up to low_lim are seen by all columns, none behind top_lim by any
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col0 = it.ct * COLS + (wc * NT + nt) * 8;
            const int j = DUP ? it.ct * COLS + (r & 3) : col0 + r;
            const int i = j / a.rep;
            const bool real = j - it.ct * COLS < there;
            const __half *src = S::QUERIES ? reinterpret_cast<const __half *>(ring + st0 * S::STAGE + S::REC) + (j - it.ct * COLS) * HD + 16 * c
                                           : a.q + (((size_t)it.b * a.m + i) * a.heads + it.h * a.rep + j % a.rep) * HD + 16 * c;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (real) x[0] = *reinterpret_cast<const uint4 *>(src + g * GROUP), x[1] = *reinterpret_cast<const uint4 *>(src + g * GROUP + 8);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t u[4] = {x[w].x, x[w].y, x[w].z, x[w].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = as_float2(u[e]);
                        sum += f.x + f.y;
                    }
                    qf[nt][g * 4][w] = prmt(u[0], u[2], 0x5410);
                    qf[nt][g * 4 + 1][w] = prmt(u[0], u[2], 0x7632);
                    qf[nt][g * 4 + 2][w] = prmt(u[1], u[3], 0x5410);
                    qf[nt][g * 4 + 3][w] = prmt(u[1], u[3], 0x7632);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= 0.015625f;
                const float p1 = __half2float(__float2half_rn(sum)), p2 = __half2float(__float2half_rn(sum - p1));
                const uint32_t h = __half_as_ushort(__float2half_rn(c == 0 ? p1 : c == 1 ? p2 : c == 2 ? sum - p1 - p2 : 0.f));
                qm[nt][g / 2] = g & 1 ? qm[nt][g / 2] | h << 16 : h;
            }
            const int l = real ? min(it.first + i, a.c.max_pages * PAGE - 1) : -2;
            low_lim = min(low_lim, (int)__reduce_min_sync(0xffffffffu, l == -2 ? 0x7fffffff : l));
            top_lim = max(top_lim, (int)__reduce_max_sync(0xffffffffu, l));
            lim[nt][0] = __shfl_sync(0xffffffffu, l, 8 * c);
            lim[nt][1] = __shfl_sync(0xffffffffu, l, 8 * c + 4);
        }
        float acc[NT][HD / 16][4], accm[NT][2][G], ref[NT][2], sum[NT][2], big[G], to_one[G];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][i][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                ref[nt][e] = 0.f, sum[nt][e] = 0.f;
#pragma unroll
                for (int g = 0; g < G; ++g) accm[nt][e][g] = 0.f;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) big[g] = 6.1035156e-5f, to_one[g] = W_ONE / big[g];     // 2**-14
        constexpr uint32_t LOOK = 0xbc00bc00u;                  // -1: no scale is that small, so the next step finds E anew
        uint32_t big_h[(G + 1) / 2];                            // the same as pairs of 16-bit numbers
#pragma unroll
        for (int i = 0; i < (G + 1) / 2; ++i) big_h[i] = 0x04000400u;
        bool first = true;                                      // nothing was added up yet
        // The tensor core rounds its sums towards zero with every product added: 5e-4 of the output after 2500 of them.  Every so many pages a
        // warp adds them to sums of its own in shared memory and begins anew.
        float *own_sums = merge + warp * S::SLOT + lane;
        bool set_aside = false;
        int since = 0;
        // the queries are read (a stage is filled again once its page is done with), s_out is written
        asm volatile("bar.sync 1, %0;" ::"n"(S::THREADS) : "memory");

        for (int p0 = 0; p0 < n; p0 += PG) {
            const int unit0 = (int)(units - left) + base + p0 + ITEM_UNITS - at;
            if (unit0 >= next_chunk) {      // two chunks are at hand: the one behind is looked up once nobody needs the one in front
                asm volatile("bar.sync 1, %0;" ::"n"(S::THREADS) : "memory");
                look_up(next_chunk / CHUNK + 1);
                next_chunk += CHUNK;
                asm volatile("bar.sync 1, %0;" ::"n"(S::THREADS) : "memory");
            }
            const int p = p0 + pg;
            if (p >= n) continue;
            const int st = (seq + p) & (S::STAGES - 1);
            if (alive) alive = mbar_wait(full + 8 * st, (seq + p) / S::STAGES & 1);
            const uint8_t *rec = ring + st * S::STAGE;
            if (++since > SET_ASIDE) {
                since = 1;
#pragma unroll
                for (int i = 0; i < S::SUMS; ++i) {
                    float &sum_i = acc[i / (HD / 4)][i / 4 % (HD / 16)][i % 4];
                    own_sums[32 * i] = set_aside ? own_sums[32 * i] + sum_i : sum_i;
                    sum_i = 0.f;
                }
                set_aside = true;
                if ((p0 / PG) % (4 * SET_ASIDE) == 0) big_h[0] = LOOK;
            }
            if (alive && sched[(unit0 + pg) & (2 * CHUNK - 1)].x >= 0) {
#pragma unroll 1
                for (int i = 0; i < 2 / WK; ++i) {
                    const int t0 = (base + p) * PAGE + 32 * (wk + WK * i);
                    if (t0 > top_lim) break;
                    const uint32_t k_at = k_lane + i * (32 * WK * R::ROW), v_at = v_lane + i * (32 * WK * R::ROW);
                    const uint8_t *par = rec + p_lane + i * (32 * WK * G * 4);
                    // 32 keys in two fragments of 16: their scores times 2**-20, lowest values times sums of q, then group by group
                    float z[2][NT][4];
                    uint32_t v0[2][G], v1[2][G];      // (scale, lowest value) of the values of this lane's keys
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
                        uint32_t k0[G], k1[G];
                        load_params<G>(k0, par + f * 16 * G * 4), load_params<G>(k1, par + (16 * f + 8) * G * 4);
                        load_params<G>(v0[f], par + R::PARAMS + f * 16 * G * 4), load_params<G>(v1[f], par + R::PARAMS + (16 * f + 8) * G * 4);
                        const uint32_t zero = 0;
                        const uint32_t a0 = G == 1 ? k0[0] >> 16 : prmt(k0[0], k0[G > 1], 0x7632), a1 = G == 1 ? k1[0] >> 16 : prmt(k1[0], k1[G > 1], 0x7632);
                        const uint32_t a2 = G == 4 ? prmt(k0[2 % G], k0[3 % G], 0x7632) : zero, a3 = G == 4 ? prmt(k1[2 % G], k1[3 % G], 0x7632) : zero;
                        float s[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816_first(s[nt], a0, a1, a2, a3, qm[nt][0], G == 4 ? qm[nt][(G + 1) / 2 - 1] : zero);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[nt][e] *= 64.f / UNIT;
                        }
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const uint8_t *at = rec + (k_at ^ (32 * g)) + f * 16 * R::ROW;
                            const uint2 x0 = *reinterpret_cast<const uint2 *>(at), x1 = *reinterpret_cast<const uint2 *>(at + 8 * R::ROW);
                            float d[NT][4];
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const uint32_t y0 = x0.x >> (8 * t), y1 = x1.x >> (8 * t), y2 = x0.y >> (8 * t), y3 = x1.y >> (8 * t);
                                const uint32_t l0 = codes_low(y0), l1 = codes_low(y1), l2 = codes_low(y2), l3 = codes_low(y3);
                                const uint32_t m0 = codes_mid(y0), m1 = codes_mid(y1), m2 = codes_mid(y2), m3 = codes_mid(y3);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const uint32_t(&b)[2] = qf[nt][g * 4 + 2 * t], (&b2)[2] = qf[nt][g * 4 + 2 * t + 1];
                                    if (t == 0) mma16816_first(d[nt], m0, m1, m2, m3, b2[0], b2[1]);
                                    else mma16816(d[nt], m0, m1, m2, m3, b2[0], b2[1]);
                                    mma16816(d[nt], l0, l1, l2, l3, b[0], b[1]);
                                }
                            }
                            const float f0 = as_float2(k0[g]).x, f1 = as_float2(k1[g]).x;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                s[nt][0] = fmaf(f0, d[nt][0], s[nt][0]);
                                s[nt][1] = fmaf(f0, d[nt][1], s[nt][1]);
                                s[nt][2] = fmaf(f1, d[nt][2], s[nt][2]);
                                s[nt][3] = fmaf(f1, d[nt][3], s[nt][3]);
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[f][nt][e] = fmaf(s[nt][e], a.scale_log2, -ref[nt][e & 1]);
                    }
                    const bool masked = t0 + 31 > low_lim;
                    if (masked) {      // what a column does not see weighs nothing, whatever its key and value are
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            const int ta = t0 + 16 * f + krow, tb = ta + 8;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (ta > lim[nt][0]) z[f][nt][0] = -INFINITY;
                                if (ta > lim[nt][1]) z[f][nt][1] = -INFINITY;
                                if (tb > lim[nt][0]) z[f][nt][2] = -INFINITY;
                                if (tb > lim[nt][1]) z[f][nt][3] = -INFINITY;
                            }
#pragma unroll
                            for (int g = 0; g < G; ++g) {
                                if (ta > top_lim) v0[f][g] = 0;
                                if (tb > top_lim) v1[f][g] = 0;
                            }
                        }
                    }
                    // A column's weights are powers relative to `ref`, which follows its largest score only when this lane's four would pass 2**8 in
                    // sum; E likewise follows the scales.  Most keys move neither, which one vote finds out.  E comes down again, to the scales of the
                    // step at hand, behind a step for some of whose positions it jumped, and every 64 pages.  A weight p * s keeps 2**-31 of E, so that
                    // E would otherwise cost all that follow a few far larger values their digits (4000 positions of weight 2**-16 behind one of 2**16 times
                    // their scale: 1 to 4 % of the largest value; now the other 31 positions of its step alone).  Asking every step costs 1 to 3 % of the time.
                    float w[2][NT][4], add[NT][2];
                    bool moved = first;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int f = 0; f < 2; ++f)
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[f][nt][e] = exp2_approx(z[f][nt][e]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            add[nt][e] = (w[0][nt][e] + w[0][nt][e + 2]) + (w[1][nt][e] + w[1][nt][e + 2]);
                            moved |= add[nt][e] > MOVE_AT;
                        }
                    }
                    if constexpr (G == 1) {
                        const __half2 x = __hmax2_nan(as_half2(prmt(v0[0][0], v1[0][0], 0x5410)), as_half2(prmt(v0[1][0], v1[1][0], 0x5410)));
                        moved |= !__hble2(x, as_half2(big_h[0]));
                    } else {
#pragma unroll
                        for (int i2 = 0; i2 < G / 2; ++i2) {
                            __half2 x = as_half2(prmt(v0[0][2 * i2], v0[0][2 * i2 + 1], 0x5410));
                            x = __hmax2_nan(x, as_half2(prmt(v1[0][2 * i2], v1[0][2 * i2 + 1], 0x5410)));
                            x = __hmax2_nan(x, __hmax2_nan(as_half2(prmt(v0[1][2 * i2], v0[1][2 * i2 + 1], 0x5410)), as_half2(prmt(v1[1][2 * i2], v1[1][2 * i2 + 1], 0x5410))));
                            moved |= !__hble2(x, as_half2(big_h[i2]));
                        }
                    }
                    if (__any_sync(0xffffffffu, moved)) {
                        float fg[G];
                        const bool anew = __any_sync(0xffffffffu, big_h[0] == LOOK);      // each lane's own
                        bool jumped = false;
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            float x = 0.f;
#pragma unroll
                            for (int f = 0; f < 2; ++f) {
                                const float x0 = fabsf(as_float2(v0[f][g]).x), x1 = fabsf(as_float2(v1[f][g]).x);
                                x = fmaxf(x, fmaxf(x0 <= 65504.f ? x0 : 0.f, x1 <= 65504.f ? x1 : 0.f));
                            }
                            const uint32_t u = (__reduce_max_sync(0xffffffffu, __float_as_uint(x)) + 0x7fffffu) & 0x7f800000u;   // up to a power of two
                            const float grown = fminf(fmaxf(__uint_as_float(u), anew ? 6.1035156e-5f : big[g]), 32768.f);
                            fg[g] = __fdividef(big[g], grown);
                            jumped |= 64.f * x < grown && fg[g] <= 0.125f;      // not for this lane's positions
                            big[g] = grown, to_one[g] = __fdividef(W_ONE, grown);
                            const uint32_t h = __half_as_ushort(__float2half_rn(grown));
                            if (G == 1) big_h[0] = h * 0x10001u;
                            else big_h[g / 2] = g & 1 ? prmt(big_h[g / 2], h, 0x5410) : prmt(big_h[g / 2], h, 0x3254);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float x = fmaxf(fmaxf(z[0][nt][e], z[0][nt][e + 2]), fmaxf(z[1][nt][e], z[1][nt][e + 2]));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                                float by = first ? 0.f : 1.f;
                                if (x > (first ? -INFINITY : 0.f)) {
                                    if (!first) by = exp2_approx(-x);
                                    ref[nt][e] += x;
#pragma unroll
                                    for (int f = 0; f < 2; ++f)
#pragma unroll
                                        for (int k = 0; k < 2; ++k) w[f][nt][e + 2 * k] = exp2_approx(z[f][nt][e + 2 * k] - x);
                                    add[nt][e] = (w[0][nt][e] + w[0][nt][e + 2]) + (w[1][nt][e] + w[1][nt][e + 2]);
                                }
                                sum[nt][e] *= by;
#pragma unroll
                                for (int g = 0; g < G; ++g) {
                                    accm[nt][e][g] *= by;
#pragma unroll
                                    for (int k = 0; k < 4; ++k) acc[nt][4 * g + k][e] *= by * fg[g], acc[nt][4 * g + k][e + 2] *= by * fg[g];
                                    if (set_aside) {
#pragma unroll
                                        for (int k = 0; k < 8; ++k) own_sums[32 * (nt * (HD / 4) + (4 * g + k / 2) * 4 + e + 2 * (k & 1))] *= by * fg[g];
                                    }
                                }
                            }
                        if (jumped) big_h[0] = LOOK;
                        first = false;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) sum[nt][0] += add[nt][0], sum[nt][1] += add[nt][1];
                    // weighted values
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            float2 f0 = as_float2(v0[f][g]), f1 = as_float2(v1[f][g]);
                            f0.y = fmaf(8.f, f0.x, f0.y), f1.y = fmaf(8.f, f1.x, f1.y);
                            const float u0 = f0.x * to_one[g], u1 = f1.x * to_one[g];
                            uint32_t b[NT][2], b2[NT][2];
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const float(&q)[4] = w[f][nt];
                                float y[4] = {q[0] * u0, q[1] * u0, q[2] * u1, q[3] * u1};
                                if (masked) {      // 0 times what is no number
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        if (q[e] == 0.f) y[e] = 0.f;
                                    accm[nt][0][g] += (q[0] == 0.f ? 0.f : q[0] * f0.y) + (q[2] == 0.f ? 0.f : q[2] * f1.y);
                                    accm[nt][1][g] += (q[1] == 0.f ? 0.f : q[1] * f0.y) + (q[3] == 0.f ? 0.f : q[3] * f1.y);
                                } else {
                                    accm[nt][0][g] = fmaf(q[0], f0.y, fmaf(q[2], f1.y, accm[nt][0][g]));
                                    accm[nt][1][g] = fmaf(q[1], f0.y, fmaf(q[3], f1.y, accm[nt][1][g]));
                                }
                                const __half2 h0 = __floats2half2_rn(y[0], y[1]), h1 = __floats2half2_rn(y[2], y[3]);
                                const float2 e0 = __half22float2(h0), e1 = __half22float2(h1);
                                if (DUP) {      // lanes 2 and 3 carry what the others' rounding left
                                    const float rest = c < 2 ? 0.f : 1.f;
                                    b[nt][0] = transposed(as_u32(c < 2 ? h0 : __floats2half2_rn(fmaf(-rest, e0.x, y[0]), fmaf(-rest, e0.y, y[1]))));
                                    b[nt][1] = transposed(as_u32(c < 2 ? h1 : __floats2half2_rn(fmaf(-rest, e1.x, y[2]), fmaf(-rest, e1.y, y[3]))));
                                } else {
                                    b[nt][0] = transposed(as_u32(h0)), b[nt][1] = transposed(as_u32(h1));
                                    b2[nt][0] = transposed(as_u32(__floats2half2_rn(y[0] - e0.x, y[1] - e0.y)));
                                    b2[nt][1] = transposed(as_u32(__floats2half2_rn(y[2] - e1.x, y[3] - e1.y)));
                                }
                            }
                            const uint8_t *at = rec + (v_at ^ (32 * g)) + f * 16 * R::ROW, *at4 = rec + (v_at ^ (32 * (g ^ R::FOUR_ON))) + f * 16 * R::ROW;
                            const uint32_t y0 = *reinterpret_cast<const uint32_t *>(at), y1 = *reinterpret_cast<const uint32_t *>(at4 + 4 * R::ROW);
                            const uint32_t y2 = *reinterpret_cast<const uint32_t *>(at + 8 * R::ROW), y3 = *reinterpret_cast<const uint32_t *>(at4 + 12 * R::ROW);
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t za = prmt(y0, y1, k ? 0x7632 : 0x5410), zb = prmt(y2, y3, k ? 0x7632 : 0x5410);
#pragma unroll
                                for (int t = 0; t < 2; ++t) {
                                    const uint32_t xa = za >> (8 * t), xb = zb >> (8 * t);
                                    const uint32_t a0 = codes_low_8(xa), a1 = codes_mid_8(xa), a2 = codes_low_8(xb), a3 = codes_mid_8(xb);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) {
                                        mma16816(acc[nt][4 * g + 2 * k + t], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                                        if (!DUP) mma16816(acc[nt][4 * g + 2 * k + t], a0, a1, a2, a3, b2[nt][0], b2[nt][1]);
                                    }
                                }
                            }
                        }
                    }
                }
            }
            // the last of the warps that are through with a page asks for the one that goes into its stage
            __syncwarp();
            unsigned done = 0;
            if (lane == 0) asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(done) : "r"(smem_u32(s_done + st)) : "memory");
            done = __shfl_sync(0xffffffffu, done, 0);
            if ((done + 1) % (WK * WC) == 0 && alive) {
                const int2 e = sched[(unit0 + pg + lane) & (2 * CHUNK - 1)];
                const unsigned pages = __ballot_sync(0xffffffffu, e.x != NOTHING);
                if (e.x != NOTHING && __popc(pages & ((1u << lane) - 1)) == S::STAGES) fetch(e, st);
            }
        }
        seq += n;

        // ---- this block's part of the item, into the output or into scratch ---------------------------------------------------------------
        const bool all = n == it.pages;
        // The blocks of an item are neighbours; a part lies in the block's first place if the item began in front of the block, else in its second.
        float *part = a.parts + ((size_t)blockIdx.x * 2 + (at == 0 ? 1 : 0)) * S::PART;
        if (set_aside) {
#pragma unroll
            for (int i = 0; i < S::SUMS; ++i) acc[i / (HD / 4)][i / 4 % (HD / 16)][i % 4] += own_sums[32 * i];
            __syncwarp();      // the part goes where the sums were
        }
        float *mine = merge + warp * S::SLOT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = sum[nt][e];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                const int col = (wc * NT + nt) * 8 + 2 * c + e;
                const float top = l == 0.f ? -INFINITY : ref[nt][e];
                if (S::PARTS > 1) {
                    if (r == 0 && (!DUP || c < 2)) mine[COLS * HD + col] = top, mine[COLS * (HD + 1) + col] = l;
                } else if (!all && r == 0) {
                    __stcg(part + COLS * HD + col, top), __stcg(part + COLS * (HD + 1) + col, l);
                }
                const float inv = 1.f / l;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float lowest = accm[nt][e][g];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) lowest += __shfl_xor_sync(0xffffffffu, lowest, o);
                    const float back = big[g] * (UNIT / W_ONE);
                    float o8[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o8[2 * i] = acc[nt][4 * g + i][e], o8[2 * i + 1] = acc[nt][4 * g + i][e + 2];
                    if (DUP) {      // first and second parts of the weights
#pragma unroll
                        for (int i = 0; i < 8; ++i) o8[i] += __shfl_xor_sync(0xffffffffu, o8[i], 2);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) o8[i] = fmaf(o8[i], back, lowest);
                    if (S::PARTS == 1 && all) {
                        if (col < there) {
                            if (l == 0.f) {      // no position: zeros
#pragma unroll
                                for (int i = 0; i < 8; ++i) o8[i] = 0.f;
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; ++i) o8[i] *= inv;
                            }
                            *reinterpret_cast<uint4 *>(a.out + s_out[col] + g * GROUP + 8 * r) =
                                make_uint4(as_u32(__floats2half2_rn(o8[0], o8[1])), as_u32(__floats2half2_rn(o8[2], o8[3])),
                                           as_u32(__floats2half2_rn(o8[4], o8[5])), as_u32(__floats2half2_rn(o8[6], o8[7])));
                        }
                    } else if (S::PARTS == 1) {
                        float4 *dst = reinterpret_cast<float4 *>(part + col * HD + g * GROUP + 8 * r);
                        if (col < there) __stcg(dst, make_float4(o8[0], o8[1], o8[2], o8[3])), __stcg(dst + 1, make_float4(o8[4], o8[5], o8[6], o8[7]));
                    } else if (!DUP || c < 2) {
                        float4 *dst = reinterpret_cast<float4 *>(mine + col * HD + g * GROUP + 8 * r);
                        dst[0] = make_float4(o8[0], o8[1], o8[2], o8[3]);
                        dst[1] = make_float4(o8[4], o8[5], o8[6], o8[7]);
                    }
                }
            }
        }
        if (S::PARTS > 1) {
            asm volatile("bar.sync 1, %0;" ::"n"(S::WARPS * 32) : "memory");
            for (int x = 4 * tid; x < there * HD; x += 4 * S::WARPS * 32) {
                const int col = x / HD;
                float t[S::PARTS], l[S::PARTS], top = -INFINITY, total = 0.f;
#pragma unroll
                for (int w = 0; w < S::PARTS; ++w) t[w] = merge[w * S::SLOT + COLS * HD + col], l[w] = merge[w * S::SLOT + COLS * (HD + 1) + col], top = fmaxf(top, t[w]);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < S::PARTS; ++w) {
                    if (l[w] == 0.f) continue;
                    const float f = exp2_approx(t[w] - top);
                    const float4 v = *reinterpret_cast<const float4 *>(merge + w * S::SLOT + x);
                    total += f * l[w];
                    o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
                }
                if (all) {
                    store_output(a.out + s_out[col] + x % HD, o, total);
                } else {
                    __stcg(reinterpret_cast<float4 *>(part + x), o);
                    if (x % HD == 0) __stcg(part + COLS * HD + col, top), __stcg(part + COLS * (HD + 1) + col, total);
                }
            }
        }
        if (!all) {
            // first and last block that has pages of this item
            const long long start = (long long)list[pair] * kvh + (long long)it.h * (it.pages + ITEM_UNITS);
            const int block0 = (int)((start + ITEM_UNITS) / per), block1 = (int)((start + ITEM_UNITS + it.pages - 1) / per);
            unsigned *counter = a.counters + (size_t)pair * kvh + it.h;
            asm volatile("bar.sync 1, %0;" ::"n"(S::WARPS * 32) : "memory");
            if (tid == 0) {
                unsigned old;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
                s_flag = old == (unsigned)(block1 - block0);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(S::WARPS * 32) : "memory");
            if (s_flag) {
                const float *parts = a.parts + (size_t)(block0 + 1) * 2 * S::PART;      // of the blocks behind the first
                const float *part0 = a.parts + ((size_t)block0 * 2 + (start >= per * block0 ? 1 : 0)) * S::PART;
                const int more = block1 - block0;
                auto add_up = [&](auto pieces, auto at_once) {      // so many pieces of four outputs per thread, so many parts of each at a time: all loads first
                    constexpr int T = decltype(pieces)::value, P = decltype(at_once)::value, STEP = 4 * S::THREADS;
                    for (int x0 = 4 * tid; x0 < there * HD; x0 += T * STEP) {
                        float4 o[T];
                        float top[T], total[T];
#pragma unroll
                        for (int i = 0; i < T; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f), top[i] = -INFINITY, total[i] = 0.f;
                        for (int k0 = -1; k0 < more; k0 += P) {
                            float4 v[T][P];
                            float t[T][P], l[T][P];
#pragma unroll
                            for (int u = 0; u < P; ++u) {
                                const int k = min(k0 + u, more - 1);
                                const float *m = k < 0 ? part0 : parts + (size_t)k * 2 * S::PART;
#pragma unroll
                                for (int i = 0; i < T; ++i) {
                                    const int x = x0 + i * STEP < there * HD ? x0 + i * STEP : x0;
                                    v[i][u] = __ldcg(reinterpret_cast<const float4 *>(m + x));
                                    t[i][u] = __ldcg(m + COLS * HD + x / HD), l[i][u] = __ldcg(m + COLS * (HD + 1) + x / HD);
                                }
                            }
#pragma unroll
                            for (int i = 0; i < T; ++i) {
                                float high = top[i];
#pragma unroll
                                for (int u = 0; u < P; ++u) {
                                    if (k0 + u >= more) l[i][u] = 0.f;
                                    if (l[i][u] != 0.f) high = fmaxf(high, t[i][u]);
                                }
                                const float old = total[i] == 0.f ? 0.f : exp2_approx(top[i] - high);
                                top[i] = high, total[i] *= old;
                                if (total[i] != 0.f) o[i].x *= old, o[i].y *= old, o[i].z *= old, o[i].w *= old;
#pragma unroll
                                for (int u = 0; u < P; ++u) {
                                    if (l[i][u] == 0.f) continue;
                                    const float w = exp2_approx(t[i][u] - high);
                                    total[i] += w * l[i][u];
                                    o[i].x += w * v[i][u].x, o[i].y += w * v[i][u].y, o[i].z += w * v[i][u].z, o[i].w += w * v[i][u].w;
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < T; ++i) {
                            const int x = x0 + i * STEP;
                            if (x < there * HD) store_output(a.out + s_out[x / HD] + x % HD, o[i], total[i]);
                        }
                    }
                };
                if (more < 4) add_up(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
                else if (more < 8 || there * HD > 4 * S::THREADS) add_up(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
                else add_up(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
                if (tid == 0) *counter = 0;      // ready for the next launch
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(S::WARPS * 32) : "memory");       // `merge` and `s_flag` are free again
    }
    if (!alive) {      // a wait ran out: the run went on without its pages, past the same barriers; what is on its way lands before the block ends
        if (lane == 0) atomicExch(a.status, SAL_E_TIMEOUT);
        for (int i = 0; i < S::STAGES; ++i) (void)mbar_wait(full + 8 * i, 0), (void)mbar_wait(full + 8 * i, 1);
    }
}

// ---- many columns: the fifth generation's tensor cores --------------------------------------------------------------------------------
//
// The same sums with the queries as rows of the products: 128 columns of an item against a page.  Codes less 8 are expanded once for all 128 into
// shared memory as 16-bit floats (exact; 64 positions x 64 numbers in rows of 128 bytes, swizzled), which serves the keys as an operand that
// runs along the dimensions and the values as one that runs along the positions.  D_g stands in tensor memory, one row a lane; two threads share a
// row, each with 32 of the page's positions.  They leave the weights p * s_g / E_g as two 16-bit parts where D_g was, from where they are the second
// product's first operand.  A page's outputs start from zero and are added to 32-bit sums in registers, so the maximum may move with every page
// and nothing is added up in the tensor core beyond a page.  E_g is the page's own.
//
// A block takes one item, or one of `splits` equal runs of its pages; the last one to arrive adds the parts up in order.  Items with the most pages are
// launched first.  Equal runs that may end inside an item, as above, cost more in parts of 128 columns and new starts than they even out: 98 us where this
// takes 79 (512 rows behind 1536 positions, 32 heads of 128: 15 GFLOP, and half as much again for the second parts).  Bound by latency at
// 16 warps an SM: 46 % of the issue slots, 1140 instructions a warp and page, most of them once per score and group.  While the tensor core works for one of the two blocks of an SM the other one expands, and within a block the next page's keys are expanded
// behind the second product's back.
template <int HD>
struct WideShape {
    static constexpr int G = HD / GROUP, COLS = 128, THREADS = 256, STAGES = 3;
    static constexpr int REC = Record<HD>::BYTES;
    static constexpr int Q_BYTES = G * COLS * 128, TILE = PAGE * 128, T_BYTES = G * TILE;      // a group of the queries, of a page
    static constexpr int SMEM = 1024 + Q_BYTES + 2 * T_BYTES + STAGES * REC + 2 * G * PAGE * 8 + 2 * (1 + G) * COLS * 4;
    static constexpr int TMEM = 2 * HD;                                // columns: D_g or weights, then outputs
    static constexpr int PART = COLS * (HD + 2);
};
constexpr int WIDE_BLOCKS = 2 * 148;      // resident at once: two of 100 KB and 128 registers a thread on an SM
constexpr int WIDE_SPLITS = 32;           // one block adds the parts up
constexpr float MOVE_BY = 8.f;            // 2**8 = MOVE_AT

__device__ __forceinline__ void tmem_load8(float *v, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(addr)
                 : "memory");
}
// two 32-bit sums or products at once
struct Two {
    unsigned long long x;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b)); }
    __device__ __forceinline__ float2 get() const {
        float2 v;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(x));
        return v;
    }
};
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.x) : "l"(a.x), "l"(b.x), "l"(c.x));
    return d;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.x) : "l"(a.x), "l"(b.x));
    return d;
}
__device__ __forceinline__ Two add(Two a, Two b) {
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.x) : "l"(a.x), "l"(b.x));
    return d;
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }      // own writes, for the tensor core
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// d[128][64] = or += a * b, a in shared memory
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(more)
                 : "memory");
}
// a in tensor memory
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
                 "r"(more)
                 : "memory");
}
// Rows of 128 bytes, eight of them an atom of 1024, 128-byte swizzle; both strides are an atom's (an operand of 64 numbers across has one of them only).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(1024 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// eight codes less 8 as 16-bit floats, in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 eight_codes(uint32_t x) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t y = x >> (8 * i);
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(o[2 * i]) : "r"(y));
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(o[2 * i + 1]) : "r"(y));
        asm("add.rn.f16x2 %0, %0, %1;" : "+r"(o[2 * i]) : "r"(0xe408e408u));                                // 1024 + c - 1032
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(o[2 * i + 1]) : "r"(0x2c002c00u), "r"(0xd480d480u));      // (1024 + 16 c) / 16 - 72
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int HD>
__global__ void __launch_bounds__(WideShape<HD>::THREADS, 2) attention_wide_kernel(AttnArgs a) {
    using S = WideShape<HD>;
    using R = Record<HD>;
    constexpr int G = S::G, COLS = S::COLS, N = HD / 2;      // outputs of a thread
    extern __shared__ __align__(1024) uint8_t wide_smem[];
    __shared__ uint64_t bars[S::STAGES + 2];
    __shared__ uint32_t s_tmem;
    __shared__ float s_back[G];
    __shared__ int s_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, half = tid / COLS, row = tid % COLS;
    uint8_t *smem = wide_smem + ((1024u - (smem_u32(wide_smem) & 1023u)) & 1023u);
    const uint32_t q_tile = smem_u32(smem), k_tile = q_tile + S::Q_BYTES, v_tile = k_tile + S::T_BYTES;
    uint8_t *ring = smem + S::Q_BYTES + 2 * S::T_BYTES;
    float *kp = reinterpret_cast<float *>(ring + S::STAGES * S::REC), *vp = kp + 2 * G * PAGE;      // of [group][pair of positions]: two scales, two lowest + 8 scales
    float *swap = reinterpret_cast<float *>(vp + 2 * G * PAGE);      // [half][1 + G][row]
    const uint32_t full = smem_u32(bars), bar_s = full + 8 * S::STAGES, bar_o = bar_s + 8;

    // The tensor memory is taken behind the wait for the launch in front and before the next one may start: neither then holds what the other waits for.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int kvh = a.c.kv_heads, split = blockIdx.x % a.splits, item = blockIdx.x / a.splits;
    Item it = {};
    it.h = item % kvh;
    if (!item_of<COLS>(a, item / kvh % a.batch, a.col_tiles - 1 - item / kvh / a.batch, it)) return;
    const int pair = it.b * a.col_tiles + it.ct;
    const int splits = min(a.splits, (it.pages + 3) / 4);      // a run has four pages at least, or the item one run
    if (split >= splits) return;
    const int page1 = (int)((long long)it.pages * (split + 1) / splits);
    const int32_t *table = a.c.table + (size_t)it.b * a.c.max_pages;
    auto next_page = [&](int p) {      // the next one that exists
        for (; p < page1; ++p) {
            const int x = table[p];
            if (x >= 0 && x < a.c.pages) break;
        }
        return p;
    };
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(S::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    } else if (tid == 32) {
        for (int i = 0; i < S::STAGES + 2; ++i) mbar_init(full + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = s_tmem, mine = tmem + ((uint32_t)(warp & 3) << 21);      // lanes of this warp: 32 of them

    int p = next_page((int)((long long)it.pages * split / splits));
    int to_fetch = p;      // of one thread
    auto fetch = [&](int st) {
        if (to_fetch >= page1) return;
        mbar_expect_tx(full + 8 * st, S::REC);
        bulk_copy(smem_u32(ring + st * S::REC), a.c.pool + ((size_t)table[to_fetch] * kvh + it.h) * S::REC, S::REC, full + 8 * st);
        to_fetch = next_page(to_fetch + 1);
    };
    if (tid == 32)
        for (int st = 0; st < S::STAGES; ++st) fetch(st);
    __syncwarp();

    // ---- queries: rows of the first operand, zero where there is no column ---------------------------------------------------------------
    const int col = it.ct * COLS + row, i_row = col / a.rep;
    const bool real = col < a.m * a.rep && i_row < it.rows;
    const size_t at = (((size_t)it.b * a.m + i_row) * a.heads + it.h * a.rep + col % a.rep) * HD + half * N;
    float qsum[G];
    {
        const int g = half * N / GROUP, chunk0 = half * N % GROUP / 8;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (real) x = *reinterpret_cast<const uint4 *>(a.q + at + 8 * i);
            const float2 f0 = as_float2(x.x), f1 = as_float2(x.y), f2 = as_float2(x.z), f3 = as_float2(x.w);
            sum += f0.x + f0.y + f1.x + f1.y + f2.x + f2.y + f3.x + f3.y;
            *reinterpret_cast<uint4 *>(smem + g * COLS * 128 + row * 128 + (((chunk0 + i) ^ (row & 7)) << 4)) =
                make_uint4(prmt(x.x, x.z, 0x5410), prmt(x.x, x.z, 0x7632), prmt(x.y, x.w, 0x5410), prmt(x.y, x.w, 0x7632));      // in the codes' order
        }
        swap[half * (1 + G) * COLS + row] = sum;
    }
    const int lim = real ? min(it.first + i_row, a.c.max_pages * PAGE - 1) : -2;
    const int low_lim = __reduce_min_sync(0xffffffffu, real ? lim : 0x7fffffff), top_lim = __reduce_max_sync(0xffffffffu, lim);      // of 32 rows

    // ---- a page's codes and parameters ------------------------------------------------------------------------------------------------
    const int hb = tid & 1, xg = G == 2 ? tid >> 3 & 1 : 0, xk = G == 2 ? tid >> 4 << 2 | (tid >> 1 & 3) : tid >> 1;      // 16 bytes: both sides without bank conflicts
    const int x_from = xk * R::ROW + R::place(xg, xk) * 32 + 16 * hb;
    auto expand = [&](const uint8_t *codes, uint32_t tile) {
        if (tid >= 2 * G * PAGE) return;
        const uint4 x = *reinterpret_cast<const uint4 *>(codes + x_from);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint8_t *to = smem + (tile - q_tile) + xg * S::TILE + xk * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(to + ((4 * hb + i) ^ (xk & 7)) * 16) = eight_codes(w[i]);
    };
    const float scale_log2 = a.scale_log2 * (1.f / UNIT);
    auto parameters = [&](const uint8_t *rec, int page) {      // positions behind the last one that is seen: nothing
        const __half2 *from = reinterpret_cast<const __half2 *>(rec + 2 * R::CODES);
        if (tid < G * PAGE) {
            const int k = tid % PAGE, g = tid / PAGE;
            const float2 x = page * PAGE + k <= it.last ? __half22float2(from[k * G + g]) : make_float2(0.f, 0.f);
            float *to = kp + (tid >> 1) * 4 + (tid & 1);
            to[0] = x.x * scale_log2, to[2] = fmaf(8.f, x.x, x.y) * scale_log2;
        }
        if (warp >= 4 && warp < 4 + G) {
            const int g = warp - 4;
            float2 x[2];
            float top = 6.1035156e-5f;      // 2**-14
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = lane + 32 * e;
                x[e] = page * PAGE + k <= it.last ? __half22float2(from[R::PARAMS / 4 + k * G + g]) : make_float2(0.f, 0.f);
                if (x[e].x <= 65504.f) top = fmaxf(top, x[e].x);      // one that is not finite is for the rows that see it
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float big = __uint_as_float((__float_as_uint(top) + 0x007fffffu) & 0x7f800000u);      // the power of two from there on
            const float to_one = W_ONE / big;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float *to = vp + ((g * PAGE + lane + 32 * e) >> 1) * 4 + (lane & 1);
                to[0] = x[e].x * to_one, to[2] = fmaf(8.f, x[e].x, x[e].y);
            }
            if (lane == 0) s_back[g] = big / W_ONE;
        }
    };
    constexpr uint32_t IDESC = 1u << 4 | (uint32_t)(PAGE >> 3) << 17 | (uint32_t)(COLS >> 4) << 24;      // 32-bit sums, 16-bit operands, 128 x 64
    constexpr uint32_t IDESC_V = IDESC | 1u << 16;                                                     // the second operand runs along the positions
    auto scores = [&] {
        if (warp == 0) {
            if (elect_one()) {
                fence_after();
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_smem(tmem + 64 * g, tile_desc(q_tile + g * COLS * 128) + 2 * k, tile_desc(k_tile + g * S::TILE) + 2 * k, IDESC, k);
                mma_commit(bar_s);
            }
            __syncwarp();
        }
    };
    auto outputs = [&] {
        if (warp == 0) {
            if (elect_one()) {
                fence_after();
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int x = 0; x < 8; ++x) {      // 16 positions, first or second parts of their weights
                        const int k = x >> 1;
                        mma_tmem(tmem + HD + 64 * g, tmem + 64 * g + 8 * x, tile_desc(v_tile + g * S::TILE + 16 * k * 128), IDESC_V, x);
                    }
                mma_commit(bar_o);
            }
            __syncwarp();
        }
    };

    bool alive = true;
    Two acc[N / 2], sums(0.f, 0.f);      // outputs
    float accm[G], ref = -INFINITY, back = 0.f, f = 1.f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) acc[i] = Two(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < G; ++g) accm[g] = 0.f;
    bool taken = false;      // this warp's rows see something of the page
    int seq = 0;
    auto take = [&] {      // the outputs of page seq - 1
        if (alive) alive = mbar_wait(bar_o, (seq - 1) & 1);
        __syncwarp();
        fence_after();
        if (!taken) return;
        if (__any_sync(0xffffffffu, f != 1.f)) {      // seldom
#pragma unroll
            for (int i = 0; i < N / 2; ++i) acc[i] = mul(acc[i], Two(f, f));
        }
#pragma unroll
        for (int i = 0; i < N; i += 16) {
            float v[16];
            tmem_load8(v, mine + HD + half * N + i);
            tmem_load8(v + 8, mine + HD + half * N + i + 8);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 16; e += 2) acc[(i + e) / 2] = fma(Two(v[e], v[e + 1]), Two(back, back), acc[(i + e) / 2]);
        }
    };
    if (p < page1) {
        if (alive) alive = mbar_wait(full, 0);
        __syncwarp();
        expand(ring, k_tile);
        parameters(ring, p);
    }
    fence_smem();
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g) qsum[g] = G == 2 ? swap[g * (1 + G) * COLS + row] : swap[row] + swap[(1 + G) * COLS + row];
    if (p < page1) scores();
    __syncthreads();      // `swap` is free

    for (; p < page1; ++seq) {
        const int st = seq % S::STAGES, after = next_page(p + 1);
        if (seq) take();
        expand(ring + st * S::REC + R::CODES, v_tile);
        if (alive) alive = mbar_wait(bar_s, seq & 1);
        __syncwarp();
        fence_after();
        taken = p * PAGE <= top_lim;
        if (taken) {
            const int t0 = p * PAGE + 32 * half;
            const uint32_t own = mine + 32 * half;      // this thread's columns of group 0
            const bool masked = p * PAGE + PAGE - 1 > low_lim;      // for some of the rows
            float top = -INFINITY;
            // scores into the last group's place, the registers being the outputs'
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
                float d[G][8];
#pragma unroll
                for (int g = 0; g < G; ++g) tmem_load8(d[g], own + 64 * g + k);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                float u[8];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    Two t(0.f, 0.f);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float4 x = *reinterpret_cast<const float4 *>(kp + 2 * (g * PAGE + 32 * half + k + e));
                        const Two low = g ? fma(Two(x.z, x.w), Two(qsum[g], qsum[g]), t) : mul(Two(x.z, x.w), Two(qsum[g], qsum[g]));
                        t = fma(Two(x.x, x.y), Two(d[g][e], d[g][e + 1]), low);
                    }
                    const float2 v = t.get();
                    u[e] = v.x, u[e + 1] = v.y;
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] = t0 + k + e <= lim ? u[e] : -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, u[e]);
                tmem_store8(own + 64 * (G - 1) + k, reinterpret_cast<const uint32_t *>(u));
            }
            swap[half * (1 + G) * COLS + row] = top;
            switch (warp & 3) {      // the two warps of these rows
                case 0: asm volatile("bar.sync 1, 64;" ::: "memory"); break;
                case 1: asm volatile("bar.sync 2, 64;" ::: "memory"); break;
                case 2: asm volatile("bar.sync 3, 64;" ::: "memory"); break;
                default: asm volatile("bar.sync 4, 64;" ::: "memory"); break;
            }
            top = fmaxf(ref, fmaxf(top, swap[(1 - half) * (1 + G) * COLS + row]));
            f = 1.f;
            if (top > ref + MOVE_BY) {      // weights stay below MOVE_AT
                if (ref != -INFINITY) f = exp2_approx(ref - top);
                ref = top;
            }
            const float from = ref == -INFINITY ? 0.f : ref;
            back = s_back[half * N / GROUP];
            const bool moved = __any_sync(0xffffffffu, f != 1.f);
            if (moved) sums = mul(sums, Two(f, f));
            Two low[G];
#pragma unroll
            for (int g = 0; g < G; ++g) low[g] = Two(0.f, 0.f);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            auto weights = [&](auto some) {      // where a position is not seen its parameters are not looked at either
#pragma unroll
                for (int k = 0; k < 32; k += 16) {
                    float s[16];
                    tmem_load8(s, own + 64 * (G - 1) + k), tmem_load8(s + 8, own + 64 * (G - 1) + k + 8);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    Two w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 v = add(Two(s[2 * e], s[2 * e + 1]), Two(-from, -from)).get();
                        w[e] = Two(exp2_approx(v.x), exp2_approx(v.y));
                        sums = add(sums, w[e]);
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float4 x = *reinterpret_cast<const float4 *>(vp + 2 * (g * PAGE + 32 * half + k + 2 * e));
                            if (decltype(some)::value) {
                                if (t0 + k + 2 * e > lim) x.x = 0.f, x.z = 0.f;
                                if (t0 + k + 2 * e + 1 > lim) x.y = 0.f, x.w = 0.f;
                            }
                            const Two z = mul(w[e], Two(x.x, x.y));
                            low[g] = fma(w[e], Two(x.z, x.w), low[g]);
                            const float2 v = z.get();
                            const __half2 h = __floats2half2_rn(v.x, v.y);
                            const float2 r = __half22float2(h);
                            const float2 rest = fma(Two(r.x, r.y), Two(-1.f, -1.f), z).get();
                            hi[e] = as_u32(h), lo[e] = as_u32(__floats2half2_rn(rest.x, rest.y));
                        }
                        tmem_store8(own + 64 * g + k, hi);      // where the scores of these positions were
                        tmem_store8(own + 64 * g + k + 8, lo);
                    }
                }
            };
            if (masked) weights(std::true_type{});
            else weights(std::false_type{});
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float2 v = low[g].get();
                accm[g] = fmaf(accm[g], f, v.x + v.y);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        fence_before();
        fence_smem();
        __syncthreads();
        outputs();
        if (tid == 32) fetch(st);
        __syncwarp();
        if (after < page1) {
            const int next = (seq + 1) % S::STAGES;
            if (alive) alive = mbar_wait(full + 8 * next, (seq + 1) / S::STAGES & 1);
            __syncwarp();
            expand(ring + next * S::REC, k_tile);
            parameters(ring + next * S::REC, after);
            fence_smem();
            __syncthreads();
            scores();
        }
        p = after;
    }
    if (seq) take();

    // ---- the outputs, or a part of them --------------------------------------------------------------------------------------------------
    fence_before();
    __syncthreads();
    const float2 both = sums.get();
    float sum = both.x + both.y, out[N];
    swap[half * (1 + G) * COLS + row] = sum;
#pragma unroll
    for (int g = 0; g < G; ++g) swap[(half * (1 + G) + 1 + g) * COLS + row] = accm[g];
    __syncthreads();
    {
        const int g = half * N / GROUP;
        sum = swap[row] + swap[(1 + G) * COLS + row];
        const float low = swap[(1 + g) * COLS + row] + swap[(2 + G + g) * COLS + row];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 v = acc[i / 2].get();
            out[i] = v.x + low, out[i + 1] = v.y + low;
        }
    }
    auto store = [&](auto get, float total) {      // get(i): output i, in order
        if (!real) return;
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = total == 0.f ? 0u : as_u32(__floats2half2_rn(get(i + 2 * e) * inv, get(i + 2 * e + 1) * inv));      // no position: zeros
            *reinterpret_cast<uint4 *>(a.out + at + i) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    };
    auto in_order = [&](int i) { return out[(i & ~7) + 2 * (i & 3) + (i >> 2 & 1)]; };
    if (splits == 1) {
        store(in_order, sum);
    } else {
        const size_t first = ((size_t)pair * kvh + it.h) * a.splits;
        float *part = a.parts + (first + split) * S::PART;      // [output / 4][row][4], maxima, sums
        float4 *part4 = reinterpret_cast<float4 *>(part) + half * (N / 4) * COLS + row;
#pragma unroll
        for (int i = 0; i < N; i += 4) __stcg(part4 + i / 4 * COLS, make_float4(in_order(i), in_order(i + 1), in_order(i + 2), in_order(i + 3)));
        if (half == 0) __stcg(part + COLS * HD + row, sum == 0.f ? -INFINITY : ref), __stcg(part + COLS * (HD + 1) + row, sum);
        unsigned *counter = a.counters + (size_t)pair * kvh + it.h;
        __syncthreads();
        if (tid == 0) {
            unsigned old;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
            s_flag = old == (unsigned)(splits - 1);
        }
        __syncthreads();
        if (s_flag) {
            const float *parts = a.parts + first * S::PART;
            float top = -INFINITY, total = 0.f;
            for (int k = 0; k < splits; ++k) top = fmaxf(top, __ldcg(parts + (size_t)k * S::PART + COLS * HD + row));
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = 0.f;
            for (int k = 0; k < splits; ++k) {
                const float *other = parts + (size_t)k * S::PART;
                const float l = __ldcg(other + COLS * (HD + 1) + row), t = __ldcg(other + COLS * HD + row);
                const float4 *other4 = reinterpret_cast<const float4 *>(other) + half * (N / 4) * COLS + row;
                float4 v[N / 4];
#pragma unroll
                for (int i = 0; i < N / 4; ++i) v[i] = __ldcg(other4 + i * COLS);
                if (l == 0.f) continue;
                const float w = exp2_approx(t - top);
                total = fmaf(w, l, total);
#pragma unroll
                for (int i = 0; i < N / 4; ++i) {
                    out[4 * i] = fmaf(w, v[i].x, out[4 * i]), out[4 * i + 1] = fmaf(w, v[i].y, out[4 * i + 1]);
                    out[4 * i + 2] = fmaf(w, v[i].z, out[4 * i + 2]), out[4 * i + 3] = fmaf(w, v[i].w, out[4 * i + 3]);
                }
            }
            store([&](int i) { return out[i]; }, total);
            if (tid == 0) *counter = 0;      // ready for the next launch
        }
    }
    if (!alive) {      // a wait ran out: what is on its way lands before the block ends
        if (lane == 0) atomicExch(a.status, SAL_E_TIMEOUT);
        for (int i = 0; i < S::STAGES + 2; ++i) (void)mbar_wait(full + 8 * i, 0), (void)mbar_wait(full + 8 * i, 1);
    }
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM));
    }
}

// Bound by HBM: 44.1 us for 15 pages of 32 layers, 283 MB read and written, 98 % of the copy rate.  Page copies travel as kernel arguments: a captured launch needs no list in memory that somebody would have to keep.
constexpr int MAX_PAIRS = 256;
struct PagePairs {
    int src[MAX_PAIRS], dst[MAX_PAIRS];
};
__global__ void __launch_bounds__(256) copy_pages_kernel(uint4 *pool, const __grid_constant__ PagePairs pairs, int pages, size_t page_vecs) {
    pdl_prologue();
    uint4 *layer = pool + (size_t)blockIdx.z * pages * page_vecs;
    const uint4 *src = layer + (size_t)pairs.src[blockIdx.y] * page_vecs;
    uint4 *dst = layer + (size_t)pairs.dst[blockIdx.y] * page_vecs;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < page_vecs; i += (size_t)gridDim.x * blockDim.x) dst[i] = src[i];
}

bool aligned16(const void *a, const void *b = nullptr, const void *c = nullptr, const void *d = nullptr, const void *e = nullptr) {
    return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d) |
             reinterpret_cast<uintptr_t>(e)) & 15) == 0;
}
// Blocks of the row kernels: all heads of a row side by side (y), sequences (z), and as many rows of each as fill the GPU once.
dim3 row_grid(int batch, int m, int heads, int hd, int per_sm) {
    const long long across = ((long long)heads * (hd / 8) + ROW_THREADS - 1) / ROW_THREADS, most = 148LL * per_sm / (across * batch);
    return dim3((unsigned)(m < most ? m : most > 1 ? most : 1), (unsigned)across, (unsigned)batch);
}
int check_cache(int batch, int m, int kv_heads, int hd, int max_pages, int pages) {
    if (hd != 64 && hd != 128 && hd != 256) return SAL_E_UNSUPPORTED;
    if (batch < 1 || m < 1 || kv_heads < 1 || kv_heads > MAX_KV_HEADS || max_pages < 1 || max_pages > MAX_PAGES || pages < 1) return SAL_E_SHAPE;
    if ((long long)batch * m > SAL_KV4_MAX_ROWS || (long long)pages * kv_heads > 0x7fffffff) return SAL_E_SHAPE;
    return SAL_OK;
}

enum AttnKind { FOUR_COLUMNS, EIGHT_COLUMNS, SIXTEEN_COLUMNS, MANY_COLUMNS };
struct AttnPlan {
    AttnKind kind;
    int cols;          // columns of a tile
    int col_tiles;     // of a sequence
    int pairs;         // (sequence, column tile) pairs
    int max_blocks;    // thread blocks that share the list
};
// Columns of a sequence that share a kv head decide.  The tile's width is what a page's codes are expanded for, so it follows the columns up to what the registers
// hold (16 for heads below 256, 8 for those).  Behind 64 columns the fifth generation's tensor cores take over, in tiles of 128: 79 us against
// 134 in tiles of 64 on the older path (512 rows behind 1536 positions, 32 heads of 128), 64 against 115 (4 sequences, 128 columns, 1000 to 6000 positions),
// 26 against 65 (66 columns behind 2000); for 64 columns and fewer tiles of 16 are the faster ones: 206 against 225 (64 rows, 8 sequences), 40 against 72 (up to
// 40 columns, 6 sequences).  Heads of 256 would need all of the tensor memory and stay on the older path, in tiles of 32.
AttnPlan attention_plan(int batch, int m, int rep, int hd) {
    const int cols = m * rep;
    AttnPlan p = {};
    p.kind = cols <= 4 ? FOUR_COLUMNS : cols <= (hd < 256 ? 8 : 32) ? EIGHT_COLUMNS : cols <= 64 && hd < 256 ? SIXTEEN_COLUMNS : MANY_COLUMNS;
    p.cols = p.kind == FOUR_COLUMNS ? 4 : p.kind == EIGHT_COLUMNS ? 8 : p.kind == SIXTEEN_COLUMNS ? 16 : hd < 256 ? 128 : 32;
    p.col_tiles = (cols + p.cols - 1) / p.cols;
    p.pairs = batch * p.col_tiles;
    p.max_blocks = p.kind != MANY_COLUMNS ? 448 : hd < 256 ? WIDE_BLOCKS / 2 : 320;
    return p;
}

template <int HD, int NT, bool DUP, int WK, int PG, int WC>
int launch_tiles(const AttnArgs &a, const AttnPlan &p, void *stream) {
    using S = AttnShape<HD, NT, DUP, WK, PG, WC>;
    auto kernel = attention_tiles_kernel<HD, NT, DUP, WK, PG, WC>;
    static std::atomic<bool> configured[64];
    static std::atomic<int> resident[64];
    if (sal_allow_shared_memory(kernel, configured) != cudaSuccess) return SAL_E_LAUNCH;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return SAL_E_DEVICE;
    int blocks = resident[dev].load(std::memory_order_relaxed);
    if (blocks == 0) {
        int per_sm = 0, sms = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, S::THREADS, S::SMEM) != cudaSuccess || per_sm < 1) return SAL_E_LAUNCH;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return SAL_E_LAUNCH;
        blocks = (per_sm * sms <= p.max_blocks ? per_sm : p.max_blocks / sms > 0 ? p.max_blocks / sms : 1) * sms;      // the same number on every SM
        resident[dev].store(blocks, std::memory_order_relaxed);
    }
    const unsigned grid = a.whole ? (unsigned)p.pairs * a.c.kv_heads : (unsigned)(blocks < p.max_blocks ? blocks : p.max_blocks);
    return sal_launch_pdl(kernel, dim3(grid), dim3(S::THREADS), S::SMEM, stream, a);
}
template <int HD>
int launch_wide(const AttnArgs &a, const AttnPlan &p, void *stream) {
    static std::atomic<bool> configured[64];
    if (sal_allow_shared_memory(attention_wide_kernel<HD>, configured) != cudaSuccess) return SAL_E_LAUNCH;
    return sal_launch_pdl(attention_wide_kernel<HD>, dim3((unsigned)(p.pairs * a.c.kv_heads * a.splits)), dim3(WideShape<HD>::THREADS), WideShape<HD>::SMEM, stream, a);
}
template <int HD>
int launch_attention(const AttnArgs &a, const AttnPlan &p, void *stream) {
    switch (p.kind) {
        case FOUR_COLUMNS: return launch_tiles<HD, 1, true, 2, 2, 1>(a, p, stream);
        case EIGHT_COLUMNS: return launch_tiles<HD, 1, false, 2, 2, 1>(a, p, stream);
        case SIXTEEN_COLUMNS:
            if constexpr (HD < 256) return launch_tiles<HD, 2, false, 2, 2, 1>(a, p, stream);
        default:
            if constexpr (HD < 256) return launch_wide<HD>(a, p, stream);
            else return launch_tiles<HD, 1, false, 1, 1, 4>(a, p, stream);
    }
}

}  // namespace

extern "C" {

int sal_rope_kv4_write_f16(const void *q, const void *k, const void *v, const void *cos, const void *sin, const int64_t *pos, const int32_t *rows,
                           const int32_t *table, void *pool, void *q_out, int batch, int m, int heads, int kv_heads, int hd, int max_len,
                           int max_pages, int pages, void *stream) {
    if (!q || !k || !v || !cos || !sin || !pos || !table || !pool || !q_out) return SAL_E_NULL;
    const int rc = check_cache(batch, m, kv_heads, hd, max_pages, pages);
    if (rc != SAL_OK) return rc;
    if (heads < 1 || heads > 16384 || max_len < 1) return SAL_E_SHAPE;
    if (!aligned16(q, k, v, q_out, pool) || !aligned16(cos, sin)) return SAL_E_ALIGN;
    const CacheArgs c = {reinterpret_cast<uint8_t *>(pool), table, kv_heads, max_pages, pages};
    const dim3 grid = row_grid(batch, m, heads + 2 * kv_heads, hd, 4);
    auto kernel = hd == 64 ? rope_kv4_write_kernel<64> : hd == 128 ? rope_kv4_write_kernel<128> : rope_kv4_write_kernel<256>;
    return sal_launch_pdl(kernel, grid, dim3(ROW_THREADS), 0, stream, reinterpret_cast<const __half *>(q), reinterpret_cast<const __half *>(k),
                          reinterpret_cast<const __half *>(v), reinterpret_cast<const float *>(cos), reinterpret_cast<const float *>(sin), pos, rows, c,
                          reinterpret_cast<__half *>(q_out), m, heads, max_len);
}

int sal_read_kv4(const void *pool, const int32_t *table, const int64_t *pos, void *k_out, void *v_out, int out_f32, int batch, int m, int kv_heads,
                 int hd, int max_pages, int pages, void *stream) {
    if (!pool || !table || !pos || !k_out || !v_out) return SAL_E_NULL;
    const int rc = check_cache(batch, m, kv_heads, hd, max_pages, pages);
    if (rc != SAL_OK) return rc;
    if (!aligned16(pool, k_out, v_out)) return SAL_E_ALIGN;
    const CacheArgs c = {reinterpret_cast<uint8_t *>(const_cast<void *>(pool)), table, kv_heads, max_pages, pages};
    const dim3 grid = row_grid(batch, m, 2 * kv_heads, hd, 8);
    if (out_f32) {
        auto kernel = hd == 64 ? read_kv4_kernel<64, float> : hd == 128 ? read_kv4_kernel<128, float> : read_kv4_kernel<256, float>;
        return sal_launch_pdl(kernel, grid, dim3(ROW_THREADS), 0, stream, c, pos, reinterpret_cast<float *>(k_out), reinterpret_cast<float *>(v_out), m);
    }
    auto kernel = hd == 64 ? read_kv4_kernel<64, __half> : hd == 128 ? read_kv4_kernel<128, __half> : read_kv4_kernel<256, __half>;
    return sal_launch_pdl(kernel, grid, dim3(ROW_THREADS), 0, stream, c, pos, reinterpret_cast<__half *>(k_out), reinterpret_cast<__half *>(v_out), m);
}

size_t sal_attention_kv4_workspace_bytes(int batch, int m, int heads, int kv_heads, int hd) {
    if (check_cache(batch, m, kv_heads, hd, 1, 1) != SAL_OK || heads < 1 || heads > 16384 || heads % kv_heads) return 0;
    const AttnPlan p = attention_plan(batch, m, heads / kv_heads, hd);
    return WS_HEADER + WS_COUNTERS + (size_t)p.max_blocks * 2 * p.cols * (hd + 2) * 4;
}

int sal_attention_kv4_f16(const void *q, const void *pool, const int32_t *table, const int64_t *pos, const int32_t *rows, void *out, int batch, int m,
                          int heads, int kv_heads, int hd, int max_pages, int pages, float scale, void *workspace, size_t workspace_bytes,
                          void *stream) {
    if (!q || !pool || !table || !pos || !out || !workspace) return SAL_E_NULL;
    const int rc = check_cache(batch, m, kv_heads, hd, max_pages, pages);
    if (rc != SAL_OK) return rc;
    if (heads < 1 || heads > 16384 || heads % kv_heads) return SAL_E_SHAPE;
    if (!aligned16(q, pool, out, workspace)) return SAL_E_ALIGN;
    if (workspace_bytes < sal_attention_kv4_workspace_bytes(batch, m, heads, kv_heads, hd)) return SAL_E_WORKSPACE;
    const AttnPlan p = attention_plan(batch, m, heads / kv_heads, hd);
    uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
    AttnArgs a = {};
    a.q = reinterpret_cast<const __half *>(q);
    a.c = {reinterpret_cast<uint8_t *>(const_cast<void *>(pool)), table, kv_heads, max_pages, pages};
    a.pos = pos, a.rows = rows;
    a.out = reinterpret_cast<__half *>(out);
    a.status = reinterpret_cast<int *>(ws);
    a.counters = reinterpret_cast<unsigned *>(ws + WS_HEADER);
    a.parts = reinterpret_cast<float *>(ws + WS_HEADER + WS_COUNTERS);
    a.batch = batch, a.m = m, a.heads = heads, a.rep = heads / kv_heads;
    a.col_tiles = p.col_tiles;
    a.whole = p.pairs > MAX_LIST;
    const int items = p.pairs * kv_heads, splits = WIDE_BLOCKS / items;
    a.splits = splits < 1 ? 1 : splits > WIDE_SPLITS ? WIDE_SPLITS : splits;
    a.scale_log2 = scale * (1.4426950408889634f * UNIT);
    return hd == 64 ? launch_attention<64>(a, p, stream) : hd == 128 ? launch_attention<128>(a, p, stream) : launch_attention<256>(a, p, stream);
}

int sal_copy_kv4_pages(void *pool, const int32_t *src, const int32_t *dst, int count, int layers, int pages, size_t page_bytes, void *stream) {
    if (count == 0) return SAL_OK;
    if (!pool || !src || !dst) return SAL_E_NULL;
    if (count < 0 || layers < 1 || layers > 65535 || pages < 1 || page_bytes < 16 || page_bytes % 16) return SAL_E_SHAPE;
    if (!aligned16(pool)) return SAL_E_ALIGN;
    {   // every page is written once at most, and none that is read: the copies may then run in any order
        unsigned char *written = new (std::nothrow) unsigned char[pages]();
        if (!written) return SAL_E_LAUNCH;
        bool ok = true;
        for (int i = 0; i < count && ok; ++i) ok = dst[i] >= 0 && dst[i] < pages && !written[dst[i]]++;
        for (int i = 0; i < count && ok; ++i) ok = src[i] >= 0 && src[i] < pages && !written[src[i]];
        delete[] written;
        if (!ok) return SAL_E_SHAPE;
    }
    const size_t vecs = page_bytes / 16;
    for (int i = 0; i < count; i += MAX_PAIRS) {
        PagePairs pairs = {};
        const int n = count - i < MAX_PAIRS ? count - i : MAX_PAIRS;
        for (int j = 0; j < n; ++j) pairs.src[j] = src[i + j], pairs.dst[j] = dst[i + j];
        const size_t blocks = (vecs + 1023) / 1024;
        const int rc = sal_launch_pdl(copy_pages_kernel, dim3((unsigned)(blocks > 65535 ? 65535 : blocks), n, layers), dim3(256), 0, stream,
                                      reinterpret_cast<uint4 *>(pool), pairs, pages, vecs);
        if (rc != SAL_OK) return rc;
    }
    return SAL_OK;
}

}  // extern "C"
