// A cache of keys and values in 4 bits, in pages of 64 positions (see include/sal_decode_ops.h for the format): rows are rotated,
// quantised and stored, read back, attended to, and pages copied.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <new>

#include "sal_decode_ops.h"
#include "sal_launch.h"
#include "sal_lutgemm.h"

namespace {

constexpr int PAGE = 64;          // positions of a page
constexpr int GROUP = 64;         // numbers that share a scale
constexpr int POS_LIMIT = 1 << 30;

__device__ __forceinline__ void pdl_prologue() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
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
};

// a * c - b * s to the nearest 32-bit number of the exact sum (products split into value and error), then to 16 bits: the same
// bits as 64-bit arithmetic gives, at a fraction of its price.
__device__ __forceinline__ __half turned(float a, float c, float b, float s) {
    const float p = __fmul_rn(a, c), pe = __fmaf_rn(a, c, -p);
    const float q = __fmul_rn(b, s), qe = __fmaf_rn(b, s, -q);
    const float d = __fsub_rn(p, q), bb = __fsub_rn(d, p);
    const float de = __fsub_rn(__fsub_rn(p, __fsub_rn(d, bb)), __fadd_rn(q, bb));
    const float r = __fadd_rn(d, __fadd_rn(de, __fsub_rn(pe, qe)));
    return __float2half_rn(isfinite(r) ? r : d);   // an infinite product has no error term
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

// One warp stores the HD numbers of a row: lane l holds numbers 64 g + 2 l and 64 g + 2 l + 1 of every group g.
template <int HD>
__device__ __forceinline__ void store_row(const __half2 (&x)[HD / GROUP], uint8_t *record, bool value, int p, int lane) {
    using R = Record<HD>;
    uint8_t *codes = record + (value ? R::CODES : 0) + p * R::ROW;
    __half2 *params = reinterpret_cast<__half2 *>(record + 2 * R::CODES + (value ? R::PARAMS : 0)) + p * R::G;
#pragma unroll
    for (int g = 0; g < R::G; ++g) {
        const float2 v = __half22float2(x[g]);
        float lo = fminf(v.x, v.y), hi = fmaxf(v.x, v.y);
        const bool odd = !(fabsf(v.x) <= 65504.f && fabsf(v.y) <= 65504.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const bool bad = __any_sync(0xffffffffu, odd);
        const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
        const float s = __half2float(scale);
        const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
        int a = (int)fminf(rintf(__fmul_rn(__fsub_rn(v.x, lo), inv)), 15.f);
        int b = (int)fminf(rintf(__fmul_rn(__fsub_rn(v.y, lo), inv)), 15.f);
        if (bad) a = b = 0;
        codes[R::place(g, p) * 32 + lane] = (uint8_t)(a | b << 4);
        if (lane == 0) params[g] = bad ? __half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff)) : __half2(scale, __float2half_rn(lo));
    }
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

// One warp per head of a row: query heads are turned into q_out, key heads turned and stored, value heads stored.
template <int HD>
__global__ void __launch_bounds__(256) rope_kv4_write_kernel(const __half *q, const __half *k, const __half *v, const float *cos_t, const float *sin_t,
                                                             const int64_t *pos, const int32_t *rows, CacheArgs c, __half *q_out, int m, int heads,
                                                             int max_len) {
    constexpr int G = HD / GROUP;
    pdl_prologue();
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = blockIdx.y, b = row / m, i = row % m;
    if (unit >= heads + 2 * c.kv_heads || i >= rows_of(rows, b, m)) return;
    const int p = row_position(pos[b], i);
    if (p < 0 || p >= max_len || p >= c.max_pages * PAGE) return;
    const bool is_q = unit < heads, is_v = unit >= heads + c.kv_heads;
    const int h = is_q ? unit : is_v ? unit - heads - c.kv_heads : unit - heads;
    const __half *src = is_q ? q + ((size_t)row * heads + h) * HD : (is_v ? v : k) + ((size_t)row * c.kv_heads + h) * HD;
    __half2 x[G];
#pragma unroll
    for (int g = 0; g < G; ++g) x[g] = *reinterpret_cast<const __half2 *>(src + g * GROUP + 2 * lane);
    if (!is_v) {
        const float *cs = cos_t + (size_t)p * (HD / 2), *sn = sin_t + (size_t)p * (HD / 2);
        if constexpr (G == 1) {   // the other number of a pair lies 32 numbers on: in the other half of the warp
            const __half2 y = __shfl_xor_sync(0xffffffffu, x[0], 16);
            const int d = 2 * (lane & 15);
            const float c0 = cs[d], c1 = cs[d + 1], s0 = sn[d], s1 = sn[d + 1];
            const float2 u = __half22float2(x[0]), w = __half22float2(y);
            const float sign = lane < 16 ? 1.f : -1.f;      // b * c + a * s = b * c - a * (-s)
            x[0] = __half2(turned(u.x, c0, w.x, sign * s0), turned(u.y, c1, w.y, sign * s1));
        } else {
#pragma unroll
            for (int g = 0; g < G / 2; ++g) {
                const int d = g * GROUP + 2 * lane;
                const float2 cc = *reinterpret_cast<const float2 *>(cs + d), ss = *reinterpret_cast<const float2 *>(sn + d);
                const float2 u = __half22float2(x[g]), w = __half22float2(x[g + G / 2]);
                x[g] = __half2(turned(u.x, cc.x, w.x, ss.x), turned(u.y, cc.y, w.y, ss.y));
                x[g + G / 2] = __half2(turned(w.x, cc.x, u.x, -ss.x), turned(w.y, cc.y, u.y, -ss.y));
            }
        }
    }
    if (is_q) {
        __half *dst = q_out + ((size_t)row * heads + h) * HD;
#pragma unroll
        for (int g = 0; g < G; ++g) *reinterpret_cast<__half2 *>(dst + g * GROUP + 2 * lane) = x[g];
        return;
    }
    uint8_t *record = record_of<HD>(c, b, p, h);
    if (record) store_row<HD>(x, record, is_v, p % PAGE, lane);
}

template <typename T>
__device__ __forceinline__ void store_pair(T *dst, float a, float b);
template <>
__device__ __forceinline__ void store_pair<float>(float *dst, float a, float b) { *reinterpret_cast<float2 *>(dst) = make_float2(a, b); }
template <>
__device__ __forceinline__ void store_pair<__half>(__half *dst, float a, float b) { *reinterpret_cast<__half2 *>(dst) = __floats2half2_rn(a, b); }

// The two numbers that lane l holds of group g of a row.
template <int HD>
__device__ __forceinline__ float2 row_pair(const uint8_t *record, bool value, int p, int g, int lane) {
    using R = Record<HD>;
    const uint8_t byte = record[(value ? R::CODES : 0) + p * R::ROW + R::place(g, p) * 32 + lane];
    const float2 sl = __half22float2(reinterpret_cast<const __half2 *>(record + 2 * R::CODES + (value ? R::PARAMS : 0))[p * R::G + g]);
    return make_float2(fmaf(sl.x, (float)(byte & 15), sl.y), fmaf(sl.x, (float)(byte >> 4), sl.y));
}

template <int HD, typename T>
__global__ void __launch_bounds__(256) read_kv4_kernel(CacheArgs c, const int64_t *pos, T *k_out, T *v_out, int m) {
    pdl_prologue();
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = blockIdx.y, b = row / m, i = row % m;
    if (unit >= 2 * c.kv_heads) return;
    const bool is_v = unit >= c.kv_heads;
    const int h = is_v ? unit - c.kv_heads : unit;
    const int p = row_position(pos[b], i);
    const uint8_t *record = record_of<HD>(c, b, p, h);
    T *dst = (is_v ? v_out : k_out) + ((size_t)row * c.kv_heads + h) * HD;
#pragma unroll
    for (int g = 0; g < HD / GROUP; ++g) {
        const float2 v = record ? row_pair<HD>(record, is_v, p % PAGE, g, lane) : make_float2(0.f, 0.f);
        store_pair(dst + g * GROUP + 2 * lane, v.x, v.y);
    }
}

// One thread block per query head of a row; warps over the positions, each with its own running maximum and sum.
template <int HD>
__global__ void __launch_bounds__(128) attention_kv4_kernel(const __half *q, CacheArgs c, const int64_t *pos, const int32_t *rows, __half *out, int m,
                                                            int heads, float scale) {
    constexpr int G = HD / GROUP, NW = 4;
    __shared__ float s_m[NW], s_l[NW], s_o[NW][HD];
    pdl_prologue();
    const int head = blockIdx.x, row = blockIdx.y, b = row / m, i = row % m;
    if (i >= rows_of(rows, b, m)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int last = row_position(pos[b], i);
    if (last >= c.max_pages * PAGE) last = c.max_pages * PAGE - 1;
    const int kvh = head / (heads / c.kv_heads);
    float2 qf[G], o[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        qf[g] = __half22float2(*reinterpret_cast<const __half2 *>(q + ((size_t)row * heads + head) * HD + g * GROUP + 2 * lane));
        o[g] = make_float2(0.f, 0.f);
    }
    float mx = -INFINITY, sum = 0.f;
    for (int p = warp; p <= last; p += NW) {
        const uint8_t *record = record_of<HD>(c, b, p, kvh);
        if (!record) continue;
        float d = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float2 k = row_pair<HD>(record, false, p % PAGE, g, lane);
            d += qf[g].x * k.x + qf[g].y * k.y;
        }
        d = warp_sum(d) * scale;
        if (d == -INFINITY) continue;
        const float next = fmaxf(mx, d);
        const float old = __expf(mx - next), w = __expf(d - next);
        mx = next;
        sum = sum * old + w;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float2 v = row_pair<HD>(record, true, p % PAGE, g, lane);
            o[g] = make_float2(o[g].x * old + w * v.x, o[g].y * old + w * v.y);
        }
    }
    if (lane == 0) s_m[warp] = mx, s_l[warp] = sum;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        s_o[warp][g * GROUP + 2 * lane] = o[g].x;
        s_o[warp][g * GROUP + 2 * lane + 1] = o[g].y;
    }
    __syncthreads();
    float all = s_m[0];
    for (int w = 1; w < NW; ++w) all = fmaxf(all, s_m[w]);
    float wgt[NW], total = 0.f;
    for (int w = 0; w < NW; ++w) {
        wgt[w] = s_l[w] == 0.f ? 0.f : s_m[w] == all ? 1.f : __expf(s_m[w] - all);
        total += wgt[w] * s_l[w];
    }
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
        float acc = 0.f;
        for (int w = 0; w < NW; ++w) acc += wgt[w] * s_o[w][d];
        out[((size_t)row * heads + head) * HD + d] = __float2half_rn(total == 0.f ? 0.f : acc / total);   // no position: zero
    }
}

// Page copies travel as kernel arguments: a captured launch needs no list in memory that somebody would have to keep.
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
int check_cache(int batch, int m, int kv_heads, int hd, int max_pages, int pages) {
    if (hd != 64 && hd != 128 && hd != 256) return SAL_E_UNSUPPORTED;
    if (batch < 1 || m < 1 || kv_heads < 1 || kv_heads > 1024 || max_pages < 1 || max_pages > POS_LIMIT / PAGE || pages < 1) return SAL_E_SHAPE;
    if ((long long)batch * m > SAL_KV4_MAX_ROWS) return SAL_E_SHAPE;
    return SAL_OK;
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
    const dim3 grid((heads + 2 * kv_heads + 7) / 8, batch * m);
    auto kernel = hd == 64 ? rope_kv4_write_kernel<64> : hd == 128 ? rope_kv4_write_kernel<128> : rope_kv4_write_kernel<256>;
    return sal_launch_pdl(kernel, grid, dim3(256), 0, stream, reinterpret_cast<const __half *>(q), reinterpret_cast<const __half *>(k),
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
    const dim3 grid((2 * kv_heads + 7) / 8, batch * m);
    if (out_f32) {
        auto kernel = hd == 64 ? read_kv4_kernel<64, float> : hd == 128 ? read_kv4_kernel<128, float> : read_kv4_kernel<256, float>;
        return sal_launch_pdl(kernel, grid, dim3(256), 0, stream, c, pos, reinterpret_cast<float *>(k_out), reinterpret_cast<float *>(v_out), m);
    }
    auto kernel = hd == 64 ? read_kv4_kernel<64, __half> : hd == 128 ? read_kv4_kernel<128, __half> : read_kv4_kernel<256, __half>;
    return sal_launch_pdl(kernel, grid, dim3(256), 0, stream, c, pos, reinterpret_cast<__half *>(k_out), reinterpret_cast<__half *>(v_out), m);
}

size_t sal_attention_kv4_workspace_bytes(int batch, int m, int heads, int kv_heads, int hd) {
    if (batch < 1 || m < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || hd < 1) return 0;
    return 1024;
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
    const CacheArgs c = {reinterpret_cast<uint8_t *>(const_cast<void *>(pool)), table, kv_heads, max_pages, pages};
    auto kernel = hd == 64 ? attention_kv4_kernel<64> : hd == 128 ? attention_kv4_kernel<128> : attention_kv4_kernel<256>;
    return sal_launch_pdl(kernel, dim3(heads, batch * m), dim3(128), 0, stream, reinterpret_cast<const __half *>(q), c, pos, rows,
                          reinterpret_cast<__half *>(out), m, heads, scale);
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
