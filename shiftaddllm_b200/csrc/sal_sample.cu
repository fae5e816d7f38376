// The next token of each sequence from its logits (see include/sal_decode_ops.h).
//
// A token's weight is w = exp((x - max) / temperature).  The filters keep a prefix of the tokens in the order of falling logits, equal
// ones by index: the first top_k; of these, while the weight in front is below top_p of their sum; of these, while w >= min_p.  So all that a
// row needs is where each prefix ends: a logit, and how many of the tokens that have it are still in.  The token is then the first, by
// index, at which the running sum of the kept weights exceeds u times their total.
//
// Weights are whole numbers in units of 2**-44 (the largest is 2**44, a sum of 2**18 of them fits 63 bits): sums do not depend on their
// order, so the same inputs give the same token however the work is split, and the running sum meets the total exactly.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sal_decode_ops.h"
#include "sal_launch.h"
#include "sal_lutgemm.h"

namespace {

typedef unsigned long long mass_t;
constexpr int UNIT_BITS = 44;
constexpr int MAX_VOCAB = 1 << 18;

__device__ __forceinline__ void pdl_prologue() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Larger logits have larger keys; 0 for what is never chosen: NaN and -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);      // -0 counts as 0
    return !(x > -INFINITY) ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// What the weights of a row need: its largest logit and log2(e) / temperature as the sum of two 32-bit numbers.
struct Weights {
    float top, c_hi, c_lo;
    __device__ __forceinline__ Weights(float top_, float temperature) : top(top_) {
        const double c = 1.4426950408889634 / (double)temperature;
        c_hi = c > 1e30 ? 1e30f : (float)c;
        c_lo = c > 1e30 ? 0.f : (float)(c - (double)c_hi);
    }
    // w in units of 2**-44.  The exponent is formed with its rounding errors (of the difference and of the product) and the error applied
    // to the power: 1.5e-7 relative, against the 1e-6 that a 32-bit exponent of 16 would cost.
    __device__ __forceinline__ mass_t operator()(float x) const {
        if (x == top) return 1ull << UNIT_BITS;
        const float d = x - top;
        const float bb = d - x;
        const float de = (x - (d - bb)) - (top + bb);
        const float t = d * c_hi;
        if (!(t > -46.f)) return 0;
        const float te = fmaf(d, c_hi, -t) + fmaf(d, c_lo, de * c_hi);
        const float w = exp2f(t);
        return (mass_t)__float2ll_rn(fmaf(w, te * 0.69314718f, w) * 17592186044416.f);
    }
};

template <typename T>
__device__ __forceinline__ T block_total(T v, T *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    T r = lane < nw ? red[lane] : T(0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    return r;
}

struct SampleArgs {
    const void *logits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int vocab;
    int64_t *token;
};

__device__ __forceinline__ float load_logit(const float *p, int i) { return p[i]; }
__device__ __forceinline__ float load_logit(const __half *p, int i) { return __half2float(p[i]); }

// One thread block per row: the ends of the prefixes are found bit by bit, with one pass over the row for each bit.
template <typename T>
__global__ void __launch_bounds__(1024) sample_kernel(SampleArgs a) {
    __shared__ mass_t red[32];
    __shared__ uint32_t red32[32];
    __shared__ mass_t s_warp[32];
    __shared__ int s_ties[32];
    __shared__ int s_token;
    pdl_prologue();
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(a.logits) + (size_t)row * a.vocab;
    const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
    float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    float u = a.u[row];
    uint32_t best = 0;
    for (int i = tid; i < a.vocab; i += blockDim.x) best = max(best, key_of(load_logit(x, i)));
    best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) red32[warp] = best;
    __syncthreads();
    best = __reduce_max_sync(0xffffffffu, red32[lane]);
    __syncthreads();
    if (best == 0) {   // nothing can be chosen
        if (tid == 0) a.token[row] = 0;
        return;
    }
    const bool greedy = !(temperature > 0.f);
    if (greedy) top_k = 1;
    const Weights weight(logit_of(best), greedy ? 1.f : temperature);
    uint32_t end = 1;                 // the kept prefix: keys above `end`, and the first `ties` of those that equal it
    int ties = a.vocab;
    if (top_k > 0 && top_k < a.vocab) {
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = key | 1u << bit;
            int n = 0;
            for (int i = tid; i < a.vocab; i += blockDim.x) n += key_of(load_logit(x, i)) >= trial;
            if (block_total<int>(n, reinterpret_cast<int *>(red)) >= top_k) key = trial;
        }
        if (key > 0) {
            int above = 0;
            for (int i = tid; i < a.vocab; i += blockDim.x) above += key_of(load_logit(x, i)) > key;
            end = key;
            ties = top_k - block_total<int>(above, reinterpret_cast<int *>(red));
        }
    }
    if (top_p < 1.f) {
        mass_t over = 0;
        int at = 0;
        for (int i = tid; i < a.vocab; i += blockDim.x) {
            const float v = load_logit(x, i);
            const uint32_t k = key_of(v);
            if (k > end) over += weight(v);
            at += k == end;
        }
        over = block_total<mass_t>(over, red);
        at = block_total<int>(at, reinterpret_cast<int *>(red));
        const mass_t all = over + (mass_t)min(ties, at) * (at ? weight(logit_of(end)) : 0);
        const double goal = (double)top_p * (double)all;
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = key | 1u << bit;
            if (trial < end) {
                key = trial;
                continue;
            }
            mass_t s = 0;
            for (int i = tid; i < a.vocab; i += blockDim.x) {
                const float v = load_logit(x, i);
                if (key_of(v) >= trial) s += weight(v);
            }
            s = block_total<mass_t>(s, red);
            if (trial <= best && ((double)s >= goal)) key = trial;
        }
        if (key > end || (key == end && end > 1)) {
            mass_t front = 0;
            for (int i = tid; i < a.vocab; i += blockDim.x) {
                const float v = load_logit(x, i);
                if (key_of(v) > key) front += weight(v);
            }
            front = block_total<mass_t>(front, red);
            const double w = (double)weight(logit_of(key));
            const double need = ceil((goal - (double)front) / w);
            const int n = need < 1. ? 1 : need > (double)a.vocab ? a.vocab : (int)need;
            ties = key == end ? min(ties, n) : n;
            end = key;
        }
    }
    const double floor_w = (min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.) * (double)(1ull << UNIT_BITS);
    // total of what is kept, then the place where the running sum passes u * total
    if (tid == 0) s_token = -1;
    mass_t total = 0, goal = 0;
    for (int pass = 0; pass < 2; ++pass) {
        mass_t sum = 0;
        int seen = 0;
        for (int i0 = 0; i0 < a.vocab; i0 += blockDim.x) {
            const int i = i0 + tid;
            const float v = i < a.vocab ? load_logit(x, i) : -INFINITY;
            const uint32_t k = i < a.vocab ? key_of(v) : 0;
            const unsigned ballot = __ballot_sync(0xffffffffu, k == end);
            if (lane == 0) s_ties[warp] = __popc(ballot);
            __syncthreads();
            int rank = seen + __popc(ballot & ((1u << lane) - 1));
            for (int w = 0; w < 32; ++w) {
                if (w < warp) rank += s_ties[w];
                seen += s_ties[w];
            }
            mass_t w = 0;
            if (k > end || (k == end && rank < ties)) {
                w = weight(v);
                if ((double)w < floor_w) w = 0;
            }
            mass_t run = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const mass_t t = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += t;
            }
            if (lane == 31) s_warp[warp] = run;
            __syncthreads();
            mass_t in_front = sum;
            for (int j = 0; j < 32; ++j) {
                if (j < warp) in_front += s_warp[j];
                sum += s_warp[j];
            }
            if (pass == 1 && w > 0 && in_front + run > goal && in_front + run - w <= goal) s_token = i;
            __syncthreads();
        }
        if (pass == 0) {
            total = sum;
            u = u > 0.f ? u : 0.f;
            const double g = (double)u * (double)total;
            goal = g < (double)(total - 1) ? (mass_t)g : total - 1;   // u >= 1 is the last kept token
        }
    }
    if (tid == 0) a.token[row] = s_token;
}

}  // namespace

extern "C" int sal_sample_token(const void *logits, int logits_f32, int rows, int vocab, const void *u, const void *temperature, const int32_t *top_k,
                                const void *top_p, const void *min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all,
                                int64_t *token, void *stream) {
    if (!logits || !u || !token) return SAL_E_NULL;
    if (rows < 1 || rows > 65535 || vocab < 1 || vocab > MAX_VOCAB) return SAL_E_SHAPE;
    const SampleArgs a = {logits, reinterpret_cast<const float *>(u), reinterpret_cast<const float *>(temperature), reinterpret_cast<const float *>(top_p),
                          reinterpret_cast<const float *>(min_p), top_k, temperature_all, top_p_all, min_p_all, top_k_all, vocab, token};
    if (logits_f32) return sal_launch_pdl(sample_kernel<float>, dim3(rows), dim3(1024), 0, stream, a);
    return sal_launch_pdl(sample_kernel<__half>, dim3(rows), dim3(1024), 0, stream, a);
}
