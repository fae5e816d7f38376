// The next token of each sequence from its logits (see include/sal_decode_ops.h).
//
// A token's weight is w = exp((x - max) / temperature).  The filters keep a prefix of the tokens in the order of falling logits, equal
// ones by index: the first top_k; of these, while the weight in front is below top_p of their sum; of these, while w >= min_p.  So all that a
// row needs is where each prefix ends: a logit, and how many of the tokens that have it are still in.  The token is then the first, by
// index, at which the running sum of the kept weights exceeds u times their total.
//
// A row is worked on by a cluster of thread blocks, each with a slice of the row in shared memory.  The ends of the prefixes are looked for in a
// histogram of the logits, 89 bins to a factor of two in weight: counts alone say which bin holds the k-th logit, and between which bins the weights
// in front pass top_p of the total (a bin's weights are known to 0.8 % from its number).  If many tokens lie there, a second histogram divides those
// bins further.  Only what lies in the last ones is gathered, in the order of the indexes, and ranked exactly by comparing each with each; what lies in front is summed exactly.  Where that
// is everything that can be kept, one block goes on alone.  Where so many lie there that the list does not take them (equal logits), the ends are
// found bit by bit, a pass over the slices for each.
//
// Weights are whole numbers in units of 2**-44 (the largest is 2**44, a sum of 2**18 of them fits 63 bits): sums do not depend on their
// order, so the same inputs give the same token however the work is split, and the running sum meets the total exactly.
//
// Bound by the latency of four to six passes over a row in shared memory (45 % of the issue slots, 1.3 % of HBM; 230 instructions of a thread per logit
// with top-p) and of about twelve barriers of the cluster, 1 us each: 14.4 us for a row of 32000 with top-k and top-p, 40 us for 64 such rows with all
// kinds of filters, 121 us for 48 rows of 131071 with top-p, whose 192 blocks lie two to an SM on 44 of them and one on the others.
#include <cooperative_groups.h>
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
    // w in units of 2**-44, rounded down.  The exponent is formed with its rounding errors (of the difference and of the product) and the error applied
    // to the power: 3e-7 relative, against the 1e-6 that a 32-bit exponent of 16 would cost.
    __device__ __forceinline__ mass_t operator()(float x) const {
        const float d = x - top;
        const float bb = d - x;
        const float de = (x - (d - bb)) - (top + bb);
        const float t = d * c_hi;
        const float te = fmaf(d, c_hi, -t) + fmaf(d, c_lo, de * c_hi);
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(t));
        w = t > -46.f ? fmaf(w, te * 0.69314718f, w) : 0.f;
        const uint32_t b = __float_as_uint(w);
        const mass_t m = (mass_t)(b & 0x7fffffu | 0x800000u) << (UNIT_BITS - 23) >> min(127u - (b >> 23), 63u);
        return x == top ? 1ull << UNIT_BITS : m;
    }
};

struct SampleArgs {
    const void *logits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int vocab;
    int slice;       // tokens of a block, a multiple of 8
    int64_t *token;
};

constexpr int MAX_WARPS = 32;
constexpr int BINS = 4096;
constexpr float BIN_SCALE = 89.f;                  // bins to a factor of two: 46 factors fit, behind them a weight is 0
constexpr int LIST = 1024;                         // tokens that can be ranked
constexpr int ALONE = 512;                         // so few that one block finishes, a token per thread
constexpr int FEW = 256;                           // a window of so many is ranked at once
constexpr int MAX_CLUSTER = 8;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// What the blocks of a cluster tell one another; `round` alternates the places, so that one barrier a round is enough.
struct Told {
    mass_t mass;
    double bound;
    unsigned long long best;
    int count;
};
struct Found {
    float end;          // the kept prefix: logits above `end`, and the first `ties` of those that equal it
    int ties;
    mass_t mass;        // of the kept prefix
};
struct alignas(16) SampleShared {
    Told told[2];
    Found found;
    int2 windows[2][2];     // first bin and the tokens in front of it, last bin and the tokens up to it; two places in turn
    mass_t warp_mass[MAX_WARPS];
    double warp_bound[MAX_WARPS];
    int warp_count[MAX_WARPS];
    unsigned long long warp_best[MAX_WARPS];
    mass_t block_mass;
    int block_count;
    uint32_t hist[BINS];
    float list_x[LIST];
    int list_i[LIST];
    mass_t list_w[LIST];
    mass_t list_before[LIST];
    int list_place[LIST];
};

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename V>
__device__ __forceinline__ V warp_running(V v, int lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(SampleArgs a) {
    constexpr int WARPS = THREADS / 32;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(smem);
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / blocks;
    const int2 no_first = make_int2(0, 0), no_last = make_int2(BINS - 1, 0x7fffffff);      // where no thread finds an end
    for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
    if (tid < 2) s.windows[tid][0] = no_first, s.windows[tid][1] = no_last;
    pdl_prologue();
    const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
    const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    const float u = a.u[row];

    // ---- the slice into shared memory; its largest logit, the first of equal ones ------------------------------------
    const int n0 = rank * a.slice, n = min(a.slice, a.vocab - n0);      // may be none
    const T *src = reinterpret_cast<const T *>(a.logits) + (size_t)row * a.vocab + n0;
    constexpr int VEC = 16 / sizeof(T);
    const int off = (int)(reinterpret_cast<uintptr_t>(src) & 15) / (int)sizeof(T);      // of the slice's first token in its 16 bytes
    T *const slice = reinterpret_cast<T *>(smem + sizeof(SampleShared));
    auto x = [&](int i) { return to_float(slice[off + i]); };
    float top = -INFINITY;
    int top_i = 0x7fffffff;
#pragma unroll 4
    for (int v = tid; v * VEC - off < n; v += THREADS) {
        const int i0 = v * VEC - off;
        uint4 raw;
        T *t = reinterpret_cast<T *>(&raw);
        if (i0 >= 0 && i0 + VEC <= n) {
            raw = *reinterpret_cast<const uint4 *>(src + i0);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) t[k] = i0 + k >= 0 && i0 + k < n ? src[i0 + k] : T(-INFINITY);
        }
        *reinterpret_cast<uint4 *>(slice + v * VEC) = raw;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float f = to_float(t[k]);
            if (f > top) top = f, top_i = n0 + i0 + k;      // never NaN or -infinity
        }
    }
    {
        unsigned long long best = top_i == 0x7fffffff ? 0ull : (unsigned long long)key_of(top) << 32 | (uint32_t)~top_i;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) s.warp_best[warp] = best;
        __syncthreads();
        best = lane < WARPS ? s.warp_best[lane] : 0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (tid == 0) s.told[0].best = best;
    }
    cluster.sync();
    unsigned long long best = lane < blocks ? cluster.map_shared_rank(&s.told[0], lane)->best : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    const int best_i = (int)~(uint32_t)best;
    // nothing can be chosen, or only one: 0, or the largest
    if (best == 0 || !(temperature > 0.f) || top_k == 1 || top_p <= 0.f) {
        if (rank == 0 && tid == 0) a.token[row] = best == 0 ? 0 : best_i;
        cluster.sync();      // nobody leaves while its memory may be read
        return;
    }
    top = logit_of((uint32_t)(best >> 32));
    const Weights weight(top, temperature);
    // A logit's place on the scale of the bins.  The histogram covers the coarse bins `from` .. `upto`, all of them at first.
    const float bins = weight.c_hi * BIN_SCALE;
    auto place_of = [&](float v) { return v == top ? 0.f : fminf((top - v) * bins, (float)(BINS - 1)); };
    int from = 0, upto = BINS - 1;
    float fine = 1.f;      // bins to a coarse one
    auto bin_at = [&](float t) { return fine == 1.f ? (int)t : (int)fminf((t - (float)from) * fine, (float)(BINS - 1)); };      // of a place in the range
    if (top_k <= 0 || top_k >= a.vocab) top_k = 0;
    const bool has_p = top_p < 1.f;
    const mass_t floor_w = min_p > 0.f ? (mass_t)ceil((double)fminf(min_p, 1.f) * (double)(1ull << UNIT_BITS)) : 0;
    int round = 1;
    // Sum over the cluster of what the blocks tell, and over the blocks in front.  Thread 0's numbers count.
    Told all, front;
    auto exchange = [&](mass_t mass, int count, double bound) {
        Told &mine = s.told[round & 1];
        if (tid == 0) mine.mass = mass, mine.count = count, mine.bound = bound;
        cluster.sync();
        Told t = {};
        if (lane < blocks) t = *cluster.map_shared_rank(&mine, lane);
        ++round;
        const bool before = lane < rank;
        all.mass = warp_total(t.mass), all.count = warp_total(t.count), all.bound = warp_total(t.bound);
        front.mass = warp_total(before ? t.mass : 0ull), front.count = warp_total(before ? t.count : 0), front.bound = warp_total(before ? t.bound : 0.);
    };
    // sums over the block; every thread gets them, and those of the warps in front of its own
    mass_t warps_mass;
    int warps_count;
    auto block_sums = [&](mass_t mass, int count) {      // of the whole warp each
        __syncthreads();
        if (lane == 0) s.warp_mass[warp] = mass, s.warp_count[warp] = count;
        __syncthreads();
        const mass_t m = lane < WARPS ? s.warp_mass[lane] : 0ull;
        const int c = lane < WARPS ? s.warp_count[lane] : 0;
        warps_mass = warp_total(lane < warp ? m : 0ull), warps_count = warp_total(lane < warp ? c : 0);
        if (warp == 0) {
            const mass_t bm = warp_total(m);
            const int bc = warp_total(c);
            if (lane == 0) s.block_mass = bm, s.block_count = bc;
        }
        __syncthreads();
    };
    // a warp's part of the slice: neighbouring tokens, so that its order is the order of the indexes
    const int part = ((max(n, 0) + WARPS - 1) / WARPS + 31) / 32 * 32;
    const int w0 = min(warp * part, max(n, 0)), w1 = min(w0 + part, max(n, 0));

    mass_t warp_front = 0, warp_kept = 0;      // of the warp's part: the weights in front of the bin `from`, and those of them that min_p keeps
    bool front_known = false;
    float end = -INFINITY;      // everything is kept, as far as it can be chosen
    int ties = 0;

    // ---- the ends bit by bit: the largest key at and above which there are `k` tokens, or weights of `goal` ----------------------------------
    auto by_bits = [&](bool by_mass, int k, double goal) {
        uint32_t key = 0;
        mass_t in_front_m = 0;
        int in_front_c = 0;
        for (int bit = 31; bit >= -1; --bit) {
            const uint32_t trial = bit >= 0 ? key | 1u << bit : key + 1;      // at last: what lies above the key
            mass_t m = 0;
            int c = 0;
            for (int i = tid; i < n; i += THREADS) {
                const uint32_t q = key_of(x(i));
                if (q >= trial && q > 0) m += weight(x(i)), ++c;
            }
            block_sums(warp_total(m), warp_total(c));
            exchange(s.block_mass, s.block_count, 0.);
            if (bit < 0) in_front_m = all.mass, in_front_c = all.count;
            else if (by_mass ? (double)all.mass >= goal && trial <= (uint32_t)(best >> 32) : all.count >= k) key = trial;
        }
        end = logit_of(key);
        const mass_t w = weight(end);
        int t;
        if (by_mass) {
            const double need = ceil((goal - (double)in_front_m) / (double)w);
            t = need < 1. ? 1 : need > (double)a.vocab ? a.vocab : (int)need;
        } else {
            t = k - in_front_c;
        }
        ties = t;
        return in_front_m + (mass_t)t * w;      // the weights of the prefix
    };
    // ---- tokens of the bins lo .. hi into the list of the cluster's first block, in the order of the indexes; exact weights in front ----------
    int listed;
    mass_t ahead;
    auto gather = [&](int lo, int hi, bool by_mass) {
        // places of the bins: where the histogram is a fine one, its range first
        const bool narrowed = fine != 1.f;
        const float p0 = narrowed ? (float)from : (float)lo, p1 = narrowed ? (float)(upto + 1) : (float)(hi + 1);
        auto in_window = [&](float t) {
            const int b = bin_at(t);
            return b >= lo && b <= hi;
        };
        mass_t m = 0, kept = 0;
        int c = 0;
#pragma unroll 2
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const float v = i < w1 ? x(i) : -INFINITY;
            const float t = v > -INFINITY ? place_of(v) : (float)BINS;
            bool in = t >= p0 && t < p1;
            if (narrowed && in) {
                if (bin_at(t) < lo) m += weight(v);
                in = in_window(t);
            } else if (!narrowed && by_mass && t < p0) {
                const mass_t w = weight(v);
                m += w;
                if (floor_w > 0 && w >= floor_w) kept += w;
            }
            c += __popc(__ballot_sync(0xffffffffu, in));
        }
        if (floor_w == 0) kept = m;
        m = warp_total(m);
        if (narrowed) {
            m += warp_front;
        } else if (by_mass) {
            from = lo;
            warp_front = m, warp_kept = warp_total(kept), front_known = true;
        }
        block_sums(m, c);
        exchange(s.block_mass, s.block_count, 0.);
        listed = all.count, ahead = all.mass;
        if (listed > LIST) return;
        int at = front.count + warps_count;
        SampleShared &first = *cluster.map_shared_rank(&s, 0);
        if (c > 0)
#pragma unroll 2
            for (int i0 = w0; i0 < w1; i0 += 32) {
                const int i = i0 + lane;
                const float v = i < w1 ? x(i) : -INFINITY;
                const float t = v > -INFINITY ? place_of(v) : (float)BINS;
                const bool in = t >= p0 && t < p1 && in_window(t);
                const unsigned all_in = __ballot_sync(0xffffffffu, in);
                if (in) {
                    const int to = at + __popc(all_in & ((1u << lane) - 1));
                    first.list_x[to] = v, first.list_i[to] = n0 + i, first.list_w[to] = weight(v);
                }
                at += __popc(all_in);
            }
        cluster.sync();
    };
    // Ranks of the listed tokens and the weights in front of them (equal logits: the lower index first): a token per warp, the others over its lanes.
    auto rank_all = [&](auto use) {
        const int count = min(listed, LIST);
        for (int i = warp; i < count; i += WARPS) {
            const float v = s.list_x[i];
            int place = 0;
            mass_t before = 0;
            for (int j = lane; j < count; j += 32) {
                const float o = s.list_x[j];
                if (o > v || (o == v && j < i)) ++place, before += s.list_w[j];
            }
            place = __reduce_add_sync(0xffffffffu, place), before = warp_total(before);
            if (lane == 0) use(i, place, before);
        }
    };
    // The first block finds the last kept token of the list; false if it is not there.  Rounding cannot push it out of the window (a bin's bounds are
    // off by 5e-6 where their sum matters, the window is 1e-5 wider), but nothing is made of shared memory that no thread wrote.
    mass_t prefix;      // the weights of the prefix
    auto settle = [&](bool by_mass, int k, double goal) {
        if (rank == 0) {
            if (tid == 0) s.found.ties = 0;
            __syncthreads();
            rank_all([&](int i, int place, mass_t before) {
                const mass_t w = s.list_w[i];
                // the last one kept: the k-th, or the one with which the weights pass the goal
                const bool last = by_mass ? (double)(ahead + before) < goal && (double)(ahead + before + w) >= goal : place == k - 1;
                if (last) {
                    int equal = 1;
                    for (int j = 0; j < i; ++j) equal += s.list_x[j] == s.list_x[i];
                    const Found f = {s.list_x[i], equal, ahead + before + w};
                    s.found = f;
                }
            });
        }
        cluster.sync();
        const Found f = cluster.map_shared_rank(&s, 0)->found;
        if (f.ties == 0) return false;
        end = f.end, ties = f.ties, prefix = f.mass;
        return true;
    };

    bool done = false;
    if (top_k > 0 || has_p) {
        mass_t total = 0;
        int before_c = 0, upto_c = 0;               // tokens of the histogram in front of this thread's bins, and with them
        double before_b = 0., upto_b = 0., all_b = 0., ratio = 0.;      // their weights at most; a bin's are above `ratio` of that
        const int mine = BINS / blocks, per = mine > THREADS ? mine / THREADS : 1;      // bins of a block and of a thread (of the first threads, where there are fewer bins)
        const int bin0 = rank * mine + min(tid * per, mine), bin1 = rank * mine + min(tid * per + per, mine);
        auto upper = [&](int b) { return (double)exp2f(-((float)from + (float)b / fine) / BIN_SCALE); };
        // ---- histogram, its running sums over the cluster: a block has BINS / blocks bins, a thread a few neighbouring ones ---------------------
        auto survey = [&](bool weights) {      // the weights in front of the bins, or of everything if these are all
            mass_t m = 0, kept = 0, sum = 0;
            const float lo = (float)from, hi = (float)(upto + 1);
#pragma unroll 2
            for (int i = w0 + lane; i < w1; i += 32) {
                const float v = x(i);
                if (!(v > -INFINITY)) continue;
                const float t = place_of(v);
                if (t >= lo && t < hi) atomicAdd(&s.hist[bin_at(t)], 1u);
                if (weights && (fine == 1.f || t < lo)) {
                    const mass_t w = weight(v);
                    m += w;
                    if (floor_w > 0 && w >= floor_w) kept += w;
                }
            }
            if (floor_w == 0) kept = m;
            m = warp_total(m);
            if (weights && fine != 1.f) warp_front = m, warp_kept = warp_total(kept), front_known = true;
            if (weights) {
                block_sums(m, 0);
                exchange(s.block_mass, 0, 0.);
                sum = all.mass;
            } else {
                cluster.sync();
            }
            int c = 0;
            double bound = 0.;      // no weight of a bin is above its upper end's
            for (int b = bin0; b < bin1; ++b) {
                int h = 0;
                for (int o = 0; o < blocks; ++o) h += (int)cluster.map_shared_rank(&s, o)->hist[b];
                c += h;
                bound += h * upper(b);
                if (blocks > 1) s.hist[b] = h;      // nobody else reads these of this block
            }
            const int run_c = warp_running(c, lane);
            const double run_b = warp_running(bound, lane);
            __syncthreads();
            if (lane == 31) s.warp_count[warp] = run_c, s.warp_bound[warp] = run_b;
            __syncthreads();
            const int in_c = lane < WARPS ? s.warp_count[lane] : 0;
            const double in_b = lane < WARPS ? s.warp_bound[lane] : 0.;
            const int warps_c = warp_total(lane < warp ? in_c : 0), block_c = warp_total(in_c);
            const double warps_b = warp_total(lane < warp ? in_b : 0.), block_b = warp_total(in_b);
            exchange(0ull, block_c, block_b);
            upto_c = front.count + warps_c + run_c, before_c = upto_c - c;
            upto_b = front.bound + warps_b + run_b, before_b = upto_b - bound;
            all_b = all.bound;
            ratio = (double)exp2f(-1.f / (BIN_SCALE * fine)) - 4e-6;
            return sum;
        };
        // Finds the first and the last bin that can hold the k-th token, or the one with which the weights pass a goal; each is found
        // by one thread, which tells the first block.
        int place = 0;
        int2 window[2];
        auto look = [&](bool by_mass, int k, double goal) {
            auto tell = [&](int which, int bin, int tokens) {
                cluster.map_shared_rank(&s, 0)->windows[place][which] = make_int2(bin, tokens);
            };
            place ^= 1;
            if (tid == 0) s.windows[place ^ 1][0] = no_first, s.windows[place ^ 1][1] = no_last;      // for the next time: a barrier lies between
            const double slack = 1e-5 * (all_b < goal ? all_b : goal), low = goal - slack, high = goal + slack;
            if (by_mass ? (before_b < low && upto_b >= low) || (before_b * ratio < high && upto_b * ratio >= high) : before_c < k && upto_c >= k) {
                int at = before_c;
                double w = before_b;
                for (int b = bin0; b < bin1; ++b) {
                    const int h = (int)s.hist[b];
                    const double next = w + h * upper(b);
                    if (by_mass ? w < low && next >= low : at < k && at + h >= k) tell(0, b, at);
                    if (by_mass ? w * ratio < high && next * ratio >= high : at < k && at + h >= k) tell(1, b, at + h);
                    at += h, w = next;
                }
            }
            cluster.sync();
            // one copy for all blocks: they have to agree on it, even where rounding let two threads find an end
            const SampleShared &first = *cluster.map_shared_rank(&s, 0);
            window[0] = first.windows[place][0], window[1] = first.windows[place][1];
        };
        // The same in two steps: where the window holds too many tokens to be ranked, it is surveyed again with bins that much finer.
        auto narrow = [&](bool by_mass, int k, double goal) {
            if (window[1].y - window[0].y <= FEW) return;
            const int in_front = window[0].y;
            from = window[0].x, upto = window[1].x, fine = (float)BINS / (float)(upto - from + 1);
            __syncthreads();
            for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
            __syncthreads();
            const mass_t ahead_of = survey(has_p);
            look(by_mass, k - in_front, (goal - (double)ahead_of) / (double)(1ull << UNIT_BITS));
            window[0].y += in_front;      // tokens in front of it in all
        };
        total = survey(has_p);
        if (all.count <= top_k) top_k = 0;      // no more than that can be chosen at all
        if (top_k > 0) look(false, top_k, 0.);
        else if (has_p) look(true, 0, (double)top_p * (double)total / (double)(1ull << UNIT_BITS));
        if (top_k == 0 && !has_p) {
            // nothing to look for
        } else if (window[1].y <= ALONE) {
            // ---- all that can be kept fits one block, a token per thread --------------------------------------------------------------------------
            gather(0, window[1].x, false);
            if (rank == 0) {
                int place = 0x7fffffff;
                mass_t before = 0, w = 0;
                rank_all([&](int i, int p, mass_t b) { s.list_place[i] = p, s.list_before[i] = b; });
                __syncthreads();
                if (tid < listed) {
                    place = s.list_place[tid], before = s.list_before[tid];
                    if (top_k == 0 || place < top_k) w = s.list_w[tid];
                }
                if (has_p) {
                    mass_t sum = total;
                    if (top_k > 0) block_sums(warp_total(w), 0), sum = s.block_mass;
                    if (place > 0 && !((double)before < (double)top_p * (double)sum)) w = 0;
                }
                if (w < floor_w) w = 0;
                const mass_t run = warp_running(w, lane);
                block_sums(__shfl_sync(0xffffffffu, run, 31), 0);
                const mass_t sum = s.block_mass, last = warps_mass + run;
                const double g = (double)(u > 0.f ? u : 0.f) * (double)sum;
                const mass_t goal = g < (double)(sum - 1) ? (mass_t)g : sum - 1;      // u >= 1 is the last kept token
                if (w > 0 && last > goal && last - w <= goal) a.token[row] = s.list_i[tid];
            }
            done = true;
        } else {
            if (top_k > 0) {
                narrow(false, top_k, 0.);
                const int in_front = window[0].y;
                gather(window[0].x, window[1].x, has_p);      // the prefix's weights are what top_p is of
                total = listed <= LIST && settle(false, top_k - in_front, 0.) ? prefix : by_bits(false, top_k, 0.);
            }
            if (has_p) {
                const float k_end = end;
                const int k_ties = ties;
                const double goal = (double)top_p * (double)total;
                if (top_k > 0) {
                    const bool narrowed = fine != 1.f;
                    from = 0, upto = BINS - 1, fine = 1.f, front_known = false;      // the whole range again
                    if (narrowed) {
                        __syncthreads();
                        for (int i = tid; i < BINS; i += THREADS) s.hist[i] = 0;
                        __syncthreads();
                        survey(false);
                    }
                    look(true, 0, goal / (double)(1ull << UNIT_BITS));
                }
                narrow(true, 0, goal);
                gather(window[0].x, window[1].x, true);
                if (listed > LIST || !settle(true, 0, goal)) (void)by_bits(true, 0, goal);
                if (top_k > 0 && end == k_end) ties = min(ties, k_ties);      // the second prefix is part of the first
            }
        }
    }

    if (!done) {
        // ---- what is kept, in the order of the indexes: sums of the warps, the blocks, then the place in one warp ---------------------------------
        mass_t m = 0;
        int c = 0;
        const float p0 = front_known ? (float)from : 0.f;
#pragma unroll 2
        for (int i = w0 + lane; i < w1; i += 32) {
            const float v = x(i);
            if (v > end) {
                if (place_of(v) < p0) continue;      // counted already
                const mass_t w = weight(v);
                if (w >= floor_w) m += w;
            } else if (v == end && end > -INFINITY) {
                ++c;
            }
        }
        m = warp_total(m) + (front_known ? warp_kept : 0), c = warp_total(c);
        mass_t tie_w = end > -INFINITY ? weight(end) : 0;
        if (tie_w < floor_w) tie_w = 0;
        block_sums(m, c);
        exchange(s.block_mass, s.block_count, 0.);
        // equal logits at the end: the first `ties` of them, so a block's share depends on those in front
        mass_t sum = 0, in_front = 0;
        for (int o = 0, seen = 0; o < blocks; ++o) {
            const Told &t = *cluster.map_shared_rank(&s.told[(round - 1) & 1], o);
            const mass_t all_of = t.mass + (mass_t)max(0, min(ties - seen, t.count)) * tie_w;
            if (o < rank) in_front += all_of;
            sum += all_of;
            seen += t.count;
        }
        const double g = (double)(u > 0.f ? u : 0.f) * (double)sum;
        const mass_t goal = g < (double)(sum - 1) ? (mass_t)g : sum - 1;      // u >= 1 is the last kept token
        const int seen = front.count + warps_count;
        const mass_t mine = m + (mass_t)max(0, min(ties - seen, c)) * tie_w;
        const int seen_block = front.count;
        const mass_t at = in_front + warps_mass + (mass_t)max(0, min(ties - seen_block, warps_count)) * tie_w;
        if (at <= goal && at + mine > goal) {      // this warp's part holds it
            mass_t run = at;
            int tie = seen;
            for (int i0 = w0; i0 < w1; i0 += 32) {
                const int i = i0 + lane;
                const float v = i < w1 ? x(i) : -INFINITY;
                const unsigned equal = __ballot_sync(0xffffffffu, v == end && end > -INFINITY);
                mass_t w = 0;
                if (v > end) {
                    w = weight(v);
                    if (w < floor_w) w = 0;
                } else if ((equal >> lane & 1) && tie + __popc(equal & ((1u << lane) - 1)) < ties) {
                    w = tie_w;
                }
                const mass_t upto = run + warp_running(w, lane);
                if (w > 0 && upto > goal && upto - w <= goal) a.token[row] = n0 + i;
                run = __shfl_sync(0xffffffffu, upto, 31);
                tie += __popc(equal);
                if (run > goal) break;
            }
        }
    }
    cluster.sync();      // nobody leaves while its memory may be read
}

template <typename T>
int launch_sample(SampleArgs a, int rows, void *stream) {
    // Blocks of a row: enough to fill the GPU with few rows, a slice of 4096 tokens or more each, as far as shared memory goes.
    int blocks = MAX_CLUSTER;
    while (blocks > 1 && (a.vocab / blocks < 2048 || (long long)rows * blocks > 2 * 148)) {
        if (a.vocab / (blocks / 2) > 36000) break;
        blocks /= 2;
    }
    a.slice = ((a.vocab + blocks - 1) / blocks + 7) / 8 * 8;
    const size_t smem = sizeof(SampleShared) + ((size_t)a.slice + 16) * sizeof(T);
    // Twice the threads where a block has an SM to itself and a long slice (one row of 131071, top-p: 41.5 us, 46.5 with 512; of 32000: 25.5, 22).
    const bool wide = (long long)rows * blocks <= 148 && a.slice > 8192;
    static std::atomic<bool> configured[2][64];
    auto kernel = wide ? sample_kernel<T, 1024> : sample_kernel<T, 512>;
    if (sal_allow_shared_memory(kernel, configured[wide]) != cudaSuccess) return SAL_E_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * blocks);
    cfg.blockDim = dim3(wide ? 1024 : 512);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)blocks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? SAL_OK : SAL_E_LAUNCH;
}

}  // namespace

extern "C" int sal_sample_token(const void *logits, int logits_f32, int rows, int vocab, const void *u, const void *temperature, const int32_t *top_k,
                                const void *top_p, const void *min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all,
                                int64_t *token, void *stream) {
    if (!logits || !u || !token) return SAL_E_NULL;
    if (rows < 1 || rows > 65535 || vocab < 1 || vocab > MAX_VOCAB) return SAL_E_SHAPE;
    const SampleArgs a = {logits, reinterpret_cast<const float *>(u), reinterpret_cast<const float *>(temperature), reinterpret_cast<const float *>(top_p),
                          reinterpret_cast<const float *>(min_p), top_k, temperature_all, top_p_all, min_p_all, top_k_all, vocab, 0, token};
    return logits_f32 ? launch_sample<float>(a, rows, stream) : launch_sample<__half>(a, rows, stream);
}
