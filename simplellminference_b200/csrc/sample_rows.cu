// csrc/sample_rows.cu — the next token of every row of a step, drawn with settings of the row's own from given random numbers, in one launch.
//
//   w_i = exp((x_i - max x) / temperature);  kept: x_i among the top_k largest, and the mass of the kept larger ones below top_p of all kept mass, and w_i >= min_p;
//   drawn: the first i (in index order) whose running kept mass exceeds u times the kept mass.  Equal logits are in or out together, as in sample.cu.
// Every border is a comparison of sums: a draw lies next to one of as many borders as there are candidates, so that fp32 weights (2^-24 of each) would move one draw in some ten
// thousands over a large vocabulary. Weights are computed in double and held as multiples of 2^-44: sums of these integers are exact, so nothing depends on the order of threads, and
// what is left is the rounding of a weight, 2^-45 of the largest.
// A cluster of CTAs shares a row and keeps it in shared memory: the logits are read once, whatever the settings ask for.
// The last value that stays (top_k, top_p) is found without sorting. The logits are counted in 1024 bins by their distance to the largest, 1/22 of a bit of weight each, over the cluster. By count
// that names the border's bin. By weight it bounds it: the logits of a bin weigh what its two ends do, 3 % apart, so that the borders of one to a few bins are possible; only then are the weights
// outside them added up, in registers. (Bins of exact weights took four additions in shared memory a logit.) Where more than kSrPairs logits are left, the few bins are counted once more in
// 1024 parts. The rest goes to one CTA, which compares it pair by pair; parts too full for that (hundreds of logits within 2^-14 of a bit, or beyond the last bin) are halved bit by bit.
// A top_k below 7/8 of the cluster's warps needs no bins: the top_k-th largest of the warps' largest logits bounds it from below, the candidates from there on are the first CTA's, and the draw ends there.
// Bound: chains. A row passes 4 to 10 barriers of its cluster (some 1000 clocks each), a weight is a chain of 13 double operations, and 64 rows of 128256 logits fill the shared memory of the
// machine twice, so that half of them wait for the other half. Floors and times, us (fp32 logits in a captured graph): one row of 32000 0.02 (bytes) and 9.5 (a kernel that adds to one number: 1.1);
// 64 rows of 128256 5.0, and by settings: top_k of 20 to 100 with top_p 30, top_p alone 92, min_p 19, none 41, a fifth each and a fifth at temperature 0 55.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace sllm {

namespace cg = cooperative_groups;

constexpr int kSrThreads = 512, kSrWarps = kSrThreads / 32, kSrCluster = 16;
constexpr int kSrSlice = 44 * 1024;              // logits of a CTA at most (176 KB)
constexpr int kSrBins = 1024, kSrFew = 512, kSrPairs = 128;   // bins; logits that one CTA can hold; up to which it compares them pair by pair rather than have their bins divided
constexpr double kSrOne = 17592186044416.0;      // 2^44: the weights of 720896 logits add up to less than 2^64

struct SampleRows {
    const float *logits, *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* idx;
    float* prob;
    int ld, n, slice;
};

// The weight of a row's logits, in 2^-44
struct SrRow {
    float top;                 // the largest logit
    double top_d, rate;        // and as a double; 32 log2(e) / temperature
    const double* powers;      // 2^(i / 32), i < 32
    // of one no further below the largest than some 46 bits: exp(z) = 2^(k / 32) e^g with |g| <= ln 2 / 64, the Taylor series of e^g (remainder 0.0109^6 / 6! = 2e-15), rounded by adding 2^52
    __device__ __forceinline__ uint64_t weight_of(float x) const {
        if (top == INFINITY) return x == top ? (uint64_t)kSrOne : 0;
        const double magic = 6755399441055744.0;                       // 1.5 * 2^52: adding it rounds to an integer, which the low bits then hold
        const double z = (double)x - top_d, r = fma(z, rate, magic), f = fma(z, rate, -(r - magic));
        const int k = __double2loint(r);
        constexpr double l = 0.693147180559945309417 / 32, c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5;
        const double g = f * f, a = fma(fma(c5, f, c4), g, fma(c3, f, c2)), p = fma(a, g, fma(l, f, 1.0)) * powers[k & 31];
        return (uint64_t)__double_as_longlong(__hiloint2double(__double2hiint(p) + (((k >> 5) + 44) << 20), __double2loint(p)) + 4503599627370496.0) & 0xfffffffffffffull;
    }
};

// order-preserving integer image of a float
__device__ __forceinline__ uint32_t sr_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float sr_float(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct alignas(16) SrShared {
    double powers[32];
    uint64_t slot[2][kSrCluster];        // what the CTAs of the cluster have sent, two sums in turn
    uint64_t warp[kSrWarps], before[kSrWarps];
    uint32_t count[2][kSrBins];          // this CTA's logits by bin, and by part of the bins around the border
    double2 span[kSrWarps];
    uint32_t span_n[kSrWarps];
    uint64_t aside[2][kSrCluster][2];    // weights of every CTA's logits before and behind the window
    // candidates, in the first CTA
    float x[kSrFew];
    int at[kSrFew];
    uint64_t w[kSrFew];
    uint32_t listed, lowest, top_key;
    float tops[kSrCluster * kSrWarps];   // the largest logit of every warp of the cluster
    int bins[2];                         // the first and the last bin that may hold the border
    uint32_t counts[2];                  // logits in the bins before the first, and up to the last
    float threshold, highest;            // the last value that stays, and the largest logit that was compared for it
};

__device__ __forceinline__ uint64_t sr_warp_sum(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum (or maximum) over the cluster, in every thread. `turn` alternates: a slot is written again only after a barrier behind its last read.
template <bool kMax>
__device__ __forceinline__ uint64_t sr_all(uint64_t v, SrShared& sh, int& turn, cg::cluster_group& cluster) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
        v = kMax ? (w > v ? w : v) : v + w;
    }
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
    __syncthreads();
    const int size = (int)cluster.num_blocks();
    if (threadIdx.x < 32) {
        v = threadIdx.x < kSrWarps ? sh.warp[threadIdx.x] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
            v = kMax ? (w > v ? w : v) : v + w;
        }
        if ((int)threadIdx.x < size) cluster.map_shared_rank(&sh.slot[turn][0], threadIdx.x)[cluster.block_rank()] = v;
    }
    if (size == 1) __syncthreads(); else cluster.sync();
    v = 0;
    for (int i = 0; i < size; ++i) {
        const uint64_t w = sh.slot[turn][i];
        v = kMax ? (w > v ? w : v) : v + w;
    }
    turn ^= 1;
    return v;
}

// sums over the threads in front, and over all
struct SrSpan {
    double low, high;          // of bounds of the weights
    uint32_t n;
};
__device__ __forceinline__ SrSpan sr_scan(SrSpan v, SrShared& sh, bool mass, SrSpan& total) {
    SrSpan upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const bool in = (int)(threadIdx.x & 31) >= o;
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto.n, o);
        upto.n += in ? n : 0;
        if (mass) {
            const double l = __shfl_up_sync(0xffffffffu, upto.low, o), h = __shfl_up_sync(0xffffffffu, upto.high, o);
            upto.low += in ? l : 0.0;
            upto.high += in ? h : 0.0;
        }
    }
    if ((threadIdx.x & 31) == 31) {
        sh.span_n[threadIdx.x >> 5] = upto.n;
        sh.span[threadIdx.x >> 5] = make_double2(upto.low, upto.high);
    }
    __syncthreads();
    SrSpan before{0.0, 0.0, 0};
    total = before;
#pragma unroll
    for (int i = 0; i < kSrWarps; ++i) {
        const bool in = i < (int)(threadIdx.x >> 5);
        const uint32_t n = sh.span_n[i];
        total.n += n;
        before.n += in ? n : 0;
        if (mass) {
            const double2 x = sh.span[i];
            total.low += x.x;
            total.high += x.y;
            before.low += in ? x.x : 0.0;
            before.high += in ? x.y : 0.0;
        }
    }
    return SrSpan{before.low + upto.low - v.low, before.high + upto.high - v.high, before.n + upto.n - v.n};
}

// n candidates, each looked at by so many neighbouring threads that all have work
__device__ __forceinline__ int sr_share(int n) {
    int s = 32;
    while (s * n > kSrThreads) s >>= 1;
    return s;
}
template <typename T>
__device__ __forceinline__ T sr_share_sum(T v, int share) {
    for (int o = share >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One row, by the CTAs of a cluster.
struct SrWork {
    SrShared& sh;
    cg::cluster_group& cluster;
    SrRow r;
    const float* s_x;
    int lo, hi, rank, size, turn;        // this warp's run
    float mine;                          // its largest logit
    uint64_t front;                      // after a search by weight that ended with a list: the weights of this thread's logits larger than all on it,
    float highest;                       // the largest one on it; else 0 and infinity
    float far, scale;                    // distances to the largest logit beyond which a weight is 0; bins in a distance of 1: the last one begins there
    // f(logit, place in the CTA's slice) for every logit of this warp's run, if one of them is not below `least`; four at a time
    template <typename F>
    __device__ __forceinline__ void each(float least, F f) const {
        if (mine < least) return;
        int i = lo + (int)(threadIdx.x & 31);
        for (; i + 96 < hi; i += 128) {
            const float x[4] = {s_x[i], s_x[i + 32], s_x[i + 64], s_x[i + 96]};
#pragma unroll
            for (int k = 0; k < 4; ++k) f(x[k], i + 32 * k);
        }
        for (; i < hi; i += 32) f(s_x[i], i);
    }
    // f(weight, place) of those for which is(logit); four weights at a time: their arithmetic is one long chain each
    template <typename G, typename F>
    __device__ __forceinline__ void weigh(float least, G is, F f) const {
        if (mine < least || r.top - mine > far) return;
        for (int i = lo + (int)(threadIdx.x & 31); i < hi; i += 128) {
            float x[4];
            bool in[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[k] = i + 32 * k < hi ? s_x[i + 32 * k] : -INFINITY;
                in[k] = !(r.top - x[k] > far) && x[k] > -INFINITY && is(x[k]);
            }
            if (in[0] || in[1] || in[2] || in[3]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t w = r.weight_of(x[k]);
                    f(in[k] ? w : 0, x[k]);
                }
            }
        }
    }

    __device__ __forceinline__ void barrier() { if (size == 1) __syncthreads(); else cluster.sync(); }
    __device__ __forceinline__ uint64_t weight(float x) const { return r.top - x > far || x == -INFINITY ? 0 : r.weight_of(x); }      // (inf - inf is no number: not beyond)
    __device__ __forceinline__ int bin_of(float d) const { return (int)fminf(d * scale, (float)(kSrBins - 1)); }
    // The bins (parts of bins [b0, b0 + width), kSrBins of them, where inner) that may hold the border, and the logits in front and up to the last one, into sh.bins and sh.counts; the counts
    // are complete, m0 and m1 lie in front of and behind the bins. By count the border is known. By weight, the mass in front of it is less than `share` of all, and that up to its end is not:
    // (1 - share) * front < share * rest. A bin's logits weigh between what its two ends do (3 % apart, or that by the number of parts), so that the border lies in one of very few bins.
    __device__ __forceinline__ void border(const uint32_t* count, bool by_mass, uint64_t top_k, double share, bool inner, int b0, int width, uint64_t m0, uint64_t m1, uint32_t n0) {
        uint32_t n[2] = {0, 0};
        constexpr int kAhead = 8;                                        // CTAs asked at once
        for (int k0 = 0; k0 < size; k0 += kAhead) {
            uint2 c[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) c[k] = reinterpret_cast<const uint2*>(cluster.map_shared_rank(count, min(k0 + k, size - 1)))[threadIdx.x];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                n[0] += k0 + k < size ? c[k].x : 0;
                n[1] += k0 + k < size ? c[k].y : 0;
            }
        }
        double low[2] = {0.0, 0.0}, high[2] = {0.0, 0.0};
        if (by_mass) {
            // bits of weight a bin; places are rounded to 2^-12 of a bin at most, weights to whole numbers
            const float bits = 46.0f * 1.0001f / (kSrBins - 1), step = inner ? (float)width / kSrBins : 1.0f, slack = 1.0f / 1024;
            const bool even = scale > 0.0f && scale < INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = 2 * (int)threadIdx.x + i;
                const float d = (float)b0 + at * step;
                // the last bin holds everything beyond it; a temperature whose bins have no width in fp32 (or no end) tells nothing
                const float h = even ? exp2f(-bits * (d - slack)) * 1.00001f : 1.0f, l = even && !(at == kSrBins - 1 && b0 + width == kSrBins) ? exp2f(-bits * (d + step + slack)) * 0.99999f : 0.0f;
                high[i] = n[i] * ((double)h * kSrOne + 1.0);
                low[i] = n[i] * fmax((double)l * kSrOne - 1.0, 0.0);
            }
        }
        SrSpan all;
        SrSpan v = sr_scan(SrSpan{low[0] + low[1], high[0] + high[1], n[0] + n[1]}, sh, by_mass, all);
        const double front = (double)m0, behind = (double)m1, tiny = 1e-12 * (front + behind + all.high);
        if (threadIdx.x == 0) { sh.bins[0] = kSrBins; sh.bins[1] = -1; }
        __syncthreads();
        bool may[2];
        uint32_t before[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            before[i] = v.n;
            if (by_mass) {
                const double least = front + v.low, rest = behind + (all.high - v.high);                   // in front of it at least, and from it on at most
                v.low += low[i];
                v.high += high[i];
                may[i] = (1.0 - share) * (least - tiny) < share * (rest + tiny) && (1.0 - share) * (front + v.high + tiny) >= share * (behind + (all.low - v.low) - tiny);
            } else {
                may[i] = n0 + v.n < top_k && n0 + v.n + n[i] >= top_k;
            }
            v.n += n[i];
            may[i] = may[i] && n[i] > 0;
            if (may[i]) {
                atomicMin(&sh.bins[0], 2 * (int)threadIdx.x + i);
                atomicMax(&sh.bins[1], 2 * (int)threadIdx.x + i);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = 2 * (int)threadIdx.x + i;
            if (at == sh.bins[0]) sh.counts[0] = before[i];
            if (at == sh.bins[1]) sh.counts[1] = before[i] + n[i];
        }
        __syncthreads();
    }

    // this CTA's weights before and behind the window to every CTA
    __device__ __forceinline__ void send_aside(uint64_t front, uint64_t behind, int buffer) {
        front = sr_warp_sum(front);
        behind = sr_warp_sum(behind);
        if ((threadIdx.x & 31) == 0) { sh.warp[threadIdx.x >> 5] = front; sh.before[threadIdx.x >> 5] = behind; }
        __syncthreads();
        if ((int)threadIdx.x < 2 * size) {
            const uint64_t* from = threadIdx.x & 1 ? sh.before : sh.warp;
            uint64_t v = 0;
#pragma unroll
            for (int i = 0; i < kSrWarps; ++i) v += from[i];
            cluster.map_shared_rank(&sh, threadIdx.x >> 1)->aside[buffer][rank][threadIdx.x & 1] = v;
        }
    }
    __device__ __forceinline__ void take_aside(uint64_t& front, uint64_t& behind, int buffer) const {
        for (int k = 0; k < size; ++k) { front += sh.aside[buffer][k][0]; behind += sh.aside[buffer][k][1]; }
    }

    // The least value that stays: of top_k of them (by_mass false), or of those that reach `share` of the mass of the logits from `above` on. small: a border by count that
    // leaves no more than kSrFew candidates is not looked for; they are all in the first CTA's list then, and the answer is 0.
    __device__ float find(bool by_mass, uint64_t top_k, double share, float above, bool& small) {
        for (int i = threadIdx.x; i < 2 * kSrBins; i += kSrThreads) (&sh.count[0][0])[i] = 0;
        if (threadIdx.x == 0) { sh.listed = 0; sh.lowest = 0xffffffffu; }
        __syncthreads();
        each(above, [&](float x, int) {
            if (x >= above) atomicAdd(&sh.count[0][bin_of(r.top - x)], 1u);
        });
        barrier();                                                       // every CTA's bins are there, its list is empty
        uint64_t m0 = 0, m1 = 0;
        highest = INFINITY;
        border(sh.count[0], by_mass, top_k, share, false, 0, kSrBins, 0, 0, 0);
        const int b0 = sh.bins[0], b1 = sh.bins[1];
        uint32_t n0 = sh.counts[0], upto = sh.counts[1];
        small = small && !by_mass && upto <= kSrFew;
        SrShared* first = cluster.map_shared_rank(&sh, 0);
        auto list = [&](float x, int i) {
            const uint32_t to = atomicAdd(&first->listed, 1u);
            if (to >= kSrFew) return;                                    // (the counts say that they fit)
            first->x[to] = x;
            first->at[to] = (rank << 20) | i;
        };
        front = 0;
        uint64_t behind = 0;
        if (small || upto - n0 <= kSrPairs) {                            // everything up to the border, or what lies around it
            each(above, [&](float x, int i) {
                const int b = bin_of(r.top - x);
                if (x >= above && b <= b1 && (small || b >= b0)) list(x, i);
            });
            if (by_mass) {
                weigh(above, [&](float x) { const int b = bin_of(r.top - x); return x >= above && (b < b0 || b > b1); }, [&](uint64_t y, float x) {
                    front += bin_of(r.top - x) < b0 ? y : 0;
                    behind += y;
                });
                send_aside(front, behind - front, 0);
            }
            barrier();
            if (small) return 0.0f;
            if (by_mass) take_aside(m0, m1, 0);
        } else {
            const float parts = (float)kSrBins / (b1 - b0 + 1);
            auto part_of = [&](float d) { return (int)fminf(fmaxf(fmaf(d, scale, -(float)b0) * parts, 0.0f), (float)(kSrBins - 1)); };
            each(above, [&](float x, int) {
                const int b = bin_of(r.top - x);
                if (x >= above && b >= b0 && b <= b1) atomicAdd(&sh.count[1][part_of(r.top - x)], 1u);
            });
            if (by_mass) {
                weigh(above, [&](float x) { const int b = bin_of(r.top - x); return x >= above && (b < b0 || b > b1); }, [&](uint64_t y, float x) {
                    front += bin_of(r.top - x) < b0 ? y : 0;
                    behind += y;
                });
                send_aside(front, behind - front, 0);
            }
            barrier();
            if (by_mass) take_aside(m0, m1, 0);
            const uint32_t outside = n0;
            border(sh.count[1], by_mass, top_k, share, true, b0, b1 - b0 + 1, m0, m1, n0);
            const int c0 = sh.bins[0], c1 = sh.bins[1];
            n0 = outside + sh.counts[0];
            upto = outside + sh.counts[1];
            if (upto - n0 > kSrFew) {
                front = 0;
                SrWork copy = *this;                                     // (its address is taken: the fields of this one stay in registers)
                const float found = copy.crowded(by_mass, top_k, share, above);
                turn = copy.turn;
                return found;
            }
            uint64_t inner = 0;
            behind = 0;
            each(above, [&](float x, int i) {
                const int b = bin_of(r.top - x);
                if (x < above || b < b0 || b > b1) return;
                const int c = part_of(r.top - x);
                if (c >= c0 && c <= c1) list(x, i);
                else if (by_mass) {
                    const uint64_t y = weight(x);
                    inner += c < c0 ? y : 0;
                    behind += c > c1 ? y : 0;
                }
            });
            if (by_mass) send_aside(inner, behind, 1);
            front += inner;
            barrier();
            if (by_mass) take_aside(m0, m1, 1);
        }
        if (rank == 0) {                                                 // pair by pair: one stays when what lies above it is not yet enough
            const int in = min((int)(upto - n0), kSrFew), split = sr_share(in), at = threadIdx.x / split, part = threadIdx.x % split;
            const float x = at < in ? sh.x[at] : 0.0f;
            if (at < in && part == 0) sh.w[at] = by_mass ? weight(x) : 1;
            if (threadIdx.x == 0) sh.top_key = 0;
            __syncthreads();
            uint64_t v = 0, all = 0;
            if (at < in) {
#pragma unroll 4
                for (int k = part; k < in; k += split) {
                    const uint64_t y = sh.w[k];
                    all += y;
                    v += sh.x[k] > x ? y : 0;
                }
            }
            v = (by_mass ? m0 : n0) + sr_share_sum(v, split);
            all = sr_share_sum(all, split);
            const double need = by_mass ? share * (double)(m0 + m1 + all) : (double)top_k;
            if (at < in) {
                if ((double)v < need) atomicMin(&sh.lowest, sr_key(x));
                atomicMax(&sh.top_key, sr_key(x));
            }
            __syncthreads();
            if (threadIdx.x == 0) { sh.threshold = sr_float(sh.lowest); sh.highest = sr_float(sh.top_key); }
        }
        barrier();
        if (by_mass) highest = first->highest;
        return first->threshold;
    }

    // A top_k below the number of the cluster's warps: the top_k-th largest of the warps' largest logits is no larger than the top_k-th largest of all, so that the candidates lie from there
    // on; as a rule not many more than top_k. True when the first CTA's list holds all of them.
    __device__ __forceinline__ bool few(int top_k, int groups) {
        if (top_k * 8 > groups * 7) return false;
        if (threadIdx.x == 0) { sh.listed = 0; sh.lowest = 0xffffffffu; }
        __syncthreads();
        const int split = sr_share(groups), at = threadIdx.x / split;
        if (at < groups) {
            const float x = sh.tops[at];
            int larger = 0;
#pragma unroll 8
            for (int k = threadIdx.x % split; k < groups; k += split) larger += sh.tops[k] > x;
            larger = sr_share_sum(larger, split);                        // (kSrThreads / split divides groups: whole warps are here)
            if (larger < top_k) atomicMin(&sh.lowest, sr_key(x));
        }
        __syncthreads();
        const float bound = sr_float(sh.lowest);
        barrier();                                                       // the first CTA's list is empty
        SrShared* first = cluster.map_shared_rank(&sh, 0);
        each(bound, [&](float x, int i) {
            if (x >= bound) {
                const uint32_t to = atomicAdd(&first->listed, 1u);
                if (to < kSrFew) {
                    first->x[to] = x;
                    first->at[to] = (rank << 20) | i;
                }
            }
        });
        barrier();
        const bool all = cluster.map_shared_rank(&sh, 0)->listed <= kSrFew;
        barrier();                                                       // (it has been read, before the first CTA goes on)
        return all;
    }

    // The border lies among more candidates than the list holds: all alike, or halved bit by bit
    __device__ __noinline__ float crowded(bool by_mass, uint64_t top_k, double share, float above) {
        uint64_t high = 0, low = 0, all = 0;
        each(above, [&](float x, int) {
            if (x < above) return;
            high = max(high, (uint64_t)sr_key(x));
            low = max(low, (uint64_t)~sr_key(x));
            all += by_mass ? weight(x) : 0;
        });
        high = sr_all<true>(high, sh, turn, cluster);
        low = (uint32_t)~(uint32_t)sr_all<true>(low, sh, turn, cluster);
        const double need = by_mass ? share * (double)sr_all<false>(all, sh, turn, cluster) : (double)top_k;
        // the largest key from `low` on at which there is enough; at `low` there is
        uint32_t from = (uint32_t)low, to = (uint32_t)high;
        while (from < to) {
            const uint32_t mid = from + (to - from + 1) / 2;
            uint64_t v = 0;
            each(above, [&](float x, int) {
                if (sr_key(x) >= mid && x >= above) v += by_mass ? weight(x) : 1;
            });
            if ((double)sr_all<false>(v, sh, turn, cluster) >= need) from = mid; else to = mid - 1;
        }
        return sr_float(from);
    }
};

__global__ void __launch_bounds__(kSrThreads, 2) sample_rows_kernel(SampleRows p) {
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // waited for before anything is sent: every CTA of the cluster runs by then (nothing is handed over)
    after_previous();
    extern __shared__ __align__(16) uint8_t sr_raw[];
    SrShared& sh = *reinterpret_cast<SrShared*>(sr_raw);
    float* s_x = reinterpret_cast<float*>(sr_raw + sizeof(SrShared));
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / size, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = min(p.n, rank * p.slice), count = min(p.n, first + p.slice) - first;
    const float* x = p.logits + (size_t)row * p.ld + first;
    int turn = 0;
    // NaN counts as -infinity
    float best = -INFINITY;
    auto take = [&](float v) {
        v = v == v ? v : -INFINITY;
        best = fmaxf(best, v);
        return v;
    };
    // a warp owns a run of neighbouring logits
    const int run = ((count + kSrWarps - 1) / kSrWarps + 3) / 4 * 4, lo = min(count, warp * run), hi = min(count, lo + run);
    if (threadIdx.x < 32) sh.powers[threadIdx.x] = exp2(threadIdx.x / 32.0);
    {
        const int off = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 4, head = min(hi - lo, off), body = (hi - lo - head) / 4;      // up to a multiple of 16 bytes; 16 bytes a load
        s_x += (4 - off) & 3;                                        // so that they are stored 16 bytes at a time, too
        const float* from = x + lo + head;
        float* to = s_x + lo + head;
        if (lane < head) s_x[lo + lane] = take(x[lo + lane]);
        constexpr int kAhead = 4;
        for (int c = lane; c < body; c += kAhead * 32) {
            float4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (c + k * 32 < body) v[k] = *reinterpret_cast<const float4*>(from + 4 * (c + k * 32));
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (c + k * 32 >= body) break;
                *reinterpret_cast<float4*>(to + 4 * (c + k * 32)) = make_float4(take(v[k].x), take(v[k].y), take(v[k].z), take(v[k].w));
            }
        }
        for (int i = lo + head + 4 * body + lane; i < hi; i += 32) s_x[i] = take(x[i]);
    }
    const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f, u = p.u[row];
    const int top_k = p.top_k ? p.top_k[row] : 0;
    // the largest of every warp to all CTAs: the largest of all, and (below) a bound for the top_k largest
    best = warp_max(best);
    cluster.barrier_wait();
    if (size == 1) {
        if (lane == 0) sh.tops[warp] = best;
        __syncthreads();
    } else {
        if (lane < size) cluster.map_shared_rank(&sh, lane)->tops[rank * kSrWarps + warp] = best;
        cluster.sync();
    }
    const int groups = size * kSrWarps;
    SrRow r;
    r.top = -INFINITY;
    for (int i = lane; i < groups; i += 32) r.top = fmaxf(r.top, sh.tops[i]);
    r.top = warp_max(r.top);
    r.top_d = (double)r.top;
    if (!(temperature > 0.0f) || r.top == -INFINITY) {
        // the first place that has it
        uint64_t place = 0;
        if (best == r.top)
            for (int i = lo + lane; i < hi; i += 32)
                if (s_x[i] == r.top) place = max(place, (uint64_t)(uint32_t)~(first + i));
        place = sr_all<true>(place, sh, turn, cluster);
        if (rank == 0 && threadIdx.x == 0) {
            p.idx[row] = r.top == -INFINITY ? 0 : (int)~(uint32_t)place;
            if (p.prob) p.prob[row] = r.top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    r.rate = 32 * 1.4426950408889634074 / (double)temperature;
    r.powers = sh.powers;
    const uint64_t least = min_p > 0.0f ? (uint64_t)__double2ll_ru(fmin((double)min_p, 1.0) * kSrOne) : 0;
    // beyond this distance a weight is below 2^-45 (or well below min_p: log2 in fp32 is off by less than a thousandth of that here)
    const float bits = min_p > 0.0f ? fminf(46.0f, -log2f(fminf(min_p, 1.0f)) + 0.01f) : 46.0f;
    const float reach = 46.0f * 0.6931472f * temperature * 1.0001f;
    SrWork w{sh, cluster, r, s_x, lo, hi, rank, size, turn, best, 0, INFINITY, reach, (float)(kSrBins - 1) / reach};
    const float far = bits * 0.6931472f * temperature * 1.0001f;
    float thr = -INFINITY;                                          // kept: from there on
    if (r.top < INFINITY) {                                         // (of infinite logits all are kept, and nothing else weighs anything)
        if (top_k > 0 && top_k < p.n) {
            bool small = true;
            thr = w.few(top_k, groups) ? 0.0f : w.find(false, (uint64_t)top_k, 0.0, -INFINITY, small);
            if (small) {                                            // the first CTA has all that may stay
                if (rank != 0) return;
                const int n = (int)sh.listed, split = sr_share(n), i = threadIdx.x / split, part = threadIdx.x % split;
                const bool is = i < n;
                const float mine = is ? sh.x[i] : -INFINITY;
                const int at = is ? (sh.at[i] >> 20) * p.slice + (sh.at[i] & 0xfffff) : 0x7fffffff;
                int above = 0;
                if (is) {
#pragma unroll 4
                    for (int k = part; k < n; k += split) above += sh.x[k] > mine;
                }
                above = sr_share_sum(above, split);
                uint64_t mass = is && above < top_k ? w.weight(mine) : 0;
                __syncthreads();
                if (is && part == 0) { sh.w[i] = mass; sh.at[i] = at; }
                __syncthreads();
                uint64_t all = 0, higher = 0;
                if (top_p > 0.0f && top_p < 1.0f) {
                    if (is) {
#pragma unroll 4
                        for (int k = part; k < n; k += split) {
                            const uint64_t y = sh.w[k];
                            all += y;
                            higher += sh.x[k] > mine ? y : 0;
                        }
                    }
                    all = sr_share_sum(all, split);
                    higher = sr_share_sum(higher, split);
                    if (!((double)higher < (double)top_p * (double)all)) mass = 0;
                }
                if (mass < least) mass = 0;
                __syncthreads();
                if (is && part == 0) sh.w[i] = mass;
                __syncthreads();
                uint64_t before = 0;
                all = 0;
                if (is) {
#pragma unroll 4
                    for (int k = part; k < n; k += split) {
                        const uint64_t y = sh.w[k];
                        all += y;
                        before += sh.at[k] < at ? y : 0;
                    }
                }
                all = sr_share_sum(all, split);
                before = sr_share_sum(before, split);
                const double to = u > 0.0f ? fmin((double)u, 1.0) * (double)all : 0.0;
                uint64_t target = (uint64_t)to;
                if (target >= all) target = all - 1;
                if (is && part == 0 && before <= target && target < before + mass) {
                    p.idx[row] = at;
                    if (p.prob) p.prob[row] = (float)((double)mass / (double)all);
                }
                return;
            }
        }
        if (top_p > 0.0f && top_p < 1.0f) {
            bool small = false;
            thr = fmaxf(thr, w.find(true, 0, (double)top_p, thr, small));
        }
    }
    turn = w.turn;
    w.far = far;
    auto kept = [&](float v) -> uint64_t {
        if (v < thr || r.top - v > far || v == -INFINITY) return 0;
        const uint64_t y = r.weight_of(v);
        return y >= least ? y : 0;
    };
    // the mass of the warp's run first (a search for top_p's border has weighed what lies above it already), then the warp in whose run the target lies walks it
    const bool known = least == 0 && w.highest < INFINITY;
    uint64_t mine = known ? w.front : 0;
    const float high = known ? w.highest : INFINITY;
    w.weigh(thr, [&](float v) { return v >= thr && v <= high; }, [&](uint64_t y, float) { mine += y >= least ? y : 0; });
    mine = sr_warp_sum(mine);
    if (lane == 0) sh.before[warp] = mine;
    const uint64_t all = sr_all<false>(lane == 0 ? mine : 0, sh, turn, cluster);
    uint64_t before = 0;
    for (int i = 0; i < rank; ++i) before += sh.slot[turn ^ 1][i];
    for (int i = 0; i < warp; ++i) before += sh.before[i];
    const double at = u > 0.0f ? fmin((double)u, 1.0) * (double)all : 0.0;
    uint64_t target = (uint64_t)at;                                 // running > at is running > floor(at) for whole numbers
    if (target >= all) target = all - 1;
    if (before <= target && target < before + mine) {
        // a lane adds up a run of its own (an odd number of logits: no two lanes meet in a bank) to find the one with the target in it, which is then looked at logit by logit
        const int each = ((hi - lo + 31) / 32) | 1, from = min(hi, lo + lane * each), to = min(hi, from + each);
        uint64_t own = 0;
#pragma unroll 4
        for (int i = from; i < to; ++i) own += kept(s_x[i]);
        uint64_t past_own = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t z = __shfl_up_sync(0xffffffffu, past_own, o);
            if (lane >= o) past_own += z;
        }
        const int who = __ffs(__ballot_sync(0xffffffffu, before + past_own > target)) - 1, end = __shfl_sync(0xffffffffu, to, who);
        before += __shfl_sync(0xffffffffu, past_own - own, who);
        for (int i = __shfl_sync(0xffffffffu, from, who); i < end; i += 32) {
            const uint64_t y = i + lane < end ? kept(s_x[i + lane]) : 0;
            uint64_t upto = y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t z = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += z;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    p.idx[row] = first + i + lane;
                    if (p.prob) p.prob[row] = (float)((double)y / (double)all);
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
}

}  // namespace sllm

using namespace sllm;

extern "C" int sllm_sample_rows(const float* logits, int32_t ld, int32_t rows, int32_t n, const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                const float* u, int32_t* idx_dev, float* prob_dev, sllm_stream_t stream) {
    SLLM_REQUIRE(logits && u && idx_dev && rows > 0 && n > 0, SLLM_EINVAL, "sample_rows: null pointer, no rows or no logits");
    SLLM_REQUIRE(ld >= n, SLLM_EINVAL, "sample_rows: rows of %d logits lie %d apart", n, ld);
    SLLM_REQUIRE(n <= kSrCluster * kSrSlice, SLLM_ENOTSUP, "sample_rows: %d logits in a row, %d at most", n, kSrCluster * kSrSlice);
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SrShared) + kSrSlice * 4 + 16));
            return SLLM_OK;
        }))
        return rc;
    // CTAs of a row: until one holds no more than 16384 logits, and then as long as the machine has room for twice as many and they have 2048 each. The five kinds of settings in turn over 128256
    // logits, with 4, 8 and 16 CTAs, us: 64 rows 63, 55 and 67 (of 16 only 14 clusters fit at once, of the others 33), 16 rows 53, 36 and 33.
    int cs = 1;
    while (cs < kSrCluster && ((n + cs - 1) / cs > 16384 || ((long long)rows * cs < 2 * sm_count() && n / cs >= 2048))) cs *= 2;
    SampleRows p{logits, temperature, top_p, min_p, u, top_k, idx_dev, prob_dev, ld, n, ((n + cs - 1) / cs + 3) / 4 * 4};
    SLLM_REQUIRE((long long)rows * cs <= 0x7fffffffLL, SLLM_ENOTSUP, "sample_rows: too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)rows * cs);
    cfg.blockDim = dim3(kSrThreads);
    cfg.dynamicSmemBytes = sizeof(SrShared) + (size_t)p.slice * 4 + 16;
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SLLM_CUDA(cudaLaunchKernelEx(&cfg, overlapping(sample_rows_kernel), p));
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}
