// csrc/sample_rows.cu — the next token of every row of a step, drawn with settings of the row's own from given random numbers, in one launch.
//
//   w_i = exp((x_i - max x) / temperature);  kept: x_i among the top_k largest, and the mass of the kept larger ones below top_p of all kept mass, and w_i >= min_p;
//   drawn: the first i (in index order) whose running kept mass exceeds u times the kept mass.  Equal logits are in or out together, as in sample.cu.
// Every border is a comparison of sums: a draw lies next to one of as many borders as there are candidates, so that fp32 weights (2^-24 of each) would move one draw in some ten
// thousands over a large vocabulary. Weights are computed in double and held as multiples of 2^-44: sums of these integers are exact, so nothing depends on the order of threads, and
// what is left is the rounding of a weight, 2^-45 of the largest.
// A cluster of CTAs shares a row and keeps it in shared memory: the logits are read once, whatever the settings ask for.
// The last value that stays (top_k, top_p) is found without sorting: a histogram of the distance to the largest logit, 1024 bins of 1/8 (integers: sums of counts, or of weights in three
// parts of 16 bits, so that shared memory's 32-bit additions do), added over the cluster; if the bin that holds the border is full, once more over its 1024 parts. What is left goes to one
// CTA, which compares it pair by pair. Where a top_k leaves no more than kSrFew candidates all of them go there, and the draw ends there. Only parts too full for that (hundreds of logits
// within 2^-13 that are not all equal, or beyond the last bin) are halved bit by bit.
// Bound: barriers of the cluster and what lies between them; bytes (4 a logit) and double arithmetic (some 20 instructions a weight) come to about a quarter of it over large batches.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace sllm {

namespace cg = cooperative_groups;

constexpr int kSrThreads = 512, kSrWarps = kSrThreads / 32, kSrCluster = 16;
constexpr int kSrSlice = 44 * 1024;              // logits of a CTA at most (176 KB)
constexpr int kSrBins = 1024, kSrFew = 512;      // bins; logits that one CTA compares pair by pair
constexpr double kSrOne = 17592186044416.0;      // 2^44: the weights of 720896 logits add up to less than 2^64

struct SampleRows {
    const float *logits, *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* idx;
    float* prob;
    int ld, n, slice;
};

// 2^t for -64 <= t <= 0 to 1e-14 of its value: 2^round(t) times the Taylor series of 2^f, |f| <= 1/2 (remainder 0.3466^12 / 12! = 6e-15)
__device__ __forceinline__ double sr_exp2(double t) {
    const double magic = 6755399441055744.0;                       // 1.5 * 2^52: adding it rounds to an integer, which the low bits then hold
    const double r = t + magic, f = t - (r - magic);
    const int n = __double2loint(r);
    constexpr double l = 0.693147180559945309417;
    constexpr double c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6, c7 = c6 * l / 7, c8 = c7 * l / 8, c9 = c8 * l / 9, c10 = c9 * l / 10, c11 = c10 * l / 11;
    double p = c11;
    p = fma(p, f, c10); p = fma(p, f, c9); p = fma(p, f, c8); p = fma(p, f, c7); p = fma(p, f, c6); p = fma(p, f, c5); p = fma(p, f, c4); p = fma(p, f, c3); p = fma(p, f, c2);
    p = fma(p, f, l);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
}

// The weight of a row's logits, in 2^-44
struct SrRow {
    float top;                 // the largest logit
    double rate;               // log2(e) / temperature
    __device__ __forceinline__ uint64_t weight_of(float x) const {
        if (x == top) return (uint64_t)kSrOne;
        if (x == -INFINITY || top == INFINITY) return 0;
        const double t = ((double)x - (double)top) * rate;
        return t < -64.0 ? 0 : (uint64_t)__double2ll_rn(sr_exp2(t) * kSrOne);
    }
};

// order-preserving integer image of a float
__device__ __forceinline__ uint32_t sr_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SrShared {
    uint64_t slot[2][kSrCluster];        // what the CTAs of the cluster have sent, two sums in turn
    uint64_t warp[kSrWarps], before[kSrWarps];
    // bins: counts and weights of this CTA's logits; sums over the cluster for the bins this CTA adds up, and of all CTAs' bins
    uint32_t count[kSrBins], part[3][kSrBins];
    uint64_t all_mass[kSrBins];
    uint32_t all_count[kSrBins];
    uint64_t cta_mass[kSrCluster];
    uint32_t cta_count[kSrCluster];
    // candidates, in the first CTA
    float x[kSrFew];
    int at[kSrFew];
    uint64_t w[kSrFew];
    uint32_t listed, lowest;
    // where a border lies: the bin, and what lies in bins before it and in it
    int bin;
    uint64_t mass_before;
    uint32_t count_before, count_in;
    uint32_t threshold;
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

// exclusive sum over the CTA, and the total
template <typename T>
__device__ __forceinline__ T sr_scan(T v, T* warps, T& total) {
    T upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, upto, o);
        if ((int)(threadIdx.x & 31) >= o) upto += x;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) warps[threadIdx.x >> 5] = upto;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSrWarps; ++i) {
        const T x = warps[i];
        if (i < (int)(threadIdx.x >> 5)) before += x;
        total += x;
    }
    return before + upto - v;
}

// One row, by the CTAs of a cluster.
struct SrWork {
    SrShared& sh;
    cg::cluster_group& cluster;
    SrRow r;
    const float* s_x;
    int count, rank, size, turn;
    float far;                           // distances to the largest logit beyond which a weight is 0

    __device__ __forceinline__ void barrier() { if (size == 1) __syncthreads(); else cluster.sync(); }
    __device__ __forceinline__ uint64_t weight(float x) const { return r.top - x > far ? 0 : r.weight_of(x); }      // (inf - inf is no number: not beyond)
    static __device__ __forceinline__ int bin_of(float d) { return (int)fminf(d * 8.0f, (float)(kSrBins - 1)); }
    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < kSrBins; i += kSrThreads) sh.count[i] = sh.part[0][i] = sh.part[1][i] = sh.part[2][i] = 0;
        if (threadIdx.x == 0) { sh.listed = 0; sh.lowest = 0xffffffffu; }
        __syncthreads();
    }
    __device__ __forceinline__ void add(int bin, uint64_t w, bool mass) {
        atomicAdd(&sh.count[bin], 1u);
        if (!mass) return;
        const uint32_t a = (uint32_t)w & 0xffffu, b = (uint32_t)(w >> 16) & 0xffffu, c = (uint32_t)(w >> 32);
        if (a) atomicAdd(&sh.part[0][bin], a);
        if (b) atomicAdd(&sh.part[1][bin], b);
        if (c) atomicAdd(&sh.part[2][bin], c);
    }
    static __device__ __forceinline__ uint64_t join(uint32_t a, uint32_t b, uint32_t c) { return (uint64_t)a + ((uint64_t)b << 16) + ((uint64_t)c << 32); }

    // The bin at which what has been counted (or weighed) reaches `need`, of two neighbouring bins a thread (the first one those from first_bin on): into sh.bin and what lies before it
    __device__ __forceinline__ void border(const uint64_t (&mass)[2], const uint32_t (&n)[2], int first_bin, uint64_t mass0, uint32_t n0, bool by_mass, double need) {
        uint64_t all_m;
        uint32_t all_n;
        const uint64_t m = mass0 + sr_scan(mass[0] + mass[1], sh.warp, all_m);
        const uint32_t c = n0 + sr_scan(n[0] + n[1], reinterpret_cast<uint32_t*>(sh.before), all_n);
        uint64_t mb = m;
        uint32_t cb = c;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double from = by_mass ? (double)mb : (double)cb, to = by_mass ? (double)(mb + mass[i]) : (double)(cb + n[i]);
            if (from < need && to >= need) {
                sh.bin = first_bin + 2 * (int)threadIdx.x + i;
                sh.mass_before = mb;
                sh.count_before = cb;
                sh.count_in = n[i];
            }
            mb += mass[i];
            cb += n[i];
        }
        __syncthreads();
    }

    // which bin of 1/8 (outer < 0), or which part of bin `outer`, a logit belongs to; -1: none
    __device__ __forceinline__ int place(float x, int outer) const {
        const float d = r.top - x;
        if (outer < 0) return bin_of(d);
        return bin_of(d) == outer ? (int)fminf(fmaxf((d - outer * 0.125f) * (8.0f * kSrBins), 0.0f), (float)(kSrBins - 1)) : -1;
    }

    // The least value that stays, as a key: top_k of them (by_mass false), or those that reach `share` of the mass of the logits with keys from `above` on. small: a border by count that
    // leaves no more than kSrFew candidates is not looked for; they are all in the first CTA's list then, and the answer is 0.
    __device__ uint32_t find(bool by_mass, uint64_t top_k, double share, uint32_t above, bool& small) {
        double need = (double)top_k;
        uint64_t m0 = 0;
        uint32_t n0 = 0;
        int outer = -1;
        for (;;) {
            clear();
            for (int i = threadIdx.x; i < count; i += kSrThreads) {
                const float x = s_x[i];
                const int bin = sr_key(x) >= above ? place(x, outer) : -1;
                if (bin >= 0) add(bin, by_mass ? weight(x) : 0, by_mass);
            }
            barrier();                                                   // every CTA's bins are there
            const int own = kSrBins / size, b0 = rank * own;
            uint64_t mass = 0;
            uint32_t n = 0;
            for (int i = threadIdx.x; i < own; i += kSrThreads) {
                uint32_t c = 0;
                uint64_t m = 0;
                for (int k = 0; k < size; ++k) {
                    const SrShared* o = cluster.map_shared_rank(&sh, k);
                    c += o->count[b0 + i];
                    if (by_mass) m += join(o->part[0][b0 + i], o->part[1][b0 + i], o->part[2][b0 + i]);
                }
                sh.all_count[i] = c;
                sh.all_mass[i] = m;
                mass += m;
                n += c;
            }
            uint64_t all_m;
            uint32_t all_n;
            sr_scan(mass, sh.warp, all_m);
            sr_scan(n, reinterpret_cast<uint32_t*>(sh.before), all_n);
            if ((int)threadIdx.x < size) {
                SrShared* o = cluster.map_shared_rank(&sh, threadIdx.x);
                o->cta_mass[rank] = all_m;
                o->cta_count[rank] = all_n;
            }
            barrier();
            if (by_mass && outer < 0) {
                uint64_t total = 0;
                for (int k = 0; k < size; ++k) total += sh.cta_mass[k];
                need = share * (double)total;
            }
            // the CTA whose bins hold the border; everybody looks at them
            int owner = 0;
            for (; owner < size - 1; ++owner) {
                const double to = by_mass ? (double)(m0 + sh.cta_mass[owner]) : (double)(n0 + sh.cta_count[owner]);
                if (to >= need) break;
                m0 += sh.cta_mass[owner];
                n0 += sh.cta_count[owner];
            }
            const SrShared* o = cluster.map_shared_rank(&sh, owner);
            uint64_t mm[2];
            uint32_t nn[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = 2 * threadIdx.x + i;
                mm[i] = at < own ? o->all_mass[at] : 0;
                nn[i] = at < own ? o->all_count[at] : 0;
            }
            border(mm, nn, owner * own, m0, n0, by_mass, need);
            const int bin = sh.bin;
            const uint32_t in = sh.count_in;
            m0 = sh.mass_before;
            n0 = sh.count_before;
            small = small && !by_mass && outer < 0 && n0 + in <= kSrFew;
            if (!small && in > kSrFew) {
                if (outer >= 0 || bin == kSrBins - 1) return crowded(by_mass, need, above, outer, bin);
                outer = bin;
                continue;
            }
            // candidates to the first CTA: the border's bin, or everything up to it
            SrShared* first = cluster.map_shared_rank(&sh, 0);
            for (int i = threadIdx.x; i < count; i += kSrThreads) {
                const float x = s_x[i];
                const int b = sr_key(x) >= above ? place(x, outer) : -1;
                if (b >= 0 && (small ? b <= bin : b == bin)) {
                    const uint32_t to = atomicAdd(&first->listed, 1u);
                    first->x[to] = x;
                    first->at[to] = (rank << 20) | i;
                }
            }
            barrier();
            if (small) return 0;
            if (rank == 0) {                                             // pair by pair: one stays when what lies above it is not yet enough
                const bool is = threadIdx.x < in;
                const float x = is ? sh.x[threadIdx.x] : 0.0f;
                if (is) sh.w[threadIdx.x] = by_mass ? weight(x) : 1;
                __syncthreads();
                uint64_t v = by_mass ? m0 : n0;
                for (uint32_t k = 0; k < in; ++k) v += sh.x[k] > x ? sh.w[k] : 0;
                if (is && (double)v < need) atomicMin(&sh.lowest, sr_key(x));
                __syncthreads();
                if (threadIdx.x == 0) sh.threshold = sh.lowest;
            }
            barrier();
            return cluster.map_shared_rank(&sh, 0)->threshold;
        }
    }

    // The border lies among more candidates than the list holds: all alike, or halved bit by bit
    __device__ __noinline__ uint32_t crowded(bool by_mass, double need, uint32_t above, int outer, int bin) {
        uint64_t high = 0, low = 0;
        for (int i = threadIdx.x; i < count; i += kSrThreads) {
            const float x = s_x[i];
            if (sr_key(x) < above || place(x, outer) != bin) continue;
            high = max(high, (uint64_t)sr_key(x));
            low = max(low, (uint64_t)~sr_key(x));
        }
        high = sr_all<true>(high, sh, turn, cluster);
        low = (uint32_t)~(uint32_t)sr_all<true>(low, sh, turn, cluster);
        // the largest key from `low` on at which there is enough; at `low` there is
        uint32_t from = (uint32_t)low, to = (uint32_t)high;
        while (from < to) {
            const uint32_t mid = from + (to - from + 1) / 2;
            uint64_t v = 0;
            for (int i = threadIdx.x; i < count; i += kSrThreads) {
                const float x = s_x[i];
                if (sr_key(x) >= mid && sr_key(x) >= above) v += by_mass ? weight(x) : 1;
            }
            if ((double)sr_all<false>(v, sh, turn, cluster) >= need) from = mid; else to = mid - 1;
        }
        return from;
    }
};

__global__ void __launch_bounds__(kSrThreads, 2) sample_rows_kernel(SampleRows p) {
    after_previous();
    extern __shared__ __align__(16) uint8_t sr_raw[];
    SrShared& sh = *reinterpret_cast<SrShared*>(sr_raw);
    float* s_x = reinterpret_cast<float*>(sr_raw + sizeof(SrShared));
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / size, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = min(p.n, rank * p.slice), count = min(p.n, first + p.slice) - first;
    const float* x = p.logits + (size_t)row * p.ld + first;
    int turn = 0;
    // the largest logit and the first place that has it, as one number; NaN counts as -infinity
    uint64_t best = 0;
    auto take = [&](float v, int i) {
        v = v == v ? v : -INFINITY;
        const uint64_t k = ((uint64_t)sr_key(v) << 32) | (uint32_t)~(first + i);
        best = k > best ? k : best;
        return v;
    };
    {
        const int head = min(count, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 4), body = (count - head) / 4;      // up to a multiple of 16 bytes; 16 bytes a load
        if ((int)threadIdx.x < head) s_x[threadIdx.x] = take(x[threadIdx.x], threadIdx.x);
        constexpr int kAhead = 4;
        for (int c = threadIdx.x; c < body; c += kAhead * kSrThreads) {
            float4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (c + k * kSrThreads < body) v[k] = *reinterpret_cast<const float4*>(x + head + 4 * (c + k * kSrThreads));
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int at = head + 4 * (c + k * kSrThreads);
                if (c + k * kSrThreads >= body) break;
                s_x[at] = take(v[k].x, at);
                s_x[at + 1] = take(v[k].y, at + 1);
                s_x[at + 2] = take(v[k].z, at + 2);
                s_x[at + 3] = take(v[k].w, at + 3);
            }
        }
        for (int i = head + 4 * body + threadIdx.x; i < count; i += kSrThreads) s_x[i] = take(x[i], i);
    }
    const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f, u = p.u[row];
    const int top_k = p.top_k ? p.top_k[row] : 0;
    best = sr_all<true>(best, sh, turn, cluster);
    const int arg = (int)~(uint32_t)best;
    const uint32_t top_key = (uint32_t)(best >> 32);
    SrRow r;
    r.top = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
    if (!(temperature > 0.0f) || r.top == -INFINITY) {
        if (rank == 0 && threadIdx.x == 0) {
            p.idx[row] = r.top == -INFINITY ? 0 : arg;
            if (p.prob) p.prob[row] = r.top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    r.rate = 1.4426950408889634074 / (double)temperature;
    const uint64_t least = min_p > 0.0f ? (uint64_t)__double2ll_ru(fmin((double)min_p, 1.0) * kSrOne) : 0;
    // beyond this distance a weight is below 2^-45 (or well below min_p: log2 in fp32 is off by less than a thousandth of that here)
    const float bits = min_p > 0.0f ? fminf(46.0f, -log2f(fminf(min_p, 1.0f)) + 0.01f) : 46.0f;
    SrWork w{sh, cluster, r, s_x, count, rank, size, turn, 46.0f * 0.6931472f * temperature * 1.0001f};
    const float far = bits * 0.6931472f * temperature * 1.0001f;
    uint32_t thr = 0;                                               // kept: key >= thr
    if (r.top < INFINITY) {                                         // (of infinite logits all are kept, and nothing else weighs anything)
        if (top_k > 0 && top_k < p.n) {
            bool small = true;
            thr = w.find(false, (uint64_t)top_k, 0.0, 0, small);
            if (small) {                                            // the first CTA has all that may stay
                if (rank != 0) return;
                const int n = (int)sh.listed, i = threadIdx.x;
                const float mine = i < n ? sh.x[i] : -INFINITY;
                const int at = i < n ? (sh.at[i] >> 20) * p.slice + (sh.at[i] & 0xfffff) : 0x7fffffff;
                int above = 0;
                for (int k = 0; k < n; ++k) above += sh.x[k] > mine;
                uint64_t mass = i < n && above < top_k ? w.weight(mine) : 0;
                __syncthreads();
                if (i < n) { sh.w[i] = mass; sh.at[i] = at; }
                __syncthreads();
                uint64_t all = 0, higher = 0;
                for (int k = 0; k < n; ++k) {
                    const uint64_t y = sh.w[k];
                    all += y;
                    higher += sh.x[k] > mine ? y : 0;
                }
                if (top_p > 0.0f && top_p < 1.0f && !((double)higher < (double)top_p * (double)all)) mass = 0;
                if (mass < least) mass = 0;
                __syncthreads();
                if (i < n) sh.w[i] = mass;
                __syncthreads();
                uint64_t before = 0;
                all = 0;
                for (int k = 0; k < n; ++k) {
                    const uint64_t y = sh.w[k];
                    all += y;
                    before += sh.at[k] < at ? y : 0;
                }
                const double to = u > 0.0f ? fmin((double)u, 1.0) * (double)all : 0.0;
                uint64_t target = (uint64_t)to;
                if (target >= all) target = all - 1;
                if (i < n && before <= target && target < before + mass) {
                    p.idx[row] = at;
                    if (p.prob) p.prob[row] = (float)((double)mass / (double)all);
                }
                return;
            }
        }
        if (top_p > 0.0f && top_p < 1.0f) {
            bool small = false;
            thr = max(thr, w.find(true, 0, (double)top_p, thr, small));
        }
    }
    turn = w.turn;
    auto kept = [&](float v) -> uint64_t {
        if (sr_key(v) < thr || r.top - v > far) return 0;
        const uint64_t y = r.weight_of(v);
        return y >= least ? y : 0;
    };
    // a warp owns a run of neighbouring logits: its mass first, then the one in whose run the target lies walks it
    const int run = (count + kSrWarps - 1) / kSrWarps, lo = min(count, warp * run), hi = min(count, lo + run);
    uint64_t mine = 0;
    for (int i = lo + lane; i < hi; i += 32) mine += kept(s_x[i]);
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
        for (int i = lo; i < hi; i += 32) {
            const uint64_t y = i + lane < hi ? kept(s_x[i + lane]) : 0;
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
    static bool ready = false;
    if (!ready) {
        SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SrShared) + kSrSlice * 4));
        ready = true;
    }
    int cs = 1;
    while (cs < kSrCluster && ((n + cs - 1) / cs > 16384 || ((long long)rows * cs < 2 * sm_count() && n / cs >= 2048))) cs *= 2;
    SampleRows p{logits, temperature, top_p, min_p, u, top_k, idx_dev, prob_dev, ld, n, ((n + cs - 1) / cs + 3) / 4 * 4};
    SLLM_REQUIRE((long long)rows * cs <= 0x7fffffffLL, SLLM_ENOTSUP, "sample_rows: too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)rows * cs);
    cfg.blockDim = dim3(kSrThreads);
    cfg.dynamicSmemBytes = sizeof(SrShared) + (size_t)p.slice * 4;
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
