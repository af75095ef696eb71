// csrc/sample_rows.cu — the next token of every row of a step, drawn with settings of the row's own from given random numbers, in one launch.
//
//   w_i = exp((x_i - max x) / temperature);  kept: x_i among the top_k largest, and the mass of the kept larger ones below top_p of all kept mass, and w_i >= min_p;
//   drawn: the first i (in index order) whose running kept mass exceeds u times the kept mass.  Equal logits are in or out together, as in sample.cu.
// Every border is a comparison of sums: a draw lies next to one of as many borders as there are candidates, so that fp32 weights (2^-24 of each) would move one draw in some ten
// thousands over a large vocabulary. Weights are computed in double and held as multiples of 2^-44: sums of these integers are exact, so nothing depends on the order of threads, and
// what is left is the rounding of a weight, 2^-45 of the largest.
// A cluster of CTAs shares a row and keeps it in shared memory: the logits are read once, whatever the settings ask for.
// The last value that stays (top_k, top_p) is found without sorting: a histogram of the distance to the largest logit, 1024 bins of 1/22 of a bit of weight (integers: sums of counts, or of weights in three
// parts of 16 bits, so that shared memory's 32-bit additions do), added over the cluster; if the bin that holds the border is full, once more over its 1024 parts. What is left goes to one
// CTA, which compares it pair by pair. Where a top_k leaves no more than kSrFew candidates all of them go there, and the draw ends there. Only parts too full for that (hundreds of logits
// within 2^-14 of a bit that are not all equal, or beyond the last bin) are halved bit by bit.
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
    float tops[kSrCluster * kSrWarps];   // the largest logit of every warp of the cluster
    // where a border lies: the bin, and what lies in bins before it and in it
    int bin;
    uint64_t mass_before;
    uint32_t count_before, count_in;
    float threshold;
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
    int lo, hi, rank, size, turn;        // this warp's run
    float mine;                          // its largest logit
    float far, scale;                    // distances to the largest logit beyond which a weight is 0; bins in a distance of 1: the last one begins there
    // f(logit, place in the CTA's slice) for every logit of this warp's run, if one of them is not below `least`
    template <typename F>
    __device__ __forceinline__ void each(float least, F f) const {
        if (mine < least) return;
        for (int i = lo + (int)(threadIdx.x & 31); i < hi; i += 32) f(s_x[i], i);
    }

    __device__ __forceinline__ void barrier() { if (size == 1) __syncthreads(); else cluster.sync(); }
    __device__ __forceinline__ uint64_t weight(float x) const { return r.top - x > far ? 0 : r.weight_of(x); }      // (inf - inf is no number: not beyond)
    __device__ __forceinline__ int bin_of(float d) const { return (int)fminf(d * scale, (float)(kSrBins - 1)); }
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

    // which bin (outer < 0), or which part of bin `outer`, a logit belongs to; -1: none
    __device__ __forceinline__ int place(float x, int outer) const {
        const float d = r.top - x;
        if (outer < 0) return bin_of(d);
        return bin_of(d) == outer ? (int)fminf(fmaxf(fmaf(d, scale, -(float)outer) * kSrBins, 0.0f), (float)(kSrBins - 1)) : -1;
    }

    // The least value that stays: of top_k of them (by_mass false), or of those that reach `share` of the mass of the logits from `above` on. small: a border by count that
    // leaves no more than kSrFew candidates is not looked for; they are all in the first CTA's list then, and the answer is 0.
    __device__ float find(bool by_mass, uint64_t top_k, double share, float above, bool& small) {
        double need = (double)top_k;
        uint64_t m0 = 0;
        uint32_t n0 = 0;
        int outer = -1;
        for (;;) {
            clear();
            each(above, [&](float x, int) {
                const int bin = x >= above ? place(x, outer) : -1;
                if (bin >= 0) add(bin, by_mass ? weight(x) : 0, by_mass);
            });
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
            each(above, [&](float x, int i) {
                const int b = x >= above ? place(x, outer) : -1;
                if (b >= 0 && (small ? b <= bin : b == bin)) {
                    const uint32_t to = atomicAdd(&first->listed, 1u);
                    first->x[to] = x;
                    first->at[to] = (rank << 20) | i;
                }
            });
            barrier();
            if (small) return 0.0f;
            if (rank == 0) {                                             // pair by pair: one stays when what lies above it is not yet enough
                const bool is = threadIdx.x < in;
                const float x = is ? sh.x[threadIdx.x] : 0.0f;
                if (is) sh.w[threadIdx.x] = by_mass ? weight(x) : 1;
                __syncthreads();
                uint64_t v = by_mass ? m0 : n0;
                for (uint32_t k = 0; k < in; ++k) v += sh.x[k] > x ? sh.w[k] : 0;
                if (is && (double)v < need) atomicMin(&sh.lowest, sr_key(x));
                __syncthreads();
                if (threadIdx.x == 0) sh.threshold = sr_float(sh.lowest);
            }
            barrier();
            return cluster.map_shared_rank(&sh, 0)->threshold;
        }
    }

    // A top_k below the number of the cluster's warps: the top_k-th largest of the warps' largest logits is no larger than the top_k-th largest of all, so that the candidates lie from there
    // on; as a rule not many more than top_k. True when the first CTA's list holds all of them.
    __device__ __forceinline__ bool few(int top_k, int groups) {
        if (top_k * 8 > groups * 7) return false;
        if (threadIdx.x == 0) { sh.listed = 0; sh.lowest = 0xffffffffu; }
        __syncthreads();
        if ((int)threadIdx.x < groups) {
            const float x = sh.tops[threadIdx.x];
            int above = 0;
            for (int k = 0; k < groups; ++k) above += sh.tops[k] > x;
            if (above < top_k) atomicMin(&sh.lowest, sr_key(x));
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
    __device__ __noinline__ float crowded(bool by_mass, double need, float above, int outer, int bin) {
        uint64_t high = 0, low = 0;
        each(above, [&](float x, int) {
            if (x < above || place(x, outer) != bin) return;
            high = max(high, (uint64_t)sr_key(x));
            low = max(low, (uint64_t)~sr_key(x));
        });
        high = sr_all<true>(high, sh, turn, cluster);
        low = (uint32_t)~(uint32_t)sr_all<true>(low, sh, turn, cluster);
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
    after_previous();
    extern __shared__ __align__(16) uint8_t sr_raw[];
    SrShared& sh = *reinterpret_cast<SrShared*>(sr_raw);
    float* s_x = reinterpret_cast<float*>(sr_raw + sizeof(SrShared));
    cg::cluster_group cluster = cg::this_cluster();
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
    SrWork w{sh, cluster, r, s_x, lo, hi, rank, size, turn, best, reach, (float)(kSrBins - 1) / reach};
    const float far = bits * 0.6931472f * temperature * 1.0001f;
    float thr = -INFINITY;                                          // kept: from there on
    if (r.top < INFINITY) {                                         // (of infinite logits all are kept, and nothing else weighs anything)
        if (top_k > 0 && top_k < p.n) {
            bool small = true;
            thr = w.few(top_k, groups) ? 0.0f : w.find(false, (uint64_t)top_k, 0.0, -INFINITY, small);
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
            thr = fmaxf(thr, w.find(true, 0, (double)top_p, thr, small));
        }
    }
    turn = w.turn;
    auto kept = [&](float v) -> uint64_t {
        if (v < thr || r.top - v > far) return 0;
        const uint64_t y = r.weight_of(v);
        return y >= least ? y : 0;
    };
    // the mass of the warp's run first, then the warp in whose run the target lies walks it
    uint64_t mine = 0;
    if (best >= thr && !(r.top - best > far))
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
        SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SrShared) + kSrSlice * 4 + 16));
        ready = true;
    }
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
