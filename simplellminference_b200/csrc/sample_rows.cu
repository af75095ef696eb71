// csrc/sample_rows.cu — the next token of every row of a step, drawn with settings of the row's own from given random numbers, in one launch.
//
//   w_i = exp((x_i - max x) / temperature);  kept: x_i among the top_k largest, and the mass of the kept larger ones below top_p of all kept mass, and w_i >= min_p;
//   drawn: the first i (in index order) whose running kept mass exceeds u times the kept mass.  Equal logits are in or out together, as in sample.cu.
// Every border is a comparison of sums: a draw lies next to one of as many borders as there are candidates, so that fp32 weights (2^-24 of each) would move one draw in some ten
// thousands over a large vocabulary. Weights are computed in double and held as multiples of 2^-44: sums of these integers are exact, so nothing depends on the order of threads, and
// what is left is the rounding of a weight, 2^-45 of the largest.
// A cluster of CTAs shares a row and keeps it in shared memory: the logits are read once, whatever the settings ask for.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace sllm {

namespace cg = cooperative_groups;

constexpr int kSrThreads = 512, kSrWarps = kSrThreads / 32, kSrCluster = 16;
constexpr int kSrSlice = 48 * 1024;              // logits of a CTA at most (192 KB)
constexpr double kSrOne = 17592186044416.0;      // 2^44: the weights of 786432 logits add up to less than 2^64

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

__global__ void __launch_bounds__(kSrThreads) sample_rows_kernel(SampleRows p) {
    after_previous();
    extern __shared__ __align__(16) float s_x[];
    __shared__ SrShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / size, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = min(p.n, rank * p.slice), count = min(p.n, first + p.slice) - first;
    const float* x = p.logits + (size_t)row * p.ld + first;
    int turn = 0;
    // the largest logit and the first place that has it, as one number; NaN counts as -infinity
    uint64_t best = 0;
    for (int i = threadIdx.x; i < count; i += kSrThreads) {
        float v = x[i];
        v = v == v ? v : -INFINITY;
        s_x[i] = v;
        const uint64_t k = ((uint64_t)sr_key(v) << 32) | (uint32_t)~(first + i);
        best = k > best ? k : best;
    }
    best = sr_all<true>(best, sh, turn, cluster);
    const int arg = (int)~(uint32_t)best;
    const uint32_t top_key = (uint32_t)(best >> 32);
    SrRow r;
    r.top = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    if (!(temperature > 0.0f) || r.top == -INFINITY) {
        if (rank == 0 && threadIdx.x == 0) {
            p.idx[row] = r.top == -INFINITY ? 0 : arg;
            if (p.prob) p.prob[row] = r.top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    r.rate = 1.4426950408889634074 / (double)temperature;
    const int top_k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
    uint32_t thr = 0;                                               // kept: key >= thr
    if (top_k > 0 && top_k < p.n) {
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = thr | (1u << bit);
            uint64_t c = 0;
            for (int i = threadIdx.x; i < count; i += kSrThreads) c += sr_key(s_x[i]) >= cand;
            if (sr_all<false>(c, sh, turn, cluster) >= (uint64_t)top_k) thr = cand;
        }
    }
    if (top_p > 0.0f && top_p < 1.0f) {
        uint64_t w = 0;
        for (int i = threadIdx.x; i < count; i += kSrThreads)
            if (sr_key(s_x[i]) >= thr) w += r.weight_of(s_x[i]);
        const double need = (double)top_p * (double)sr_all<false>(w, sh, turn, cluster);
        uint32_t cut = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = cut | (1u << bit);
            w = 0;
            for (int i = threadIdx.x; i < count; i += kSrThreads) {
                const uint32_t k = sr_key(s_x[i]);
                if (k >= cand && k >= thr) w += r.weight_of(s_x[i]);
            }
            if ((double)sr_all<false>(w, sh, turn, cluster) >= need) cut = cand;
        }
        thr = max(thr, cut);
    }
    const uint64_t least = min_p > 0.0f ? (uint64_t)__double2ll_ru(fmin((double)min_p, 1.0) * kSrOne) : 0;
    auto kept = [&](float v) {
        const uint64_t w = sr_key(v) >= thr ? r.weight_of(v) : 0;
        return w >= least ? w : 0;
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
    const float u = p.u[row];
    const double at = u > 0.0f ? fmin((double)u, 1.0) * (double)all : 0.0;
    uint64_t target = (uint64_t)at;                                 // running > at is running > floor(at) for whole numbers
    if (target >= all) target = all - 1;
    if (before <= target && target < before + mine) {
        for (int i = lo; i < hi; i += 32) {
            const uint64_t w = i + lane < hi ? kept(s_x[i + lane]) : 0;
            uint64_t upto = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    p.idx[row] = first + i + lane;
                    if (p.prob) p.prob[row] = (float)((double)w / (double)all);
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
        SLLM_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSrSlice * 4));
        ready = true;
    }
    int cs = 1;
    while (cs < kSrCluster && ((n + cs - 1) / cs > 8192 || ((long long)rows * cs < sm_count() && n / cs >= 2048))) cs *= 2;
    SampleRows p{logits, temperature, top_p, min_p, u, top_k, idx_dev, prob_dev, ld, n, ((n + cs - 1) / cs + 3) / 4 * 4};
    SLLM_REQUIRE((long long)rows * cs <= 0x7fffffffLL, SLLM_ENOTSUP, "sample_rows: too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)rows * cs);
    cfg.blockDim = dim3(kSrThreads);
    cfg.dynamicSmemBytes = (size_t)p.slice * 4;
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
