// csrc/logprobs.cu — what a row of logits says about a given token and the most likely ones, in one launch and one pass over the logits.
//
//   M = max x,  S = sum exp(x - M);  log p_t = (x_t - M) - log S;  entropy = log S + sum exp(x - M) (M - x) / S;  rank of t: logits in front of it (larger ones, equal ones with a lower
//   index);  alternatives: the `top` first logits in that order.
// S is held as 1 + R with the largest logit itself left out of R: log1p(R) and both terms of the entropy, neither of them negative, keep their bits where one token has nearly all the weight.
// A cluster of up to eight CTAs shares a row; a CTA takes 16384 logits at a time into its registers. The threads' largest logits give, beside M, a bound that at least `top` logits
// reach (the least of the warps' first or second largest), so that a few dozen logits are left to be put in order, by counting for each how many are in front of it. Data that defeat the
// bound (hundreds of equal logits, nearly everything banned) are searched `top` times for the next one instead. Nothing depends on the order of threads but the fp32 sums' fixed tree.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace sllm {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32, kLpValues = 32, kLpChunk = kLpThreads * kLpValues, kLpCluster = 8;
constexpr int kLpTop = 32, kLpFew = 1024;        // alternatives at most; logits that are put in order by counting
constexpr float kLpLog2e = 1.4426950408889634f;

struct LogprobArgs {
    const float* logits;
    const int32_t* token;
    float *logprob, *entropy, *top_logprob;
    int32_t *rank, *top_idx;
    int64_t ld;
    int n, top, slice;
};

// A logit in its place of the order as one number: larger logits first, of equal ones the lower index; NaN behind everything else, nothing is 0.
__device__ __forceinline__ uint64_t lp_entry(float x, int i) {
    const uint32_t u = __float_as_uint(x + 0.0f);                        // -0 is 0
    const uint32_t key = x != x ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (uint64_t)key << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float lp_value(uint64_t e) {
    const uint32_t k = (uint32_t)(e >> 32);
    return k == 0 ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ int lp_index(uint64_t e) { return (int)(0xffffffffu - (uint32_t)e); }
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The sum of exp(x - M) over all logits but those that are M, and of the same times (x - M); how many are M; logits in front of the token.
struct LpSums {
    float largest, rest, spread;
    int before, has;
};

struct alignas(16) LpShared {
    uint64_t few[kLpFew], list[kLpTop], next[kLpTop];
    uint64_t all[kLpCluster * kLpTop];           // of the first CTA: every CTA's list
    LpSums sums[kLpCluster];                     // and sums
    uint64_t warp64[kLpWarps];
    float warp_top[kLpWarps], warp_second[kLpWarps], part[2][kLpWarps];
    int before[kLpWarps], has[kLpWarps];
    int count;
    float log_sum;
};

// The sums from one reference to a larger one: the logits that were the largest come in.
__device__ __forceinline__ void lp_move(float& rest, float& spread, int& has, float from, float to) {
    if (from == to) return;
    if (from == -INFINITY) {                     // nothing but -infinity so far (times zero: NaN stays NaN)
        rest *= 0.0f;
        spread *= 0.0f;
    } else {
        const float d = fmaxf(from - to, -300.0f), f = expf(d);
        rest += (float)has;
        spread = f * fmaf(d, rest, spread);
        rest *= f;
    }
    has = 0;
}

template <bool kVec>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(LogprobArgs p) {
    after_previous();
    __shared__ LpShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / size;
    const float* x = p.logits + row * p.ld;
    const int tok = p.token ? p.token[row] : -1;
    const bool known = tok >= 0 && tok < p.n;
    const float mine = known ? x[tok] : NAN;
    // logits in front of the token: those above a bound, which for indices before the token's is the next float below
    const bool plain = known && mine == mine;
    const float just_below = !plain || mine == -INFINITY ? mine : mine == 0.0f ? -1.4012984643e-45f : __uint_as_float(__float_as_uint(mine) + (mine > 0.0f ? -1 : 1));
    const int lo = min(p.n, rank * p.slice), hi = min(p.n, lo + p.slice);
    const int second = p.top > kLpWarps;         // two logits of every warp are needed for `top` of them
    float largest = -INFINITY, rest = 0.0f, spread = 0.0f;
    int before = 0, has = 0, listed = 0;
    if (tid < kLpTop) sh.list[tid] = 0;
    for (int at = lo; at < hi; at += kLpChunk) {
        const int groups = (min(hi - at, kLpChunk) + 4 * kLpThreads - 1) / (4 * kLpThreads);
        auto index = [&](int k, int e) { return kVec ? at + (k * kLpThreads + tid) * 4 + e : at + (4 * k + e) * kLpThreads + tid; };
        float v[kLpValues];
#pragma unroll
        for (int k = 0; k < kLpValues / 4; ++k) {
            if (kVec && index(k, 3) < hi) {
                const uint4 q = ld_stream(x + index(k, 0));
                v[4 * k] = __uint_as_float(q.x); v[4 * k + 1] = __uint_as_float(q.y); v[4 * k + 2] = __uint_as_float(q.z); v[4 * k + 3] = __uint_as_float(q.w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * k + e] = k < groups && index(k, e) < hi ? x[index(k, e)] : -INFINITY;
            }
        }
        float own = -INFINITY;
#pragma unroll
        for (int k = 0; k < kLpValues; ++k) own = fmaxf(own, v[k]);
        const float top = warp_max(own);
        const unsigned who = __ballot_sync(0xffffffffu, own == top);
        const float below = second ? warp_max(who && lane == __ffs(who) - 1 ? -INFINITY : own) : top;
        __syncthreads();                         // the last turn's readers are through
        if (lane == 0) {
            sh.warp_top[warp] = top;
            sh.warp_second[warp] = below;
        }
        if (tid == 0) sh.count = 0;
        __syncthreads();
        float m = largest, bound = INFINITY;
#pragma unroll
        for (int w = 0; w < kLpWarps; ++w) {
            m = fmaxf(m, sh.warp_top[w]);
            bound = fminf(bound, sh.warp_second[w]);
        }
        lp_move(rest, spread, has, largest, m);
        largest = m;
        const float ref = m == -INFINITY ? 0.0f : m;
        auto add = [&](float y) {                // -infinity adds nothing, NaN makes everything NaN
            const float z = y - ref, e = lp_exp2(z * kLpLog2e);
            rest += e;
            spread = fmaf(e, fmaxf(z, -300.0f), spread);
        };
        if (own == m) {                          // few threads: the others need not look
#pragma unroll
            for (int k = 0; k < kLpValues; ++k) {
                if (v[k] == m) ++has;
                else add(v[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kLpValues; ++k) add(v[k]);
        }
        if (plain) {
#pragma unroll
            for (int k = 0; k < kLpValues / 4; ++k) {
                if (kVec) {
                    const float above = index(k, 3) < tok ? just_below : mine;
#pragma unroll
                    for (int e = 0; e < 4; ++e) before += v[4 * k + e] > above;
                    if (index(k, 0) < tok && index(k, 3) >= tok) {
#pragma unroll
                        for (int e = 0; e < 3; ++e) before += index(k, e) < min(tok, hi) && v[4 * k + e] == mine;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) before += v[4 * k + e] > mine || (v[4 * k + e] == mine && index(k, e) < min(tok, hi));
                }
            }
            if (kVec && mine == -INFINITY) {     // nothing is below it: equal ones are counted one by one
#pragma unroll
                for (int k = 0; k < kLpValues; ++k) before += index(k / 4, k % 4) < min(hi, tok) && index(k / 4, 3) < tok && v[k] == mine;
            }
        } else if (known) {                      // NaN comes behind everything else
#pragma unroll
            for (int k = 0; k < kLpValues; ++k) before += index(k / 4, k % 4) < hi && (v[k] == v[k] || index(k / 4, k % 4) < tok);
        }
        if (p.top == 0) continue;
        if (listed == p.top) bound = fmaxf(bound, lp_value(sh.list[p.top - 1]));
#pragma unroll
        for (int k = 0; k < kLpValues / 4; ++k) {
            if (fmaxf(fmaxf(v[4 * k], v[4 * k + 1]), fmaxf(v[4 * k + 2], v[4 * k + 3])) < bound) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[4 * k + e] >= bound && index(k, e) < hi) {
                    const int to = atomicAdd(&sh.count, 1);
                    if (to < kLpFew) sh.few[to] = lp_entry(v[4 * k + e], index(k, e));
                }
        }
        __syncthreads();
        const int found = sh.count, want = min(p.top, listed + min(hi - at, kLpChunk));
        if (found + listed <= kLpFew && found + listed >= want) {
            if (tid < kLpTop) sh.next[tid] = 0;
            if (tid < listed) sh.few[found + tid] = sh.list[tid];
            __syncthreads();
            for (int i = tid; i < found + listed; i += kLpThreads) {
                const uint64_t e = sh.few[i];
                int ahead = 0;
                for (int j = 0; j < found + listed; ++j) ahead += sh.few[j] > e;
                if (ahead < p.top) sh.next[ahead] = e;
            }
            __syncthreads();
        } else {
            uint64_t last = ~0ull;
            for (int i = 0; i < p.top; ++i) {    // the largest one below the last
                uint64_t best = 0;
                if (tid < listed && sh.list[tid] < last) best = sh.list[tid];
#pragma unroll
                for (int k = 0; k < kLpValues; ++k) {
                    if (index(k / 4, k % 4) >= hi) continue;
                    const uint64_t e = lp_entry(v[k], index(k / 4, k % 4));
                    if (e < last && e > best) best = e;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t e = __shfl_xor_sync(0xffffffffu, best, o);
                    best = e > best ? e : best;
                }
                if (lane == 0) sh.warp64[warp] = best;
                __syncthreads();
                best = 0;
                for (int w = 0; w < kLpWarps; ++w) best = sh.warp64[w] > best ? sh.warp64[w] : best;
                if (tid == 0) sh.next[i] = best;
                last = best;                     // 0: there is none left, now or later
                __syncthreads();
            }
        }
        if (tid < p.top) sh.list[tid] = sh.next[tid];
        listed = want;
        __syncthreads();
    }
    // this CTA's sums
    rest = warp_sum(rest);
    spread = warp_sum(spread);
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        has += __shfl_xor_sync(0xffffffffu, has, o);
    }
    if (lane == 0) {
        sh.part[0][warp] = rest;
        sh.part[1][warp] = spread;
        sh.before[warp] = before;
        sh.has[warp] = has;
    }
    __syncthreads();
    cluster.barrier_wait();    // every CTA of the cluster runs
    LpShared* first = cluster.map_shared_rank(&sh, 0);
    if (warp == 0) {
        LpSums s{largest, warp_sum(lane < kLpWarps ? sh.part[0][lane] : 0.0f), warp_sum(lane < kLpWarps ? sh.part[1][lane] : 0.0f), lane < kLpWarps ? sh.before[lane] : 0,
                 lane < kLpWarps ? sh.has[lane] : 0};
        for (int o = 16; o > 0; o >>= 1) {
            s.before += __shfl_xor_sync(0xffffffffu, s.before, o);
            s.has += __shfl_xor_sync(0xffffffffu, s.has, o);
        }
        if (lane == 0) first->sums[rank] = s;
    }
    if (tid >= 32 && tid < 32 + p.top) first->all[rank * p.top + tid - 32] = sh.list[tid - 32];
    cluster.sync();
    if (rank != 0) return;
    if (tid == 0) {
        float m = -INFINITY;
        for (int i = 0; i < size; ++i) m = fmaxf(m, sh.sums[i].largest);
        float r = 0.0f, s = 0.0f;
        int ahead = 0, tops = 0;
        for (int i = 0; i < size; ++i) {
            LpSums a = sh.sums[i];
            lp_move(a.rest, a.spread, a.has, a.largest, m);
            r += a.rest;
            s += a.spread;
            tops += a.has;
            ahead += a.before;
        }
        r += (float)(tops - 1);
        float log_sum = log1pf(r), entropy = log_sum - s / (1.0f + r);
        if (m == -INFINITY) log_sum = entropy = NAN;
        if (p.entropy) p.entropy[row] = entropy;
        if (p.rank) p.rank[row] = known ? ahead : -1;
        if (p.logprob) p.logprob[row] = (mine == m ? 0.0f : mine - m) - log_sum;
        sh.log_sum = log_sum;
        sh.part[0][0] = m;
    }
    __syncthreads();
    const float log_sum = sh.log_sum, m = sh.part[0][0];
    for (int i = tid; i < size * p.top; i += kLpThreads) {
        const uint64_t e = sh.all[i];
        if (e == 0) continue;
        int ahead = 0;
        for (int j = 0; j < size * p.top; ++j) ahead += sh.all[j] > e;
        if (ahead < p.top) {
            const float z = lp_value(e);
            p.top_idx[row * p.top + ahead] = lp_index(e);
            if (p.top_logprob) p.top_logprob[row * p.top + ahead] = (z == m ? 0.0f : z - m) - log_sum;
        }
    }
}

}  // namespace sllm

using namespace sllm;

extern "C" int sllm_token_logprobs(const float* logits, int64_t ld, int32_t rows, int32_t n, const int32_t* token, float* logprob, float* entropy, int32_t* rank, int32_t top, int32_t* top_idx,
                                   float* top_logprob, sllm_stream_t stream) {
    SLLM_REQUIRE(logits && rows > 0 && n > 0, SLLM_EINVAL, "token_logprobs: null pointer, no rows or no logits");
    SLLM_REQUIRE(ld >= n, SLLM_EINVAL, "token_logprobs: rows of %d logits lie %lld apart", n, (long long)ld);
    SLLM_REQUIRE(token || (!logprob && !rank), SLLM_EINVAL, "token_logprobs: a log probability and a rank are those of a given token");
    SLLM_REQUIRE(top >= 0 && top <= n, SLLM_EINVAL, "token_logprobs: %d alternatives of %d logits", top, n);
    SLLM_REQUIRE(top <= kLpTop, SLLM_ENOTSUP, "token_logprobs: %d alternatives, %d at most", top, kLpTop);
    SLLM_REQUIRE(top ? top_idx != nullptr : !top_idx && !top_logprob, SLLM_EINVAL, "token_logprobs: alternatives need a place, and a number of them");
    SLLM_REQUIRE(logprob || entropy || rank || top, SLLM_EINVAL, "token_logprobs: nothing is asked for");
    // CTAs of a row: as many as leave one no more than it holds in registers, and more while the machine has room and they have 2048 logits each
    int cs = 1;
    while (cs < kLpCluster && ((n + cs - 1) / cs > kLpChunk || ((long long)rows * cs < 2 * sm_count() && n / cs >= 4096))) cs *= 2;
    SLLM_REQUIRE((long long)rows * cs <= 0x7fffffffLL, SLLM_ENOTSUP, "token_logprobs: too many rows");
    const int slice = (int)(((int64_t)n + cs - 1) / cs + 3) / 4 * 4;
    LogprobArgs p{logits, token, logprob, entropy, top_logprob, rank, top_idx, ld, n, top, slice};
    const bool vec = slice >= 4 * kLpThreads && ld % 4 == 0 && ((uintptr_t)logits % 16) == 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * cs));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (vec) SLLM_CUDA(cudaLaunchKernelEx(&cfg, overlapping(token_logprobs_kernel<true>), p));
    else SLLM_CUDA(cudaLaunchKernelEx(&cfg, overlapping(token_logprobs_kernel<false>), p));
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}
