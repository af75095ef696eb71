// csrc/logprobs.cu — what a row of logits says about a given token and the most likely ones, in one launch and one pass over the logits.
//
//   M = max x,  S = sum exp(x - M);  log p_t = (x_t - M) - log S;  entropy = log S + sum exp(x - M) (M - x) / S;  rank of t: logits in front of it (larger ones, equal ones with a lower
//   index);  alternatives: the `top` first logits in that order.
// S is held as 1 + R with the largest logit itself left out of R: log1p(R) and both terms of the entropy, neither of them negative, keep their bits where one token has nearly all the weight.
// A cluster of up to eight CTAs shares a row; a CTA takes 8192 logits at a time into its registers (2048 where its part of the row is no longer than 4096), so that they are read once. A warp's sums
// are relative to its own largest so far. The threads' largest logits give a bound that at least `top` logits reach, so that a few dozen of the first turn's are left to be put in order, by counting for each how many are in front of it; after that only
// what is larger than the last of the list. Data that defeat the bound (hundreds of equal logits, nearly everything banned) are searched `top` times for the next one instead. Nothing depends on the
// order of threads but the fp32 sums' fixed tree.
// Bound: a turn is a chain (loads 2000 to 3000 clocks, largest and bound 1500, rank 1200, sums 1200, list 2000) that four CTAs an SM hide in part, and a row ends with two barriers of its cluster
// and 4000 clocks for the lists. One row of 32000 logits, two turns of 2048 a CTA, 6.2 us (floor 0.02), 64 rows of 128256 with 20 alternatives 19.7 (5.0; the same in one turn of 16384 a CTA 23.5),
// 1000 rows 114 (78.2: 4.5 TB/s). A round of the machine is 592 CTAs: 592 rows of 128256 take 65 us, 600 90, 1184 127, so that some rows more than a round holds are the dearest.
#include <cooperative_groups.h>

#include <type_traits>

#include "seq_common.cuh"

namespace sllm {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32, kLpCluster = 8;
constexpr int kLpMany = 32, kLpSome = 8;         // logits a thread takes at a time
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
__device__ __forceinline__ float lp_max3(float a, float b, float c) {    // NaN if one of them is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two fp32 operations at once, each rounded as the single one
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) { uint64_t d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ uint64_t lp_mul2(uint64_t a, uint64_t b) { uint64_t d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ void lp_split(uint64_t v, float& lo, float& hi) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    lo = __uint_as_float(a);
    hi = __uint_as_float(b);
}

// The sum of exp(x - M) over all logits but those that are M, and of the same times (x - M); how many are M; logits in front of the token.
struct LpSums {
    float largest, rest, spread;
    int before, has;
};

struct alignas(16) LpShared {
    uint64_t few[kLpFew], list[2][kLpTop];
    uint64_t all[kLpCluster * kLpTop];           // of the first CTA: every CTA's list
    LpSums sums[kLpCluster];                     // and sums
    LpSums warp[kLpWarps];
    uint64_t warp64[kLpWarps];
    uint32_t tops[kLpWarps];
    int count[2];
    float log_sum, largest;
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

// a float's place among the others as a whole number; NaN is 0
__device__ __forceinline__ uint32_t lp_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float lp_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ LpSums lp_warp_sums(LpSums a) {               // over the warp's lanes, relative to the largest of all
    const float m = warp_max(a.largest);
    lp_move(a.rest, a.spread, a.has, a.largest, m);
    return {m, warp_sum(a.rest), warp_sum(a.spread), __reduce_add_sync(0xffffffffu, a.before), __reduce_add_sync(0xffffffffu, a.has)};
}

// kValues: logits a thread takes at a time. kVec: rows start at multiples of 16 bytes, four neighbours a load; else every kLpThreads-th logit
template <bool kVec, int kValues>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(LogprobArgs p) {
    after_previous();
    constexpr int kGroup = 4 * kLpThreads, kGroups = kValues / 4, kTurn = kLpThreads * kValues;      // four of a thread's logits, and the CTA's neighbouring ones with them; logits a turn
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
    const bool plain = known && mine == mine && mine != -INFINITY;
    const float just_below = mine == 0.0f ? -1.4012984643e-45f : __uint_as_float(__float_as_uint(mine) + (mine > 0.0f ? -1 : 1));
    const int lo = min(p.n, rank * p.slice), hi = min(p.n, lo + p.slice);
    float largest = -INFINITY, rest = 0.0f, spread = 0.0f;               // of the warp
    int before = 0, has = 0, listed = 0, turn = 0;
    if (tid < kLpTop) sh.list[0][tid] = sh.list[1][tid] = 0;
    if (tid < 2) sh.count[tid] = 0;
    for (int at = lo; at < hi; at += kTurn) {
        auto index = [&](int k, int e) { return kVec ? at + k * kGroup + tid * 4 + e : at + k * kGroup + e * kLpThreads + tid; };
        float v[kValues];
        // every address is one of the row's, so that nothing is asked before a load (behind a condition each waited for the one before); what is behind the end is replaced afterwards
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            if constexpr (kVec) {
                const uint4 q = ld_stream(x + min(index(k, 0), (hi & ~3) - 4));
                v[4 * k] = __uint_as_float(q.x); v[4 * k + 1] = __uint_as_float(q.y); v[4 * k + 2] = __uint_as_float(q.z); v[4 * k + 3] = __uint_as_float(q.w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * k + e] = x[min(index(k, e), hi - 1)];
            }
        }
        if (at + kTurn > hi) {
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                if (at + (k + 1) * kGroup <= hi) continue;
                const bool part = kVec && index(k, 0) < hi && index(k, 3) >= hi;             // the row's last one to three
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (index(k, e) >= hi) v[4 * k + e] = -INFINITY;
                    else if (part) v[4 * k + e] = x[index(k, e)];
                }
            }
        }
        float own = -INFINITY;
#pragma unroll
        for (int k = 0; k < kValues; k += 2) own = lp_max3(own, v[k], v[k + 1]);
        if (own != own) rest = own;              // NaN: so are this row's sums
        const uint32_t key = lp_key(own), top = __reduce_max_sync(0xffffffffu, key);
        const float m = fmaxf(largest, top ? lp_unkey(top) : -INFINITY);
        lp_move(rest, spread, has, largest, m);
        largest = m;
        bool pushed = false;
        if (p.top > 0) {
            float bound;
            if (listed == p.top) {               // the list is full: only what is larger than its last one (an equal one has a higher index), so the next float above
                const uint64_t last = sh.list[turn][p.top - 1];
                bound = last >> 32 == 0 ? -INFINITY : lp_unkey((uint32_t)(last >> 32) + 1);         // (NaN, which nothing reaches, above infinity)
            } else {                             // the first turn: behind it the list is full, or there is no second one
                static_assert(kTurn >= kLpTop, "a turn fills the list");
                // `top` logits reach the `top`-th largest of the warps' largest threads, or half (a quarter) as many warps with two (four) each their second (fourth) (NaN is below everything)
                const int each = p.top <= kLpWarps ? 1 : p.top <= 2 * kLpWarps ? 2 : 4;
                uint32_t left = key, least = top;
                for (int i = 1; i < each; ++i) {
                    if (lane == __ffs(__ballot_sync(0xffffffffu, left == least)) - 1) left = 0;
                    least = __reduce_max_sync(0xffffffffu, left);
                }
                __syncthreads();
                if (lane == 0) sh.tops[warp] = least;
                __syncthreads();
                const uint32_t one = sh.tops[lane & (kLpWarps - 1)];
                int ahead = 0;
#pragma unroll
                for (int w = 0; w < kLpWarps; ++w) {
                    const uint32_t other = sh.tops[w];
                    ahead += other > one || (other == one && w < (lane & (kLpWarps - 1)));
                }
                const uint32_t reached = __shfl_sync(0xffffffffu, one, __ffs(__ballot_sync(0xffffffffu, ahead == (p.top + each - 1) / each - 1)) - 1);
                bound = reached ? lp_unkey(reached) : -INFINITY;
            }
            if (own >= bound || own != own) {
#pragma unroll
                for (int k = 0; k < kValues; ++k) {
                    if (!(v[k] >= bound) || index(k / 4, k % 4) >= hi) continue;
                    const int to = atomicAdd(&sh.count[turn], 1);
                    if (to < kLpFew) sh.few[to] = lp_entry(v[k], index(k / 4, k % 4));
                    pushed = true;
                }
            }
        }
        if (plain) {
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const int first = at + k * kGroup;
                if (first + kGroup <= tok || first > tok) {              // a group before the token or behind it
                    const float above = first > tok ? mine : just_below;
#pragma unroll
                    for (int e = 0; e < 4; ++e) before += v[4 * k + e] > above;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) before += v[4 * k + e] > mine || (v[4 * k + e] == mine && index(k, e) < tok);
                }
            }
        } else if (known) {                      // -infinity, behind which there is NaN alone; NaN, behind which there is nothing
#pragma unroll 4
            for (int k = at + tid; k < min(hi, at + kTurn); k += kLpThreads) before += mine == mine ? x[k] > mine || (x[k] == mine && k < tok) : x[k] == x[k] || k < tok;
        }
        // sums. A thread that has one of the largest leaves it out
        const float ref = m == -INFINITY ? 0.0f : m;
        if (own == m) {
#pragma unroll
            for (int k = 0; k < kValues; ++k) {
                if (v[k] == m) {
                    ++has;
                    v[k] = -INFINITY;
                }
            }
        }
        uint64_t rest2 = 0, spread2 = 0;
        const uint64_t ref2 = pair_f32(-ref, -ref), log2e2 = pair_f32(kLpLog2e, kLpLog2e);
#pragma unroll
        for (int k = 0; k < kValues; k += 2) {   // -infinity adds nothing
            float z0, z1, t0, t1;
            lp_split(lp_add2(pair_f32(v[k], v[k + 1]), ref2), z0, z1);
            const uint64_t z = pair_f32(fmaxf(z0, -300.0f), fmaxf(z1, -300.0f));
            lp_split(lp_mul2(z, log2e2), t0, t1);
            const uint64_t e = pair_f32(lp_exp2(t0), lp_exp2(t1));
            rest2 = lp_add2(rest2, e);
            fma_pair(spread2, e, z);
        }
        rest += pair_sum(rest2);
        spread += pair_sum(spread2);
        if (p.top == 0) continue;
        const int want = min(p.top, listed + min(hi - at, kTurn));
        if (!__syncthreads_or(pushed) && listed == want) continue;       // nothing came in front of the last one of the list
        const int found = sh.count[turn];
        uint64_t* to = sh.list[turn ^ 1];
        if (found + listed <= kLpFew && found + listed >= want) {
            if (listed > 0) {
                if (tid < listed) sh.few[found + tid] = sh.list[turn][tid];
                __syncthreads();
            }
            for (int i = tid; i < found + listed; i += kLpThreads) {
                const uint64_t e = sh.few[i];
                int ahead = 0;
#pragma unroll 8
                for (int j = 0; j < found + listed; ++j) ahead += sh.few[j] > e;
                if (ahead < p.top) to[ahead] = e;
            }
        } else {
            // (from memory: this is rare, and the code is read by every CTA)
            uint64_t last = ~0ull;
#pragma unroll 1
            for (int i = 0; i < p.top; ++i) {    // the largest one below the last
                uint64_t best = 0;
                if (tid < listed && sh.list[turn][tid] < last) best = sh.list[turn][tid];
#pragma unroll 4
                for (int k = at + tid; k < min(hi, at + kTurn); k += kLpThreads) {
                    const uint64_t e = lp_entry(x[k], k);
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
                if (tid == 0) to[i] = best;
                last = best;                     // 0: there is none left, now or later
                __syncthreads();
            }
        }
        listed = want;
        __syncthreads();
        if (tid < kLpTop) sh.list[turn][tid] = 0;
        if (tid == 0) sh.count[turn] = 0;
        turn ^= 1;
    }
    // this CTA's sums
    const LpSums w = {largest, warp_sum(rest), warp_sum(spread), __reduce_add_sync(0xffffffffu, before), __reduce_add_sync(0xffffffffu, has)};
    if (lane == 0) sh.warp[warp] = w;
    __syncthreads();
    cluster.barrier_wait();                      // every CTA of the cluster runs
    LpShared* first = cluster.map_shared_rank(&sh, 0);
    if (warp == 0) {
        const LpSums s = lp_warp_sums(lane < kLpWarps ? sh.warp[lane] : LpSums{-INFINITY, 0.0f, 0.0f, 0, 0});
        if (lane == 0) first->sums[rank] = s;
    }
    if (tid >= 32 && tid < 32 + p.top) first->all[rank * p.top + tid - 32] = sh.list[turn][tid - 32];
    if (size == 1) __syncthreads(); else cluster.sync();
    if (rank != 0) return;
    if (warp == 0) {
        const LpSums s = lp_warp_sums(lane < size ? sh.sums[lane] : LpSums{-INFINITY, 0.0f, 0.0f, 0, 0});
        if (lane == 0) {
            const float r = s.rest + (float)(s.has - 1), m = s.largest;
            float log_sum = log1pf(r), entropy = log_sum - s.spread / (1.0f + r);
            if (m == -INFINITY) log_sum = entropy = NAN;
            if (p.entropy) p.entropy[row] = entropy;
            if (p.rank) p.rank[row] = known ? s.before : -1;
            if (p.logprob) p.logprob[row] = (mine == m ? 0.0f : mine - m) - log_sum;
            sh.log_sum = log_sum;
            sh.largest = m;
        }
    }
    if (p.top == 0) return;
    // of the lists together
    static_assert(kLpCluster * kLpTop <= kLpThreads, "an entry a thread");
    const uint64_t e = tid < size * p.top ? sh.all[tid] : 0;
    int ahead = 0;
    if (e != 0) {
#pragma unroll 8
        for (int j = 0; j < size * p.top; ++j) ahead += sh.all[j] > e;
    }
    __syncthreads();
    if (e != 0 && ahead < p.top) {
        const float z = lp_value(e);
        p.top_idx[row * p.top + ahead] = lp_index(e);
        if (p.top_logprob) p.top_logprob[row * p.top + ahead] = (z == sh.largest ? 0.0f : z - sh.largest) - sh.log_sum;
    }
}

}  // namespace sllm

using namespace sllm;

extern "C" int sllm_token_logprobs(const float* logits, int64_t ld, int32_t rows, int32_t n, const int32_t* token, float* logprob, float* entropy, int32_t* rank, int32_t top, int32_t* top_idx,
                                   float* top_logprob, sllm_stream_t stream) {
    SLLM_REQUIRE(logits && rows > 0 && n > 0, SLLM_EINVAL, "token_logprobs: null pointer, no rows or no logits");
    SLLM_REQUIRE(n <= 1 << 30, SLLM_ENOTSUP, "token_logprobs: rows of %d logits", n);      // (indices go on to the end of a turn)
    SLLM_REQUIRE(ld >= n, SLLM_EINVAL, "token_logprobs: rows of %d logits lie %lld apart", n, (long long)ld);
    SLLM_REQUIRE(token || (!logprob && !rank), SLLM_EINVAL, "token_logprobs: a log probability and a rank are those of a given token");
    SLLM_REQUIRE(top >= 0 && top <= n, SLLM_EINVAL, "token_logprobs: %d alternatives of %d logits", top, n);
    SLLM_REQUIRE(top <= kLpTop, SLLM_ENOTSUP, "token_logprobs: %d alternatives, %d at most", top, kLpTop);
    SLLM_REQUIRE(top ? top_idx != nullptr : !top_idx && !top_logprob, SLLM_EINVAL, "token_logprobs: alternatives need a place, and a number of them");
    SLLM_REQUIRE(logprob || entropy || rank || top, SLLM_EINVAL, "token_logprobs: nothing is asked for");
    // CTAs of a row: what a CTA does once (its bound, its list, what the cluster puts together) costs as much as some 8000 logits, so no more than fill the machine once. us, until there are
    // 1, 4, 8 and 16 CTAs an SM: 64 rows of 128256 21.8, 19.6, 19.7, 19.6; 1000 rows 114, 114, 121, 140
    int cs = 1;
    while (cs < kLpCluster && (long long)rows * cs < 4 * sm_count() && n / cs >= 4096) cs *= 2;
    SLLM_REQUIRE((long long)rows * cs <= 0x7fffffffLL, SLLM_ENOTSUP, "token_logprobs: too many rows");
    const int64_t each = ((int64_t)n + cs - 1) / cs;
    const bool vec = each >= 4 * kLpThreads && ld % 4 == 0 && ((uintptr_t)logits % 16) == 0;
    const int slice = (int)(vec ? (each + 4 * kLpThreads - 1) / (4 * kLpThreads) * (4 * kLpThreads) : each);      // whole groups: only the last CTA has a part of one
    LogprobArgs p{logits, token, logprob, entropy, top_logprob, rank, top_idx, ld, n, top, slice};
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
    auto launch = [&](auto whole, auto values) { return cudaLaunchKernelEx(&cfg, overlapping(token_logprobs_kernel<whole.value, values.value>), p); };
    using yes = std::true_type;
    using no = std::false_type;
    using some = std::integral_constant<int, kLpSome>;
    using many = std::integral_constant<int, kLpMany>;
    if (slice <= 2 * kLpSome * kLpThreads) SLLM_CUDA(vec ? launch(yes{}, some{}) : launch(no{}, some{}));
    else SLLM_CUDA(vec ? launch(yes{}, many{}) : launch(no{}, many{}));
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}
