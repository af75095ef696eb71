// csrc/seq_attn_shared.cuh — what the kernels of attention behind shared first positions have in common (seq_attn_shared.cu).
#pragma once
#include <cfloat>

#include "seq_attn.cuh"

namespace sllm {

// the kernel for pools in bf16 and heads of 64 or 128 (seq_attn_shared_tc.cu)
struct SharedArgs;
int launch_attention_shared_tc(const SharedArgs& p, cudaStream_t st);
int64_t attention_shared_tc_flush_floats(int dk, int dv);      // what its CTAs need to move their accumulators to

// A step whose segments come in groups: the first group_len[g] positions of all segments group_start[g] .. group_start[g + 1] - 1 are the same and are read through the block table of the group's
// first segment; the positions behind them through each segment's own.
struct SharedArgs {
    sllm_seq_batch b;
    int n_groups;
    const int32_t *group_start, *group_len;
    const float* q;
    int ldq, heads, kv_heads, dk, dv;
    float scale;
    const void *k_pool, *v_pool;
    int n_pages, window, keep_first;
    float softcap;
    const float* slopes;
    int shares, own;                     // records of a (token, head) at most: of the shared positions, of its own
    int table_len;                       // positions that a row of the block table has room for
    uint32_t page_magic;                 // ceil(2^32 / page_len): the page of a position without a division (page_of)
    int least, own_least;                // keys of a share at least (least: of the kernel that does not plan it itself)
    int* plan;                           // of every listed tile: its records of shared positions, and its own ones << 16
    float* ws;
    float* flush;                        // of the kernel on the tensor cores: what its CTAs' accumulators held, a tile of rows each
    float* out;
    int ldo;
    uint16_t* out16;
};

// What a CTA leaves of the keys it has seen, for a (token, head): the reference of the weights as a power of two, their sum, and the weighted sum of the values. Records lie
// [token][head][shares + own][dv + 4].
constexpr int kShHead = 4;               // floats in front of the values (16 bytes, so that these are aligned)
// positions of a table at most: added to the keys of a share, whole tiles and the like, 2^26 at most, they stay within 32 bits
constexpr int kShMostPositions = 0x7fffffff - (1 << 26);
// bytes in front of the records: the plan
inline int64_t sh_plan_bytes(int n_qtiles) { return ((int64_t)n_qtiles * 4 + 15) / 16 * 16; }

#ifdef __CUDACC__

__device__ __forceinline__ float* sh_record(const SharedArgs& p, int t, int h, int which) {
    return p.ws + (((size_t)t * p.heads + h) * (p.shares + p.own) + which) * (p.dv + kShHead);
}
// the page of a position (-1 where the table has none that exists) and the position's place in it
__device__ __forceinline__ int sh_page(const SharedArgs& p, int slot, int pos, int& in_page) {
    const int at = page_of(pos, p.b.page_len, p.page_magic, in_page);
    if (slot < 0 || at >= p.b.max_pages) return -1;
    const int page = p.b.block_table[(size_t)slot * p.b.max_pages + at];
    return page >= 0 && page < p.n_pages ? page : -1;
}
// tokens [first, first + n) of a group
__device__ __forceinline__ void sh_group_tokens(const SharedArgs& p, int g, int& first, int& n) {
    const int s0 = p.group_start[g], s1 = min(p.group_start[g + 1], p.b.nseg);
    first = n = 0;
    if (s0 < 0 || s0 >= s1) return;
    first = p.b.seg_start[s0];
    n = max(0, min(p.b.seg_start[s1 - 1] + p.b.seg_len[s1 - 1], p.b.T) - first);
}
// positions that a group shares, whatever it says: those that a table has room for, since none of the others has a page
__device__ __forceinline__ int sh_group_len(const SharedArgs& p, int g) { return min(max(0, p.group_len[g]), p.table_len); }
// positions that segment `seg` shares with its group (by whole warps)
__device__ __forceinline__ int sh_shared_len(const SharedArgs& p, int seg) {
    int upto = 0;                        // groups that begin at or before the segment
    for (int i = threadIdx.x & 31; i - (int)(threadIdx.x & 31) < p.n_groups; i += 32) upto += __popc(__ballot_sync(0xffffffffu, i < p.n_groups && p.group_start[i] <= seg));
    return upto > 0 ? sh_group_len(p, upto - 1) : 0;
}
// The group that holds row tile `tile` of tiles of `tokens` tokens, group after group, its first token and how many it has; `tile` becomes the tile's number in it (by whole warps). -1: there
// are not so many.
__device__ __forceinline__ int sh_find_group(const SharedArgs& p, int tokens, int& tile, int& first, int& n) {
    const int lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        first = n = 0;
        if (g0 + lane < p.n_groups) sh_group_tokens(p, g0 + lane, first, n);
        const int tiles = (n + tokens - 1) / tokens;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, upto > tile);
        if (past) {
            const int who = __ffs(past) - 1;
            tile -= __shfl_sync(0xffffffffu, upto - tiles, who);
            first = __shfl_sync(0xffffffffu, first, who);
            n = __shfl_sync(0xffffffffu, n, who);
            return g0 + who;
        }
        tile -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return -1;
}
// How many of the step's shares a range of keys is cut into: none smaller than `least` keys.
__device__ __forceinline__ int sh_cuts(int keys, int least, int most) { return keys <= 0 ? 0 : min(most, (keys + least - 1) / least); }

// a score after its scale: capped, charged for its distance
__device__ __forceinline__ float sh_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}
// Weights and the factors that carry sums to another reference are never zero, but 32 bits may hold no more than a zero for one: for finite numbers that is what it is, an infinity (or NaN) stays what
// it is. (A least weight instead of the zero brought 1e36 times 2^-126 into results of size 1.)
__device__ __forceinline__ float sh_carried(float sum, float factor) { return fabsf(sum) <= FLT_MAX ? sum * factor : sum; }
__device__ __forceinline__ float sh_add(float sum, float w, float x) { return fabsf(x) <= FLT_MAX ? fmaf(w, x, sum) : sum + x; }

#endif

}  // namespace sllm
