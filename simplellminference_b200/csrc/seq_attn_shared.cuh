// csrc/seq_attn_shared.cuh — what the kernels of attention behind shared first positions have in common (seq_attn_shared.cu).
#pragma once
#include "seq_attn.cuh"

namespace sllm {

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
    int shares, own;                     // records of a (token, head): of the shared positions, of its own
    float* ws;
    float* out;
    int ldo;
    uint16_t* out16;
};

// What a CTA leaves of the keys it has seen, for a (token, head): the reference of the weights as a power of two, their sum, and the weighted sum of the values. Records lie
// [token][head][shares + own][dv + 4].
constexpr int kShHead = 4;               // floats in front of the values (16 bytes, so that these are aligned)

#ifdef __CUDACC__

__device__ __forceinline__ float* sh_record(const SharedArgs& p, int t, int h, int which) {
    return p.ws + (((size_t)t * p.heads + h) * (p.shares + p.own) + which) * (p.dv + kShHead);
}
// the page of a position, -1 where the table has none that exists
__device__ __forceinline__ int sh_page(const SharedArgs& p, int slot, int pos) {
    const int at = pos / p.b.page_len;
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
// positions that segment `seg` shares with its group
__device__ __forceinline__ int sh_shared_len(const SharedArgs& p, int seg) {
    int lo = 0, hi = p.n_groups;         // group_start[lo] <= seg < group_start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.group_start[mid] <= seg) lo = mid; else hi = mid;
    }
    return max(0, p.group_len[lo]);
}
// a score after its scale: capped, charged for its distance
__device__ __forceinline__ float sh_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}

#endif

}  // namespace sllm
