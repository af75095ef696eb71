// csrc/seq_kv8.cu — keys and values appended to the 8-bit paged cache, the rotation applied on the way (kv8.cuh has the format).
//
// One launch, two kinds of CTAs. The first part of the grid writes the cache: a CTA per (block of 32 positions that a segment writes to, kv head, keys or values) turns up to 32 rows,
// keeps them in registers, takes their largest magnitude and stores codes and scale; where the block holds earlier rows and its scale grows, their codes move to the new one.
// No other CTA touches the block, so nothing is atomic and the result does not depend on the order of CTAs. The others turn a token's queries.
// Angles come as a table (sllm_seq_angles): made once a step for all layers, they cost a layer 8 bytes a pair and token here instead of a sine and a cosine in double per head.
// Bound: bytes; queries in and out are most of them (32 heads over 8: 32 of 43 KB a token). Prompts of 3896 tokens, 32 heads over 8 of 128: 39.4 us, 26 at the rate of a copy (4.3 TB/s; loads wait
// for memory, and the queries' stream shares registers and block size with the cache's part); 64 requests of one token 3.9 us, one 2.8 (a kernel that adds to one number takes 1.1).
#include <climits>

#include "kv8.cuh"

namespace sllm {

struct Kv8Args {
    sllm_seq_batch b;
    const float *q, *k, *v, *angles;
    float *q_out, *k_scale, *v_scale;
    uint8_t *k_pool, *v_pool;
    int ldq, ldk, ldv, ldqo, heads, kv_heads, dk, dv, n_freq, n_pages;
    int units, q_split;              // (segment, block) pairs the grid has room for; CTAs that share a token's queries
    int32_t* status;
};

constexpr int kKv8Threads = 128;

// A job is eight columns of a row: four neighbouring pairs of a turned row (both halves of each), eight neighbouring columns elsewhere. The first column of its two runs of four:
template <bool kVec, int kLayout>
__device__ __forceinline__ int kv8_column(int job, int n_freq, int run) {
    return kVec && kLayout == 1 && job < n_freq / 4 ? (run ? n_freq + 4 * job : 4 * job) : 8 * job + 4 * run;
}
// kVec: rows are 16-byte aligned and n_freq is a multiple of four, so that a run is one load; else every column for itself.
template <bool kVec, int kLayout>
__device__ __forceinline__ void kv8_load(const float* row, const float* angles, int n_freq, int job, float (&x)[8]) {
    if constexpr (kVec) {
        const float4 a = *reinterpret_cast<const float4*>(row + kv8_column<kVec, kLayout>(job, n_freq, 0)), c = *reinterpret_cast<const float4*>(row + kv8_column<kVec, kLayout>(job, n_freq, 1));
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
        if (job < n_freq / 4) {
            const float4 t0 = *reinterpret_cast<const float4*>(angles + 8 * job), t1 = *reinterpret_cast<const float4*>(angles + 8 * job + 4);
            const float cs[4] = {t0.x, t0.z, t1.x, t1.z}, sn[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                constexpr int kStep = kLayout ? 1 : 2, kOther = kLayout ? 4 : 1;
                const float u = x[kStep * i], w = x[kStep * i + kOther];
                // products and sums rounded one by one: a code does not depend on where a compiler contracts
                x[kStep * i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(w, sn[i]));
                x[kStep * i + kOther] = __fadd_rn(__fmul_rn(w, cs[i]), __fmul_rn(u, sn[i]));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = 8 * job + i;
            x[i] = row[c];
            if (c < 2 * n_freq) {
                const bool first = kLayout ? c < n_freq : !(c & 1);
                const int m = kLayout ? (first ? c : c - n_freq) : c >> 1, other = kLayout ? (first ? c + n_freq : c - n_freq) : c ^ 1;
                const float cs = angles[2 * m], sn = angles[2 * m + 1], o = row[other];
                x[i] = first ? __fsub_rn(__fmul_rn(x[i], cs), __fmul_rn(o, sn)) : __fadd_rn(__fmul_rn(x[i], cs), __fmul_rn(o, sn));
            }
        }
    }
}

// The part of one segment's rows that lies in the block at `lo` (a multiple of 32), for one head of one pool, by the whole CTA.
template <bool kVec, int kLayout, int kJobs>
__device__ __forceinline__ void kv8_block(const Kv8Args& p, int tok0, int pos0, int len, int slot, int lo, int g, const float* src, int ld, int width, int n_freq, uint8_t* pool,
                                          float* scales, float* red) {
    const sllm_seq_batch& b = p.b;
    const int page = kv8_page(b, p.n_pages, slot, lo);
    if (page < 0) {                                                        // nowhere to write: reported, the memory stays as it is
        if (threadIdx.x == 0) *reinterpret_cast<volatile int32_t*>(p.status) = kStatusPages;
        return;
    }
    const int in_page = lo % b.page_len, first = max(lo, pos0), rows = min(lo + kKv8Block, pos0 + len) - first, per_row = width / 8, jobs = rows * per_row;
    const int tok = tok0 + first - pos0;
    float* scale = scales + kv8_scale_at(page, p.kv_heads, g, b.page_len, in_page);
    uint8_t* dst = pool + seq_pool_row(page, p.kv_heads, g, b.page_len, in_page, width);
    const float was = first > lo ? *scale : 0.0f;                          // without earlier rows the block begins anew
    float x[kJobs][8], top = 0.0f;
#pragma unroll
    for (int j = 0; j < kJobs; ++j) {
        const int i = threadIdx.x + j * kKv8Threads;
        if (i >= jobs) break;
        const int t = tok + i / per_row;
        kv8_load<kVec, kLayout>(src + (size_t)t * ld + (size_t)g * width, p.angles + (size_t)t * 2 * n_freq, n_freq, i % per_row, x[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(x[j][e]);
            if (a < INFINITY) top = fmaxf(top, a);
            else x[j][e] = __int_as_float(0x7fffffff);                     // e4m3 has no infinity: it becomes NaN, as NaN does, and does not move the scale
        }
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float fresh = kv8_pow2(kv8_exponent(top)), now = fmaxf(was, fresh), inv = 1.0f / now;
    if (now > was && first > lo) {
        const float f = was / now;
        for (int i = threadIdx.x; i < (first - lo) * width / 4; i += kKv8Threads) {
            uint32_t* word = reinterpret_cast<uint32_t*>(dst) + i;
            const float2 a = kv8_float2(*word & 0xffffu), c = kv8_float2(*word >> 16);
            *word = kv8_pack4(a.x * f, a.y * f, c.x * f, c.y * f);
        }
    }
    if (threadIdx.x == 0) *scale = now;
#pragma unroll
    for (int j = 0; j < kJobs; ++j) {
        const int i = threadIdx.x + j * kKv8Threads;
        if (i >= jobs) break;
        uint8_t* row = dst + (size_t)(first - lo + i / per_row) * width;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float* y = x[j] + 4 * h;
            *reinterpret_cast<uint32_t*>(row + kv8_column<kVec, kLayout>(i % per_row, n_freq, h)) = kv8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        }
    }
    __syncthreads();                                                       // red is used again
}

// kJobs: jobs of a thread for 32 rows
// Eight CTAs an SM, though their 64 registers spill 50 words (as do 128): 39.4 us for the prompts above, with six of 80 registers and one division a thread instead of one a job 42.3, with the layout an argument 51.7.
template <bool kVec, int kLayout, int kJobs>
__global__ void __launch_bounds__(kKv8Threads, kJobs == 4 ? 8 : 4) seq_rotary_kv8_kernel(Kv8Args p) {
    after_previous();
    __shared__ float red[kKv8Threads / 32];
    const sllm_seq_batch& b = p.b;
    const int per_unit = 2 * p.kv_heads;
    const unsigned cache = (unsigned)p.units * per_unit;
    if (blockIdx.x < cache) {
        const int unit = blockIdx.x / per_unit, g = blockIdx.x % per_unit >> 1, values = blockIdx.x & 1, lane = threadIdx.x & 31;
        int seg = unit, from = 0, n_blocks = INT_MAX;                      // single tokens: a CTA per segment (all its blocks)
        if (b.T != b.nseg) {
            // the segment that holds this block, counted over all of them, 32 at a time
            int before = 0, s0 = 0;
            seg = -1;
            for (; s0 < b.nseg; s0 += 32) {
                const int s = s0 + lane, len = s < b.nseg ? b.seg_len[s] : 0, pos0 = s < b.nseg ? b.seg_pos0[s] : 0;
                const int mine = len > 0 ? (pos0 + len - 1) / kKv8Block - pos0 / kKv8Block + 1 : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + upto > unit);
                if (past) {
                    const int l = __ffs(past) - 1;
                    seg = s0 + l;
                    from = unit - before - __shfl_sync(0xffffffffu, upto - mine, l);
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (seg < 0) return;
            n_blocks = 1;
        }
        const int tok0 = b.seg_start[seg], len = b.seg_len[seg], pos0 = b.seg_pos0[seg], slot = b.seg_slot[seg];
        if (len <= 0 || slot < 0) return;
        // two segments of one sequence would write the same scales: reported, nothing of theirs is written
        bool twice = false;
        for (int s = threadIdx.x; s < b.nseg; s += kKv8Threads) twice |= s != seg && b.seg_slot[s] == slot && b.seg_len[s] > 0;
        if (__syncthreads_or(twice)) {
            if (threadIdx.x == 0) *reinterpret_cast<volatile int32_t*>(p.status) = kStatusTwice;
            return;
        }
        const int lo0 = pos0 / kKv8Block * kKv8Block + from * kKv8Block;
        for (int i = 0; i < n_blocks && lo0 + i * kKv8Block < pos0 + len; ++i) {
            if (values) kv8_block<kVec, kLayout, kJobs>(p, tok0, pos0, len, slot, lo0 + i * kKv8Block, g, p.v, p.ldv, p.dv, 0, p.v_pool, p.v_scale, red);
            else kv8_block<kVec, kLayout, kJobs>(p, tok0, pos0, len, slot, lo0 + i * kKv8Block, g, p.k, p.ldk, p.dk, p.n_freq, p.k_pool, p.k_scale, red);
        }
        return;
    }
    const int t = (blockIdx.x - cache) / p.q_split, part = (blockIdx.x - cache) % p.q_split;
    const bool token = b.tok_slot[t] >= 0;                                 // or a place without one: its row is read, but nothing is stored (asked for beside the rows, not in front)
    const float *q = p.q + (size_t)t * p.ldq, *angles = p.angles + (size_t)t * 2 * p.n_freq;
    float* out = p.q_out + (size_t)t * p.ldqo;
    // in place only what turns has to move
    const int per_head = q == out ? (2 * p.n_freq + 7) / 8 : p.dk / 8, jobs = p.heads * per_head;
    constexpr int kAhead = 4;                                              // rows may be turned in place: loads are asked for before the stores in front of them
    if constexpr (kVec) {
        for (int i0 = part * kKv8Threads + threadIdx.x; i0 < jobs; i0 += kAhead * p.q_split * kKv8Threads) {
            float x[kAhead][8];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = i0 + j * p.q_split * kKv8Threads;
                if (i < jobs) kv8_load<true, kLayout>(q + (size_t)(i / per_head) * p.dk, angles, p.n_freq, i % per_head, x[j]);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = i0 + j * p.q_split * kKv8Threads;
                if (i >= jobs || !token) break;
                float* row = out + (size_t)(i / per_head) * p.dk;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4*>(row + kv8_column<true, kLayout>(i % per_head, p.n_freq, h)) = make_float4(x[j][4 * h], x[j][4 * h + 1], x[j][4 * h + 2], x[j][4 * h + 3]);
            }
        }
    } else {                                                               // pair by pair: both halves belong to one thread, so that rows may be turned in place
        if (!token) return;
        const int pairs = p.heads * p.n_freq;
        for (int i = part * kKv8Threads + threadIdx.x; i < pairs; i += p.q_split * kKv8Threads) {
            const int h = i / p.n_freq, m = i % p.n_freq, ia = kLayout ? m : 2 * m, ib = kLayout ? m + p.n_freq : 2 * m + 1;
            const float u = q[(size_t)h * p.dk + ia], w = q[(size_t)h * p.dk + ib], cs = angles[2 * m], sn = angles[2 * m + 1];
            out[(size_t)h * p.dk + ia] = __fsub_rn(__fmul_rn(u, cs), __fmul_rn(w, sn));
            out[(size_t)h * p.dk + ib] = __fadd_rn(__fmul_rn(w, cs), __fmul_rn(u, sn));
        }
        const int rest = p.dk - 2 * p.n_freq;
        if (q != out)
            for (int i = part * kKv8Threads + threadIdx.x; i < p.heads * rest; i += p.q_split * kKv8Threads) {
                const size_t at = (size_t)(i / rest) * p.dk + 2 * p.n_freq + i % rest;
                out[at] = q[at];
            }
    }
}

template <bool kVec, int kLayout>
static void launch_rotary_kv8(const Kv8Args& p, unsigned grid, cudaStream_t st) {
    if (max(p.dk, p.dv) <= 128) overlapping(seq_rotary_kv8_kernel<kVec, kLayout, 4>)<<<grid, kKv8Threads, 0, st>>>(p);
    else overlapping(seq_rotary_kv8_kernel<kVec, kLayout, 8>)<<<grid, kKv8Threads, 0, st>>>(p);
}

}  // namespace sllm

using namespace sllm;

extern "C" int sllm_seq_rotary_kv8(const sllm_seq_batch* b, const float* q, int32_t ldq, int32_t heads, int32_t dk, const float* k, int32_t ldk, int32_t kv_heads, const float* v,
                                   int32_t ldv, int32_t dv, const float* angles, int32_t n_freq, int32_t layout, float* q_out, int32_t ldqo, void* k_pool, float* k_scale,
                                   void* v_pool, float* v_scale, int32_t n_pages, sllm_stream_t stream) {
    SLLM_REQUIRE(b && b->T > 0 && b->nseg > 0 && b->tok_slot && b->seg_start && b->seg_len && b->seg_slot && b->seg_pos0 && b->block_table && b->max_pages > 0, SLLM_EINVAL,
                 "seq_rotary_kv8: incomplete batch description");
    SLLM_REQUIRE(q && k && v && q_out && k_pool && k_scale && v_pool && v_scale && n_pages > 0, SLLM_EINVAL, "seq_rotary_kv8: null pointer or no pages");
    SLLM_REQUIRE(heads > 0 && kv_heads > 0 && dk > 0 && dv > 0, SLLM_EINVAL, "seq_rotary_kv8: bad sizes");
    SLLM_REQUIRE(dk % 16 == 0 && dv % 16 == 0 && dk <= 256 && dv <= 256, SLLM_ENOTSUP, "seq_rotary_kv8: head widths %d and %d are not multiples of 16 up to 256", dk, dv);
    SLLM_REQUIRE(b->page_len > 0 && b->page_len % kKv8Block == 0, SLLM_ENOTSUP, "seq_rotary_kv8: pages of a multiple of %d positions", kKv8Block);
    SLLM_REQUIRE(n_freq >= 0 && 2 * n_freq <= dk && (n_freq == 0 || angles), SLLM_EINVAL, "seq_rotary_kv8: %d rotary pairs do not fit %d dimensions", n_freq, dk);
    SLLM_REQUIRE(layout == 0 || layout == 1, SLLM_EINVAL, "seq_rotary_kv8: layout 0 (interleaved) or 1 (halves)");
    SLLM_REQUIRE(ldq >= heads * dk && ldqo >= heads * dk && ldk >= kv_heads * dk && ldv >= kv_heads * dv, SLLM_EINVAL, "seq_rotary_kv8: a row is shorter than its heads");
    SLLM_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) % 16) == 0, SLLM_EINVAL, "seq_rotary_kv8: pools have to start at a multiple of 16 bytes");
    SLLM_REQUIRE(q != q_out || ldq == ldqo, SLLM_EINVAL, "seq_rotary_kv8: queries in place keep their row stride");
    Kv8Args p{*b, q, k, v, angles, q_out, k_scale, v_scale, (uint8_t*)k_pool, (uint8_t*)v_pool, ldq, ldk, ldv, ldqo, heads, kv_heads, dk, dv, n_freq, n_pages, 0, 1, nullptr};
    // a segment of n tokens touches (n + 62) / 32 blocks at most, and no more than it has tokens
    p.units = b->T == b->nseg ? b->nseg : (int)std::min<long long>(b->T, (b->T + 62LL * b->nseg) / kKv8Block);
    constexpr int kMostSplit = 8;
    SLLM_REQUIRE((long long)p.units * 2 * kv_heads + (long long)b->T * kMostSplit <= INT_MAX, SLLM_ENOTSUP, "seq_rotary_kv8: %d tokens of %d heads are too many for one launch", b->T,
                 kv_heads);
    if (int rc = status_check()) return rc;
    if (int rc = status_word(&p.status)) return rc;
    const int jobs = heads * (dk / 8);
    // A token's queries are divided where the tokens alone do not fill the machine, us with 1, 2, 4 and 8 CTAs a token: one token of 32 heads of 128 3.04, 2.97, 2.97, 3.02; 64 of them 4.28, 3.97, 4.06, 4.58;
    // 664 tokens of 32 heads of 64 5.52, 4.85, 5.05, 5.99; 3896 of 128 39.7, 41.3, 45.7, 50.3
    p.q_split = b->T >= 8 * sm_count() ? 1 : std::max(1, std::min(b->T >= 2 * sm_count() ? 2 : kMostSplit, (jobs + kKv8Threads - 1) / kKv8Threads));
    const unsigned grid = (unsigned)(p.units * 2 * kv_heads + b->T * p.q_split);
    const bool vec = ((ldq | ldqo | ldk | ldv | n_freq) % 4) == 0 && (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)angles) % 16) == 0;
    cudaStream_t st = as_stream(stream);
    if (layout) vec ? launch_rotary_kv8<true, 1>(p, grid, st) : launch_rotary_kv8<false, 1>(p, grid, st);
    else vec ? launch_rotary_kv8<true, 0>(p, grid, st) : launch_rotary_kv8<false, 0>(p, grid, st);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}
