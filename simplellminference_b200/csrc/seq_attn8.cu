// csrc/seq_attn8.cu — softmax attention of the ragged token batch over the 8-bit paged cache (kv8.cuh has the format).
//
//   s_j = scale * 2^ek * (q . code_j),  p = softmax over the visible j,  o = sum_j p_j 2^ev code'_j
// A block's scales are one number each for 32 keys, so they multiply scores and weights, never codes: the codes enter the products as they are.
// Keys whose page the block table does not have are hidden; a query that sees no key gives zeros.
#include <cfloat>

#include "seq_attn8.cuh"

namespace sllm {

// Any head width: CTA = (tile of up to 32 queries of a segment, query head), a warp per query in turn. A lane owns one of a block's 32 keys for the scores and every 32nd group
// of four columns for the weighted sum; fp32 throughout.
constexpr int kA8Warps = 4;

template <int kGroups>       // groups of 128 value columns
__global__ void __launch_bounds__(kA8Warps * 32) seq_attention8_kernel(Attn8Args p, int least) {
    after_previous();
    __shared__ __align__(16) float s_q[kA8Warps][256];
    const sllm_seq_batch& b = p.b;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, g = h / (p.heads / p.kv_heads);
    const int seg = b.qt_seg[blockIdx.x], off = b.qt_off[blockIdx.x], n = min(kBQ, b.seg_len[seg] - off), slot = b.seg_slot[seg];
    const float slope = p.slopes ? p.slopes[h] : 0.0f;
    if (n < least) return;                                     // another kernel's
    for (int i = warp; i < n; i += kA8Warps) {
        const int t = b.seg_start[seg] + off + i, pos = b.seg_pos0[seg] + off + i, wnd = seq_row_window(pos, p.window, p.chunk);
        const float* q = p.q + (size_t)t * p.ldq + (size_t)h * p.dk;
        __syncwarp();
        for (int c = lane; c < p.dk; c += 32) s_q[warp][c] = q[c] * p.scale;
        __syncwarp();
        float m = -INFINITY, l = 0.0f, o[kGroups][4] = {};
        const TileList tiles(pos, pos, wnd, p.keep_first, kKv8Block);
        for (int x = 0; x < tiles.n; ++x) {
            const int j0 = tiles.tile_of(x) * kKv8Block, page = kv8_page(b, p.n_pages, slot, j0), in_page = j0 % b.page_len;
            if (page < 0) continue;
            const float ks = p.k_scale[kv8_scale_at(page, p.kv_heads, g, b.page_len, in_page)], vs = p.v_scale[kv8_scale_at(page, p.kv_heads, g, b.page_len, in_page)];
            const uint8_t* kr = p.k_pool + seq_pool_row(page, p.kv_heads, g, b.page_len, in_page + lane, p.dk);
            const uint8_t* vr = p.v_pool + seq_pool_row(page, p.kv_heads, g, b.page_len, in_page, p.dv);
            const bool sees = seq_sees(pos, j0 + lane, wnd, p.keep_first);
            float s = -INFINITY;
            if (sees) {
                float sum[4] = {};
                for (int c = 0; c < p.dk; c += 16) {
                    const uint4 w = *reinterpret_cast<const uint4*>(kr + c);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 a = kv8_float2(ws[e] & 0xffffu), d = kv8_float2(ws[e] >> 16);
                        const float4 qq = *reinterpret_cast<const float4*>(&s_q[warp][c + 4 * e]);
                        sum[e] = fmaf(qq.w, d.y, fmaf(qq.z, d.x, fmaf(qq.y, a.y, fmaf(qq.x, a.x, sum[e]))));
                    }
                }
                s = attn8_score(((sum[0] + sum[1]) + (sum[2] + sum[3])) * ks, p.softcap, slope, pos, j0 + lane);
            }
            const float mn = fmaxf(m, warp_max(s));
            const float corr = mn == -INFINITY ? 1.0f : expf(m - mn), w = s == -INFINITY ? 0.0f : expf(s - mn);
            m = mn;
            l = l * corr + warp_sum(w);
#pragma unroll
            for (int c = 0; c < kGroups; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][e] *= corr;
            const unsigned seen = __ballot_sync(0xffffffffu, sees);
            for (int k = 0; k < kKv8Block; ++k) {
                if (!(seen >> k & 1)) continue;                // a hidden row may hold anything
                const float wk = __shfl_sync(0xffffffffu, w, k) * vs;
#pragma unroll
                for (int c = 0; c < kGroups; ++c) {
                    const int col = c * 128 + 4 * lane;
                    if (col >= p.dv) break;
                    const uint32_t v = *reinterpret_cast<const uint32_t*>(vr + (size_t)k * p.dv + col);
                    const float2 a = kv8_float2(v & 0xffffu), d = kv8_float2(v >> 16);
                    o[c][0] = fmaf(wk, a.x, o[c][0]); o[c][1] = fmaf(wk, a.y, o[c][1]); o[c][2] = fmaf(wk, d.x, o[c][2]); o[c][3] = fmaf(wk, d.y, o[c][3]);
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < kGroups; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = c * 128 + 4 * lane + e;
                if (col >= p.dv) break;
                if (p.out) p.out[(size_t)t * p.ldo + (size_t)h * p.dv + col] = o[c][e] * inv;
                if (p.out16) p.out16[((size_t)t * p.heads + h) * p.dv + col] = f32_to_bf16_bits(o[c][e] * inv);
            }
    }
}

}  // namespace sllm

using namespace sllm;

extern "C" {

int64_t sllm_seq_attention8_ws_bytes(const sllm_seq_batch* b, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv) {
    SLLM_REQUIRE(b && b->T > 0 && b->nseg > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && dk > 0 && dv > 0, SLLM_EINVAL, "seq_attention8_ws_bytes: bad argument");
    return (int64_t)kA8Ws;
}

int sllm_seq_attention8(const sllm_seq_batch* b, const float* q, int32_t ldq, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv, float scale, const void* k_pool,
                        const float* k_scale, const void* v_pool, const float* v_scale, int32_t n_pages, void* ws, int64_t ws_bytes, const sllm_seq_attn_opts* opts, float* out,
                        int32_t ldo, void* out16, sllm_stream_t stream) {
    SLLM_REQUIRE(b && b->T > 0 && b->nseg > 0 && b->seg_start && b->seg_len && b->seg_slot && b->seg_pos0 && b->block_table && b->max_pages > 0 && b->qt_seg && b->qt_off &&
                     b->n_qtiles > 0,
                 SLLM_EINVAL, "seq_attention8: incomplete batch description");
    SLLM_REQUIRE(q && k_pool && k_scale && v_pool && v_scale && n_pages > 0 && (out || out16), SLLM_EINVAL, "seq_attention8: null pointer, no pages or no output");
    SLLM_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, SLLM_EINVAL, "seq_attention8: %d query heads over %d kv heads", heads, kv_heads);
    SLLM_REQUIRE(dk > 0 && dv > 0 && dk % 16 == 0 && dv % 16 == 0 && dk <= 256 && dv <= 256, SLLM_ENOTSUP, "seq_attention8: head widths %d and %d are not multiples of 16 up to 256",
                 dk, dv);
    SLLM_REQUIRE(heads <= 65535, SLLM_ENOTSUP, "seq_attention8: %d heads", heads);
    SLLM_REQUIRE(scale > 0.0f && scale <= FLT_MAX, SLLM_EINVAL, "seq_attention8: scores need a positive finite scale");
    SLLM_REQUIRE(b->page_len > 0 && b->page_len % kKv8Block == 0, SLLM_ENOTSUP, "seq_attention8: pages of a multiple of %d positions", kKv8Block);
    SLLM_REQUIRE(ldq >= heads * dk && (!out || ldo >= heads * dv), SLLM_EINVAL, "seq_attention8: a row is shorter than its heads");
    SLLM_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) % 16) == 0, SLLM_EINVAL, "seq_attention8: pools have to start at a multiple of 16 bytes");
    SLLM_REQUIRE(ws && ((uintptr_t)ws % 16) == 0 && ws_bytes >= sllm_seq_attention8_ws_bytes(b, heads, kv_heads, dk, dv), SLLM_EINVAL, "seq_attention8: the workspace is too small or not aligned");
    SLLM_REQUIRE(!opts || (opts->window >= 0 && opts->keep_first >= 0 && opts->softcap >= 0.0f && opts->chunk >= 0), SLLM_EINVAL, "seq_attention8: bad options");
    SLLM_REQUIRE(!opts || !opts->chunk || !opts->window, SLLM_EINVAL, "seq_attention8: a window or chunks, not both");
    SLLM_REQUIRE(!opts || (!opts->values_in_keys && !opts->logdist && !opts->cross_values), SLLM_ENOTSUP,
                 "seq_attention8: values in keys, charges on the logarithm of the distance and values of every head are not part of this form");
    Attn8Args p{*b, q, ldq, heads, kv_heads, dk, dv, scale, (const uint8_t*)k_pool, (const uint8_t*)v_pool, k_scale, v_scale, n_pages, INT_MAX, 0, 0, 0.0f, nullptr, out, ldo,
                (uint16_t*)out16};
    if (opts) {
        if (opts->window > 0) {
            p.window = opts->window;
            p.keep_first = opts->keep_first;
        }
        p.chunk = opts->chunk;
        p.softcap = opts->softcap;
        p.slopes = opts->slopes;
    }
    if (int rc = status_check()) return rc;
    cudaStream_t st = as_stream(stream);
    const bool narrow = dk <= 128 && dv <= 128 && (unsigned long long)n_pages * kv_heads * b->page_len < 1ull << 31;
    if (narrow) {
        const bool single = b->T == b->nseg;
        const bool tc = !single && attention8_tc_takes(p);
        if (int rc = launch_attention8_decode(p, single, tc ? attention8_tc_width(p) : 0, ws, st)) return rc;
        if (single) return SLLM_OK;
        if (tc) return launch_attention8_tc(p, ws, st);
    }
    const dim3 grid(b->n_qtiles, heads);
    const int least = narrow ? 2 : 1;
    if (dv <= 128) overlapping(seq_attention8_kernel<1>)<<<grid, kA8Warps * 32, 0, st>>>(p, least);
    else overlapping(seq_attention8_kernel<2>)<<<grid, kA8Warps * 32, 0, st>>>(p, least);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

}  // extern "C"
