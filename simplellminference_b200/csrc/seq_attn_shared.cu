// csrc/seq_attn_shared.cu — softmax attention of requests whose first positions are the same (several answers to one prompt, questions behind a common text).
//
//   s_j = scale * (q . k_j),  p = softmax over the visible j,  o = sum_j p_j v_j
// The keys j below the group's shared length are read once for all tokens of the group: the query heads of a kv head and all the tokens are the rows of one product. The keys from there on are each
// segment's own. Both leave (reference, sum, weighted values) of every row, and a last kernel puts them together. A hidden key's values may be anything: they reach no row that does not see it.
#include "seq_attn_shared.cuh"

namespace sllm {

// Any head width, pools in fp32 or bf16: a CTA takes 4 * kRw rows of a (group or segment, kv head) and a share of the keys, 32 at a time through shared memory; a warp has kRw rows, a lane one
// key of them for the scores and four columns of the values for the sums; fp32 throughout.
// Bound: a chain. Four answers of 16 heads of 64 behind 1500 positions 19 us with the last kernel, which are, in clocks: whose share it is 2900, queries and pages 3000, for each of its two key
// tiles keys and values 3800, scores 1600, weights 1800 (the rows' shuffles side by side), sums 2000 (a key's four weights read together, nothing asked in between; with a question per key and row
// they took 9500).
constexpr int kShWarps = 4, kShKeys = 32;

struct ShSpan {                          // rows and keys of a CTA
    int tok0, n_rows, slot, key0, key1;  // rows: (token, head of the kv head) from tok0 on; keys [key0, key1)
    int which;                           // of the records
};

// load(i) for the CTA's i < n in turn, kAhead of a thread on their way before the first is handed to store(i, value)
template <int kAhead, class L, class S>
__device__ __forceinline__ void sh_stage(int n, L load, S store) {
    constexpr int kThreads = kShWarps * 32;
    for (int i0 = threadIdx.x; i0 < n; i0 += kAhead * kThreads) {
        decltype(load(0)) x[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) x[k] = load(min(i0 + k * kThreads, n - 1));
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i0 + k * kThreads < n) store(i0 + k * kThreads, x[k]);
    }
}
__device__ __forceinline__ void sh_floats(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void sh_floats(const uint4& v, float (&x)[8]) {
    x[0] = bf16_lo(v.x); x[1] = bf16_hi(v.x); x[2] = bf16_lo(v.y); x[3] = bf16_hi(v.y); x[4] = bf16_lo(v.z); x[5] = bf16_hi(v.z); x[6] = bf16_lo(v.w); x[7] = bf16_hi(v.w);
}

template <typename T, int kRw>
__device__ __forceinline__ void sh_rows(const SharedArgs& p, const ShSpan& sp, int g, float* smem) {
    constexpr int kRows = kShWarps * kRw, kPer = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = p.heads / p.kv_heads;
    const int ldk = p.dk + 4, cols = (p.dv + 127) / 128;
    float *s_q = smem, *s_k = s_q + kRows * p.dk, *s_v = s_k + kShKeys * ldk, *s_p = s_v + kShKeys * p.dv;      // s_p: [warp][key][row]
    for (int r0 = 0; r0 < sp.n_rows; r0 += kRows) {
        int in_page, page = sh_page(p, sp.slot, sp.key0 / kShKeys * kShKeys, in_page);           // (pages are a multiple of 32 positions)
        int pos[kRw];
        float m[kRw], l[kRw], o[kRw][2][4], slope[kRw];
        bool infinite = false;                                           // a tile so far had values that are no numbers
#pragma unroll
        for (int i = 0; i < kRw; ++i) {
            const int r = r0 + warp * kRw + i;
            pos[i] = r < sp.n_rows ? p.b.tok_pos[sp.tok0 + r / per] : -1;
            slope[i] = p.slopes ? p.slopes[g * per + r % per] : 0.0f;
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; ++c) o[i][c / 4][c % 4] = 0.0f;
        }
        __syncthreads();
        // (rows behind the last one are the last one again; nothing asks for their results)
        sh_stage<4>(kRows * p.dk / 4, [&](int i) {
            const int r = min(r0 + 4 * i / p.dk, sp.n_rows - 1), c = 4 * i % p.dk;
            const float* src = p.q + (size_t)(sp.tok0 + r / per) * p.ldq + (size_t)(g * per + r % per) * p.dk + c;
            return make_float4(src[0], src[1], src[2], src[3]);
        }, [&](int i, const float4& x) {
            // as the products on the tensor cores take it
            *reinterpret_cast<float4*>(s_q + 4 * i) = sizeof(T) == 2 ? make_float4(seq_round_bf16(x.x), seq_round_bf16(x.y), seq_round_bf16(x.z), seq_round_bf16(x.w)) : x;
        });
        for (int j0 = sp.key0 / kShKeys * kShKeys; j0 < sp.key1; j0 += kShKeys) {
            if (j0 > sp.key0) page = sh_page(p, sp.slot, j0, in_page);
            // hidden from every row of the CTA: before its window, or no page
            int seen = 0;
#pragma unroll
            for (int i = 0; i < kRw; ++i) seen |= pos[i] >= j0 && (pos[i] - (j0 + kShKeys - 1) < p.window || j0 < p.keep_first);
            if (!__syncthreads_or(seen && page >= 0)) continue;          // (behind it the last tile has been read, and the queries are there)
            // All rows of the tile are the page's, whatever part of them is the share's: nothing is asked before they are loaded. Scores of the others are hidden, their values zeros.
            int odd = 0;                                                 // a value that is infinite or NaN
            const T *kr = reinterpret_cast<const T*>(p.k_pool) + seq_pool_row(page, p.kv_heads, g, p.b.page_len, in_page, p.dk);
            const T *vr = reinterpret_cast<const T*>(p.v_pool) + seq_pool_row(page, p.kv_heads, g, p.b.page_len, in_page, p.dv);
            const int n_k = kShKeys * p.dk / kPer;
            sh_stage<8>(n_k + kShKeys * p.dv / kPer, [&](int i) { return ld_stream(i < n_k ? kr + i * kPer : vr + (i - n_k) * kPer); }, [&](int i, const uint4& v) {
                float x[kPer];
                sh_floats(v, x);
                float* to;
                if (i < n_k) {
                    const int at = i * kPer, k = at / p.dk;
                    to = s_k + k * ldk + at - k * p.dk;
                } else {
                    const int at = (i - n_k) * kPer, k = j0 + at / p.dv;
                    const bool in = k >= sp.key0 && k < sp.key1;
                    to = s_v + at;
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        x[e] = in ? x[e] : 0.0f;
                        odd |= !(fabsf(x[e]) <= FLT_MAX);
                    }
                }
#pragma unroll
                for (int e = 0; e < kPer; e += 4) *reinterpret_cast<float4*>(to + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            });
            odd = __syncthreads_or(odd);
            infinite |= odd != 0;
            const int key = j0 + lane;
            float s[kRw] = {};
#pragma unroll 4
            for (int c = 0; c < p.dk; c += 4) {
                const float4 k = *reinterpret_cast<const float4*>(s_k + lane * ldk + c);
#pragma unroll
                for (int i = 0; i < kRw; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(s_q + (warp * kRw + i) * p.dk + c);
                    s[i] = fmaf(x.w, k.w, fmaf(x.z, k.z, fmaf(x.y, k.y, fmaf(x.x, k.x, s[i]))));
                }
            }
            unsigned sees[kRw];
            float top[kRw], f[kRw];
#pragma unroll
            for (int i = 0; i < kRw; ++i) {
                const bool here = key >= sp.key0 && key < sp.key1 && seq_sees(pos[i], key, p.window, p.keep_first);
                sees[i] = __ballot_sync(0xffffffffu, here);
                s[i] = here ? sh_score(s[i] * p.scale, p.softcap, slope[i], pos[i], key) : -INFINITY;
                top[i] = s[i];
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2)              // (the rows side by side: each step waits for the one before)
#pragma unroll
                for (int i = 0; i < kRw; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
#pragma unroll
            for (int i = 0; i < kRw; ++i) {
                top[i] = fmaxf(m[i], top[i]);
                f[i] = top[i] == -INFINITY ? 1.0f : expf(m[i] - top[i]);
                const float w = s[i] == -INFINITY ? 0.0f : expf(s[i] - top[i]);
                m[i] = top[i];
                l[i] = fmaf(l[i], f[i], w);              // of this lane's keys
                if (!infinite) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) o[i][c / 4][c % 4] *= f[i];
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c) o[i][c / 4][c % 4] = sh_carried(o[i][c / 4][c % 4], f[i]);
                }
                s_p[(warp * kShKeys + lane) * kRw + i] = w;
            }
            __syncwarp();
            static_assert(kRw == 4, "a key's weights are read together");
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = c * 128 + 4 * lane;
                if (c >= cols || col >= p.dv) break;
                auto add = [&](int i, float x, const float4& v) {
                    o[i][c][0] = fmaf(x, v.x, o[i][c][0]); o[i][c][1] = fmaf(x, v.y, o[i][c][1]); o[i][c][2] = fmaf(x, v.z, o[i][c][2]); o[i][c][3] = fmaf(x, v.w, o[i][c][3]);
                };
                if (!odd) {
#pragma unroll 8
                    for (int k = 0; k < kShKeys; ++k) {
                        const float4 w = *reinterpret_cast<const float4*>(s_p + (warp * kShKeys + k) * kRw), v = *reinterpret_cast<const float4*>(s_v + k * p.dv + col);
                        add(0, w.x, v); add(1, w.y, v); add(2, w.z, v); add(3, w.w, v);
                    }
                } else {
                    for (int k = 0; k < kShKeys; ++k) {
                        const float4 v = *reinterpret_cast<const float4*>(s_v + k * p.dv + col);
#pragma unroll
                        for (int i = 0; i < kRw; ++i)
                            if (sees[i] >> k & 1) {
                                const float w = s_p[(warp * kShKeys + k) * kRw + i], x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[i][c][e] = sh_add(o[i][c][e], w, x[e]);
                            }
                    }
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < kRw; ++i) {
            const int r = r0 + warp * kRw + i;
            if (r >= sp.n_rows) break;
            float* rec = sh_record(p, sp.tok0 + r / per, g * per + r % per, sp.which);
            const float sum = warp_sum(l[i]);
            if (lane == 0) {
                rec[0] = m[i] * 1.4426950408889634f;
                rec[1] = sum;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = c * 128 + 4 * lane;
                if (col < p.dv) *reinterpret_cast<float4*>(rec + kShHead + col) = make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
            }
        }
    }
}

// The grid's x: row tiles of the groups (as many as there can be; the ones there are not have nothing to do), then the listed tiles of queries. y: kv heads; z: shares of the keys.
template <typename T, int kRw>
__global__ void __launch_bounds__(kShWarps * 32) seq_attention_shared_kernel(SharedArgs p, int group_tiles) {
    after_previous();
    extern __shared__ __align__(16) float sh_smem[];
    constexpr int kRows = kShWarps * kRw;
    const int g = blockIdx.y, per = p.heads / p.kv_heads, z = blockIdx.z, tokens = max(1, kRows / per);      // of a row tile
    ShSpan sp;
    if ((int)blockIdx.x < group_tiles) {
        if (z >= p.shares) return;
        int tile = blockIdx.x, first, n;
        const int i = sh_find_group(p, tokens, tile, first, n);
        if (i < 0) return;
        const int len = sh_group_len(p, i), tiles = (len + kShKeys - 1) / kShKeys, cuts = sh_cuts(len, p.least, p.shares);
        if (z >= cuts) return;
        sp.tok0 = first + tile * tokens;
        sp.n_rows = min(tokens, n - tile * tokens) * per;
        sp.slot = p.b.seg_slot[p.group_start[i]];
        sp.key0 = tiles * z / cuts * kShKeys;
        sp.key1 = min(len, tiles * (z + 1) / cuts * kShKeys);
        sp.which = z;
    } else {
        if (z >= p.own) return;
        const int x = blockIdx.x - group_tiles, seg = p.b.qt_seg[x], off = p.b.qt_off[x];
        const int n = min(kBQ, p.b.seg_len[seg] - off), end = p.b.seg_pos0[seg] + off + n;
        const int shared = sh_shared_len(p, seg), from = min(shared, end);
        const int t0 = from / kShKeys, tiles = (end + kShKeys - 1) / kShKeys - t0, cuts = sh_cuts(end - from, p.own_least, p.own);
        if (g == 0 && z == 0 && threadIdx.x == 0) p.plan[x] = sh_cuts(shared, p.least, p.shares) | cuts << 16;
        if (z >= cuts) return;
        sp.tok0 = p.b.seg_start[seg] + off;
        sp.n_rows = n * per;
        sp.slot = p.b.seg_slot[seg];
        sp.key0 = max(from, (t0 + tiles * z / cuts) * kShKeys);
        sp.key1 = min(end, (t0 + tiles * (z + 1) / cuts) * kShKeys);
        sp.which = p.shares + z;
    }
    sh_rows<T, kRw>(p, sp, g, sh_smem);
}

// The records of a (token, head) put together: a warp each. Bound: loads one behind the other (the tile, its segment, kAhead records at a time).
template <bool kVec, int kAhead>         // results 16 bytes at a time; records on their way at once
__global__ void __launch_bounds__(128) seq_attention_shared_merge_kernel(SharedArgs p) {
    after_previous();
    const int seg = p.b.qt_seg[blockIdx.x], off = p.b.qt_off[blockIdx.x], cuts = (int)__vminu2(p.plan[blockIdx.x], p.shares | p.own << 16), lane = threadIdx.x & 31;
    // (no more records than there are places for, whatever the plan may say)
    const int n = min(kBQ, p.b.seg_len[seg] - off), t0 = p.b.seg_start[seg] + off, first = cuts & 0xffff, count = first + (cuts >> 16), step = p.dv + kShHead;
    for (int i = blockIdx.y * 4 + (threadIdx.x >> 5); i < n * p.heads; i += gridDim.y * 4) {
        const int t = t0 + i / p.heads, h = i % p.heads;
        const float* recs = sh_record(p, t, h, 0);
        auto place = [&](int k) { return recs + (size_t)(k < first ? k : p.shares + k - first) * step; };
        // at most 48 records: references and sums two a lane
        float2 head[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int k = lane + 32 * x;
            head[x] = *reinterpret_cast<const float2*>(place(min(k, max(count, 1) - 1)));
            if (k >= count) head[x] = make_float2(-INFINITY, 0.0f);
        }
        // kAhead records' columns at a time, the first of them on their way while the factors are made
        float4 x[kAhead];
        auto fetch = [&](int k0, int c) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = *reinterpret_cast<const float4*>(place(min(k0 + k, max(count, 1) - 1)) + kShHead + min(c * 128 + 4 * lane, p.dv - 4));
        };
        fetch(0, 0);
        const float top = warp_max(fmaxf(head[0].x, head[1].x));
        float f[2], sum = 0.0f, o[2][4] = {};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            f[x] = head[x].x == -INFINITY && head[x].y == 0.0f ? 0.0f : exp2f(head[x].x - top);      // nothing seen: nothing (a sum of NaN goes on)
            sum = fmaf(f[x], head[x].y, sum);
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (c * 128 >= p.dv) break;
            for (int k0 = 0; k0 < count; k0 += kAhead) {
                if (c + k0 > 0) fetch(k0, c);
                float w[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) w[k] = __shfl_sync(0xffffffffu, k0 < 32 ? f[0] : f[1], (k0 + k) & 31);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    if (k0 + k >= count) break;
                    o[c][0] = fmaf(w[k], x[k].x, o[c][0]); o[c][1] = fmaf(w[k], x[k].y, o[c][1]); o[c][2] = fmaf(w[k], x[k].z, o[c][2]); o[c][3] = fmaf(w[k], x[k].w, o[c][3]);
                }
            }
        }
        // NaN: as a rule an infinity times a factor that 32 bits have no number for, which is to stay an infinity. Once more, asking for each
        bool none = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) none |= o[e / 4][e % 4] != o[e / 4][e % 4];
        if (__any_sync(0xffffffffu, none)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e / 4][e % 4] = 0.0f;
#pragma unroll 1
            for (int k = 0; k < count; ++k) {
                const float w = __shfl_sync(0xffffffffu, k < 32 ? f[0] : f[1], k & 31);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (c * 128 + 4 * lane >= p.dv) break;
                    const float4 y = *reinterpret_cast<const float4*>(place(k) + kShHead + c * 128 + 4 * lane);
                    o[c][0] = sh_add(o[c][0], w, y.x); o[c][1] = sh_add(o[c][1], w, y.y); o[c][2] = sh_add(o[c][2], w, y.z); o[c][3] = sh_add(o[c][3], w, y.w);
                }
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = c * 128 + 4 * lane;
            if (col >= p.dv) break;
            const float y[4] = {o[c][0] * inv, o[c][1] * inv, o[c][2] * inv, o[c][3] * inv};
            if (p.out) {
                float* to = p.out + (size_t)t * p.ldo + (size_t)h * p.dv + col;
                if constexpr (kVec) {
                    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = y[e];
                }
            }
            if (p.out16) {
                uint16_t* to = p.out16 + ((size_t)t * p.heads + h) * p.dv + col;
                if constexpr (kVec) {
                    *reinterpret_cast<uint2*>(to) = make_uint2((uint32_t)f32_to_bf16_bits(y[0]) | (uint32_t)f32_to_bf16_bits(y[1]) << 16,
                                                               (uint32_t)f32_to_bf16_bits(y[2]) | (uint32_t)f32_to_bf16_bits(y[3]) << 16);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = f32_to_bf16_bits(y[e]);
                }
            }
        }
    }
}

static int sh_merge(const SharedArgs& p, cudaStream_t st) {
    const int most = (p.b.T == p.b.nseg ? p.heads : kBQ * p.heads) / 4 + 1;
    const bool vec = p.ldo % 4 == 0 && ((uintptr_t)p.out % 16) == 0 && ((uintptr_t)p.out16 % 8) == 0;
    LaunchCfg lc(dim3(p.b.n_qtiles, std::min(most, 256)), dim3(128), 0, st, true);
    // records on their way: few rows have many records each and wait for them, many rows few, and CTAs enough to wait beside one another. us of the whole call, 4 | 16: 4 answers behind 1500 positions
    // in fp32 20.2 | 18.6, 64 behind 8000 62.8 | 60.7, 512 rows behind 4000 110.6 | 119.5
    const bool few = (long long)p.b.T * p.heads < 16LL * sm_count();
    auto launch = [&](auto whole, auto ahead) { return cudaLaunchKernelEx(&lc.cfg, overlapping(seq_attention_shared_merge_kernel<whole.value, ahead.value>), p); };
    using four = std::integral_constant<int, 4>;
    using sixteen = std::integral_constant<int, 16>;
    SLLM_CUDA(vec ? few ? launch(std::true_type{}, sixteen{}) : launch(std::true_type{}, four{}) : few ? launch(std::false_type{}, sixteen{}) : launch(std::false_type{}, four{}));
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

template <typename T, int kRw>
static int sh_launch(const SharedArgs& p, cudaStream_t st) {
    constexpr int kRows = kShWarps * kRw;
    const int tokens = std::max(1, kRows / (p.heads / p.kv_heads));
    const size_t smem = ((size_t)kRows * p.dk + (size_t)kShKeys * (p.dk + 4 + p.dv) + kShWarps * kShKeys * kRw) * sizeof(float);
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(seq_attention_shared_kernel<T, kRw>, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024));
            return SLLM_OK;
        }))
        return rc;
    const long long tiles = (p.b.T + tokens - 1) / tokens + p.n_groups;
    SLLM_REQUIRE(tiles + p.b.n_qtiles <= 0x7fffffffLL, SLLM_ENOTSUP, "seq_attention_shared: too many tokens");
    overlapping(seq_attention_shared_kernel<T, kRw>)<<<dim3((unsigned)tiles + p.b.n_qtiles, p.kv_heads, std::max(p.shares, p.own)), kShWarps * 32, smem, st>>>(p, (int)tiles);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

}  // namespace sllm

using namespace sllm;

// Shares of the keys at most, the same for every call with these sizes: enough CTAs for the machine, however few rows there are.
static void shared_plan(int64_t T, int n_qtiles, int n_groups, int heads, int kv_heads, int* shares, int* own) {
    const int64_t tiles = (T * (heads / kv_heads) / 128 + n_groups) * kv_heads, tiles_own = (int64_t)n_qtiles * kv_heads;
    *shares = (int)std::min<int64_t>(32, std::max<int64_t>(1, (4 * sm_count() + tiles - 1) / tiles));
    // (two at a time, two CTAs an SM: where there are several, one more than fits would take a second round, 8 tokens behind 3000 positions 46 us instead of 38; where there are one or two, a second
    // share is what evens long ones out: with one the mixed step of 52 tiles took 229 us instead of 204)
    const int64_t fit = 4 * sm_count() / tiles_own;
    *own = (int)std::min<int64_t>(16, fit >= 4 ? fit : std::max<int64_t>(1, (4 * sm_count() + tiles_own - 1) / tiles_own));
}

extern "C" {

int64_t sllm_seq_attention_shared_ws_bytes(const sllm_seq_batch* b, int32_t n_groups, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv) {
    SLLM_REQUIRE(b && b->T > 0 && b->nseg > 0 && b->n_qtiles > 0 && n_groups > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && dk > 0 && dv > 0, SLLM_EINVAL,
                 "seq_attention_shared_ws_bytes: bad argument");
    int shares, own;
    shared_plan(b->T, b->n_qtiles, n_groups, heads, kv_heads, &shares, &own);
    return ((int64_t)b->T * heads * (shares + own) * (dv + kShHead) + attention_shared_tc_flush_floats(dk, dv)) * (int64_t)sizeof(float) + sh_plan_bytes(b->n_qtiles);
}

int sllm_seq_attention_shared(const sllm_seq_batch* b, int32_t n_groups, const int32_t* group_start, const int32_t* group_len, const float* q, int32_t ldq, int32_t heads, int32_t kv_heads,
                              int32_t dk, int32_t dv, float scale, const void* k_pool, const void* v_pool, int32_t kv_dtype, int32_t n_pages, void* ws, int64_t ws_bytes,
                              const sllm_seq_attn_opts* opts, float* out, int32_t ldo, void* out16, sllm_stream_t stream) {
    SLLM_REQUIRE(b && b->T > 0 && b->nseg > 0 && b->tok_pos && b->seg_start && b->seg_len && b->seg_slot && b->seg_pos0 && b->block_table && b->max_pages > 0 && b->qt_seg && b->qt_off &&
                     b->n_qtiles > 0,
                 SLLM_EINVAL, "seq_attention_shared: incomplete batch description");
    SLLM_REQUIRE(n_groups > 0 && n_groups <= b->nseg && group_start && group_len, SLLM_EINVAL, "seq_attention_shared: %d groups of %d segments", n_groups, b->nseg);
    SLLM_REQUIRE(q && k_pool && v_pool && n_pages > 0 && (out || out16), SLLM_EINVAL, "seq_attention_shared: null pointer, no pages or no output");
    SLLM_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, SLLM_EINVAL, "seq_attention_shared: %d query heads over %d kv heads", heads, kv_heads);
    SLLM_REQUIRE(kv_dtype == SLLM_F32 || kv_dtype == SLLM_BF16, SLLM_ENOTSUP, "seq_attention_shared: fp32 or bf16 pools");
    SLLM_REQUIRE(dk > 0 && dv > 0 && dk % 8 == 0 && dv % 8 == 0 && dk <= 256 && dv <= 256, SLLM_ENOTSUP, "seq_attention_shared: head widths %d and %d are not multiples of 8 up to 256", dk, dv);
    SLLM_REQUIRE(kv_heads <= 65535, SLLM_ENOTSUP, "seq_attention_shared: %d kv heads", kv_heads);
    SLLM_REQUIRE(scale > 0.0f && scale <= FLT_MAX, SLLM_EINVAL, "seq_attention_shared: scores need a positive finite scale");
    SLLM_REQUIRE(b->page_len > 0 && b->page_len % kBK == 0, SLLM_ENOTSUP, "seq_attention_shared: pages of a multiple of %d positions", kBK);
    SLLM_REQUIRE((int64_t)b->max_pages * b->page_len <= kShMostPositions, SLLM_ENOTSUP, "seq_attention_shared: tables of up to %d positions", kShMostPositions);
    SLLM_REQUIRE(ldq >= heads * dk && (!out || ldo >= heads * dv), SLLM_EINVAL, "seq_attention_shared: a row is shorter than its heads");
    SLLM_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool) % 16) == 0, SLLM_EINVAL, "seq_attention_shared: pools have to start at a multiple of 16 bytes");
    SLLM_REQUIRE(ws && ((uintptr_t)ws % 16) == 0 && ws_bytes >= sllm_seq_attention_shared_ws_bytes(b, n_groups, heads, kv_heads, dk, dv), SLLM_EINVAL,
                 "seq_attention_shared: the workspace is too small or not aligned");
    SLLM_REQUIRE(!opts || (opts->window >= 0 && opts->keep_first >= 0 && opts->softcap >= 0.0f && opts->softcap <= FLT_MAX), SLLM_EINVAL, "seq_attention_shared: bad options");
    SLLM_REQUIRE(!opts || (!opts->values_in_keys && !opts->logdist && !opts->cross_values && !opts->chunk), SLLM_ENOTSUP,
                 "seq_attention_shared: values in keys, charges on the logarithm of the distance, values of every head and chunks are not part of this form");
    SharedArgs p{*b, n_groups, group_start, group_len, q, ldq, heads, kv_heads, dk, dv, scale, k_pool, v_pool, n_pages, INT_MAX, 0, 0.0f, nullptr, 0, 0,
                 b->max_pages * b->page_len,
                 (uint32_t)(((1ull << 32) + b->page_len - 1) / b->page_len), 0, 0, (int*)ws,
                 (float*)((char*)ws + sh_plan_bytes(b->n_qtiles)), nullptr, out, ldo, (uint16_t*)out16};
    if (opts) {
        if (opts->window > 0) {
            p.window = opts->window;
            p.keep_first = opts->keep_first;
        }
        p.softcap = opts->softcap;
        p.slopes = opts->slopes;
    }
    shared_plan(b->T, b->n_qtiles, n_groups, heads, kv_heads, &p.shares, &p.own);
    p.flush = p.ws + (int64_t)b->T * heads * (p.shares + p.own) * (dv + kShHead);
    if (int rc = status_check()) return rc;
    cudaStream_t st = as_stream(stream);
    const bool tc = kv_dtype == SLLM_BF16 && dk == dv && (dk == 64 || dk == 128);
    p.least = 64;
    // On the tensor cores' kernel a share of a segment's own keys costs as much as some hundred keys at its beginning and end, so it has 512 unless there are too few segments to occupy two CTAs an SM.
    // us, 512 always | like this: a token behind 2000 positions of its own 29.9 | 17.5, four behind 1000 31.6 | 17.7, 16 behind 500 and 1000 shared ones 32.6 | 28.2, a portion of 512 37.0 | 33.0;
    // half as long where there are segments enough, that portion took 40.5.
    const int64_t units = (int64_t)b->n_qtiles * kv_heads;
    p.own_least = tc ? (int)std::min<int64_t>(512, std::max<int64_t>(128, (512 * units / (2 * sm_count()) + 63) / 64 * 64)) : 64;
    const int rc = tc ? launch_attention_shared_tc(p, st) : kv_dtype == SLLM_F32 ? sh_launch<float, 4>(p, st) : sh_launch<uint16_t, 4>(p, st);
    return rc ? rc : sh_merge(p, st);
}

}  // extern "C"
