// csrc/seq_attn8_decode.cu — attention of single tokens over the 8-bit paged cache, heads of up to 128 columns: one launch, whatever the contexts are.
//
// Bound: the cache's bytes. Everything else is arranged so that they keep coming:
//   Work. A unit is one block of 32 keys for the query heads of a kv head (up to 8 at a time). All units of a step lie in one row, request by request and head by head, and every CTA
//   takes an equal share of it, found from the contexts on the device: requests of 77 and of 8000 positions fill the machine alike. A request's head that several CTAs share is put
//   together by the one of them that is done last (a counter), in the order of its parts.
//   Loads. A unit is two boxes of 32 rows (TMA, swizzled so that the reads below meet no bank twice) into a ring of the warp's own; a warp takes every fourth unit of its CTA's share and
//   waits for nobody else's.
//   Products on mma.sync m16n8k16 with fp16 operands: e4m3 codes are fp16 numbers, so keys and values enter exactly, two codes an instruction. Keys are the A operand (16 of them x 16
//   columns), queries the B operand: its eight columns are four heads twice, a query's value being the sum of two fp16 numbers (22 bits of the head's largest, which a power of two brings to
//   1 .. 2). Both terms' scores then lie side by side in one lane. The softmax's weights are split the same way, transposed by movmatrix, and are the B operand of the second product, whose A
//   operand is the values, turned on the way from shared memory by two byte permutations for four codes. Which key is which row, and which column which k, is free as long
//   as both operands agree: the order is the one in which a lane's 16-byte reads deliver them.
//   Sums. The tensor core truncates as it accumulates: a chain is two instructions long before it is added to an fp32 register with ordinary rounding.
//   Scales are numbers of a unit: a key scale multiplies scores, a value scale the weights. Weights are relative to the largest of (score + exponent of the value scale), kept as a
//   whole number R, so that they are at most 2 whatever the scales are and changing R is exact; the denominator has a reference of its own.
#include "seq_attn8.cuh"
#include "tcgen05.cuh"

namespace sllm {

constexpr int kD8Warps = 4, kD8Least = 8;       // warps of a CTA; units of a CTA's share at least

template <int D>
struct D8Tile {
    static constexpr int kRows = kKv8Block * D, kStage = 2 * kRows, kRing = D == 128 ? 3 : 6;      // bytes of a unit's keys; of keys and values; stages of a warp
    static constexpr int kSmem = 1024 + kD8Warps * kRing * kStage;
};

struct D8Args {
    Attn8Args a;
    int only;                    // the launch is the step's only one: it has no tiles of more than one query
    int sets, per_set;           // groups of query heads that a kv head's are divided into, and how many of them one holds
    int* counters;
    float* records;
    int32_t* status;
    unsigned polls;
};

__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_round(float x) { return __half2float(__float2half_rn(x)); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
// byte offset of 16-byte chunk `chunk` of row `row` in a box
template <int D>
__device__ __forceinline__ uint32_t d8_at(int row, int chunk) {
    return (uint32_t)(row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4));
}

// References are whole numbers (of log2). Beyond +-10^9, where scores in fp32 are 64 apart, exponents stop there and the rest is carried by the reference alone.
constexpr float kD8Far = 1e9f;
constexpr int kD8None = -1100000000;         // exponent of sums that hold nothing yet
__device__ __forceinline__ int d8_whole(float x) { return (int)fmaxf(-kD8Far, fminf(kD8Far, x)); }
__device__ __forceinline__ float d8_factor(float from, float to) {        // 2^(from - to) but for what the exponents say
    return from == to ? 1.0f : tc_exp2((from - (float)d8_whole(from)) - (to - (float)d8_whole(to)));
}

// What a tile of the list has to do here: units of one head set, 0 when it holds more than one query (or none)
__device__ __forceinline__ int d8_units(const D8Args& da, int tile) {
    const Attn8Args& p = da.a;
    const int seg = p.b.qt_seg[tile], off = p.b.qt_off[tile], n = p.b.seg_len[seg] - off;
    if (n > 1 && da.only) *reinterpret_cast<volatile int32_t*>(da.status) = kStatusSingle;
    if (n != 1) return 0;
    const int pos = p.b.seg_pos0[seg] + off;
    return pos < 0 ? 0 : TileList(pos, pos, seq_row_window(pos, p.window, p.chunk), p.keep_first, kKv8Block).n;
}

template <int D, int NT>       // column width of a head, rounded up; groups of four query heads
__global__ void __launch_bounds__(kD8Warps * 32, 2) seq_attention8_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const D8Args da) {
    using Tile = D8Tile<D>;
    constexpr int kRing = Tile::kRing, kChunk = D / 8, kSteps = D / 16, kMt = D / 16, kHeads = 4 * NT;   // bytes of a value row a lane reads; k-steps of a score; 16-column tiles of a result
    const Attn8Args& p = da.a;
    const sllm_seq_batch& b = p.b;
    extern __shared__ uint8_t d8_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(d8_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[kD8Warps][kRing];
    __shared__ int s_page[kD8Warps][kRing];
    __shared__ float2 s_scale[kD8Warps][kRing];
    __shared__ long long s_sum[kD8Warps];
    __shared__ int s_tile, s_gave_up, s_last;
    __shared__ long long s_before;
    __shared__ float s_ref[kD8Warps][kHeads], s_l[kD8Warps][kHeads];
    __shared__ int s_R[kD8Warps][kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    volatile int* gave_up = &s_gave_up;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kD8Warps; ++w)
            for (int i = 0; i < kRing; ++i) mb_init(&bars[w][i], 1);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    after_previous();

    // ---- the row of all units, and this CTA's share of it ----
    const int per_tile = p.kv_heads * da.sets, n_tiles = b.n_qtiles;
    const int per_thread = (n_tiles + kD8Warps * 32 - 1) / (kD8Warps * 32), t0 = min(n_tiles, (int)threadIdx.x * per_thread), t1 = min(n_tiles, t0 + per_thread);
    long long mine = 0;
    for (int i = t0; i < t1; ++i) mine += d8_units(da, i);
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < kD8Warps; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    total *= per_tile;
    before *= per_tile;
    const int ctas = (int)min((long long)gridDim.x, (total + kD8Least - 1) / kD8Least);
    if ((int)blockIdx.x >= ctas) return;
    auto share = [&](int x) { return (long long)x * total / ctas; };
    auto owner = [&](long long u) { return (int)(((u + 1) * ctas - 1) / total); };
    const long long begin = share(blockIdx.x), end = share(blockIdx.x + 1);
    if (begin >= before && begin < before + mine * per_tile) {
        long long at = before;
        for (int i = t0; i < t1; ++i) {
            const long long n = (long long)d8_units(da, i) * per_tile;
            if (begin < at + n) {
                s_tile = i;
                s_before = at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    int tile = s_tile;
    long long tile0 = s_before;

    const uint32_t ring = s_addr(smem) + warp * (kRing * Tile::kStage);
    uint32_t turns = 0;                    // units this warp has taken so far: stage and parity
    int fresh = 1;                         // no shared memory written by ordinary stores since the last copies
    // ---- pieces: this CTA's part of one head set of one tile ----
    for (long long u = begin; u < end;) {
        const int seg = b.qt_seg[tile], off = b.qt_off[tile], t = b.seg_start[seg] + off, pos = b.seg_pos0[seg] + off, slot = b.seg_slot[seg];
        const int wnd = seq_row_window(pos, p.window, p.chunk);
        const TileList blocks(pos, pos, wnd, p.keep_first, kKv8Block);
        if (u >= tile0 + (long long)blocks.n * per_tile || b.seg_len[seg] - off != 1 || pos < 0) {       // the next tile (this one may have nothing to do here)
            if (b.seg_len[seg] - off == 1 && pos >= 0) tile0 += (long long)blocks.n * per_tile;
            ++tile;
            continue;
        }
        const int set = (int)((u - tile0) / blocks.n), gkv = set / da.sets, h0 = gkv * (p.heads / p.kv_heads) + (set % da.sets) * da.per_set;
        const int G = min(da.per_set, (gkv + 1) * (p.heads / p.kv_heads) - h0);                       // query heads of this set
        const long long item0 = tile0 + (long long)set * blocks.n, item1 = item0 + blocks.n;
        const int j0 = (int)(u - item0), j1 = (int)(min(end, item1) - item0), n_mine = max(0, (j1 - j0 - warp + kD8Warps - 1) / kD8Warps);
        if (!fresh) {                      // the last piece's sums were written where copies land: in front of them for everybody
            fence_async_smem();
            __syncthreads();
            fresh = 1;
        }
        // ---- loads: unit i of this warp ----
        int ahead_page = -1;               // lane l: page of unit 32 * x + l
        auto issue = [&](int i) {
            if ((i & 31) == 0) {
                const int at = i + lane;
                ahead_page = at < n_mine ? kv8_page(b, p.n_pages, slot, blocks.tile_of(j0 + warp + at * kD8Warps) * kKv8Block) : -1;
            }
            const int page = __shfl_sync(0xffffffffu, ahead_page, i & 31);
            if (i < n_mine) {
                const int stage = (int)((turns + i) % kRing), in_page = blocks.tile_of(j0 + warp + i * kD8Warps) * kKv8Block % b.page_len;
                if (lane == 0) {
                    s_page[warp][stage] = page;
                    if (page >= 0) {
                        const int row = (page * p.kv_heads + gkv) * b.page_len + in_page;
                        uint8_t* dst = smem + (warp * kRing + stage) * Tile::kStage;
                        mb_expect(&bars[warp][stage], Tile::kStage);
                        tma_load_2d(dst, &tmK, 0, row, &bars[warp][stage]);
                        tma_load_2d(dst + Tile::kRows, &tmV, 0, row, &bars[warp][stage]);
                    } else {
                        mb_arrive(&bars[warp][stage]);
                    }
                } else if (lane <= 2 && page >= 0) {
                    const float* src = (lane == 1 ? p.k_scale : p.v_scale) + kv8_scale_at(page, p.kv_heads, gkv, b.page_len, in_page);
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s_addr(&s_scale[warp][stage]) + (lane - 1) * 4), "l"(src) : "memory");
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) issue(i);
        // ---- queries: two fp16 terms of q * 2^-e, e from the head's largest ----
        uint32_t qb[NT][kSteps][2];
        float factor[NT];                  // what a sum of products times a key scale is multiplied by
        float slope[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const int h = 4 * x + (g >> 1);
            const bool live = h < G;
            const float* q = p.q + (size_t)t * p.ldq + (size_t)(h0 + (live ? h : 0)) * p.dk;
            float v[kSteps][4], top = 0.0f;
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
                const int col = 16 * (c + 4 * (ks / 4)) + 4 * (ks % 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[ks][e] = live && col < p.dk ? q[col + e] : 0.0f;
                    top = fmaxf(top, fabsf(v[ks][e]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int ex = top < INFINITY ? max((int)(__float_as_uint(top) >> 23) - 127, -100) : 0;
            const float down = kv8_pow2(-ex), up = kv8_pow2(ex);
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = v[ks][e] * down, hi = f16_round(y);
                    w[e] = g & 1 ? y - hi : hi;
                }
                qb[x][ks][0] = pack_f16(w[0], w[1]);
                qb[x][ks][1] = pack_f16(w[2], w[3]);
            }
            // scores are head c's on this lane: its scale comes from the lanes that hold its queries
            factor[x] = p.scale * __shfl_sync(0xffffffffu, up, 8 * c + c);
            slope[x] = p.slopes && 4 * x + c < G ? p.slopes[h0 + 4 * x + c] : 0.0f;
        }
        float ref[NT], l[NT], o[NT][kMt][2];
        int R[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            ref[x] = -INFINITY;
            l[x] = 0.0f;
            R[x] = kD8None;
#pragma unroll
            for (int i = 0; i < kMt; ++i) o[x][i][0] = o[x][i][1] = 0.0f;
        }
        const int fg = g ^ ((g & 1) << 2);                          // key of row g: rows of a read lie in different banks
        bool ok = true;
        for (int i = 0; i < n_mine; ++i) {
            issue(i + kRing - 1);                                   // (the stage of unit i - 1, which every lane has read)
            const int stage = (int)((turns + i) % kRing);
            cp_async_wait<kRing - 1>();
            ok = tc_wait_warp(&bars[warp][stage], (uint32_t)((turns + i) / kRing) & 1, gave_up, da.polls);
            if (!ok) break;
            __syncwarp();
            if (s_page[warp][stage] < 0) continue;
            const float ks_ = s_scale[warp][stage].x, vs_ = s_scale[warp][stage].y;
            const uint32_t kb = ring + stage * Tile::kStage, vb = kb + Tile::kRows;
            const int key0 = blocks.tile_of(j0 + warp + i * kD8Warps) * kKv8Block;
            // ---- scores: two tiles of 16 keys ----
            float w[NT][4];                                          // weights of keys fg, fg + 8, fg + 16, fg + 24 for head c (and 4 + c)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                float s[NT][4];
#pragma unroll
                for (int x = 0; x < NT; ++x) s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.0f;
#pragma unroll
                for (int half = 0; half < D / 64; ++half) {
                    const int r0 = 16 * mt + fg;
                    const uint4 lo = lds16(kb + d8_at<D>(r0, c + 4 * half)), hi = lds16(kb + d8_at<D>(r0 + 8, c + 4 * half));
                    const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, d[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        float part[NT][4];
                        const uint32_t f0[4] = {kv8_half2(a[e] & 0xffffu), kv8_half2(d[e] & 0xffffu), kv8_half2(a[e] >> 16), kv8_half2(d[e] >> 16)};
                        const uint32_t f1[4] = {kv8_half2(a[e + 1] & 0xffffu), kv8_half2(d[e + 1] & 0xffffu), kv8_half2(a[e + 1] >> 16), kv8_half2(d[e + 1] >> 16)};
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            mma_f16_zero(part[x], f0, qb[x][4 * half + e][0], qb[x][4 * half + e][1]);
                            mma_f16(part[x], f1, qb[x][4 * half + e + 1][0], qb[x][4 * half + e + 1][1]);
#pragma unroll
                            for (int y = 0; y < 4; ++y) s[x][y] += part[x][y];
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    w[x][2 * mt] = s[x][0] + s[x][1];
                    w[x][2 * mt + 1] = s[x][2] + s[x][3];
                }
            }
            const bool masked = key0 + kKv8Block - 1 > pos || (pos - key0 >= wnd && key0 + kKv8Block > p.keep_first);
            const int ev = (int)(__float_as_uint(vs_) >> 23 & 0xff) - 127;
            const float mant = __uint_as_float((__float_as_uint(vs_) & 0x7fffffu) | 0x3f800000u);        // 1 for the scales the append leaves
            uint32_t pb[NT][4];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                const float f = factor[x] * ks_;
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = w[x][e] * f;
                    if (p.softcap > 0.0f || p.slopes) v = attn8_score(v, p.softcap, slope[x], pos, key0 + fg + 8 * e);
                    v *= 1.4426950408889634f;
                    if (masked && !seq_sees(pos, key0 + fg + 8 * e, wnd, p.keep_first)) v = -INFINITY;
                    w[x][e] = v;
                    mx = fmaxf(mx, v);
                }
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                const float up = ceilf(mx);
                if (up > ref[x]) {
                    const float less = tc_exp2(ref[x] - up);
                    l[x] *= less;
                    if (fabsf(up) > kD8Far)
#pragma unroll
                        for (int k = 0; k < kMt; ++k) {
                            o[x][k][0] *= less;
                            o[x][k][1] *= less;
                        }
                    ref[x] = up;
                }
                const int want = d8_whole(up) + ev;
                if (up > -INFINITY && want > R[x]) {
                    const float down = want - R[x] > 126 ? 0.0f : kv8_pow2(R[x] - want);
#pragma unroll
                    for (int k = 0; k < kMt; ++k) {
                        o[x][k][0] *= down;
                        o[x][k][1] *= down;
                    }
                    R[x] = want;
                }
                const float base = ref[x] == -INFINITY ? 0.0f : ref[x];                              // nothing seen yet: every weight is 0
                const int d = ev + d8_whole(ref[x]) - R[x];
                const float lift = mant * kv8_pow2(max(-126, min(126, d)));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float q = tc_exp2(w[x][e] - base);
                    l[x] += q;
                    const float y = q * lift, hi = f16_round(y);
                    pb[x][e] = movmatrix_trans(pack_f16(hi, y - hi));
                }
            }
            // ---- values: two runs of 16 keys ----
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                uint32_t v[4][kChunk / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 2 * c + (e & 1), key = 16 * ks + 8 * (e >> 1) + (row ^ ((row & 1) << 2));
                    if constexpr (D == 128) {
                        const uint4 y = lds16(vb + d8_at<D>(key, g));
                        v[e][0] = y.x; v[e][1] = y.y; v[e][2] = y.z; v[e][3] = y.w;
                    } else {
                        const uint2 y = lds8(vb + d8_at<D>(key, g >> 1) + 8 * (g & 1));
                        v[e][0] = y.x; v[e][1] = y.y;
                    }
                    if (masked && !seq_sees(pos, key0 + key, wnd, p.keep_first)) {                   // a hidden row may hold anything
#pragma unroll
                        for (int k = 0; k < kChunk / 4; ++k) v[e][k] = 0u;
                    }
                }
#pragma unroll
                for (int k = 0; k < kChunk / 4; ++k) {
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd) {
                        const uint32_t sel = odd ? 0x7362u : 0x5140u, y = __byte_perm(v[0][k], v[1][k], sel), z = __byte_perm(v[2][k], v[3][k], sel);
                        const uint32_t a[4] = {kv8_half2(y & 0xffffu), kv8_half2(y >> 16), kv8_half2(z & 0xffffu), kv8_half2(z >> 16)};
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            float part[4];
                            mma_f16_zero(part, a, pb[x][2 * ks], pb[x][2 * ks + 1]);
                            o[x][2 * k + odd][0] += part[0] + part[1];
                            o[x][2 * k + odd][1] += part[2] + part[3];
                        }
                    }
                }
            }
            __syncwarp();
        }
        turns += n_mine;
        // ---- the four warps' sums together ----
        cp_async_wait<0>();
        __syncthreads();                   // every stage has been read
        if (s_gave_up) break;
        float* sums = reinterpret_cast<float*>(smem);                       // [warp][head][D]
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], s);
            const int h = 4 * x + c;
            if (g == 0) {
                s_ref[warp][h] = ref[x];
                s_l[warp][h] = l[x];
                s_R[warp][h] = R[x];
            }
            float* dst = sums + (warp * kHeads + h) * D + kChunk * g;
#pragma unroll
            for (int i = 0; i < kMt; i += 2) *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[x][i][0], o[x][i][1], o[x][i + 1][0], o[x][i + 1][1]);
        }
        fresh = 0;
        __syncthreads();
        // reference, sum and exponent of a head over `n` parts; then a column's value from them
        const int first_cta = owner(item0), last_cta = owner(item1 - 1), parts = last_cta - first_cta + 1;
        float* record = da.records + (size_t)(2 * blockIdx.x + (begin >= item0 ? 0 : 1)) * kA8Record;
        constexpr int kTail = kA8MaxHeads * 128;                               // where a record's references, sums and exponents begin
        auto store = [&](int h, int col, float v) {
            if (p.out) p.out[(size_t)t * p.ldo + (size_t)(h0 + h) * p.dv + col] = v;
            if (p.out16) p.out16[((size_t)t * p.heads + h0 + h) * p.dv + col] = f32_to_bf16_bits(v);
        };
        auto result = [&](float sum, float den, float r, int e) {              // sum * 2^e / (den * 2^r); a query that sees no key gives 0
            if (den == 0.0f) return 0.0f;
            const int d = e - d8_whole(r);
            return sum / den * kv8_pow2(max(-126, min(126, d)));
        };
        for (int i = threadIdx.x; i < G * D; i += kD8Warps * 32) {
            const int h = i / D, col = i % D;
            float r = -INFINITY, den = 0.0f, sum = 0.0f;
            int e = kD8None;
#pragma unroll
            for (int w = 0; w < kD8Warps; ++w) {
                r = fmaxf(r, s_ref[w][h]);
                e = max(e, s_R[w][h]);
            }
#pragma unroll
            for (int w = 0; w < kD8Warps; ++w) {
                const int d = s_R[w][h] - e;
                den += s_l[w][h] * (s_ref[w][h] == r ? 1.0f : tc_exp2(s_ref[w][h] - r));
                sum += sums[(w * kHeads + h) * D + col] * (d < -126 ? 0.0f : kv8_pow2(d) * d8_factor(s_ref[w][h], r));
            }
            if (parts == 1) {
                if (col < p.dv) store(h, col, result(sum, den, r, e));
            } else {
                record[h * 128 + col] = sum;
                if (col == 0) {
                    record[kTail + 4 * h] = r;
                    record[kTail + 4 * h + 1] = den;
                    record[kTail + 4 * h + 2] = __int_as_float(e);
                }
            }
        }
        if (parts > 1) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                s_last = atomicAdd(da.counters + first_cta, 1) == parts - 1;
                if (s_last) da.counters[first_cta] = 0;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {                  // all parts are there: in the order of the units, whoever was last
                const float* rest = da.records + (size_t)2 * first_cta * kA8Record;
                auto part = [&](int i) { return rest + (size_t)(2 * i + (i == 0 && share(first_cta) < item0 ? 1 : 0)) * kA8Record; };
                for (int i = threadIdx.x; i < G * D; i += kD8Warps * 32) {
                    const int h = i / D, col = i % D;
                    float r = -INFINITY, den = 0.0f, sum = 0.0f;
                    int e = kD8None;
#pragma unroll 8
                    for (int x = 0; x < parts; ++x) {
                        r = fmaxf(r, __ldcg(part(x) + kTail + 4 * h));
                        e = max(e, __float_as_int(__ldcg(part(x) + kTail + 4 * h + 2)));
                    }
#pragma unroll 8
                    for (int x = 0; x < parts; ++x) {
                        const float rx = __ldcg(part(x) + kTail + 4 * h);
                        const int d = __float_as_int(__ldcg(part(x) + kTail + 4 * h + 2)) - e;
                        den += __ldcg(part(x) + kTail + 4 * h + 1) * (rx == r ? 1.0f : tc_exp2(rx - r));
                        sum += __ldcg(part(x) + h * 128 + col) * (d < -126 ? 0.0f : kv8_pow2(d) * d8_factor(rx, r));
                    }
                    if (col < p.dv) store(h, col, result(sum, den, r, e));
                }
            }
        }
        u = item0 + j1;
    }
    __syncthreads();
    if (s_gave_up) tc_gave_up(da.status);
}

template <int D, int NT>
static int d8_launch(D8Args& a, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    auto* kernel = seq_attention8_decode_kernel<D, NT>;
    static bool ready = false;
    if (!ready) {
        SLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, D8Tile<D>::kSmem));
        ready = true;
    }
    overlapping(kernel)<<<std::min(kA8Workers, 2 * sm_count()), kD8Warps * 32, D8Tile<D>::kSmem, st>>>(tmK, tmV, a);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

int launch_attention8_decode(const Attn8Args& p, bool only, void* ws, cudaStream_t st) {
    D8Args a{};
    a.a = p;
    a.only = only;
    const int group = p.heads / p.kv_heads;
    a.sets = (group + kA8MaxHeads - 1) / kA8MaxHeads;
    a.per_set = (group + a.sets - 1) / a.sets;
    a.sets = (group + a.per_set - 1) / a.per_set;
    a.counters = (int*)ws;
    a.records = (float*)(a.counters + kA8Workers);
    if (int rc = status_word(&a.status)) return rc;
    a.polls = (unsigned)g_tune_tc_polls;
    const int D = std::max(p.dk, p.dv) <= 64 ? 64 : 128;
    CUtensorMap tmK, tmV;
    const uint64_t rows = (uint64_t)p.n_pages * p.kv_heads * p.b.page_len;
    if (int rc = tc_encode_bytes(&tmK, p.k_pool, rows, p.dk, kKv8Block, D)) return rc;
    if (int rc = tc_encode_bytes(&tmV, p.v_pool, rows, p.dv, kKv8Block, D)) return rc;
    if (D == 128) return a.per_set <= 4 ? d8_launch<128, 1>(a, tmK, tmV, st) : d8_launch<128, 2>(a, tmK, tmV, st);
    return a.per_set <= 4 ? d8_launch<64, 1>(a, tmK, tmV, st) : d8_launch<64, 2>(a, tmK, tmV, st);
}

}  // namespace sllm
