// csrc/seq_attn8_decode.cu — attention of single tokens over the 8-bit paged cache, heads of up to 128 columns: one launch, whatever the contexts are.
//
// Bound: the cache's bytes. 64 requests of up to 8191 positions, 32 heads over 8 of 128: 98 us, 80 at the rate of a copy (5.3 TB/s); eight of 76 to 8000 17.4, of which 7.3; one of 8000 13.8, of
// which 2.5: the launch, the look at the contexts, an item's beginning and end and the joining of parts through global memory take 11 us here whatever the contexts are, which is this kernel's way
// and no floor (the kernel over bf16 pools, whose clusters join parts in shared memory, serves eight requests of 64 positions in 7.0). Everything else is arranged so that the bytes keep coming:
//   Work. A unit is one block of 32 keys for the query heads of a kv head (up to 8 at a time). All units of a step lie in one row, request by request and head by head, and every CTA
//   takes an equal share of it, found from the contexts on the device: requests of 77 and of 8000 positions fill the machine alike. A request's head that several CTAs share is put
//   together by the one of them that is done last (a counter), in the order of its parts.
//   Loads. A unit is two boxes of 32 rows (TMA, swizzled so that the reads below meet no bank twice) into a ring of the warp's own; a warp takes every fourth unit of its CTA's share and
//   waits for nobody else's.
//   Products on mma.sync m16n8k16 with fp16 operands: e4m3 codes are fp16 numbers, so keys and values enter exactly, two codes an instruction. Keys are the A operand (16 of them x 16
//   columns), queries the B operand: its eight columns are four heads twice, a query's value being the sum of two fp16 numbers (22 bits of the head's largest, which a power of two brings to
//   1 .. 2). Both terms' scores then lie side by side in one lane. The softmax's weights are split the same way (2^14 times as large, kA8Lift), transposed by movmatrix, and are the B operand of the second product, whose A
//   operand is the values, turned on the way from shared memory by two byte permutations for four codes. Which key is which row, and which column which k, is free as long
//   as both operands agree: the order is the one in which a lane's 16-byte reads deliver them.
//   Sums. The tensor core truncates as it accumulates: a chain of scores is four instructions long (64 columns), one of values two, before it is added to fp32 registers with ordinary rounding.
//   Scales are numbers of a unit: a key scale multiplies scores, a value scale the weights. Weights are relative to the largest of (score + exponent of the value scale), kept as a
//   whole number R, so that they are at most 2 whatever the scales are and changing R is exact; the denominator has a reference of its own.
#include "seq_attn8.cuh"
#include "tcgen05.cuh"

namespace sllm {

constexpr int kD8Warps = 4, kD8Ctas = 3;        // warps of a CTA, CTAs of an SM
// Beginning and ending an item takes a CTA as long as some eight units (queries to fragments, four warps' sums together): every item counts that many more, in front of its first one.
// Without them a CTA with 34 short items took 208 us where others took 76 (64 requests of up to 8192 positions).
constexpr int kD8Extra = 8, kD8Least = 8;       // units that an item counts more; units of a CTA's share at least

template <int D>
struct D8Tile {
    static constexpr int kRows = kKv8Block * D, kStage = 2 * kRows, kRing = D == 128 ? 2 : 4;      // bytes of a unit's keys; of keys and values; stages of a warp
    static constexpr int kSmem = 1024 + kD8Warps * kRing * kStage;
};

struct D8Args {
    Attn8Args a;
    int plan_width;              // of the other kernel's plan, which CTA 0 makes (0: it is a worker like the others)
    A8Plan* plan;
    int only;                    // the launch is the step's only one: it has no tiles of more than one query
    int sets, per_set;           // groups of query heads that a kv head's are divided into, and how many of them one holds
    int vec_q;                   // rows of queries can be read 16 bytes at a time
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

// A tile of the list as this kernel sees it: its query, and how many units a head set of it has; none when it holds more than one query (or none).
struct D8Tile1 { int t, pos, slot, units; };
__device__ __forceinline__ D8Tile1 d8_tile(const D8Args& da, int tile) {
    const Attn8Args& p = da.a;
    const int seg = p.b.qt_seg[tile], off = p.b.qt_off[tile], n = p.b.seg_len[seg] - off, pos = p.b.seg_pos0[seg] + off;
    D8Tile1 r{p.b.seg_start[seg] + off, pos, p.b.seg_slot[seg], 0};
    if (n > 1 && da.only) *reinterpret_cast<volatile int32_t*>(da.status) = kStatusSingle;
    if (n == 1 && pos >= 0) r.units = TileList(pos, pos, seq_row_window(pos, p.window, p.chunk), p.keep_first, kKv8Block).n;
    return r;
}

template <int D, int NT>       // column width of a head, rounded up; groups of four query heads
__global__ void __launch_bounds__(kD8Warps * 32, kD8Ctas) seq_attention8_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                                           const __grid_constant__ D8Args da) {
    using Tile = D8Tile<D>;
    constexpr int kRing = Tile::kRing, kChunk = D / 8, kSteps = D / 16, kMt = D / 16, kHeads = 4 * NT;   // bytes of a value row a lane reads; k-steps of a score; 16-column tiles of a result
    const Attn8Args& p = da.a;
    const sllm_seq_batch& b = p.b;
    extern __shared__ uint8_t d8_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(d8_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bars[kD8Warps][kRing];
    __shared__ long long s_sum[kD8Warps];
    constexpr int kKnown = 128;            // tiles kept at hand
    __shared__ D8Tile1 s_known[kKnown];
    __shared__ int s_tile, s_gave_up, s_last;
    __shared__ long long s_before;
    __shared__ float4 s_head[kD8Warps + 1][kHeads];      // of a warp and head, and of all: reference, sum, exponent
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    volatile int* gave_up = &s_gave_up;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kD8Warps; ++w)
            for (int i = 0; i < kRing; ++i) mb_init(&bars[w][i], 1);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    after_previous();
    static_assert(kA8PlanSmem <= Tile::kSmem - 1024, "room for the plan");
    if (da.plan_width && blockIdx.x == 0) {
        a8_plan<kD8Warps * 32>(p, da.plan_width, da.plan, smem);
        return;
    }
    const int worker = blockIdx.x - (da.plan_width != 0), workers = gridDim.x - (da.plan_width != 0);

    // ---- the row of all units, and this CTA's share of it ----
    const int per_tile = p.kv_heads * da.sets, n_tiles = b.n_qtiles;
    const int per_thread = (n_tiles + kD8Warps * 32 - 1) / (kD8Warps * 32), t0 = min(n_tiles, (int)threadIdx.x * per_thread), t1 = min(n_tiles, t0 + per_thread);
    long long mine = 0;
    auto count = [&](int units) { return units > 0 ? units + kD8Extra : 0; };
    for (int i = t0; i < t1; ++i) {
        const D8Tile1 x = d8_tile(da, i);
        if (n_tiles <= kKnown) s_known[i] = x;
        mine += count(x.units);
    }
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
    const int ctas = (int)min((long long)workers, (total + kD8Least - 1) / kD8Least);
    if (worker >= ctas) return;
    auto share = [&](int x) { return (long long)x * total / ctas; };
    auto owner = [&](long long u) { return (int)(((u + 1) * ctas - 1) / total); };
    const long long begin = share(worker), end = share(worker + 1);
    if (begin >= before && begin < before + mine * per_tile) {
        long long at = before;
        for (int i = t0; i < t1; ++i) {
            const long long n = (long long)count((n_tiles <= kKnown ? s_known[i] : d8_tile(da, i)).units) * per_tile;
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
        const D8Tile1 known = n_tiles <= kKnown ? s_known[tile] : d8_tile(da, tile);
        const int t = known.t, pos = known.pos, slot = known.slot, each = count(known.units);
        if (u >= tile0 + (long long)each * per_tile) {               // the next tile
            tile0 += (long long)each * per_tile;
            ++tile;
            continue;
        }
        const int wnd = seq_row_window(pos, p.window, p.chunk);
        const TileList blocks(pos, pos, wnd, p.keep_first, kKv8Block);
        const int set = (int)((u - tile0) / each), gkv = set / da.sets, h0 = gkv * (p.heads / p.kv_heads) + (set % da.sets) * da.per_set;
        const int G = min(da.per_set, (gkv + 1) * (p.heads / p.kv_heads) - h0);                       // query heads of this set
        const long long item0 = tile0 + (long long)set * each + kD8Extra, item1 = item0 + blocks.n;    // its units
        const int j0 = max(0, (int)(u - item0)), j1 = (int)(min(end, item1) - item0), n_mine = max(0, (j1 - j0 - warp + kD8Warps - 1) / kD8Warps);
        if (j1 <= 0) break;                // the share ends before the first of them
        if (!fresh) {                      // the last piece's sums were written where copies land: in front of them for everybody
            fence_async_smem();
            __syncthreads();
            fresh = 1;
        }
        // ---- loads: unit i of this warp; lane l knows the pool row (-1: no page) and the scales of unit 32 * x + l ----
        int rows = -1;
        float ks_l = 0.0f, vs_l = 0.0f, ks_before = 0.0f, vs_before = 0.0f;
        auto look_up = [&](int i) {
            const int at = i + lane;
            ks_before = ks_l;
            vs_before = vs_l;
            rows = -1;
            if (at < n_mine) {
                const int key0 = blocks.tile_of(j0 + warp + at * kD8Warps) * kKv8Block, page = kv8_page(b, p.n_pages, slot, key0);
                if (page >= 0) {
                    rows = (page * p.kv_heads + gkv) * b.page_len + key0 % b.page_len;
                    ks_l = p.k_scale[rows / kKv8Block];
                    vs_l = p.v_scale[rows / kKv8Block];
                } else {
                    ks_l = -1.0f;
                }
            }
        };
        auto issue = [&](int i) {
            const int row = __shfl_sync(0xffffffffu, rows, i & 31);
            if (i < n_mine && lane == 0) {
                const int stage = (int)((turns + i) % kRing);
                if (row >= 0) {
                    uint8_t* dst = smem + (warp * kRing + stage) * Tile::kStage;
                    mb_expect(&bars[warp][stage], Tile::kStage);
                    tma_load_2d(dst, &tmK, 0, row, &bars[warp][stage]);
                    tma_load_2d(dst + Tile::kRows, &tmV, 0, row, &bars[warp][stage]);
                } else {
                    mb_arrive(&bars[warp][stage]);
                }
            }
        };
        look_up(0);
        // ---- queries: asked for before the table has answered; then two fp16 terms of q * 2^-e, e from the head's largest ----
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
                const bool take = live && col < p.dk;
                if (da.vec_q) {
                    const float4 y = take ? *reinterpret_cast<const float4*>(q + col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    v[ks][0] = y.x; v[ks][1] = y.y; v[ks][2] = y.z; v[ks][3] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[ks][e] = take ? q[col + e] : 0.0f;
                }
            }
            if (x == 0) {
#pragma unroll
                for (int i = 0; i < kRing - 1; ++i) issue(i);
            }
#pragma unroll
            for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[ks][e]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int ex = top < INFINITY ? min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126) : 0;      // so that 2^-ex is a normal number, too
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
            // scores are head c's on this lane: its scale comes from a lane that holds its queries
            factor[x] = p.scale * __shfl_sync(0xffffffffu, up, 8 * c);
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
        const int va = 2 * c, vo = (2 * c + 1) ^ 4;      // and of k 2c, 2c + 1
        bool ok = true;
        for (int i = 0; i < n_mine; ++i) {
            if (((i + kRing - 1) & 31) == 0) look_up(i + kRing - 1);
            issue(i + kRing - 1);                                   // (the stage of unit i - 1, which every lane has read)
            const int stage = (int)((turns + i) % kRing);
            ok = tc_wait_warp(&bars[warp][stage], (uint32_t)((turns + i) / kRing) & 1, gave_up, da.polls);
            if (!ok) break;
            // (the batch of units that is being issued may be the one behind this unit's)
            const bool older = ((i + kRing - 1) & ~31) != (i & ~31);
            const float ks_ = __shfl_sync(0xffffffffu, older ? ks_before : ks_l, i & 31), vs_ = __shfl_sync(0xffffffffu, older ? vs_before : vs_l, i & 31);
            if (ks_ < 0.0f) continue;                               // no page: its keys are hidden
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
                    float part[NT][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t f[4] = {kv8_half2(a[e] & 0xffffu), kv8_half2(d[e] & 0xffffu), kv8_half2(a[e] >> 16), kv8_half2(d[e] >> 16)};
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            if (e == 0) mma_f16_zero(part[x], f, qb[x][4 * half][0], qb[x][4 * half][1]);
                            else mma_f16(part[x], f, qb[x][4 * half + e][0], qb[x][4 * half + e][1]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int y = 0; y < 4; ++y) s[x][y] += part[x][y];
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
                const float lift = mant * kv8_pow2(max(-126, min(126, d + kA8Lift)));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float q = tc_exp2(w[x][e] - base);
                    l[x] += q;
                    const float y = q * lift, hi = f16_round(y);
                    pb[x][e] = movmatrix_trans(pack_f16(hi, y - hi));
                }
            }
            // ---- values: two runs of 16 keys, one chain ----
            uint32_t v[8][kChunk / 4];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = 8 * (e >> 1) + (e & 1 ? vo : va);
                if constexpr (D == 128) {
                    const uint4 y = lds16(vb + d8_at<D>(key, g));
                    v[e][0] = y.x; v[e][1] = y.y; v[e][2] = y.z; v[e][3] = y.w;
                } else {
                    const uint2 y = lds8(vb + d8_at<D>(key, g >> 1) + 8 * (g & 1));
                    v[e][0] = y.x; v[e][1] = y.y;
                }
                if (masked && !seq_sees(pos, key0 + key, wnd, p.keep_first)) {                       // a hidden row may hold anything
#pragma unroll
                    for (int k = 0; k < kChunk / 4; ++k) v[e][k] = 0u;
                }
            }
#pragma unroll
            for (int k = 0; k < kChunk / 4; ++k) {
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    const uint32_t sel = odd ? 0x7362u : 0x5140u;
                    uint32_t y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = __byte_perm(v[2 * e][k], v[2 * e + 1][k], sel);
                    const uint32_t a0[4] = {kv8_half2(y[0] & 0xffffu), kv8_half2(y[0] >> 16), kv8_half2(y[1] & 0xffffu), kv8_half2(y[1] >> 16)};
                    const uint32_t a1[4] = {kv8_half2(y[2] & 0xffffu), kv8_half2(y[2] >> 16), kv8_half2(y[3] & 0xffffu), kv8_half2(y[3] >> 16)};
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        float part[4];
                        mma_f16_zero(part, a0, pb[x][0], pb[x][1]);
                        mma_f16(part, a1, pb[x][2], pb[x][3]);
                        o[x][2 * k + odd][0] += part[0] + part[1];
                        o[x][2 * k + odd][1] += part[2] + part[3];
                    }
                }
            }
            __syncwarp();
        }
        turns += n_mine;
        // ---- the four warps' sums together ----
        __syncthreads();                   // every stage has been read
        if (s_gave_up) break;
        float* sums = reinterpret_cast<float*>(smem);                       // [warp][head][D]
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], s);
            const int h = 4 * x + c;
            if (g == 0) s_head[warp][h] = make_float4(ref[x], l[x], __int_as_float(R[x]), 0.0f);
            float* dst = sums + (warp * kHeads + h) * D + kChunk * g;
#pragma unroll
            for (int i = 0; i < kMt; i += 2) *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[x][i][0], o[x][i][1], o[x][i + 1][0], o[x][i + 1][1]);
        }
        fresh = 0;
        __syncthreads();
        const int first_cta = owner(item0), last_cta = owner(item1 - 1), parts = last_cta - first_cta + 1;
        float* record = da.records + (size_t)(2 * worker + (begin >= item0 ? 0 : 1)) * kA8Record;
        constexpr int kTail = kA8MaxHeads * 128;                               // where a record's references, sums and exponents begin
        // Sums of parts with references and exponents of their own, brought to the largest of each. A column's result: sum * 2^e / (den * 2^r); a query that sees no key gives 0.
        auto store = [&](int h, int col, float4 sum, float r, float den, int e) {
            const float f = den == 0.0f ? 0.0f : kv8_pow2(max(-126, min(126, e - d8_whole(r) - kA8Lift))) / den;
            const float y[4] = {sum.x * f, sum.y * f, sum.z * f, sum.w * f};
            if (col >= p.dv) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (p.out) p.out[(size_t)t * p.ldo + (size_t)(h0 + h) * p.dv + col + i] = y[i];
                if (p.out16) p.out16[((size_t)t * p.heads + h0 + h) * p.dv + col + i] = f32_to_bf16_bits(y[i]);
            }
        };
        auto weight = [&](float4 part, float r, int e) {
            const int d = __float_as_int(part.z) - e;
            return d < -126 ? 0.0f : kv8_pow2(d) * d8_factor(part.x, r);
        };
        auto add = [](float4& sum, float4 v, float f) {
            sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y); sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
        };
        for (int i = threadIdx.x; i < G * (D / 4); i += kD8Warps * 32) {
            const int h = i / (D / 4), col = i % (D / 4) * 4;
            float r = -INFINITY, den = 0.0f;
            int e = kD8None;
#pragma unroll
            for (int w = 0; w < kD8Warps; ++w) {
                r = fmaxf(r, s_head[w][h].x);
                e = max(e, __float_as_int(s_head[w][h].z));
            }
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kD8Warps; ++w) {
                const float4 part = s_head[w][h];
                den += part.y * (part.x == r ? 1.0f : tc_exp2(part.x - r));
                add(sum, *reinterpret_cast<const float4*>(sums + (w * kHeads + h) * D + col), weight(part, r, e));
            }
            if (parts == 1) {
                store(h, col, sum, r, den, e);
            } else {
                *reinterpret_cast<float4*>(record + h * 128 + col) = sum;
                if (col == 0) *reinterpret_cast<float4*>(record + kTail + 4 * h) = make_float4(r, den, __int_as_float(e), 0.0f);
            }
        }
        if (parts > 1) {
            __syncthreads();
            if (threadIdx.x == 0) {        // what the CTA has stored before the barrier comes before this, and what others have stored before theirs, before what follows
                int before_me;
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before_me) : "l"(da.counters + first_cta) : "memory");
                s_last = before_me == parts - 1;
                if (s_last) da.counters[first_cta] = 0;
            }
            __syncthreads();
            if (s_last) {                  // all parts are there: in the order of the units, whoever was last
                const int later = share(first_cta) < item0;
                const float* rest = da.records + (size_t)2 * first_cta * kA8Record;
                __threadfence();
                auto part = [&](int x) { return reinterpret_cast<const float4*>(rest + (size_t)(2 * x + (x == 0 ? later : 0)) * kA8Record); };
                float* weights = sums;     // [head][part]: at most 8 x 512 of them, the ring holds more
                for (int h = warp; h < G; h += kD8Warps) {
                    float r = -INFINITY, den = 0.0f;
                    int e = kD8None;
                    for (int x = lane; x < parts; x += 32) {
                        const float4 v = __ldcg(part(x) + kTail / 4 + h);
                        r = fmaxf(r, v.x);
                        e = max(e, __float_as_int(v.z));
                    }
                    r = warp_max(r);
                    e = __reduce_max_sync(0xffffffffu, e);
                    for (int x = lane; x < parts; x += 32) {
                        const float4 v = __ldcg(part(x) + kTail / 4 + h);
                        den += v.y * (v.x == r ? 1.0f : tc_exp2(v.x - r));
                        weights[h * kA8Workers + x] = weight(v, r, e);
                    }
                    den = warp_sum(den);
                    if (lane == 0) s_head[kD8Warps][h] = make_float4(r, den, __int_as_float(e), 0.0f);
                }
                __syncthreads();
                for (int i = threadIdx.x; i < G * (D / 4); i += kD8Warps * 32) {
                    const int h = i / (D / 4), col = i % (D / 4) * 4;
                    const float4 head = s_head[kD8Warps][h];
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    int x = 0;
                    for (; x + 8 <= parts; x += 8) {
                        float4 v[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) v[y] = __ldcg(part(x + y) + (h * 128 + col) / 4);
#pragma unroll
                        for (int y = 0; y < 8; ++y) add(sum, v[y], weights[h * kA8Workers + x + y]);
                    }
                    for (; x < parts; ++x) add(sum, __ldcg(part(x) + (h * 128 + col) / 4), weights[h * kA8Workers + x]);
                    store(h, col, sum, head.x, head.y, __float_as_int(head.z));
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
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, D8Tile<D>::kSmem));
            return SLLM_OK;
        }))
        return rc;
    overlapping(kernel)<<<std::min(kA8Workers, kD8Ctas * sm_count()), kD8Warps * 32, D8Tile<D>::kSmem, st>>>(tmK, tmV, a);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

int launch_attention8_decode(const Attn8Args& p, bool only, int plan_width, void* ws, cudaStream_t st) {
    D8Args a{};
    a.a = p;
    a.only = only;
    a.plan_width = plan_width;
    a.plan = reinterpret_cast<A8Plan*>((uint8_t*)ws + kA8PlanAt);
    const int group = p.heads / p.kv_heads;
    a.sets = (group + kA8MaxHeads - 1) / kA8MaxHeads;
    a.per_set = (group + a.sets - 1) / a.sets;
    a.sets = (group + a.per_set - 1) / a.per_set;
    a.vec_q = p.ldq % 4 == 0 && ((uintptr_t)p.q % 16) == 0;
    a.counters = (int*)ws;
    a.records = (float*)((uint8_t*)ws + kA8RecordsAt);
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
