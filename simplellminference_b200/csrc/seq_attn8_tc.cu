// csrc/seq_attn8_tc.cu — attention of prompt portions over the 8-bit paged cache on the 5th-generation tensor cores, heads of up to 128 columns.
//
// 128 rows = the query heads of a kv head (four, two or one) x 32, 64 or 128 neighbouring queries are a tile; a CTA has two tiles at a time, neighbours in the sequence (a run), that share
// tiles of 64 keys and values. fp16 operands, since fp16 holds every e4m3 code: keys and values enter exactly, and block scales multiply scores and weights.
//   warp 0 (one lane)   TMA producer: boxes of 32 rows of codes, looked up in the block table, into a ring;
//   warps 2, 3          codes to fp16 rows in the 128B swizzle (keys K-major, values as they lie); value rows that the run must not see, and NaN codes among values, become zeros;
//   warp 1 (one lane)   MMA issuer: S = Q K^T, O += P V with P read from TMEM; P has columns of its own, so that the next scores are made while the softmax takes its exponentials;
//   warps 4-7, 8-11     softmax of tile 0 / 1: queries to fp16 once an item; then, a thread per row, maximum, weights and their sum of every key tile;
//   warps 12-15         O of both tiles: rescaled where a maximum has grown, results or parts of them written.
// Queries and weights are the sum of two fp16 numbers each (22 bits), and O is added to an fp32 copy of the CTA's own every kT8Flush tiles, because the tensor core truncates as it accumulates.
// Results in bf16 are those in fp32, rounded: with one fp16 number for a query and a weight 15 % of them were another bf16 number (now 0.06 %, as far as fp32 sums let them), and they
// depended on whether fp32 results were asked for as well; the prompts below took 170 us then.
// Weights are relative to the largest of score + log2(value scale) so far, rounded up to a whole number: differences of exponents are exact then, and O is rescaled by powers of two, and
// seldom; as operands, and in O, they are 2^14 times as large (kA8Lift). The denominator takes the value scale out again, block by block.
// A value's NaN code must reach exactly the rows that see it, but 0 * NaN is NaN: the converters replace it and say so, and rows of such an item look for NaN among their keys' values
// at the end.
// Shares. A CTA per item would leave most SMs idle where few queries follow a long context. The key tiles of all items lie in one row, made by a CTA of the kernel in front from what the
// device knows (contexts, listed tiles); every CTA takes an equal run of it. Items that a cut goes through leave O, reference and sum as parts, which a kernel behind puts together (done by
// the last of an item's CTAs, one SM reading what up to ten had left, that took as long as all the rest).
// Bound: the chain of a step (64 keys for 256 rows): 2.6 us, 3.8 with capped scores (18 portions of 64 queries behind 4000 and 8100 positions), of which the tensor pipe needs 2048 clocks and the
// exponentials 1024; an item's beginning and end, 10 us (1184 items of one step); some 20 us of launches, plan and first queries. Prompts of 2048, 1300 behind 700, 311 and 37 behind 4000 tokens,
// 32 heads over 8 of 128, bf16 results: 276 us, 41 at the rate of a large product and 81 with the two terms. A portion of 256 behind 6000 and 12 decoding requests, capped, fp32: 148 us, 32 with two
// terms.
#include <type_traits>

#include "seq_attn8.cuh"
#include "tcgen05.cuh"

namespace sllm {

constexpr int kT8Rows = 128, kT8Keys = kA8Keys, kT8Threads = 512; // rows of a tile, keys of a tile
// Key tiles that an item's beginning and end count for (4, 6 and 8: 280, 278 and 280 us for prompts, 151, 152 and 152 for a portion); key tiles of a CTA's share at least; key tiles after which O
// leaves tensor memory, which truncates as it adds, all one way. Prompts, fp32 results, 16, 8, 4 and 2 tiles: 262, 271, 282 and 299 us, off by 1.4e-6, 1.0e-6, 0.7e-6 and 0.5e-6 of the norm; the portion
// 141, 143, 147 and 148 us, off by 1.4e-6, 0.9e-6, 0.6e-6 and 0.5e-6, where fp32 arithmetic throughout is off by 1.1e-6.
constexpr int kT8Extra = kA8Extra, kT8Least = 4, kT8Flush = 4;
constexpr int kT8Known = 16;                    // key tiles whose scales are kept at hand: more than the producer is ever ahead of the softmax (the rings' stages and two)
constexpr uint32_t kT8Tmem = 512, kT8S = 0, kT8P = 128, kT8O = 256;           // columns: S0 S1 | P0 P1 | O0 O1

struct T8Args {
    Attn8Args a;
    int hpc, hpc_log2, queries;          // query heads and queries of a tile: hpc * queries = 128
    int sets;                            // head sets of a step: kv_heads * (group / hpc)
    int vec_q;
    const A8Plan* plan;
    struct T8Item* cuts;                 // of every CTA: the item it has the first part of and others the rest (parts 0: none)
    float* parts;
    int32_t* status;
    unsigned polls;
};

// An item of a CTA's share, as all its roles see it.
struct T8Item {
    int k0, k1, n;                           // its key tiles that are this CTA's, of so many
    int tok0, pos0, slot, gkv, h0;           // first token and position of the run; kv head, first query head
    int lo, hi;                              // first and last listed query of the run
    int keys[2];                             // how many of k0 .. k1 either tile has to see: those up to its last listed query's
    int first_cta, parts, slot_of, later;    // the CTAs that share it; which of this CTA's two places its part takes, and the first CTA's
    uint32_t m[8];                           // listed queries
    __device__ __forceinline__ bool listed(int q) const { return m[q >> 5] >> (q & 31) & 1; }
};
static_assert(sizeof(T8Item) <= kA8Cut, "the workspace's cuts");
constexpr int kT8Items = 48;                 // of a share, kept in shared memory; the ones behind are worked out where they are needed

// A CTA's share of the row of all key tiles: items first_item, first_item + 1, ... of the step (run by run, head set by head set)
struct T8Share {
    const T8Args& p;
    long long total, begin, end;
    int ctas, first_item, count;
    const int* before;                   // of the plan, or a copy of it
    __device__ __forceinline__ long long share(int c) const { return (long long)c * total / ctas; }
    __device__ __forceinline__ int owner(long long v) const { return (int)(((v + 1) * ctas - 1) / total); }
    __device__ __forceinline__ T8Share(const T8Args& args, int n_ctas, long long all, const int* plan_before) : p(args), total(all), ctas(n_ctas), before(plan_before) {
        begin = share(blockIdx.x);
        end = share(blockIdx.x + 1);
    }
    __device__ __forceinline__ int item_of(long long u, int runs) const {          // the item that unit u (beginnings counted) belongs to
        int lo = 0, hi = runs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((long long)before[mid] * p.sets <= u) lo = mid; else hi = mid;
        }
        const int b0 = before[lo], each = before[lo + 1] - b0;
        return lo * p.sets + (int)((u - (long long)b0 * p.sets) / each);
    }
    __device__ __noinline__ void work_out(int i, T8Item& it) const {     // k1 <= 0: the share ends before its first tile
        const int x = (first_item + i) / p.sets, y = (first_item + i) % p.sets;
        const int b0 = before[x], each = before[x + 1] - b0;
        const long long item0 = (long long)b0 * p.sets + (long long)y * each + kT8Extra;
        it.n = each - kT8Extra;
        it.k0 = (int)max(0ll, begin - item0);
        it.k1 = (int)(min(end, item0 + it.n) - item0);
        const sllm_seq_batch& b = p.a.b;
        const int seg = p.plan->seg[x], first = p.plan->first[x], group = p.a.heads / p.a.kv_heads, per = group / p.hpc;
        it.tok0 = b.seg_start[seg] + first;
        it.pos0 = b.seg_pos0[seg] + first;
        it.slot = b.seg_slot[seg];
        it.gkv = y / per;
        it.h0 = it.gkv * group + y % per * p.hpc;
        it.lo = it.hi = -1;
        int last[2] = {-1, -1};
        for (int w = 0; w < 8; ++w) {
            it.m[w] = p.plan->mask[x][w];
            if (!it.m[w]) continue;
            if (it.lo < 0) it.lo = 32 * w + __ffs(it.m[w]) - 1;
            it.hi = 32 * w + 31 - __clz(it.m[w]);
            last[32 * w >= p.queries] = it.hi;
        }
        for (int j = 0; j < 2; ++j) {
            const int n = last[j] < 0 ? 0 : it.n - ((it.pos0 + it.hi) / kT8Keys - (it.pos0 + last[j]) / kT8Keys);
            it.keys[j] = max(0, min(it.k1, n) - it.k0);
        }
        it.first_cta = owner(item0);
        it.parts = owner(item0 + it.n - 1) - it.first_cta + 1;
        it.slot_of = begin >= item0 ? 0 : 1;
        it.later = share(it.first_cta) < item0;
    }
};

constexpr float kT8Down = 1.0f / (1 << kA8Lift);          // of weights, and of O
constexpr int kT8Terms = 2;                      // fp16 numbers that a query, or a weight, is the sum of
template <int HD>
struct T8Shape {
    static constexpr int kBlocks = HD / 64, kK = 2, kV = 1, kRaw = 2;         // stages of keys, of values, of codes
    static constexpr int kBlock = kT8Keys * 128, kTile = kBlocks * kBlock;    // fp16: 64 columns of all keys; all columns
    static constexpr int kCodes = kT8Keys * HD;                              // bytes of a tile of codes
    static constexpr int kQBlock = kT8Rows * 128, kQTerm = kBlocks * kQBlock, kQTile = kT8Terms * kQTerm;
    static constexpr int kItems = (kT8Items * (int)sizeof(T8Item) + 127) / 128 * 128;
    static constexpr int kSmem = 1024 + (kK + kV) * kTile + 2 * kRaw * kCodes + 2 * kQTile + 512 + 8 * kT8Rows * (int)sizeof(float) + kItems;
};
constexpr int kT8PartTile = kT8Rows * (128 + 2), kT8Part = 2 * kT8PartTile;   // floats of a part: per tile O as [HD / 4][128][4], references, sums
static_assert(kT8Part == kA8Part, "the workspace's parts");

// what the producer knows of a key tile: per 32 keys the key scale, log2 of the value scale, the pool row (-1: no page)
struct T8Tile { float ks[2], ev[2]; int row[2], pad[2]; };

// pool row of 32 keys, or -1 where they have no page (or lie behind the last listed query)
__device__ __forceinline__ int t8_row(const Attn8Args& p, int slot, int gkv, int key0, int last_pos) {
    if (key0 > last_pos) return -1;
    const int page = kv8_page(p.b, p.n_pages, slot, key0);
    return page < 0 ? -1 : (page * p.kv_heads + gkv) * p.b.page_len + key0 % p.b.page_len;
}
__device__ __forceinline__ uint32_t t8_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 t8_unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// of a scale; exact for powers of two, as the append leaves them
__device__ __forceinline__ float t8_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__uint_as_float((__float_as_uint(x) & 0x7fffffu) | 0x3f800000u)));
    return y + (float)((int)(__float_as_uint(x) >> 23 & 0xff) - 127);
}
__device__ __forceinline__ uint4 t8_lds(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void t8_sts(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The roles' code together has to stay near what the instruction caches hold (with everything in line it was 172 KB, and an item's beginning took 14000 clocks): what is seldom run is a function.
__device__ __noinline__ bool t8_wait_long(uint64_t* bar, uint32_t parity, volatile int* gave_up, unsigned polls) { return tc_wait(bar, parity, gave_up, polls); }
__device__ __forceinline__ bool t8_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, unsigned polls) {
    uint32_t done = 0;
    if (polls)
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(s_addr(bar)), "r"(parity) : "memory");
    return done || t8_wait_long(bar, parity, gave_up, polls);
}
__device__ __forceinline__ bool t8_wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up, unsigned polls) {
    return __all_sync(0xffffffffu, t8_wait(bar, parity, gave_up, polls));
}
// fp16 operands: the bf16 descriptor without its types
__host__ __device__ constexpr uint32_t t8_idesc(int M, int N) { return umma_idesc_bf16(M, N) & ~((1u << 7) | (1u << 10)); }

// Where the result of a row of tile j goes, or whether it has none
struct T8Out { float* out; uint16_t* out16; bool listed, wide; };
__device__ __forceinline__ T8Out t8_out(const T8Args& p, const T8Item& it, int j, int row) {
    const Attn8Args& a = p.a;
    const int q = j * p.queries + (row >> p.hpc_log2), h = it.h0 + (row & (p.hpc - 1));
    const size_t t = it.tok0 + q;
    T8Out r{a.out ? a.out + t * a.ldo + (size_t)h * a.dv : nullptr, a.out16 ? a.out16 + (t * a.heads + h) * a.dv : nullptr, it.listed(q), false};
    r.wide = ((reinterpret_cast<uintptr_t>(r.out) | reinterpret_cast<uintptr_t>(r.out16)) & 15) == 0;
    return r;
}
__device__ __noinline__ void t8_store_narrow(float* out, uint16_t* out16, float4 x, float4 y) {
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (out) out[e] = v[e];
        if (out16) out16[e] = f32_to_bf16_bits(v[e]);
    }
}
// eight columns
__device__ __forceinline__ void t8_store(const T8Out& to, int c, float4 x, float4 y) {
    if (!to.wide) {
        t8_store_narrow(to.out ? to.out + c : nullptr, to.out16 ? to.out16 + c : nullptr, x, y);
        return;
    }
    if (to.out) {
        *reinterpret_cast<float4*>(to.out + c) = x;
        *reinterpret_cast<float4*>(to.out + c + 4) = y;
    }
    if (to.out16) *reinterpret_cast<uint4*>(to.out16 + c) = make_uint4(tc_pack(x.x, x.y), tc_pack(x.z, x.w), tc_pack(y.x, y.y), tc_pack(y.z, y.w));
}
// Rare: a row whose keys' values may hold NaN codes has its result; it becomes NaN in the columns c0 .. c1 - 1 where one of the values that it sees is.
__device__ __noinline__ void t8_poison(const T8Args& p, const T8Item& it, int j, int row, int c0, int c1) {
    const Attn8Args& a = p.a;
    const T8Out to = t8_out(p, it, j, row);
    if (!to.listed) return;
    const int pos = it.pos0 + j * p.queries + (row >> p.hpc_log2), wnd = seq_row_window(pos, a.window, a.chunk);
    const TileList mine(pos, pos, wnd, a.keep_first, kKv8Block);
    for (int x = 0; x < mine.n; ++x) {
        const int key0 = mine.tile_of(x) * kKv8Block, r = t8_row(a, it.slot, it.gkv, key0, pos);
        if (r < 0) continue;
        for (int e = 0; e < kKv8Block; ++e) {
            if (!seq_sees(pos, key0 + e, wnd, a.keep_first)) continue;
            const uint8_t* v = a.v_pool + (size_t)(r + e) * a.dv;
            for (int c = c0; c < c1; ++c) {
                if ((v[c] & 0x7f) != 0x7f) continue;
                if (to.out) to.out[c] = __int_as_float(0x7fffffff);
                if (to.out16) to.out16[c] = 0x7fff;
            }
        }
    }
}
// The parts of the items that were cut, brought to one reference and added, in the order of the key tiles. CTA (x, y): the item that CTA x of the kernel in front had the first part of,
// if there is one; a thread per row of one tile, 16 columns.
constexpr int kT8JoinCols = 16, kT8JoinCtas = 2 * 128 / kT8JoinCols;
__global__ void __launch_bounds__(kT8Rows) seq_attention8_join_kernel(const __grid_constant__ T8Args p) {
    after_previous();
    const int row = threadIdx.x, j = blockIdx.y / (kT8JoinCtas / 2), c0 = blockIdx.y % (kT8JoinCtas / 2) * kT8JoinCols;
    const T8Item& it = p.cuts[blockIdx.x];
    const int parts = it.parts;
    if (parts < 2 || c0 >= p.a.dv) return;
    const T8Out to = t8_out(p, it, j, row);
    if (!to.listed) return;
    const float* first = p.parts + (size_t)(2 * it.first_cta + it.later) * kT8Part + j * kT8PartTile;
    const float* rest = p.parts + (size_t)(2 * it.first_cta) * kT8Part + j * kT8PartTile;
    auto from = [&](int x) { return x == 0 ? first : rest + (size_t)(2 * x) * kT8Part; };
    float top = -INFINITY, l = 0.0f;
#pragma unroll 8
    for (int x = 0; x < parts; ++x) top = fmaxf(top, from(x)[128 * kT8Rows + row]);
    bool wild = false;
    float4 y[kT8JoinCols / 4] = {};
    constexpr int kAhead = 4;                              // parts asked for at once, without a branch between them
    for (int x0 = 0; x0 < parts; x0 += kAhead) {
        float r[kAhead], sum[kAhead];
        float4 v[kAhead][kT8JoinCols / 4];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const float* part = from(min(x0 + x, parts - 1));
            r[x] = part[128 * kT8Rows + row];
            sum[x] = part[129 * kT8Rows + row];
#pragma unroll
            for (int i = 0; i < kT8JoinCols / 4; ++i) v[x][i] = reinterpret_cast<const float4*>(part)[(c0 / 4 + i) * kT8Rows + row];
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            // where none of a part's keys is visible its O may never have been written
            if (x0 + x >= parts) continue;
            wild |= __float_as_uint(sum[x]) >> 31;
            if (r[x] == -INFINITY && sum[x] == 0.0f) continue;
            const float f = r[x] == top ? 1.0f : tc_exp2(r[x] - top);
            l += fabsf(sum[x]) * f;
#pragma unroll
            for (int i = 0; i < kT8JoinCols / 4; ++i) {
                y[i].x = fmaf(v[x][i].x, f, y[i].x); y[i].y = fmaf(v[x][i].y, f, y[i].y); y[i].z = fmaf(v[x][i].z, f, y[i].z); y[i].w = fmaf(v[x][i].w, f, y[i].w);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kT8JoinCols / 4; i += 2) {
        if (c0 + 4 * i >= p.a.dv) break;
        const float4 u = y[i], v = y[i + 1];
        t8_store(to, c0 + 4 * i, make_float4(u.x * inv, u.y * inv, u.z * inv, u.w * inv), make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
    if (wild) t8_poison(p, it, j, row, c0, min(p.a.dv, c0 + kT8JoinCols));
}

template <int HD, bool kOpts>
__global__ void __launch_bounds__(kT8Threads, 1) seq_attention8_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ T8Args p) {
    using Sh = T8Shape<HD>;
    constexpr int SK = Sh::kK, SV = Sh::kV, RS = Sh::kRaw;
    extern __shared__ uint8_t t8_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(t8_smem) + 1023) & ~(uintptr_t)1023);
    uint8_t *sK = smem, *sV = sK + SK * Sh::kTile, *sQ = sV + SV * Sh::kTile, *sRaw = sQ + 2 * Sh::kQTile;      // sRaw: keys, then values, of each stage
    uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + 2 * RS * Sh::kCodes);
    uint64_t *rfull = bars, *rempty = rfull + RS, *kfull = rempty + RS, *kempty = kfull + SK, *vfull = kempty + SK, *vempty = vfull + SV;
    // per tile: queries written / scores written / scores read / factors for O written / weights written and O rescaled / product with the values done / sums written, and read
    uint64_t *qready = vempty + SV, *sfull = qready + 2, *sread = sfull + 2, *factors = sread + 2, *pready = factors + 2, *odone = pready + 2, *lready = odone + 2, *lread = lready + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(lread + 2);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_start = reinterpret_cast<int*>(tmem_slot + 2);                        // the first item and how many
    int* s_last = reinterpret_cast<int*>(tmem_slot + 4);
    volatile int* s_nan = reinterpret_cast<volatile int*>(tmem_slot + 5);        // [8]: at i % 8 the number (from 1) of an item that had NaN among its values; the converters are fewer items ahead
    float* factor = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);        // [2][128]
    float *s_ref = factor + 2 * kT8Rows, *s_sum = s_ref + 2 * kT8Rows;                        // [2][128] each
    T8Tile* s_tile = reinterpret_cast<T8Tile*>(s_sum + 2 * kT8Rows);                           // [kT8Known]
    T8Item* s_items = reinterpret_cast<T8Item*>(factor + 8 * kT8Rows);                         // [kT8Items]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Attn8Args& a = p.a;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < RS; ++i) { mb_init(rfull + i, 1); mb_init(rempty + i, 2); }
        for (int i = 0; i < SK; ++i) { mb_init(kfull + i, 2); mb_init(kempty + i, 1); }
        for (int i = 0; i < SV; ++i) { mb_init(vfull + i, 2); mb_init(vempty + i, 1); }
        for (int j = 0; j < 2; ++j) {
            mb_init(qready + j, 128); mb_init(sfull + j, 1); mb_init(sread + j, 128); mb_init(factors + j, 128); mb_init(pready + j, 256); mb_init(odone + j, 1); mb_init(lready + j, 128); mb_init(lread + j, 128);
        }
        *gave_up = 0;
        for (int i = 0; i < 8; ++i) s_nan[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tc_alloc(tmem_slot, kT8Tmem);
    after_previous();
    // this CTA's share of the row of all key tiles, and its items
    const int runs = p.plan->runs;
    int* s_before = reinterpret_cast<int*>(smem);                              // where operands come later
    static_assert((kA8Runs + 1) * 4 <= (SK + SV) * Sh::kTile + 2 * RS * Sh::kCodes, "room for the plan");
    for (int i = threadIdx.x; i <= runs; i += kT8Threads) s_before[i] = p.plan->before[i];
    __syncthreads();
    const long long total = (long long)s_before[runs] * p.sets;
    const int ctas = (int)min((long long)gridDim.x, (total + kT8Least - 1) / kT8Least);
    const bool work = (int)blockIdx.x < ctas;
    T8Share w(p, ctas, total, s_before);
    if (work && warp >= 2 && warp < 4) {
        w.first_item = w.item_of(w.begin, runs);
        const int n = w.item_of(w.end - 1, runs) - w.first_item + 1, i = threadIdx.x - 64;
        if (i < min(n, kT8Items)) w.work_out(i, s_items[i]);
        if (i == 0) { s_start[0] = w.first_item; s_start[1] = n; }
        if (i == 63) {                           // the last one may go on in the next CTA
            T8Item last;
            w.work_out(n - 1, last);
            if (last.first_cta != (int)blockIdx.x || last.parts == 1) last.parts = 0;
            p.cuts[blockIdx.x] = last;
        }
    } else if (!work && threadIdx.x == 127) {
        p.cuts[blockIdx.x].parts = 0;
    }
    fence_async_smem();                                                        // (s_before has been read before the first copy writes there)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    w.first_item = s_start[0];
    w.count = s_start[1];
    w.before = p.plan->before;
    // the i-th item, or false behind the last one (whose first tile the share may end before)
    auto item_at = [&](int i, T8Item& more) -> const T8Item* {
        if (i >= w.count) return nullptr;
        const T8Item* it = s_items + i;
        if (i >= kT8Items) {
            w.work_out(i, more);
            it = &more;
        }
        return it->k1 > 0 ? it : nullptr;
    };
    auto tiles_of = [&](const T8Item& it) { return TileList(it.pos0 + it.lo, it.pos0 + it.hi, seq_row_window(it.pos0 + it.lo, a.window, a.chunk), a.keep_first, kT8Keys); };

    if (!work) {
    } else if (warp == 0) {   // ===== TMA producer: lane l knows key tile 32 * x + l of the item =====
        T8Item more;
        int g = 0;                               // key tiles so far
        bool ok = true;
        for (int n_item = 0; ok; ++n_item) {
            const T8Item* at = item_at(n_item, more);
            if (!at) break;
            const T8Item& it = *at;
            const TileList tiles = tiles_of(it);
            T8Tile mine{};
            for (int k = it.k0, k1 = it.k1; k < k1; ++k, ++g) {
                if (((k - it.k0) & 31) == 0 && k + lane < it.k1) {
                    const int key0 = tiles.tile_of(k + lane) * kT8Keys;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int row = t8_row(a, it.slot, it.gkv, key0 + x * kKv8Block, it.pos0 + it.hi);
                        mine.row[x] = row;
                        mine.ks[x] = row >= 0 ? a.k_scale[row / kKv8Block] : 1.0f;
                        mine.ev[x] = row >= 0 ? t8_log2(a.v_scale[row / kKv8Block]) : 0.0f;
                    }
                }
                const int s = g % RS, from = (k - it.k0) & 31;
                const int row[2] = {__shfl_sync(0xffffffffu, mine.row[0], from), __shfl_sync(0xffffffffu, mine.row[1], from)};
                ok = t8_wait_warp(rempty + s, ((uint32_t)(g / RS) & 1) ^ 1, gave_up, p.polls);
                if (!ok) break;
                if (lane == from) s_tile[g % kT8Known] = mine;
                __syncwarp();
                if (lane == 0) {
                    const int boxes = (row[0] >= 0) + (row[1] >= 0);
                    if (boxes) mb_expect(rfull + s, (uint32_t)(boxes * 2 * kKv8Block * HD));
                    else mb_arrive(rfull + s);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (row[x] < 0) continue;
                        tma_load_2d(sRaw + 2 * s * Sh::kCodes + x * kKv8Block * HD, &tmK, 0, row[x], rfull + s);
                        tma_load_2d(sRaw + (2 * s + 1) * Sh::kCodes + x * kKv8Block * HD, &tmV, 0, row[x], rfull + s);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {   // ===== MMA issuer =====
            constexpr uint32_t idesc_s = t8_idesc(kT8Rows, kT8Keys), idesc_o = t8_idesc(kT8Rows, HD) | (1u << 16);      // B MN-major
            const uint64_t q_desc = umma_desc_sw128(sQ), k_desc = umma_desc_sw128(sK), v_desc = umma_desc_mn_sw128(sV, Sh::kBlock);     // + bytes / 16: another place
            uint32_t made[2] = {0, 0}, done[2] = {0, 0}, items[2] = {0, 0};     // scores, products and items of either tile
            auto scores = [&](int j, int g) {    // behind the softmax's reading of the ones before
                if (made[j] && !t8_wait(sread + j, (made[j] - 1) & 1, gave_up, p.polls)) return false;
                ++made[j];
                tc_fence_after();
                const uint64_t k = k_desc + (uint32_t)(g % SK) * (Sh::kTile / 16);
#pragma unroll
                for (int term = kT8Terms - 1; term >= 0; --term) {         // the small products first: the tensor core truncates by the size of what it adds to
                    const uint64_t q = q_desc + (uint32_t)j * (Sh::kQTile / 16) + (uint32_t)term * (Sh::kQTerm / 16);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        tc_mma_bf16(tmem + kT8S + 64 * j, q + (uint32_t)((ks / 4) * (Sh::kQBlock / 16) + 2 * (ks % 4)), k + (uint32_t)((ks / 4) * (Sh::kBlock / 16) + 2 * (ks % 4)), idesc_s,
                                    term != kT8Terms - 1 || ks != 0);
                }
                tc_commit(sfull + j);
                return true;
            };
            auto values = [&](int j, int g, bool more) {
                const uint64_t v = v_desc + (uint32_t)(g % SV) * (Sh::kTile / 16);
#pragma unroll
                for (int ks = 0; ks < kT8Terms * kT8Keys / 16; ++ks)       // first terms, then second ones, against the same values
                    tc_mma_bf16_ts(tmem + kT8O + 128 * j, tmem + kT8P + 64 * j + 8 * ks, v + (uint32_t)((ks % (kT8Keys / 16)) * 128), idesc_o, more || ks != 0);
                tc_commit(odone + j);
            };
            T8Item more;
            int g = 0;                           // key tiles so far
            bool ok = true;
            for (int n_item = 0; ok; ++n_item) {
                const T8Item* at = item_at(n_item, more);
                if (!at) break;
                const int n = at->k1 - at->k0, nkt[2] = {at->keys[0], at->keys[1]};
                ok = t8_wait(kfull + g % SK, (uint32_t)(g / SK) & 1, gave_up, p.polls);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (ok && nkt[j]) ok = t8_wait(qready + j, items[j]++ & 1, gave_up, p.polls) && scores(j, g);
                if (!ok) break;
                tc_commit(kempty + g % SK);
                for (int kt = 0; ok && kt < n; ++kt, ++g) {
                    if (kt + 1 < n) ok = t8_wait(kfull + (g + 1) % SK, (uint32_t)((g + 1) / SK) & 1, gave_up, p.polls);
                    // Either tile's next scores, then its product with these values: so the tiles come to lie half a step apart, and one's exponentials run during the other's products.
                    bool values_there = false;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (ok && kt + 1 < nkt[j]) ok = scores(j, g + 1);
                        if (!ok || kt >= nkt[j]) continue;
                        if (!values_there) ok = t8_wait(vfull + g % SV, (uint32_t)(g / SV) & 1, gave_up, p.polls);
                        values_there = true;
                        ok = ok && t8_wait(pready + j, done[j] & 1, gave_up, p.polls);
                        if (!ok) continue;
                        ++done[j];
                        tc_fence_after();
                        values(j, g, kt % kT8Flush != 0);
                    }
                    if (!ok) break;
                    tc_commit(vempty + g % SV);
                    if (kt + 1 < n) tc_commit(kempty + (g + 1) % SK);
                }
            }
        }
    } else if (warp < 4) {   // ===== codes to fp16 =====
        T8Item more;
        int g = 0;
        bool ok = true;
        const int me = (warp - 2) * 32 + lane, r8 = me & 7, c0 = me >> 3;       // row of eight, first chunk: neighbouring lanes' chunks lie in different banks, read and written
        constexpr int kChunks = HD / 16, kPer = 8 / kChunks;                    // chunks of a row; rows of eight that 64 threads take at a time: 1 or 2
        // wild: rows that the run must not see become zeros, and NaN codes, which are reported
        auto convert = [&](int key0, int last_pos, int x, const uint8_t* raw, uint8_t* tile, auto values_, auto wild_) {
            constexpr bool values = decltype(values_)::value, wild = decltype(wild_)::value;
            const uint32_t from = s_addr(raw), to = s_addr(tile);
            uint32_t any = 0;
            // all reads in front of all writes: a round's own chain, eight times over, took 1080 clocks a tile of keys and 1380 of values, and the product with the values waited for it
            constexpr int kRounds = kT8Keys / (8 * kPer);
            uint4 codes[kRounds];
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                const int row = i * 8 * kPer + r8 + 8 * (c0 / kChunks), chunk = c0 % kChunks;
                codes[i] = t8_lds(from + row * HD + ((HD == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4));
            }
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                const int row = i * 8 * kPer + r8 + 8 * (c0 / kChunks), chunk = c0 % kChunks;
                uint4 v = codes[i];
                if (values) {
                    const bool take = !wild || (key0 + row <= last_pos && s_tile[x % kT8Known].row[row >= kKv8Block] >= 0);
                    auto look = [&](uint32_t y) {
                        if (wild && !take) y = 0u;
                        const uint32_t n = (y & 0x7f7f7f7fu) + 0x01010101u;                  // the top bit of every NaN
                        any |= n;
                        return wild ? y & ~(((n & 0x80808080u) >> 7) * 0xffu) : y;
                    };
                    v.x = look(v.x); v.y = look(v.y); v.z = look(v.z); v.w = look(v.w);
                }
                const uint32_t at = to + (chunk / 4) * Sh::kBlock + row * 128, c = (chunk % 4) * 2;
                t8_sts(at + ((c ^ (row & 7)) << 4), kv8_half2(v.x & 0xffffu), kv8_half2(v.x >> 16), kv8_half2(v.y & 0xffffu), kv8_half2(v.y >> 16));
                t8_sts(at + (((c + 1) ^ (row & 7)) << 4), kv8_half2(v.z & 0xffffu), kv8_half2(v.z >> 16), kv8_half2(v.w & 0xffffu), kv8_half2(v.w >> 16));
            }
            return __any_sync(0xffffffffu, any & 0x80808080u);
        };
        auto publish = [&]() {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        for (int n_item = 0; ok; ++n_item) {
            const T8Item* at = item_at(n_item, more);
            if (!at) break;
            const TileList tiles = tiles_of(*at);
            const int last_pos = at->pos0 + at->hi;
            auto keys = [&](int x) {               // keys of this CTA's tile x
                ok = t8_wait_warp(rfull + x % RS, (uint32_t)(x / RS) & 1, gave_up, p.polls) && t8_wait_warp(kempty + x % SK, ((uint32_t)(x / SK) & 1) ^ 1, gave_up, p.polls);
                if (!ok) return;
                convert(0, 0, 0, sRaw + 2 * (x % RS) * Sh::kCodes, sK + x % SK * Sh::kTile, std::false_type{}, std::false_type{});
                publish();
                if (lane == 0) mb_arrive(kfull + x % SK);
            };
            keys(g);
            for (int k = at->k0, k1 = at->k1; ok && k < k1; ++k, ++g) {
                const int s = g % RS, tv = g % SV, key0 = tiles.tile_of(k) * kT8Keys;
                if (k + 1 < k1) keys(g + 1);       // a tile ahead of the values: the scores come first
                if (!ok) break;
                ok = t8_wait_warp(vempty + tv, ((uint32_t)(g / SV) & 1) ^ 1, gave_up, p.polls);
                if (!ok) break;
                const uint8_t* codes = sRaw + (2 * s + 1) * Sh::kCodes;
                bool whole = key0 + kT8Keys - 1 <= last_pos && s_tile[g % kT8Known].row[0] >= 0 && s_tile[g % kT8Known].row[1] >= 0;
                if (whole) whole = !convert(key0, last_pos, g, codes, sV + tv * Sh::kTile, std::true_type{}, std::false_type{});
                if (!whole && convert(key0, last_pos, g, codes, sV + tv * Sh::kTile, std::true_type{}, std::true_type{})) {
                    s_nan[n_item & 7] = n_item + 1;          // read behind the product with these values
                    __threadfence_block();
                }
                publish();
                if (lane == 0) { mb_arrive(vfull + tv); mb_arrive(rempty + s); }
            }
        }
    } else if (warp >= 12) {   // ===== O of both tiles =====
        const int quad = warp & 3, row = quad * 32 + lane;
        T8Item more;
        uint32_t done0 = 0, done1 = 0, items0 = 0, items1 = 0;
        bool ok = true;
        for (int n_item = 0; ok; ++n_item) {
            const T8Item* at = item_at(n_item, more);
            if (!at) break;
            const T8Item& it = *at;
            const int n = it.k1 - it.k0, nkt[2] = {it.keys[0], it.keys[1]};
            const bool whole = it.parts == 1;
            float* part = p.parts + (size_t)(2 * blockIdx.x + it.slot_of) * kT8Part;
            float since0 = 1.0f, since1 = 1.0f;                                // what the references have grown by since O was flushed
            for (int kt = 0; ok && kt < n; ++kt)
#pragma unroll 1
                for (int j = 0; j < 2; ++j) {
                    if (!ok || kt >= (j ? nkt[1] : nkt[0])) continue;
                    float since = j ? since1 : since0;
                    const uint32_t so_far = j ? done1 : done0;
                    ok = t8_wait_warp(factors + j, so_far & 1, gave_up, p.polls);       // (the softmax has waited for the product before)
                    if (ok && kt > 0) ok = t8_wait_warp(odone + j, (so_far - 1) & 1, gave_up, p.polls);
                    if (!ok) continue;
                    (j ? done1 : done0) = so_far + 1;
                    tc_fence_after();
                    const float f = factor[j * kT8Rows + row];
                    const uint32_t o_tmem = tmem + ((uint32_t)(quad * 32) << 16) + kT8O + 128 * j;
                    if (kt > 0 && kt % kT8Flush == 0) {         // O so far, relative to the reference before this tile's
                        uint4* acc = reinterpret_cast<uint4*>(part + j * kT8PartTile);
                        const float s = kt > kT8Flush ? since : 0.0f;
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            uint4 v[8];
                            tc_ld32_async(o_tmem + c, o);
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[i] = kt > kT8Flush ? acc[(c / 4 + i) * kT8Rows + row] : make_uint4(0u, 0u, 0u, 0u);
                            tc_arrived(o);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                auto sum = [&](uint32_t x, uint32_t y) { return __float_as_uint(fmaf(__uint_as_float(x), s, __uint_as_float(y))); };
                                acc[(c / 4 + i) * kT8Rows + row] = make_uint4(sum(v[i].x, o[4 * i]), sum(v[i].y, o[4 * i + 1]), sum(v[i].z, o[4 * i + 2]), sum(v[i].w, o[4 * i + 3]));
                            }
                        }
                        since = f;
                    } else {
                        since *= f;
                        if (kt > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
                            for (int c = 0; c < HD; c += 32) {
                                uint32_t o[32];
                                tc_ld32_async(o_tmem + c, o);
                                tc_arrived(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc_st32(o_tmem + c, o);
                            }
                            tc_wait_st();
                        }
                    }
                    (j ? since1 : since0) = since;
                    tc_fence_before();
                    mb_arrive(pready + j);
                }
            if (!ok) break;
            // ---- results, or this CTA's part of them ----
#pragma unroll 1
            for (int j = 0; ok && j < 2; ++j) {
                const int mine = j ? nkt[1] : nkt[0];
                const float since = j ? since1 : since0;
                if (mine == 0) {
                    if (!whole) {                                              // none of this part's keys is visible to this tile
                        part[j * kT8PartTile + 128 * kT8Rows + row] = -INFINITY;
                        part[j * kT8PartTile + 129 * kT8Rows + row] = 0.0f;
                    }
                    continue;
                }
                ok = t8_wait_warp(lready + j, (j ? items1 : items0) & 1, gave_up, p.polls) && t8_wait_warp(odone + j, ((j ? done1 : done0) - 1) & 1, gave_up, p.polls);
                if (j) ++items1; else ++items0;
                if (!ok) break;
                tc_fence_after();
                const float ref = s_ref[j * kT8Rows + row], l = s_sum[j * kT8Rows + row], inv = l == 0.0f ? 0.0f : kT8Down / l;
                mb_arrive(lread + j);
                const bool nan_here = s_nan[n_item & 7] == n_item + 1;         // (behind the last product: every value has been converted)
                const uint32_t o_tmem = tmem + ((uint32_t)(quad * 32) << 16) + kT8O + 128 * j;
                uint4* acc = reinterpret_cast<uint4*>(part + j * kT8PartTile);
                const bool flushed = mine > kT8Flush;
                const T8Out to = t8_out(p, it, j, row);
                const float f = whole ? inv : kT8Down;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tc_ld32_async(o_tmem + c, o);
                    if (flushed) {
                        uint4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = acc[(c / 4 + i) * kT8Rows + row];
                        tc_arrived(o);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            auto sum = [&](uint32_t x, uint32_t& y) { y = __float_as_uint(fmaf(__uint_as_float(x), since, __uint_as_float(y))); };
                            sum(v[i].x, o[4 * i]); sum(v[i].y, o[4 * i + 1]); sum(v[i].z, o[4 * i + 2]); sum(v[i].w, o[4 * i + 3]);
                        }
                    } else {
                        tc_arrived(o);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        auto four = [&](int e) { return make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f); };
                        const float4 x = four(i), y = four(i + 4);
                        if (!whole) {
                            reinterpret_cast<float4*>(acc)[((c + i) / 4) * kT8Rows + row] = x;
                            reinterpret_cast<float4*>(acc)[((c + i) / 4 + 1) * kT8Rows + row] = y;
                        } else if (to.listed && c + i < a.dv) {
                            t8_store(to, c + i, x, y);
                        }
                    }
                    __syncwarp();
                }
                if (whole && nan_here) t8_poison(p, it, j, row, 0, a.dv);
                if (!whole) {
                    part[j * kT8PartTile + 128 * kT8Rows + row] = ref;
                    part[j * kT8PartTile + 129 * kT8Rows + row] = nan_here ? -l : l;      // (sums are not negative: the sign says that there was NaN)
                }
            }
            if (!ok) break;
            tc_fence_before();
        }
    } else {   // ===== softmax: TMEM lane quadrant = warp % 4 =====
        const int j = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16, s_tmem = tmem + lanes + kT8S + 64 * j, p_tmem = tmem + lanes + kT8P + 64 * j;
        const int q = j * p.queries + (row >> p.hpc_log2);
        T8Item more;
        uint32_t done = 0, items = 0;
        int g0 = 0, g1 = 0;                      // key tiles of the CTA in front of this item, and of the next
        bool ok = true;
        for (int n_item = 0; ok; ++n_item) {
            const T8Item* at = item_at(n_item, more);
            if (!at) break;
            const T8Item& it = *at;
            const int n = it.keys[j];
            g0 = g1;
            g1 += it.k1 - it.k0;
            if (n == 0) continue;
            const bool live = it.listed(q);
            const int qpos = it.pos0 + (live ? q : it.hi), h = it.h0 + (row & (p.hpc - 1));
            const TileList tiles = tiles_of(it);
            // ---- queries: fp16, brought to 1 .. 2 by a power of two of the row's largest; every score of the item before has been made ----
            float up;
            {
                // By copies to where fp16 rows come to lie: theirs, and those of the second term. Two lanes convert a row, sixteen rows at a time, once all of it is in registers: few instructions
                // (by whole rows, each with a reduction, and in line for all of them it was 20 KB of code run once an item, and took 5000 to 20000 clocks).
                constexpr int kLanes = HD / 4, kPer = 32 / kLanes, kLoads = 16 / kPer, kChunks = HD / 8;       // lanes of a row, rows of a load, loads of sixteen rows; a lane's chunks of four columns
                const int mine = it.tok0 + (live ? q : it.hi), col = (lane % kLanes) * 4, sub = lane / kLanes;      // (a row without a query reads another)
                const float* src = a.q + (size_t)it.h0 * a.dk + col;
                // row 8 i + r of a block lies 1024 i + 128 r further, its chunks of 16 bytes exchanged by r
                const uint32_t own = s_addr(sQ) + j * Sh::kQTile + quad * 4096;
                auto piece = [&](int x, int n) { return own + (n >> 1) * Sh::kQBlock + x * 2048 + (n & 1) * Sh::kQTerm; };      // 2 KB, a quarter (HD 64: half) of sixteen rows
                int ex = 127;
                {
                    auto address = [&](int i) {
                        const int r = i * kPer + sub;
                        return src + (size_t)(uint32_t)__shfl_sync(0xffffffffu, mine, r) * (uint32_t)a.ldq + (uint32_t)((r & (p.hpc - 1)) * a.dk);
                    };
                    auto place = [&](int i) { return piece(i / kLoads, i % kLoads / 4) + (i & 3) * 512 + lane * 16; };
                    const bool take = col < a.dk;
                    if (p.vec_q) {                                 // (no branch between the copies: they go out one behind the other)
#pragma unroll
                        for (int i = 0; i < kLoads * 2; ++i) {
                            const float* at = address(i);
                            asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %2, 0;\n@p cp.async.cg.shared.global [%0], [%1], 16;\n}\n" ::"r"(place(i)), "l"(at), "r"((uint32_t)take) : "memory");
                        }
                    } else {
#pragma unroll 1
                        for (int i = 0; i < kLoads * 2; ++i) {
                            const float* at = address(i);
                            if (take) t8_sts(place(i), __float_as_uint(at[0]), __float_as_uint(at[1]), __float_as_uint(at[2]), __float_as_uint(at[3]));
                        }
                    }
                    if (!take) {
#pragma unroll 1
                        for (int i = 0; i < kLoads * 2; ++i) t8_sts(place(i), 0u, 0u, 0u, 0u);
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();                                  // a copy is seen by its own lane after the wait, by the others behind this
                }
#pragma unroll 1
                for (int x = 0; x < 2; ++x) {
                    // lane r of either half takes its chunks of four columns in the order 0 ^ r, 1 ^ r, ...: no two meet in a bank
                    constexpr int kRow = HD * 4, kOf = 2048 / kRow;                            // bytes of a row, rows of a piece
                    const int n = lane & 15, r = 16 * x + n, turn = n & (kChunks - 1);
                    const uint32_t from = piece(x, n / kOf) + n % kOf * kRow + (lane >> 4) * (kRow / 2);
                    uint32_t v[kChunks][4];
                    float most = 0.0f;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        const uint4 w = t8_lds(from + ((c ^ turn) << 4));
                        v[c][0] = w.x; v[c][1] = w.y; v[c][2] = w.z; v[c][3] = w.w;
                        auto of = [](uint32_t y) { return fabsf(__uint_as_float(y)); };
                        most = tc_max3(tc_max3(most, of(w.x), of(w.y)), of(w.z), of(w.w));
                    }
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                    const int of = (int)(__float_as_uint(most) >> 23), e = of == 255 ? 127 : min(max(of, 27), 253);      // exponent + 127 (an infinity among them: 0), so that its reciprocal is a normal number
                    if (lane >> 4 == x) ex = e;
                    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    __syncwarp();                                  // all have read
#pragma unroll
                    for (int d = 0; d < kChunks / 2; ++d) {        // eight columns; in an odd lane the second four come first
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float y = __uint_as_float(v[2 * d + k / 2][2 * k & 3]) * down, z = __uint_as_float(v[2 * d + k / 2][(2 * k & 3) + 1]) * down;
                            hi[k] = t8_pack(y, z);
                            const float2 w = t8_unpack(hi[k]);
                            lo[k] = t8_pack(y - w.x, z - w.y);
                        }
                        const bool odd = turn & 1;
                        const int chunk = (lane >> 4) * (kChunks / 2) + (d ^ (turn >> 1));
                        const uint32_t to = own + (chunk >> 3) * Sh::kQBlock + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
                        t8_sts(to, odd ? hi[2] : hi[0], odd ? hi[3] : hi[1], odd ? hi[0] : hi[2], odd ? hi[1] : hi[3]);
                        t8_sts(to + Sh::kQTerm, odd ? lo[2] : lo[0], odd ? lo[3] : lo[1], odd ? lo[0] : lo[2], odd ? lo[1] : lo[3]);
                    }
                    __syncwarp();
                }
                up = __uint_as_float((uint32_t)ex << 23);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mb_arrive(qready + j);
                // the next item's queries come into the L2 meanwhile: each lane asks for a row's
                if (n_item + 1 < min(w.count, kT8Items)) {
                    const T8Item& after = s_items[n_item + 1];
                    if (after.k1 > 0 && after.keys[j] > 0) {
                        const char* at = reinterpret_cast<const char*>(a.q + (size_t)(after.tok0 + (after.listed(q) ? q : after.hi)) * a.ldq + (size_t)(after.h0 + (row & (p.hpc - 1))) * a.dk);
#pragma unroll
                        for (int c = 0; c < HD * 4; c += 128)
                            if (c < a.dk * 4) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + c));
                    }
                }
            }
            const int wnd = seq_row_window(qpos, a.window, a.chunk);
            const float slope = kOpts && a.slopes ? a.slopes[h] : 0.0f, mul = a.scale * up * (kOpts ? 1.0f : kTcLog2e);
            float ref = -INFINITY, l = 0.0f;
            for (int kt = 0; kt < n; ++kt) {
                const int key0 = tiles.tile_of(it.k0 + kt) * kT8Keys;
                ok = t8_wait_warp(sfull + j, done & 1, gave_up, p.polls);
                if (!ok) break;
                ++done;
                tc_fence_after();
                uint32_t s[64];
                tc_ld32_async(s_tmem, s);
                tc_ld32_async(s_tmem + 32, s + 32);
                const T8Tile known = s_tile[(g0 + kt) % kT8Known];
                const bool gone[2] = {known.row[0] < 0, known.row[1] < 0};
                const float ev[2] = {known.ev[0], known.ev[1]};
                // every key of the tile is visible to every row of the warp
                const bool all = __all_sync(0xffffffffu, !gone[0] && !gone[1] && key0 + kT8Keys - 1 <= qpos && (qpos - key0 < wnd || key0 + kT8Keys <= a.keep_first));
                tc_arrived(s);
                tc_arrived(s + 32);
                tc_fence_before();
                mb_arrive(sread + j);              // the next scores may be made
                // (2^-100 at least, which adds nothing to a score: queries and keys of nothing but zeros have scales of 2^-100 each, and a hidden score of -inf times 0 were no number)
                float f[2] = {fmaxf(known.ks[0] * mul, 7.9e-31f), fmaxf(known.ks[1] * mul, 7.9e-31f)};
                if (kOpts) {
                    if (a.softcap > 0.0f) {        // s becomes what times f is the capped score
                        const float inv[2] = {f[0] / a.softcap, f[1] / a.softcap};
                        float most[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                t0 = tc_max3(t0, fabsf(__uint_as_float(s[32 * x + e])), fabsf(__uint_as_float(s[32 * x + e + 1])));
                                t1 = tc_max3(t1, fabsf(__uint_as_float(s[32 * x + e + 2])), fabsf(__uint_as_float(s[32 * x + e + 3])));
                            }
                            most[x] = fmaxf(t0, t1);
                        }
                        // scores below the cap, as nearly all are: tanh x = x g(x^2), g through Chebyshev's eight points of [0, 1] (9e-9 of its value; with its roundings 1.1e-7), two scores
                        // at a time: 5 instructions a score, where tc_tanh takes 13 and two of the special function unit. Where one of the warp's scores is not, that of a hidden key (which may be
                        // anything) among them, the others still go through the same series: it shows in no bit of theirs.
                        constexpr float k7 = -0.00035232809f, k6 = 0.0022786476f, k5 = -0.0079124849f, k4 = 0.0214614104f, k3 = -0.0538697056f, k2 = 0.1333213896f, k1 = -0.333332777f;
                        if (__any_sync(0xffffffffu, !(fmaxf(most[0] * inv[0], most[1] * inv[1]) < 1.0f))) {
                            const float back[2] = {a.softcap / f[0], a.softcap / f[1]};
#pragma unroll
                            for (int e = 0; e < 64; ++e) {
                                const float v = __uint_as_float(s[e]), x = __fmul_rn(v, inv[e / 32]), u = __fmul_rn(x, x);
                                const float t = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, k7, k6), k5), k4), k3), k2), k1);
                                s[e] = __float_as_uint(fabsf(x) < 1.0f ? __fmul_rn(v, fmaf(u, t, 1.0f)) : back[e / 32] * tc_tanh(x));
                            }
                        } else {
                            auto both = [](float v) { return tc_two(__float_as_uint(v), __float_as_uint(v)); };
                            const uint64_t c7 = both(k7), c6 = both(k6), c5 = both(k5), c4 = both(k4), c3 = both(k3), c2 = both(k2), c1 = both(k1), one = both(1.0f);
#pragma unroll
                            for (int e = 0; e < 64; e += 2) {
                                const uint64_t v = tc_two(s[e], s[e + 1]), x = tc_mul2(v, both(inv[e / 32])), u = tc_mul2(x, x);
                                uint64_t t = tc_fma2(u, c7, c6);
                                t = tc_fma2(u, t, c5);
                                t = tc_fma2(u, t, c4);
                                t = tc_fma2(u, t, c3);
                                t = tc_fma2(u, t, c2);
                                t = tc_fma2(u, t, c1);
                                float y, z;
                                tc_split(tc_mul2(v, tc_fma2(u, t, one)), y, z);
                                s[e] = __float_as_uint(y);
                                s[e + 1] = __float_as_uint(z);
                            }
                        }
                    }
                    if (a.slopes) {
                        const float dist = (float)(qpos - key0);
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(fmaf(-slope, dist - (float)e, __uint_as_float(s[e]) * f[e / 32]));
                        f[0] = f[1] = 1.0f;
                    }
                    f[0] *= kTcLog2e;
                    f[1] *= kTcLog2e;
                }
                if (!all) {        // the columns this row sees, as bits
                    const int hi = qpos - key0, lo = wnd > qpos ? -1 : qpos - wnd - key0, keep = a.keep_first - key0;
                    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };       // bits 0 .. n - 1
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t seen = gone[x] ? 0u : below(hi + 1 - 32 * x) & (~below(lo + 1 - 32 * x) | below(keep - 32 * x));
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[32 * x + e] = seen & (1u << e) ? s[32 * x + e] : 0xff800000u;        // -inf
                    }
                }
                {
                    float top[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            t0 = tc_max3(t0, __uint_as_float(s[32 * x + e]), __uint_as_float(s[32 * x + e + 1]));
                            t1 = tc_max3(t1, __uint_as_float(s[32 * x + e + 2]), __uint_as_float(s[32 * x + e + 3]));
                        }
                        top[x] = fmaxf(t0, t1);
                    }
                    const float m0 = fmaf(top[0], f[0], ev[0]), m1 = fmaf(top[1], f[1], ev[1]);
                    float mx = fmaxf(m0, m1);
                    // Rare, with one vote for both: scores so large that a rounded product and one inside a multiply-add are far apart, and a value scale's exponent is less than their steps: every
                    // product is rounded then, its reference, rounded down, taken from it in front of the exponent, and what is above 1 still is 1 (the largest one's weight: rounded to nearest
                    // the reference could be a step above or below, and the weight out of fp16's range); and a block whose weights come out below 2^-60 because its value scale is that much
                    // smaller than others' (`far`).
                    float far[2] = {0.0f, 0.0f};
                    const bool rare = __any_sync(0xffffffffu, fabsf(mx) > 65536.0f ? mx != -INFINITY : fminf(m0, m1) < fmaxf(ref, mx) - 60.0f);
                    bool large = false;
                    if (rare) {
                        large = __any_sync(0xffffffffu, fabsf(mx) > 65536.0f && mx != -INFINITY);
                        if (large) {
                            top[0] *= f[0];
                            top[1] *= f[1];
                            mx = fmaxf(__fadd_rd(top[0], ev[0]), __fadd_rd(top[1], ev[1]));
                        }
                        // Nothing to O (2^-60 is far below the last step of fp16, too), but the denominator has their weights without the scale: they are taken 2^far larger, so that they do not vanish.
                        const float base = fmaxf(ref, ceilf(mx)), from = base == -INFINITY ? 0.0f : base;
                        auto relative = [&](float product, int x) {        // 2^.. of a weight without the value scale, of a large score
                            const float y = __fsub_rn(product, from);
                            return y > -ev[x] ? -ev[x] : y;                // (NaN stays)
                        };
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float most = large ? relative(top[x], x) + ev[x] : fmaf(top[x], f[x], ev[x]) - base;
                            far[x] = most < -60.0f && most > -1e6f ? floorf(-most) : 0.0f;
                        }
                        if (large) {
#pragma unroll
                            for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(relative(__fmul_rn(__uint_as_float(s[e]), f[e / 32]), e / 32));
                            f[0] = f[1] = 1.0f;
                        }
                    }
                    const float nr = fmaxf(ref, ceilf(mx)), less = kt == 0 || nr == ref ? 1.0f : tc_exp2(ref - nr);
                    // the product with the last weights has been made: their place is free, and their factors have been used
                    if (done > 1) ok = t8_wait_warp(odone + j, (done - 2) & 1, gave_up, p.polls);
                    if (!ok) break;
                    tc_fence_after();
                    factor[j * kT8Rows + row] = less;
                    mb_arrive(factors + j);
                    l = kt == 0 ? 0.0f : l * less;
                    ref = nr;
                    // where every score so far is -inf, -inf - ref were no number: relative to 0 their weights are 0
                    const float base = ref == -INFINITY || large ? 0.0f : ref;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float neg = ev[x] - base + (far[x] + (float)kA8Lift);
                        const uint64_t f2 = tc_two(__float_as_uint(f[x]), __float_as_uint(f[x])), neg2 = tc_two(__float_as_uint(neg), __float_as_uint(neg));
                        uint64_t sum = 0;
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float y, z;
                            tc_split(tc_fma2(tc_two(s[32 * x + 2 * e], s[32 * x + 2 * e + 1]), f2, neg2), y, z);
                            y = tc_exp2(y);
                            z = tc_exp2(z);
                            sum = tc_add2(sum, tc_two(__float_as_uint(y), __float_as_uint(z)));
                            hi[e] = t8_pack(y, z);
                            const float2 u = t8_unpack(hi[e]);
                            lo[e] = t8_pack(y - u.x, z - u.y);
                        }
                        if (rare) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                hi[e] = far[x] != 0.0f ? 0u : hi[e];
                                lo[e] = far[x] != 0.0f ? 0u : lo[e];
                            }
                        }
                        tc_st16(p_tmem + 16 * x, hi);
                        tc_st16(p_tmem + 32 + 16 * x, lo);
                        float s0, s1;
                        tc_split(sum, s0, s1);
                        l = fmaf((s0 + s1) * kT8Down, tc_exp2(-ev[x] - far[x]), l);         // without the value scale
                    }
                }
                tc_wait_st();
                tc_fence_before();
                mb_arrive(pready + j);
            }
            if (!ok) break;
            if (items) ok = t8_wait_warp(lread + j, (items - 1) & 1, gave_up, p.polls);
            if (!ok) break;
            s_ref[j * kT8Rows + row] = ref;
            s_sum[j * kT8Rows + row] = l;
            ++items;
            mb_arrive(lready + j);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*gave_up) tc_gave_up(p.status);
    if (warp == 1) {
        tc_fence_after();
        tc_dealloc(tmem, kT8Tmem);
    }
}

template <int HD, bool kOpts>
static int t8_launch(const T8Args& a, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    using Sh = T8Shape<HD>;
    auto* kernel = seq_attention8_tc_kernel<HD, kOpts>;
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
            return SLLM_OK;
        }))
        return rc;
    LaunchCfg lc(dim3(std::min(kA8TcWorkers, sm_count())), dim3(kT8Threads), Sh::kSmem, st, true);        // its beginning while the plan is made
    SLLM_CUDA(cudaLaunchKernelEx(&lc.cfg, overlapping(kernel), tmK, tmV, a));
    LaunchCfg join(dim3(lc.cfg.gridDim.x, kT8JoinCtas), dim3(kT8Rows), 0, st, true);
    SLLM_CUDA(cudaLaunchKernelEx(&join.cfg, overlapping(seq_attention8_join_kernel), a));
    g_launches += 2;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

static int t8_hpc(const Attn8Args& p) {
    const int group = p.heads / p.kv_heads;
    return group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
}

int attention8_tc_width(const Attn8Args& p) { return 2 * kT8Rows / t8_hpc(p); }

bool attention8_tc_takes(const Attn8Args& p) {
    const int width = attention8_tc_width(p);
    return p.dk <= 128 && p.dv <= 128 && p.b.nseg <= kA8Segs && p.b.T / width + p.b.nseg <= kA8Runs;
}

int launch_attention8_tc(const Attn8Args& p, void* ws, cudaStream_t st) {
    T8Args a{};
    a.a = p;
    a.hpc = t8_hpc(p);
    a.hpc_log2 = a.hpc / 2;
    a.queries = kT8Rows / a.hpc;
    a.sets = p.heads / a.hpc;
    a.vec_q = p.ldq % 4 == 0 && ((uintptr_t)p.q % 16) == 0;
    a.plan = reinterpret_cast<const A8Plan*>((uint8_t*)ws + kA8PlanAt);
    a.cuts = reinterpret_cast<T8Item*>((uint8_t*)ws + kA8CutsAt);
    a.parts = (float*)((uint8_t*)ws + kA8PartsAt);
    if (int rc = status_word(&a.status)) return rc;
    a.polls = (unsigned)g_tune_tc_polls;
    const int HD = std::max(p.dk, p.dv) <= 64 ? 64 : 128;
    CUtensorMap tmK, tmV;
    const uint64_t rows = (uint64_t)p.n_pages * p.kv_heads * p.b.page_len;
    if (int rc = tc_encode_bytes(&tmK, p.k_pool, rows, p.dk, kKv8Block, HD)) return rc;
    if (int rc = tc_encode_bytes(&tmV, p.v_pool, rows, p.dv, kKv8Block, HD)) return rc;
    const bool opts = p.softcap > 0.0f || p.slopes;
    if (HD == 128) return opts ? t8_launch<128, true>(a, tmK, tmV, st) : t8_launch<128, false>(a, tmK, tmV, st);
    return opts ? t8_launch<64, true>(a, tmK, tmV, st) : t8_launch<64, false>(a, tmK, tmV, st);
}

}  // namespace sllm
