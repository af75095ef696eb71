// csrc/seq_attn8_tc.cu — attention of prompt portions over the 8-bit paged cache on the 5th-generation tensor cores, heads of up to 128 columns.
//
// 128 rows = the query heads of a kv head (four, two or one) x 32, 64 or 128 neighbouring queries are a tile; a CTA has two tiles at a time, neighbours in the sequence (a run), that share
// tiles of 64 keys and values. fp16 operands, since fp16 holds every e4m3 code: keys and values enter exactly, and block scales multiply scores and weights.
//   warp 0 (one lane)   TMA producer: boxes of 32 rows of codes, looked up in the block table, into a ring;
//   warps 2, 3          codes to fp16 rows in the 128B swizzle (keys K-major, values as they lie); value rows that the run must not see, and NaN codes among values, become zeros;
//   warp 1 (one lane)   MMA issuer: S = Q K^T with Q read from TMEM (shared memory has to feed the codes' conversion, too: from there Q alone would take its bandwidth), O += P V with P over S;
//   warps 4-7, 8-11     softmax of tile 0 / 1, a thread per row: queries to fp16 in TMEM once an item, then per key tile maximum, weights and their sum;
//   warps 12-15         O of both tiles: rescaled where a maximum has grown, results written, parts of shared items put together.
// Results in bf16 (kTerms = 1): queries and weights are one fp16 number each (2^-12 of a value on average less than the 2^-9 of the result's own rounding). Results in fp32 (kTerms = 2): both are
// the sum of two (22 bits; the second query term is read from shared memory), and O is added to an fp32 copy of the CTA's own every kT8Flush tiles, because the tensor core truncates as it
// accumulates.
// Weights are relative to the largest of score + log2(value scale) so far, rounded up to a whole number: differences of exponents are exact then, and O is rescaled by powers of two, and
// seldom. The denominator takes the value scale out again, block by block.
// A value's NaN code must reach exactly the rows that see it, but 0 * NaN is NaN: the converters replace it and say so, and rows of such an item look for NaN among their keys' values
// at the end.
// Shares. A CTA per item would leave most SMs idle where few queries follow a long context. The key tiles of all items lie in one row, made by a small kernel in front from what the
// device knows (contexts, listed tiles); every CTA takes an equal run of it. Items that a cut goes through leave O, reference and sum as parts for the one of their CTAs that is done last.
#include <type_traits>

#include "seq_attn8.cuh"
#include "tcgen05.cuh"

namespace sllm {

constexpr int kT8Rows = 128, kT8Keys = 64, kT8Threads = 512, kT8Raw = 4;      // rows of a tile, keys of a tile, stages of the codes' ring
constexpr int kT8Extra = 4, kT8Least = 4;       // key tiles that an item's beginning and end count for; key tiles of a CTA's share at least
constexpr int kT8Flush = 16;
constexpr uint32_t kT8Tmem = 512, kT8S = 0, kT8Q = 128, kT8O = 256;           // columns: S0 S1 | Q0 Q1 | O0 O1

template <int HD, int kTerms>
struct T8Shape {
    static constexpr int kBlocks = HD / 64, kStages = kTerms == 1 ? 3 : 2;
    static constexpr int kBlock = kT8Keys * 128, kTile = kBlocks * kBlock;    // fp16: 64 columns of all keys; all columns
    static constexpr int kCodes = kT8Keys * HD;                              // bytes of a tile of codes
    static constexpr int kQBlock = kT8Rows * 128, kQTile = kTerms == 2 ? kBlocks * kQBlock : 0;
    static constexpr int kSmem = 1024 + 2 * kStages * kTile + 2 * kT8Raw * kCodes + 2 * kQTile + 512 + 8 * kT8Rows * (int)sizeof(float);
};
constexpr int kT8PartTile = kT8Rows * (128 + 2), kT8Part = 2 * kT8PartTile;   // floats of a part: per tile O as [HD / 4][128][4], references, sums
static_assert(kT8Part == kA8Part, "the workspace's parts");

struct T8Args {
    Attn8Args a;
    int hpc, hpc_log2, queries;          // query heads and queries of a tile: hpc * queries = 128
    int sets;                            // head sets of a step: kv_heads * (group / hpc)
    int vec_q;
    const A8Plan* plan;
    int* counters;
    float* parts;
    int32_t* status;
    unsigned polls;
};

// ---- the plan: which runs of 2 * queries neighbouring queries have listed tiles, and how many key tiles each ----
// One CTA. Tiles of one query are the other kernel's.
__global__ void __launch_bounds__(1024) seq_attention8_plan_kernel(Attn8Args p, int width, A8Plan* plan) {
    after_previous();
    const sllm_seq_batch& b = p.b;
    __shared__ int s_base[kA8Segs + 1];
    __shared__ int s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](int v, int& total) {         // exclusive sum over the CTA
        int upto = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = upto;
        __syncthreads();
        int before = 0;
        total = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += s_warp[w];
            total += s_warp[w];
        }
        return before + upto - v;
    };
    int runs = 0;
    for (int s0 = 0; s0 < b.nseg; s0 += 1024) {
        const int s = s0 + threadIdx.x, len = s < b.nseg ? b.seg_len[s] : 0;
        int total;
        const int at = scan(len > 1 ? (len + width - 1) / width : 0, total);
        if (s < b.nseg) s_base[s] = runs + at;
        runs += total;
    }
    runs = min(runs, kA8Runs);                   // (the host has made sure)
    for (int i = threadIdx.x; i < runs * 8; i += 1024) plan->mask[i / 8][i % 8] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < b.nseg; i += 1024) {
        const int len = b.seg_len[i], n = len > 1 ? (len + width - 1) / width : 0;
        for (int r = 0; r < n && s_base[i] + r < runs; ++r) {
            plan->seg[s_base[i] + r] = i;
            plan->first[s_base[i] + r] = r * width;
        }
    }
    for (int i = threadIdx.x; i < b.n_qtiles; i += 1024) {
        const int seg = b.qt_seg[i], off = b.qt_off[i], n = min(kBQ, b.seg_len[seg] - off);
        if (n <= 1 || off < 0) continue;
        for (int q = off; q < off + n;) {        // a word of a run's mask at a time
            const int run = s_base[seg] + q / width, bit = q % width, count = min(off + n - q, 32 - bit % 32);
            if (run < runs) atomicOr(&plan->mask[run][bit / 32], (count == 32 ? 0xffffffffu : (1u << count) - 1) << (bit % 32));
            q += count;
        }
    }
    __syncthreads();
    __threadfence_block();
    int all = 0;
    for (int r0 = 0; r0 < runs; r0 += 1024) {
        const int r = r0 + threadIdx.x;
        int units = 0;
        if (r < runs) {
            int lo = -1, hi = -1;
            for (int w = 0; w < 8; ++w) {
                const uint32_t m = *reinterpret_cast<volatile uint32_t*>(&plan->mask[r][w]);
                if (!m) continue;
                if (lo < 0) lo = 32 * w + __ffs(m) - 1;
                hi = 32 * w + 31 - __clz(m);
            }
            const int seg = plan->seg[r], pos0 = b.seg_pos0[seg] + plan->first[r];
            if (lo >= 0 && pos0 >= 0) units = TileList(pos0 + lo, pos0 + hi, seq_row_window(pos0 + lo, p.window, p.chunk), p.keep_first, kT8Keys).n + kT8Extra;
        }
        int total;
        const int at = scan(units, total);
        if (r < runs) plan->before[r] = all + at;
        all += total;
    }
    if (threadIdx.x == 0) {
        plan->before[runs] = all;
        plan->runs = runs;
    }
}

// What a role knows of the item it is at. Every role walks its CTA's share by itself.
struct T8Item {
    int x, y;                                // run, head set
    int k0, k1, n;                           // its key tiles that are this CTA's, of so many
    int tok0, pos0, slot, gkv, h0;           // first token and position of the run; kv head, first query head
    int lo, hi;                              // first and last listed query of the run
    uint32_t m[8];
};

struct T8Walk {
    const T8Args& p;
    long long begin, end, u;
    int x, ctas;
    long long total;
    __device__ __forceinline__ T8Walk(const T8Args& args, int start_run, int n_ctas, long long all) : p(args), x(start_run), ctas(n_ctas), total(all) {
        begin = share(blockIdx.x);
        end = share(blockIdx.x + 1);
        u = begin;
    }
    __device__ __forceinline__ long long share(int c) const { return (long long)c * total / ctas; }
    __device__ __forceinline__ int owner(long long v) const { return (int)(((v + 1) * ctas - 1) / total); }
    __device__ __forceinline__ bool next(T8Item& it) {
        for (; u < end;) {
            const int b0 = p.plan->before[x], each = p.plan->before[x + 1] - b0;
            const long long at = (long long)b0 * p.sets;
            if (u >= at + (long long)each * p.sets) { ++x; continue; }
            it.x = x;
            it.y = (int)((u - at) / each);
            it.n = each - kT8Extra;
            const long long item0 = at + (long long)it.y * each + kT8Extra;
            it.k0 = (int)max(0ll, u - item0);
            it.k1 = (int)(min(end, item0 + it.n) - item0);
            if (it.k1 <= 0) return false;        // the share ends before the item's first tile
            u = item0 + it.k1;
            const sllm_seq_batch& b = p.a.b;
            const int seg = p.plan->seg[x], first = p.plan->first[x], group = p.a.heads / p.a.kv_heads, per = group / p.hpc;
            it.tok0 = b.seg_start[seg] + first;
            it.pos0 = b.seg_pos0[seg] + first;
            it.slot = b.seg_slot[seg];
            it.gkv = it.y / per;
            it.h0 = it.gkv * group + it.y % per * p.hpc;
            it.lo = it.hi = -1;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                it.m[w] = p.plan->mask[x][w];
                if (it.m[w]) {
                    if (it.lo < 0) it.lo = 32 * w + __ffs(it.m[w]) - 1;
                    it.hi = 32 * w + 31 - __clz(it.m[w]);
                }
            }
            return true;
        }
        return false;
    }
    __device__ __forceinline__ TileList tiles(const T8Item& it) const {
        return TileList(it.pos0 + it.lo, it.pos0 + it.hi, seq_row_window(it.pos0 + it.lo, p.a.window, p.a.chunk), p.a.keep_first, kT8Keys);
    }
    // how many of its key tiles k0 .. k1 a tile has to see: those up to its last listed query's
    __device__ __forceinline__ int keys(const T8Item& it, int j) const {
        int last = -1;
        const int q0 = j * p.queries, q1 = q0 + p.queries;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            if (32 * w >= q0 && 32 * w < q1 && it.m[w]) last = 32 * w + 31 - __clz(it.m[w]);
        if (last < 0) return 0;
        const int n = it.n - ((it.pos0 + it.hi) / kT8Keys - (it.pos0 + last) / kT8Keys);
        return max(0, min(it.k1, n) - it.k0);
    }
};

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
// fp16 operands: the bf16 descriptor without its types
__host__ __device__ constexpr uint32_t t8_idesc(int M, int N) { return umma_idesc_bf16(M, N) & ~((1u << 7) | (1u << 10)); }

template <int HD, int kTerms, bool kOpts>
__global__ void __launch_bounds__(kT8Threads, 1) seq_attention8_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ T8Args p) {
    using Sh = T8Shape<HD, kTerms>;
    constexpr int ST = Sh::kStages, RS = kT8Raw;
    extern __shared__ uint8_t t8_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(t8_smem) + 1023) & ~(uintptr_t)1023);
    uint8_t *sK = smem, *sV = sK + ST * Sh::kTile, *sQ = sV + ST * Sh::kTile, *sRaw = sQ + 2 * Sh::kQTile;      // sRaw: keys, then values, of each stage
    uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + 2 * RS * Sh::kCodes);
    uint64_t *rfull = bars, *rempty = rfull + RS, *kfull = rempty + RS, *kempty = kfull + ST, *vfull = kempty + ST, *vempty = vfull + ST;
    // per tile: queries written / scores written / factors for O written / weights written and O rescaled / product with the values done / sums written, and read
    uint64_t *qready = vempty + ST, *sfull = qready + 2, *factors = sfull + 2, *pready = factors + 2, *odone = pready + 2, *lready = odone + 2, *lread = lready + 2;
    uint64_t* meet = lread + 2;              // of warps 12-15
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(meet + 1);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_start = reinterpret_cast<int*>(tmem_slot + 2);
    int* s_last = reinterpret_cast<int*>(tmem_slot + 3);
    volatile int* s_nan = reinterpret_cast<volatile int*>(tmem_slot + 4);        // [8]: at i % 8 the number (from 1) of an item that had NaN among its values; the converters are fewer items ahead
    float* factor = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);        // [2][128]
    float *s_ref = factor + 2 * kT8Rows, *s_sum = s_ref + 2 * kT8Rows;                        // [2][128] each
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Attn8Args& a = p.a;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < RS; ++i) { mb_init(rfull + i, 1); mb_init(rempty + i, 2); }
        for (int i = 0; i < ST; ++i) { mb_init(kfull + i, 2); mb_init(kempty + i, 1); mb_init(vfull + i, 2); mb_init(vempty + i, 1); }
        for (int j = 0; j < 2; ++j) {
            mb_init(qready + j, 128); mb_init(sfull + j, 1); mb_init(factors + j, 128); mb_init(pready + j, 256); mb_init(odone + j, 1); mb_init(lready + j, 128); mb_init(lread + j, 128);
        }
        *gave_up = 0;
        for (int i = 0; i < 8; ++i) s_nan[i] = 0;
        mb_init(meet, 128);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tc_alloc(tmem_slot, kT8Tmem);
    after_previous();
    // this CTA's share: the run it begins in
    const int runs = p.plan->runs;
    const long long total = (long long)p.plan->before[runs] * p.sets;
    const int ctas = (int)min((long long)gridDim.x, (total + kT8Least - 1) / kT8Least);
    const bool work = (int)blockIdx.x < ctas;
    if (work && threadIdx.x == 0) {
        const long long first = (long long)blockIdx.x * total / ctas;
        int lo = 0, hi = runs;                   // before[lo] * sets <= first < before[hi] * sets
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((long long)p.plan->before[mid] * p.sets <= first) lo = mid; else hi = mid;
        }
        *s_start = lo;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (!work) {
    } else if (warp == 0) {
        if (elect_one()) {   // ===== TMA producer =====
            T8Walk w(p, *s_start, ctas, total);
            T8Item it;
            int g = 0;                           // key tiles so far
            bool ok = true;
            while (ok && w.next(it)) {
                const TileList tiles = w.tiles(it);
                for (int k = it.k0; k < it.k1; ++k, ++g) {
                    const int s = g % RS, key0 = tiles.tile_of(k) * kT8Keys;
                    int row[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) row[x] = t8_row(a, it.slot, it.gkv, key0 + x * kKv8Block, it.pos0 + it.hi);
                    ok = tc_wait(rempty + s, ((uint32_t)(g / RS) & 1) ^ 1, gave_up, p.polls);
                    if (!ok) break;
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
            auto scores = [&](int j, int g) {
                const uint64_t k = k_desc + (uint32_t)(g % ST) * (Sh::kTile / 16), q = q_desc + (uint32_t)j * (Sh::kQTile / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    tc_mma_bf16_ts(tmem + kT8S + 64 * j, tmem + kT8Q + 64 * j + 8 * ks, k + (uint32_t)((ks / 4) * (Sh::kBlock / 16) + 2 * (ks % 4)), idesc_s, ks != 0);
                if constexpr (kTerms == 2) {
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        tc_mma_bf16(tmem + kT8S + 64 * j, q + (uint32_t)((ks / 4) * (Sh::kQBlock / 16) + 2 * (ks % 4)), k + (uint32_t)((ks / 4) * (Sh::kBlock / 16) + 2 * (ks % 4)), idesc_s, 1);
                }
                tc_commit(sfull + j);
            };
            auto values = [&](int j, int g, bool more) {
                const uint64_t v = v_desc + (uint32_t)(g % ST) * (Sh::kTile / 16);
#pragma unroll
                for (int ks = 0; ks < kTerms * kT8Keys / 16; ++ks)       // first terms, then second ones, against the same values
                    tc_mma_bf16_ts(tmem + kT8O + 128 * j, tmem + kT8S + 64 * j + 8 * ks, v + (uint32_t)((ks % (kT8Keys / 16)) * 128), idesc_o, more || ks != 0);
                tc_commit(odone + j);
            };
            T8Walk w(p, *s_start, ctas, total);
            T8Item it;
            int g = 0;                           // key tiles so far; products and items of either tile
            uint32_t done[2] = {0, 0}, items[2] = {0, 0};
            bool ok = true;
            while (ok && w.next(it)) {
                const int n = it.k1 - it.k0, nkt[2] = {w.keys(it, 0), w.keys(it, 1)};
                ok = tc_wait(kfull + g % ST, (uint32_t)(g / ST) & 1, gave_up, p.polls);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (!ok || nkt[j] == 0) continue;
                    ok = tc_wait(qready + j, items[j]++ & 1, gave_up, p.polls);
                    // they land where the last weights of the item before lie
                    if (ok && done[j]) ok = tc_wait(odone + j, (done[j] - 1) & 1, gave_up, p.polls);
                    if (!ok) continue;
                    tc_fence_after();
                    scores(j, g);
                }
                if (!ok) break;
                tc_commit(kempty + g % ST);
                for (int kt = 0; kt < n; ++kt, ++g) {
                    ok = tc_wait(vfull + g % ST, (uint32_t)(g / ST) & 1, gave_up, p.polls);
                    bool keys = false;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (!ok || kt >= nkt[j]) continue;
                        ok = tc_wait(pready + j, done[j] & 1, gave_up, p.polls);
                        if (!ok) continue;
                        tc_fence_after();
                        values(j, g, kTerms == 1 ? kt != 0 : kt % kT8Flush != 0);
                        ++done[j];
                        if (kt + 1 >= nkt[j]) continue;
                        if (!keys) {
                            ok = tc_wait(kfull + (g + 1) % ST, (uint32_t)((g + 1) / ST) & 1, gave_up, p.polls);
                            keys = true;
                        }
                        // the next scores land where the weights lie that this product is still reading
                        ok = ok && tc_wait(odone + j, (done[j] - 1) & 1, gave_up, p.polls);
                        if (!ok) continue;
                        tc_fence_after();
                        scores(j, g + 1);
                    }
                    if (!ok) break;
                    tc_commit(vempty + g % ST);
                    if (kt + 1 < n) {
                        if (!keys) ok = tc_wait(kfull + (g + 1) % ST, (uint32_t)((g + 1) / ST) & 1, gave_up, p.polls);     // (nobody needed these keys; never so while a tile goes on)
                        tc_commit(kempty + (g + 1) % ST);
                    }
                }
            }
        }
    } else if (warp < 4) {   // ===== codes to fp16 =====
        T8Walk w(p, *s_start, ctas, total);
        T8Item it;
        int g = 0, item = 0;
        bool ok = true;
        const int me = (warp - 2) * 32 + lane, r8 = me & 7, c0 = me >> 3;       // row of eight, first chunk: neighbouring lanes' chunks lie in different banks, read and written
        constexpr int kChunks = HD / 16, kPer = 8 / kChunks;                    // chunks of a row; rows of eight that 64 threads take at a time: 1 or 2
        while (ok && w.next(it)) {
            ++item;
            const TileList tiles = w.tiles(it);
            const int last_pos = it.pos0 + it.hi;
            bool bad = false;
            for (int k = it.k0; k < it.k1; ++k, ++g) {
                const int s = g % RS, t = g % ST, key0 = tiles.tile_of(k) * kT8Keys;
                const uint32_t par = (uint32_t)(g / ST) & 1;
                ok = tc_wait_warp(rfull + s, (uint32_t)(g / RS) & 1, gave_up, p.polls) && tc_wait_warp(kempty + t, par ^ 1, gave_up, p.polls);
                if (!ok) break;
                auto convert = [&](const uint8_t* raw, uint8_t* tile, auto values_) {
                    constexpr bool values = decltype(values_)::value;
                    const uint32_t from = s_addr(raw), to = s_addr(tile);
                    bool there[2];                 // (keys without a page are hidden by the softmax, whatever they are)
                    if (values) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) there[x] = t8_row(a, it.slot, it.gkv, key0 + x * kKv8Block, last_pos) >= 0;
                    }
#pragma unroll
                    for (int r0 = 0; r0 < kT8Keys; r0 += 8 * kPer) {
                        const int row = r0 + r8 + 8 * (c0 / kChunks), chunk = c0 % kChunks;
                        uint4 v = t8_lds(from + row * HD + ((HD == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4));
                        if (values) {
                            const bool take = there[r0 + 8 * (c0 / kChunks) >= kKv8Block] && key0 + row <= last_pos;
                            uint32_t* y = &v.x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                y[e] = take ? y[e] : 0u;
                                const uint32_t n = ((y[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;       // the top bit of every NaN
                                if (n) {
                                    bad = true;
                                    y[e] &= ~((n >> 7) * 0xffu);
                                }
                            }
                        }
                        const uint32_t at = to + (chunk / 4) * Sh::kBlock + row * 128, c = (chunk % 4) * 2;
                        t8_sts(at + ((c ^ (row & 7)) << 4), kv8_half2(v.x & 0xffffu), kv8_half2(v.x >> 16), kv8_half2(v.y & 0xffffu), kv8_half2(v.y >> 16));
                        t8_sts(at + (((c + 1) ^ (row & 7)) << 4), kv8_half2(v.z & 0xffffu), kv8_half2(v.z >> 16), kv8_half2(v.w & 0xffffu), kv8_half2(v.w >> 16));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                };
                convert(sRaw + 2 * s * Sh::kCodes, sK + t * Sh::kTile, std::false_type{});
                if (lane == 0) mb_arrive(kfull + t);
                ok = tc_wait_warp(vempty + t, par ^ 1, gave_up, p.polls);
                if (!ok) break;
                convert(sRaw + (2 * s + 1) * Sh::kCodes, sV + t * Sh::kTile, std::true_type{});
                if (bad) s_nan[item & 7] = item;   // read behind the product with these values
                __threadfence_block();
                __syncwarp();
                if (lane == 0) { mb_arrive(vfull + t); mb_arrive(rempty + s); }
            }
        }
    } else if (warp >= 12) {   // ===== O of both tiles =====
        const int quad = warp & 3, row = quad * 32 + lane;
        T8Walk w(p, *s_start, ctas, total);
        T8Item it;
        uint32_t done[2] = {0, 0}, items[2] = {0, 0};
        int item = 0;
        uint32_t met = 0;
        bool ok = true;
        while (ok && w.next(it)) {
            ++item;
            const int n = it.k1 - it.k0, nkt[2] = {w.keys(it, 0), w.keys(it, 1)};
            const bool whole = it.k0 == 0 && it.k1 == it.n;
            const long long item0 = w.u - it.k1;                               // its first key tile in the row of all
            float* part = p.parts + (size_t)(2 * blockIdx.x + (w.begin >= item0 ? 0 : 1)) * kT8Part;
            float since[2] = {1.0f, 1.0f};                                     // what the references have grown by since O was flushed
            for (int kt = 0; ok && kt < n; ++kt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (!ok || kt >= nkt[j]) continue;
                    ok = tc_wait_warp(factors + j, done[j] & 1, gave_up, p.polls);
                    if (ok && kt > 0) ok = tc_wait_warp(odone + j, (done[j] - 1) & 1, gave_up, p.polls);     // long since: the scores follow that product
                    if (!ok) continue;
                    ++done[j];
                    tc_fence_after();
                    const float f = factor[j * kT8Rows + row];
                    const uint32_t o_tmem = tmem + ((uint32_t)(quad * 32) << 16) + kT8O + 128 * j;
                    if (kTerms == 2 && kt > 0 && kt % kT8Flush == 0) {         // O so far, relative to the reference before this tile's
                        uint4* acc = reinterpret_cast<uint4*>(part + j * kT8PartTile);
                        const float s = kt > kT8Flush ? since[j] : 0.0f;
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
                        since[j] = f;
                    } else {
                        since[j] *= f;
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
                    tc_fence_before();
                    mb_arrive(pready + j);
                }
            if (!ok) break;
            // ---- results, or this CTA's part of them ----
            const bool nan_here = s_nan[item & 7] == item;
            auto query = [&](int j, int& q) {                                  // this row's query, and whether it is listed
                q = j * p.queries + (row >> p.hpc_log2);
                uint32_t m = 0;
#pragma unroll
                for (int x = 0; x < 8; ++x) m = q / 32 == x ? it.m[x] : m;
                return (m >> (q & 31) & 1) != 0;
            };
            // columns c .. c + 31 of this row: o * inv; `hit`: columns that a NaN value reaches
            auto store = [&](int j, int c, const float (&o)[32], float inv, const uint32_t (&hit)[4]) {
                int q;
                if (!query(j, q) || c >= a.dv) return;
                const size_t t = it.tok0 + q;
                const int h = it.h0 + (row & (p.hpc - 1)), cols = min(32, a.dv - c);
                float y[32];
                uint32_t hits = 0;
#pragma unroll
                for (int x = 0; x < 4; ++x) hits = c / 32 == x ? hit[x] : hits;
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = hits >> i & 1 ? __int_as_float(0x7fffffff) : o[i] * inv;
                if (a.out) {
                    float* dst = a.out + t * a.ldo + (size_t)h * a.dv + c;
                    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (i < cols) *reinterpret_cast<float4*>(dst + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < cols) dst[i] = y[i];
                    }
                }
                if (a.out16) {
                    uint16_t* dst = a.out16 + (t * a.heads + h) * a.dv + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        if (i < cols) {
                            if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
                                *reinterpret_cast<uint4*>(dst + i) = make_uint4(tc_pack(y[i], y[i + 1]), tc_pack(y[i + 2], y[i + 3]), tc_pack(y[i + 4], y[i + 5]), tc_pack(y[i + 6], y[i + 7]));
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e) dst[i + e] = f32_to_bf16_bits(y[i + e]);
                            }
                        }
                }
            };
            // the columns in which a value that this row sees is NaN (rare: a walk over all its keys)
            auto search = [&](int j, uint32_t (&hit)[4]) {
                int q;
                if (!query(j, q)) return;
                const int pos = it.pos0 + q, wnd = seq_row_window(pos, a.window, a.chunk);
                const TileList mine(pos, pos, wnd, a.keep_first, kKv8Block);
                for (int x = 0; x < mine.n; ++x) {
                    const int key0 = mine.tile_of(x) * kKv8Block, r = t8_row(a, it.slot, it.gkv, key0, pos);
                    if (r < 0) continue;
                    for (int e = 0; e < kKv8Block; ++e) {
                        if (!seq_sees(pos, key0 + e, wnd, a.keep_first)) continue;
                        const uint32_t* v = reinterpret_cast<const uint32_t*>(a.v_pool + (size_t)(r + e) * a.dv);
                        for (int c = 0; c < a.dv / 4; ++c) {
                            const uint32_t m = ((v[c] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                            if (m) {
                                const uint32_t bits = (m >> 7 & 1) | (m >> 14 & 2) | (m >> 21 & 4) | (m >> 28 & 8);
#pragma unroll
                                for (int y = 0; y < 4; ++y)
                                    if (c / 8 == y) hit[y] |= bits << (4 * (c % 8));
                            }
                        }
                    }
                }
            };
#pragma unroll 1
            for (int j = 0; ok && j < 2; ++j) {
                if (nkt[j] == 0) {
                    if (!whole) {                                              // none of this part's keys is visible to this tile
                        part[j * kT8PartTile + 128 * kT8Rows + row] = -INFINITY;
                        part[j * kT8PartTile + 129 * kT8Rows + row] = 0.0f;
                    }
                    continue;
                }
                ok = tc_wait_warp(lready + j, items[j]++ & 1, gave_up, p.polls) && tc_wait_warp(odone + j, (done[j] - 1) & 1, gave_up, p.polls);
                if (!ok) break;
                tc_fence_after();
                const float ref = s_ref[j * kT8Rows + row], l = s_sum[j * kT8Rows + row], inv = l == 0.0f ? 0.0f : 1.0f / l;
                mb_arrive(lread + j);
                uint32_t hit[4] = {0u, 0u, 0u, 0u};
                if (whole && nan_here) search(j, hit);
                const uint32_t o_tmem = tmem + ((uint32_t)(quad * 32) << 16) + kT8O + 128 * j;
                uint4* acc = reinterpret_cast<uint4*>(part + j * kT8PartTile);
                const bool flushed = kTerms == 2 && nkt[j] > kT8Flush;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tc_ld32_async(o_tmem + c, o);
                    float y[32];
                    if (flushed) {
                        uint4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = acc[(c / 4 + i) * kT8Rows + row];
                        tc_arrived(o);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float s = since[j];
                            y[4 * i] = fmaf(__uint_as_float(v[i].x), s, __uint_as_float(o[4 * i])); y[4 * i + 1] = fmaf(__uint_as_float(v[i].y), s, __uint_as_float(o[4 * i + 1]));
                            y[4 * i + 2] = fmaf(__uint_as_float(v[i].z), s, __uint_as_float(o[4 * i + 2])); y[4 * i + 3] = fmaf(__uint_as_float(v[i].w), s, __uint_as_float(o[4 * i + 3]));
                        }
                    } else {
                        tc_arrived(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]);
                    }
                    if (whole) {
                        store(j, c, y, inv, hit);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) acc[(c / 4 + i) * kT8Rows + row] = make_uint4(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]), __float_as_uint(y[4 * i + 2]), __float_as_uint(y[4 * i + 3]));
                    }
                    __syncwarp();
                }
                if (!whole) {
                    part[j * kT8PartTile + 128 * kT8Rows + row] = ref;
                    part[j * kT8PartTile + 129 * kT8Rows + row] = nan_here ? -l : l;      // (sums are not negative: the sign says that there was NaN)
                }
            }
            if (!ok) break;
            tc_fence_before();
            if (!whole) {
                const int c_first = w.owner(item0), parts = w.owner(item0 + it.n - 1) - c_first + 1;
                auto together = [&]() {              // these four warps; a wait like the others, which ends
                    mb_arrive(meet);
                    ok = tc_wait_warp(meet, met++ & 1, gave_up, p.polls);
                    return ok;
                };
                if (!together()) break;
                if (threadIdx.x == 12 * 32) {        // what these warps have stored before the barrier comes before this, and what others have stored before theirs, before what follows
                    int before_me;
                    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before_me) : "l"(p.counters + c_first) : "memory");
                    *s_last = before_me == parts - 1;
                    if (before_me == parts - 1) p.counters[c_first] = 0;
                }
                if (!together()) break;
                if (*s_last) {                       // all parts are there: in the order of the key tiles, whoever was last
                    __threadfence();
                    const int later = w.share(c_first) < item0;
                    auto from = [&](int x, int j) { return p.parts + (size_t)(2 * (c_first + x) + (x == 0 ? later : 0)) * kT8Part + j * kT8PartTile; };
#pragma unroll 1
                    for (int j = 0; j < 2; ++j) {
                        int q;
                        float top = -INFINITY, l = 0.0f;
                        bool wild = false;
                        for (int x = 0; x < parts; ++x) top = fmaxf(top, __ldcg(from(x, j) + 128 * kT8Rows + row));
                        for (int x = 0; x < parts; ++x) {
                            const float r = __ldcg(from(x, j) + 128 * kT8Rows + row), s = __ldcg(from(x, j) + 129 * kT8Rows + row);
                            wild |= __float_as_uint(s) >> 31;
                            l += fabsf(s) * (r == top ? 1.0f : tc_exp2(r - top));
                        }
                        uint32_t hit[4] = {0u, 0u, 0u, 0u};
                        if (__any_sync(0xffffffffu, wild)) search(j, hit);
                        if (!query(j, q)) continue;
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float y[32] = {};
#pragma unroll 2
                            for (int x = 0; x < parts; ++x) {
                                const float r = __ldcg(from(x, j) + 128 * kT8Rows + row);
                                const bool none = r == -INFINITY && __ldcg(from(x, j) + 129 * kT8Rows + row) == 0.0f;       // its O may never have been written
                                if (none) continue;
                                const float f = r == top ? 1.0f : tc_exp2(r - top);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float4 v = __ldcg(reinterpret_cast<const float4*>(from(x, j)) + (c / 4 + i) * kT8Rows + row);
                                    y[4 * i] = fmaf(v.x, f, y[4 * i]); y[4 * i + 1] = fmaf(v.y, f, y[4 * i + 1]); y[4 * i + 2] = fmaf(v.z, f, y[4 * i + 2]); y[4 * i + 3] = fmaf(v.w, f, y[4 * i + 3]);
                                }
                            }
                            store(j, c, y, inv, hit);
                        }
                    }
                }
                if (!together()) break;              // s_last has been read
            }
        }
    } else {   // ===== softmax: TMEM lane quadrant = warp % 4 =====
        const int j = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16, s_tmem = tmem + lanes + kT8S + 64 * j, q_tmem = tmem + lanes + kT8Q + 64 * j;
        const int q = j * p.queries + (row >> p.hpc_log2);
        T8Walk w(p, *s_start, ctas, total);
        T8Item it;
        uint32_t done = 0, items = 0;
        bool ok = true;
        while (ok && w.next(it)) {
            const int n = w.keys(it, j);
            if (n == 0) continue;
            uint32_t m = 0;
#pragma unroll
            for (int x = 0; x < 8; ++x) m = q / 32 == x ? it.m[x] : m;
            const bool live = m >> (q & 31) & 1;
            const int qpos = it.pos0 + (live ? q : it.hi), h = it.h0 + (row & (p.hpc - 1)), last_pos = it.pos0 + it.hi;
            const TileList tiles = w.tiles(it);
            // ---- queries: fp16 in TMEM, brought to 1 .. 2 by a power of two of the row's largest; every score of the item before has been read ----
            float up;
            {
                const float* src = a.q + (size_t)(it.tok0 + (live ? q : it.hi)) * a.ldq + (size_t)h * a.dk;
                float top = 0.0f;
                auto load = [&](int c, float (&x)[32]) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const bool take = c + i < a.dk;
                        if (p.vec_q) {
                            const float4 v = take ? *reinterpret_cast<const float4*>(src + c + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[i + e] = take ? src[c + i + e] : 0.0f;
                        }
                    }
                };
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float x[32];
                    load(c, x);
#pragma unroll
                    for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(x[i]));
                }
                const int ex = top < INFINITY ? max((int)(__float_as_uint(top) >> 23) - 127, -100) : 0;
                const float down = kv8_pow2(-ex);
                up = kv8_pow2(ex);
                if (items) tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float x[32];
                    uint32_t hi[16];
                    load(c, x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        x[2 * i] *= down;
                        x[2 * i + 1] *= down;
                        hi[i] = t8_pack(x[2 * i], x[2 * i + 1]);
                    }
                    tc_st16(q_tmem + c / 2, hi);
                    if constexpr (kTerms == 2) {
                        uint32_t lo[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 y = t8_unpack(hi[i]);
                            lo[i] = t8_pack(x[2 * i] - y.x, x[2 * i + 1] - y.y);
                        }
                        const uint32_t at = s_addr(sQ) + j * Sh::kQTile + (c / 64) * Sh::kQBlock + row * 128;
#pragma unroll
                        for (int i = 0; i < 4; ++i) t8_sts(at + (((c % 64 / 8 + i) ^ (row & 7)) << 4), lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
                    }
                }
                tc_wait_st();
                if constexpr (kTerms == 2) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                mb_arrive(qready + j);
            }
            const int wnd = seq_row_window(qpos, a.window, a.chunk);
            const float slope = kOpts && a.slopes ? a.slopes[h] : 0.0f, mul = a.scale * up * (kOpts ? 1.0f : 1.4426950408889634f);
            float ref = -INFINITY, l = 0.0f;
            // scales of the next tile's blocks, asked for a tile ahead
            int rows[2];
            float ks[2], vs[2];
            auto look_up = [&](int k) {
                const int key0 = tiles.tile_of(k) * kT8Keys;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    rows[x] = t8_row(a, it.slot, it.gkv, key0 + x * kKv8Block, last_pos);
                    ks[x] = rows[x] >= 0 ? a.k_scale[rows[x] / kKv8Block] : 1.0f;
                    vs[x] = rows[x] >= 0 ? a.v_scale[rows[x] / kKv8Block] : 1.0f;
                }
            };
            look_up(it.k0);
            for (int kt = 0; kt < n; ++kt) {
                const int key0 = tiles.tile_of(it.k0 + kt) * kT8Keys;
                const bool gone[2] = {rows[0] < 0, rows[1] < 0};
                const float f0[2] = {ks[0] * mul, ks[1] * mul}, v0[2] = {vs[0], vs[1]};
                if (kt + 1 < n) look_up(it.k0 + kt + 1);
                ok = tc_wait_warp(sfull + j, done & 1, gave_up, p.polls);
                if (!ok) break;
                ++done;
                tc_fence_after();
                uint32_t s[64];
                tc_ld32_async(s_tmem, s);
                tc_ld32_async(s_tmem + 32, s + 32);
                float ev[2] = {t8_log2(v0[0]), t8_log2(v0[1])};
                // every key of the tile is visible to every row of the warp
                const bool all = __all_sync(0xffffffffu, !gone[0] && !gone[1] && key0 + kT8Keys - 1 <= qpos && (qpos - key0 < wnd || key0 + kT8Keys <= a.keep_first));
                tc_arrived(s);
                tc_arrived(s + 32);
                float f[2] = {f0[0], f0[1]};
                if (kOpts) {
                    const float dist = (float)(qpos - key0), inv = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
#pragma unroll
                    for (int e = 0; e < 64; ++e) {
                        float v = __uint_as_float(s[e]) * f0[e / 32];
                        if (a.softcap > 0.0f) v = a.softcap * tanhf(v * inv);
                        v = fmaf(-slope, dist - (float)e, v);
                        s[e] = __float_as_uint(v);
                    }
                    f[0] = f[1] = 1.4426950408889634f;
                }
                auto step = [&](auto masked) {
                    constexpr bool kMasked = decltype(masked)::value;
                    if (kMasked) {
                        const int hi = qpos - key0, lo = wnd > qpos ? INT_MIN : qpos - wnd - key0, keep = a.keep_first - key0;
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (e > hi || (e <= lo && e >= keep) || gone[e / 32]) s[e] = 0xff800000u;       // -inf
                    }
                    float top[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            m0 = tc_max3(m0, __uint_as_float(s[32 * x + e]), __uint_as_float(s[32 * x + e + 1]));
                            m1 = tc_max3(m1, __uint_as_float(s[32 * x + e + 2]), __uint_as_float(s[32 * x + e + 3]));
                        }
                        top[x] = fmaxf(m0, m1);
                    }
                    float mx = fmaxf(fmaf(top[0], f[0], ev[0]), fmaf(top[1], f[1], ev[1]));
                    // Scores so large that a rounded product and one inside a multiply-add are far apart: every product is rounded, so that no weight is above 1
                    if (__any_sync(0xffffffffu, fabsf(mx) > 65536.0f && mx != -INFINITY)) {
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * f[e / 32]);
                        mx = fmaxf(__fadd_rn(__fmul_rn(top[0], f[0]), ev[0]), __fadd_rn(__fmul_rn(top[1], f[1]), ev[1]));
                        top[0] *= f[0];
                        top[1] *= f[1];
                        f[0] = f[1] = 1.0f;
                    }
                    const float nr = fmaxf(ref, ceilf(mx)), less = kt == 0 || nr == ref ? 1.0f : tc_exp2(ref - nr);
                    factor[j * kT8Rows + row] = less;
                    mb_arrive(factors + j);
                    l = kt == 0 ? 0.0f : l * less;
                    ref = nr;
                    // where every score so far is -inf, -inf - ref were no number: relative to 0 their weights are 0
                    const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        // A block whose weights come out below 2^-60 because its value scale is that much smaller than others': nothing to O, but the denominator has its weights without the
                        // scale. They are taken 2^far larger, so that they do not vanish.
                        const float most = fmaf(top[x], f[x], ev[x]) - base, far = most < -60.0f && most > -1e6f ? floorf(-most) : 0.0f;
                        const float neg = ev[x] - base + far;
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
                            if constexpr (kTerms == 2) {
                                const float2 u = t8_unpack(hi[e]);
                                lo[e] = t8_pack(y - u.x, z - u.y);
                            }
                        }
                        if (__any_sync(0xffffffffu, far != 0.0f)) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                hi[e] = far != 0.0f ? 0u : hi[e];
                                if constexpr (kTerms == 2) lo[e] = far != 0.0f ? 0u : lo[e];
                            }
                        }
                        tc_st16(s_tmem + 16 * x, hi);
                        if constexpr (kTerms == 2) tc_st16(s_tmem + 32 + 16 * x, lo);
                        float s0, s1;
                        tc_split(sum, s0, s1);
                        l = fmaf(s0 + s1, tc_exp2(-ev[x] - far), l);         // without the value scale
                    }
                };
                if (all) step(std::false_type{});
                else step(std::true_type{});
                tc_wait_st();
                tc_fence_before();
                mb_arrive(pready + j);
            }
            if (!ok) break;
            if (items) ok = tc_wait_warp(lread + j, (items - 1) & 1, gave_up, p.polls);
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

template <int HD, int kTerms, bool kOpts>
static int t8_launch(const T8Args& a, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
    using Sh = T8Shape<HD, kTerms>;
    auto* kernel = seq_attention8_tc_kernel<HD, kTerms, kOpts>;
    static bool ready = false;
    if (!ready) {
        SLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
        ready = true;
    }
    overlapping(kernel)<<<std::min(kA8TcWorkers, sm_count()), kT8Threads, Sh::kSmem, st>>>(tmK, tmV, a);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

static int t8_hpc(const Attn8Args& p) {
    const int group = p.heads / p.kv_heads;
    return group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
}

bool attention8_tc_takes(const Attn8Args& p) {
    const int width = 2 * kT8Rows / t8_hpc(p);
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
    A8Plan* plan = reinterpret_cast<A8Plan*>((uint8_t*)ws + kA8PlanAt);
    a.plan = plan;
    a.counters = (int*)ws + kA8Workers;
    a.parts = (float*)((uint8_t*)ws + kA8PartsAt);
    if (int rc = status_word(&a.status)) return rc;
    a.polls = (unsigned)g_tune_tc_polls;
    const int HD = std::max(p.dk, p.dv) <= 64 ? 64 : 128;
    CUtensorMap tmK, tmV;
    const uint64_t rows = (uint64_t)p.n_pages * p.kv_heads * p.b.page_len;
    if (int rc = tc_encode_bytes(&tmK, p.k_pool, rows, p.dk, kKv8Block, HD)) return rc;
    if (int rc = tc_encode_bytes(&tmV, p.v_pool, rows, p.dv, kKv8Block, HD)) return rc;
    overlapping(seq_attention8_plan_kernel)<<<1, 1024, 0, st>>>(p, 2 * a.queries, plan);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    const bool opts = p.softcap > 0.0f || p.slopes;
#define SLLM_T8(HD_)                                                                                                                            \
    (p.out ? (opts ? t8_launch<HD_, 2, true>(a, tmK, tmV, st) : t8_launch<HD_, 2, false>(a, tmK, tmV, st))                                        \
           : (opts ? t8_launch<HD_, 1, true>(a, tmK, tmV, st) : t8_launch<HD_, 1, false>(a, tmK, tmV, st)))
    return HD == 128 ? SLLM_T8(128) : SLLM_T8(64);
#undef SLLM_T8
}

}  // namespace sllm
