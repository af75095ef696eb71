// csrc/seq_attn_shared_tc.cu — attention behind shared first positions over bf16 pools, heads of 64 or 128 columns.
//
// One launch, two kinds of CTAs. Where many rows see the same keys (the shared positions of a group, a portion's own positions) a CTA is a tile of 128 rows = the query heads of a kv head x
// neighbouring tokens, on tcgen05, against a share of the keys, 48 at a time (so that TMEM, of which two CTAs of an SM have half each, holds a tile's scores, its weights and O: the next scores are
// made while these are worked on, and their products while the next are):
//   warps 0-3  softmax, a thread per row: queries to bf16 rows in shared memory; per key tile the scores from TMEM, capped, charged and masked, fp32 maximum and sum; the weights go back to TMEM as
//              THREE bf16 terms (24 bits; two leave 2^-18 of a weight, which is more than all the rest). O stays in TMEM, rescaled only where a maximum has grown by more than 2^8; the
//              tensor core truncates as it adds, so every kStFlush tiles O moves on to the CTA's own place in the workspace, [columns / 4][rows] so that whole lines are read and written
//              (moves of 16 bytes of a row a lane, to the rows' records, with the tiles of 64 keys that were there before: the mixed step 290 us instead of 223). Between two moves 6 | 9 | 12 | 18
//              tiles: results of the mixed step 6.5e-7 | 9.0e-7 | 1.15e-6 | 1.6e-6 off (without moves 2.6e-6; the plain form in fp32 1.16e-6), 211 | 206 | 200 | 194 us;
//   warp 4     (one lane) TMA producer: boxes of 16 positions, looked up in the block table; what is behind the last position or in no page reads as zeros;
//   warp 5     (one lane) MMA issuer: S = Q K^T, O += (hi + mid + lo) V with the weights read from TMEM, V as it lies;
//   warps 6-7  zero the value rows that are not part of the share, and take infinities and NaN out of the values (0 * NaN is NaN for rows that do not see them, and the terms of a weight times
//              infinity are NaN for those that do); rows that see them get them back at the end.
// Bound of this kind: 148 SMs take a key tile of 128 rows in 1400 clocks each (2100 with a cap). Its products are 800 of them and the rest of the softmax's instructions that two CTAs cannot hide;
// an item begins with 6000 (its queries) and ends with 7500 (64 KB of records a CTA, all CTAs at once), the step's plan is 4000 to 6000 for eight answers and 5600 to 8400 for the mixed step.
// 512 rows of 32 heads behind 4000 positions 111 us (71 GFLOP with the weights' terms: 0.64 PFLOP/s). All 128 registers of a thread are in use, and 40 to 64 bytes a
// thread spilled (84 for heads of 128 with caps or charges). Tiles of 64 keys, scores and weights one over the other, took 128 us, and then one CTA an SM with two such tiles, or two threads a row, no
// less.
// Where a segment has few rows of its own (a decoding request: the query heads of one token), four warps take 16 keys in turn on mma.sync, 8 rows at a time as the columns: such work is bound by what
// it reads, and a tile of 128 rows would be empty but for four. A CTA does two items at once, since one is a chain (queries, pages, keys and values, maximum, sums, four parts put together), and the
// next keys and values are on their way to shared memory meanwhile. The columns of a head are contracted in an order of the kernel's own, 16 bytes a lane, and those of the values are dealt to the
// tiles of O so that a lane's eight neighbours are rows of four of them. 64 tokens with 200 positions each of their own 28 us, with 400 40 (4.2 TB/s between the two).
#include "seq_attn_shared.cuh"
#include "tcgen05.cuh"

namespace sllm {

constexpr int kStRows = 128, kStKeys = 48, kStThreads = 256, kStBox = 16, kStBoxes = kStKeys / kStBox, kStWarps = kStThreads / 32;
constexpr int kStFlush = 9, kStEnds = 10;
constexpr uint32_t kStTmem = 256, kStTerms = 48;       // scores at 0 .. 47, the weights' terms at 48, 72 and 96, O at 128; two CTAs share an SM's 512 columns
constexpr int kStFew = 16, kStTeam = 4, kStTeams = kStWarps / kStTeam;      // rows of a segment up to which its own positions are a team's work; warps of a team
constexpr float kStLog2e = 1.4426950408889634f;

template <int HD>
struct StShape {
    static constexpr int kBlocks = HD / 64, kQBlock = kStRows * 128, kQBytes = kBlocks * kQBlock, kKBlock = kStKeys * 128, kTile = kBlocks * kKBlock;
    static constexpr int kKeyStages = HD == 128 ? 2 : 4, kValueStages = HD == 128 ? 3 : 4;      // tiles of keys and of values on their way or in use
    static constexpr int kBars = kQBytes + (kKeyStages + kValueStages) * kTile, kPlan = kBars + 512, kSmem = 1024 + kPlan + 11 * 1024;
};

// The step's work as a CTA sees it: entries (groups, then listed tiles of queries), as many at a time as it has threads, and how many items each and those before it are.
constexpr int kStEntries = kStThreads;
struct StPlan {
    int tok0[kStEntries], n[kStEntries], slot[kStEntries], from[kStEntries], end[kStEntries], cuts[kStEntries], tiles[kStEntries], upto[kStEntries];
    int low[kStEntries], high[kStEntries];       // positions of a group's listed tokens
    int warp[kStWarps];
    int least, total;
};
static_assert(sizeof(StPlan) <= 11 * 1024, "its place");

struct StArgs {
    SharedArgs a;
    int hpc, sets, queries;                  // query heads of a tile, tiles' head sets of a kv head, tokens of a tile
    uint32_t hpc_magic;                      // ceil(2^16 / hpc): row / hpc is (row * hpc_magic) >> 16 for the rows of a tile
    int vec_q;
    int32_t* status;
    unsigned polls;
};

// What a CTA does.
struct StItem {
    int tok0, nq, slot, g, h0;               // rows: nq tokens from tok0 on x hpc heads from h0 on, of kv head g
    int pos0;                                // position of the first token where the others follow it, -1: their positions are looked up
    int key0, key1, which;                   // keys, and the record that takes the result
    int low, high;                           // no token of the rows lies before the one or behind the other position
};

__device__ __forceinline__ int st_token(const StArgs& sa, int row) { return (int)((uint32_t)row * sa.hpc_magic >> 16); }
__device__ __forceinline__ int st_pos(const StArgs& sa, const StItem& it, int token) { return it.pos0 >= 0 ? it.pos0 + token : sa.a.b.tok_pos[it.tok0 + token]; }

// columns of TMEM from registers and to registers; complete behind tc_wait_st and tc_wait_ld
__device__ __forceinline__ void st_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void st_ld16_async(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void st_ld16(uint32_t taddr, uint32_t* o) {
    st_ld16_async(taddr, o);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) asm volatile("" : "+r"(o[e]));
}
// Two bf16 values times zero, added up: zero as long as all were numbers, NaN where one was infinite or NaN.
__device__ __forceinline__ void st_times_zero(uint32_t& sum, uint32_t x) { asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u)); }
__device__ __forceinline__ void st_times_zero(uint32_t& sum, const uint4& v) {
    st_times_zero(sum, v.x);
    st_times_zero(sum, v.y);
    st_times_zero(sum, v.z);
    st_times_zero(sum, v.w);
}
__device__ __forceinline__ bool st_odd(uint32_t sum) { return (sum & 0x7fff7fffu) != 0; }
__device__ __forceinline__ uint32_t st_without(uint32_t x) {            // the pair with those replaced by zero
    return ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u) | ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu);
}
__device__ __forceinline__ uint4 st_without(const uint4& v) { return make_uint4(st_without(v.x), st_without(v.y), st_without(v.z), st_without(v.w)); }

// ---- few rows: four warps -------------------------------------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t st_turned(uint32_t x) {              // 8 x 8 values of 16 bits, transposed over the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int HD>
__device__ __forceinline__ void st_few(const StArgs& sa, const StItem& it, uint8_t* smem) {
    const SharedArgs& p = sa.a;
    constexpr int kSteps = HD / 32, kHalves = HD / 64, kTiles = HD / 16, kStage = 64 * HD;       // bytes of a warp: 16 keys, 16 values
    const int team = threadIdx.x / (32 * kStTeam), warp = threadIdx.x / 32 % kStTeam, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, n_rows = it.nq * sa.hpc;
    auto together = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(3 + team) : "memory"); };
    auto area = [&](int w) { return smem + (team * kStTeam + w) * kStage; };
    // what a lane copies it reads itself, 16 bytes beside its neighbours' 16 bytes
    uint8_t *k_stage = area(warp) + lane * 16, *v_stage = k_stage + kStage / 2;
    const uint16_t *kp = reinterpret_cast<const uint16_t*>(p.k_pool), *vp = reinterpret_cast<const uint16_t*>(p.v_pool);
    for (int r0 = 0; r0 < n_rows; r0 += 8) {
        // columns of the products: rows r0 .. r0 + 7. As an operand a lane has row g, as a result rows 2t and 2t + 1
        int pos[2];
        float slope[2], m[2] = {-INFINITY, -INFINITY}, l[4] = {}, o[kTiles][4] = {};      // l: of rows 2t, 2t + 1, twice
        bool infinite = false;               // a value so far was no number
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 2 * t + i, qi = st_token(sa, r);
            pos[i] = r < n_rows ? st_pos(sa, it, qi) : -1;
            slope[i] = p.slopes && r < n_rows ? p.slopes[it.h0 + r - qi * sa.hpc] * kStLog2e : 0.0f;
        }
        // the keys that any of the rows sees: up to the last position, and from the oldest of a window
        int last = max(pos[0], pos[1]), least = min(pos[0] < 0 ? INT_MAX : pos[0], pos[1] < 0 ? INT_MAX : pos[1]);
#pragma unroll
        for (int w = 1; w < 4; w *= 2) {
            last = max(last, __shfl_xor_sync(0xffffffffu, last, w));
            least = min(least, __shfl_xor_sync(0xffffffffu, least, w));
        }
        const int end = min(it.key1, last + 1), oldest = p.window > least ? 0 : least - p.window + 1;
        auto mine = [&](int key) { return key >= it.key0 && key < end; };
        if (r0 > 0) together();              // the rows before these have been read
        // the warp's next sixteen keys that there are, and their page
        int page = -1, in_page = 0;
        auto next = [&](int j) {
            for (; j < end; j += 16 * kStTeam) {
                if (j + 16 <= oldest && j >= p.keep_first) continue;
                page = sh_page(p, it.slot, j, in_page);              // (pages are a multiple of 32 positions)
                if (page >= 0) break;
            }
            return j;
        };
        // All sixteen rows are the page's, whatever part of them is the share's: scores of the others are replaced, their values taken out below.
        auto fetch_keys = [&](bool there) {
            if (there) {
                const uint16_t* kr = kp + seq_pool_row(page, p.kv_heads, it.g, p.b.page_len, in_page, HD) + g * HD + 8 * t;
#pragma unroll
                for (int i = 0; i < 2 * kSteps; ++i) cp_async16(k_stage + i * 512, kr + (i & 1) * 8 * HD + 32 * (i >> 1), 16);
            }
            cp_async_commit();
        };
        auto value_row = [&](int pg, int in) { return vp + seq_pool_row(pg, p.kv_heads, it.g, p.b.page_len, in, HD) + 8 * g; };
        auto fetch_values = [&](bool there) {
            if (there) {
                const uint16_t* vr = value_row(page, in_page) + 2 * t * HD;
#pragma unroll
                for (int i = 0; i < 4 * kHalves; ++i) cp_async16(v_stage + i * 512, vr + ((i & 1) + 8 * ((i >> 1) & 1)) * HD + 64 * (i >> 2), 16);
            }
            cp_async_commit();
        };
        int j0 = next(it.key0 / 16 * 16 + 16 * warp);
        fetch_keys(j0 < end);
        fetch_values(j0 < end);
        uint32_t q[kSteps][4];
        {
            const int r = min(r0 + g, n_rows - 1), qi = st_token(sa, r);
            const float* src = p.q + (size_t)(it.tok0 + qi) * p.ldq + (size_t)(it.h0 + r - qi * sa.hpc) * HD + 8 * t;
            if (sa.vec_q) {
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const float4 a = *reinterpret_cast<const float4*>(src + 32 * s), b = *reinterpret_cast<const float4*>(src + 32 * s + 4);
                    q[s][0] = pack_bf16(a.x, a.y); q[s][1] = pack_bf16(a.z, a.w); q[s][2] = pack_bf16(b.x, b.y); q[s][3] = pack_bf16(b.z, b.w);
                }
            } else {
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[s][e] = pack_bf16(src[32 * s + 2 * e], src[32 * s + 2 * e + 1]);
            }
        }
        while (j0 < end) {
            const int at_page = page, at_in = in_page, j1 = next(j0 + 16 * kStTeam);
            cp_async_wait<1>();              // the keys, not the values
            float s[4] = {};                 // (key g, rows 2t and 2t + 1), (key g + 8, the same)
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const uint4 k0 = *reinterpret_cast<const uint4*>(k_stage + (2 * e) * 512), k1 = *reinterpret_cast<const uint4*>(k_stage + (2 * e + 1) * 512);
                const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
                mma_bf16_16816(s, a0, q[e][0], q[e][1]);
                mma_bf16_16816(s, a1, q[e][2], q[e][3]);
            }
            fetch_keys(j1 < end);
            float top[2] = {m[0], m[1]};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = j0 + g + 8 * (i >> 1), row = i & 1;
                float x = s[i] * p.scale;
                if (p.softcap > 0.0f) x = p.softcap * tc_tanh(x / p.softcap);
                s[i] = mine(key) && seq_sees(pos[row], key, p.window, p.keep_first) ? fmaf(-slope[row], (float)(pos[row] - key), x * kStLog2e) : -INFINITY;
                top[row] = fmaxf(top[row], s[i]);
            }
#pragma unroll
            for (int w = 4; w < 32; w *= 2) {
                top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], w));
                top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], w));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
                const float f0 = top[0] == m[0] ? 1.0f : tc_exp2(m[0] - top[0]), f1 = top[1] == m[1] ? 1.0f : tc_exp2(m[1] - top[1]);
                l[0] *= f0; l[1] *= f1; l[2] *= f0; l[3] *= f1;
                if (!infinite) {
#pragma unroll
                    for (int c = 0; c < kTiles; ++c) { o[c][0] *= f0; o[c][1] *= f1; o[c][2] *= f0; o[c][3] *= f1; }
                } else {
#pragma unroll
                    for (int c = 0; c < kTiles; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[c][i] = sh_carried(o[c][i], i & 1 ? f1 : f0);
                }
                m[0] = top[0];
                m[1] = top[1];
            }
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = s[i] == -INFINITY ? 0.0f : tc_exp2(s[i] - m[i & 1]);
            uint32_t b[3][2];
            split3_bf16(w[0], w[1], b[0][0], b[1][0], b[2][0]);
            split3_bf16(w[2], w[3], b[0][1], b[1][1], b[2][1]);
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int i = 0; i < 2; ++i) b[x][i] = st_turned(b[x][i]);
            {       // the weights' sum by the products that O comes from, so that it is truncated like it
                const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                for (int x = 0; x < 3; ++x) mma_bf16_16816(l, ones, b[x][0], b[x][1]);
            }
            cp_async_wait<1>();              // the values, not the next keys
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                uint4 v[4];
                uint32_t odd = 0;            // a value that is no number goes by itself to the rows that see its key
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(v_stage + (4 * h + i) * 512);
                if (j0 < it.key0 || j0 + 16 > end) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!mine(j0 + 2 * t + (i & 1) + 8 * (i >> 1))) v[i] = make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) st_times_zero(odd, v[i]);
                if (__any_sync(0xffffffffu, st_odd(odd))) {
                    infinite = true;
                    const uint16_t* vr = value_row(at_page, at_in);
#pragma unroll 1
                    for (int key = 0; key < 16; ++key) {
                        if (!mine(j0 + key)) continue;
                        const bool s0 = seq_sees(pos[0], j0 + key, p.window, p.keep_first), s1 = seq_sees(pos[1], j0 + key, p.window, p.keep_first);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {      // columns 64 h + 8 g + 2 c + i, rows 2t and 2t + 1
                                const float x = seq_ld(vr + key * HD, 64 * h + 2 * c + i);
                                if (fabsf(x) <= FLT_MAX) continue;
                                if (s0) o[4 * h + c][2 * i] += x;
                                if (s1) o[4 * h + c][2 * i + 1] += x;
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = st_without(v[i]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    auto word = [&](int i) { return e == 0 ? v[i].x : e == 1 ? v[i].y : e == 2 ? v[i].z : v[i].w; };
                    const uint32_t a[4] = {__byte_perm(word(0), word(1), 0x5410), __byte_perm(word(0), word(1), 0x7632), __byte_perm(word(2), word(3), 0x5410), __byte_perm(word(2), word(3), 0x7632)};
#pragma unroll
                    for (int x = 0; x < 3; ++x) mma_bf16_16816(o[4 * h + e], a, b[x][0], b[x][1]);
                }
            }
            fetch_values(j1 < end);
            j0 = j1;
        }
        cp_async_wait<0>();
        // the warps' parts, each in its own area: [row][columns], then references and sums
        __syncwarp();
        float* part = reinterpret_cast<float*>(area(warp));
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(part + (2 * t + i) * HD + 64 * (c / 4) + 8 * g + 2 * (c % 4)) = make_float2(o[c][i], o[c][2 + i]);
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                part[8 * HD + 2 * t + i] = m[i];
                part[8 * HD + 8 + 2 * t + i] = l[i];
            }
        }
        together();
        for (int i = warp; i < min(8, n_rows - r0); i += kStTeam) {      // a warp puts a row together
            float mx = -INFINITY, all = 0.0f, f[kStTeam];
#pragma unroll
            for (int w = 0; w < kStTeam; ++w) {
                f[w] = reinterpret_cast<const float*>(area(w))[8 * HD + i];
                mx = fmaxf(mx, f[w]);
            }
#pragma unroll
            for (int w = 0; w < kStTeam; ++w) {
                const float y = reinterpret_cast<const float*>(area(w))[8 * HD + 8 + i];
                f[w] = f[w] == -INFINITY && y == 0.0f ? 0.0f : tc_exp2(f[w] - mx);
                all = fmaf(f[w], y, all);
            }
            const int qi = st_token(sa, r0 + i);
            float* rec = sh_record(p, it.tok0 + qi, it.h0 + r0 + i - qi * sa.hpc, it.which);
            if (lane == 0) {
                rec[0] = mx;
                rec[1] = all;
            }
            if (4 * lane < HD) {
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kStTeam; ++w) {      // (a part without keys is zeros)
                    const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(area(w)) + i * HD + 4 * lane);
                    y.x = fmaf(f[w], x.x, y.x); y.y = fmaf(f[w], x.y, y.y); y.z = fmaf(f[w], x.z, y.z); y.w = fmaf(f[w], x.w, y.w);
                }
                if (y.x != y.x || y.y != y.y || y.z != y.z || y.w != y.w) {      // NaN: as a rule an infinity times a factor that 32 bits have no number for, which is to stay an infinity
                    y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kStTeam; ++w) {
                        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(area(w)) + i * HD + 4 * lane);
                        y.x = sh_add(y.x, f[w], x.x); y.y = sh_add(y.y, f[w], x.y); y.z = sh_add(y.z, f[w], x.z); y.w = sh_add(y.w, f[w], x.w);
                    }
                }
                *reinterpret_cast<float4*>(rec + kShHead + 4 * lane) = y;
            }
        }
    }
}

// behind the barriers: the flag of a wait that was given up, then what an item needs beside it, then the TMEM address
template <int HD>
__device__ __forceinline__ int* st_gave_up(uint8_t* smem) { return reinterpret_cast<int*>(smem + StShape<HD>::kBars + 448); }

// the barriers, in the order in which st_many has them
template <int HD>
__device__ __forceinline__ void st_barriers(uint8_t* smem) {
    constexpr int KS = StShape<HD>::kKeyStages, VS = StShape<HD>::kValueStages;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + StShape<HD>::kBars);
    for (int i = 0; i < 2 * (KS + VS); ++i) mb_init(bar++, 1);          // keys full, keys empty, values full, values empty
    for (int i = 0; i < VS; ++i) mb_init(bar++, 2);              // values ready
    mb_init(bar++, 128);                                         // queries ready
    mb_init(bar++, 1);                                           // scores full
    mb_init(bar++, 128);                                         // weights ready
    mb_init(bar++, 128);                                         // scores read
    mb_init(bar, 1);                                             // O done
}

// ---- many rows: tcgen05 ----------------------------------------------------------------------------------------------------------------------------------------------------------------
// The key tiles of a share that any row may see: those of the first positions that stay visible behind a window, then those from the oldest key in a window on.
struct StTiles {
    int first, n_keep, lo, n;
    __device__ __forceinline__ StTiles(int key0, int key1, int oldest, int keep_first) {
        first = key0 / kStKeys;
        const int end = (key1 + kStKeys - 1) / kStKeys;
        lo = min(max(first, oldest / kStKeys), max(end, first));
        n_keep = max(0, (min(keep_first, lo * kStKeys) + kStKeys - 1) / kStKeys - first);
        n = key1 > key0 ? n_keep + max(0, end - lo) : 0;
    }
    __device__ __forceinline__ int tile_of(int i) const { return i < n_keep ? first + i : lo + i - n_keep; }
};

template <int HD, bool kOpts>
__device__ void st_many(const CUtensorMap& tmK, const CUtensorMap& tmV, const StArgs& sa, const StItem& it, uint8_t* smem, uint32_t tmem, uint32_t& done, uint32_t turn) {
    using Sh = StShape<HD>;
    constexpr int KS = Sh::kKeyStages, VS = Sh::kValueStages;
    const SharedArgs& p = sa.a;
    uint8_t *sK = smem, *sV = sK + KS * Sh::kTile, *sQ = sV + VS * Sh::kTile;
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + Sh::kBars);
    uint64_t *kempty = kfull + KS, *vfull = kempty + KS, *vempty = vfull + VS, *vready = vempty + VS, *qready = vready + VS, *sfull = qready + 1, *pready = sfull + 1, *sread = pready + 1, *odone = sread + 1;
    volatile int* gave_up = st_gave_up<HD>(smem);
    int* taken = st_gave_up<HD>(smem) + 1 + (turn & 1);          // whether values were taken out
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_rows = it.nq * sa.hpc;
    const int row = threadIdx.x, qi = min(st_token(sa, row), it.nq - 1), h = it.h0 + min(row - st_token(sa, row) * sa.hpc, sa.hpc - 1);      // (of the first four warps)
    const bool live = row < n_rows;
    if (threadIdx.x == 0) st_gave_up<HD>(smem)[1 + (~turn & 1)] = 0;      // the next item's
    const int key1 = min(it.key1, it.high + 1);
    const StTiles tiles(it.key0, key1, p.window > it.low ? 0 : it.low - p.window + 1, p.keep_first);
    const int n = tiles.n;
    const uint32_t was = done;               // key tiles of the items before: the barriers' phases go on from there
    done += n;
    if (warp < 4) {
        // the warp's 32 rows of queries, one row (or two) per load so that neighbouring lanes read neighbouring columns; sixteen loads on their way before the first of them is stored. Where a
        // row lies its own lane knows
        constexpr int kLanes = HD / 4, kPer = 32 / kLanes, kAhead = 16;
        const int col = (lane % kLanes) * 4;
        const float* from = p.q + (size_t)it.tok0 * p.ldq + (size_t)it.h0 * HD + col;
        auto queries = [&](auto load) {
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += kPer * kAhead) {
                uint4 x[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k)     // (rows of no token are some other row's: nothing asks for their results)
                {
                    const int r = min(warp * 32 + r0 + k * kPer + lane / kLanes, n_rows - 1), token = st_token(sa, r);
                    x[k] = load(from + (size_t)token * p.ldq + (r - token * sa.hpc) * HD);
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int r = warp * 32 + r0 + k * kPer + lane / kLanes;
                    *reinterpret_cast<uint2*>(sQ + (col / 64) * Sh::kQBlock + r * 128 + ((((col % 64) / 8) ^ (r & 7)) << 4) + (col % 8) * 2) =
                        make_uint2(tc_pack(__uint_as_float(x[k].x), __uint_as_float(x[k].y)), tc_pack(__uint_as_float(x[k].z), __uint_as_float(x[k].w)));
                }
            }
        };
        if (sa.vec_q) queries([](const float* src) { return ld_stream(src); });      // (left to itself the compiler had each load wait for the one before: 20000 clocks)
        else queries([](const float* src) { return make_uint4(__float_as_uint(src[0]), __float_as_uint(src[1]), __float_as_uint(src[2]), __float_as_uint(src[3])); });
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mb_arrive(qready);
    }

    if (warp == 4) {
        if (elect_one()) {   // ===== TMA producer =====
            for (int i = 0; i < n; ++i) {
                const int j0 = tiles.tile_of(i) * kStKeys;
                const uint32_t ks = (was + i) % KS, kph = (was + i) / KS & 1, vs = (was + i) % VS, vph = (was + i) / VS & 1;
                int at[kStBoxes], row[kStBoxes];
#pragma unroll
                for (int x = 0; x < kStBoxes; ++x) {
                    int in_page;
                    const int pos = j0 + x * kStBox, page = pos < key1 && pos + kStBox > it.key0 ? sh_page(p, it.slot, pos, in_page) : -1;
                    at[x] = page >= 0 ? in_page : p.b.page_len;                     // outside the map: zeros
                    row[x] = page >= 0 ? page * p.kv_heads + it.g : 0;
                }
                if (!tc_wait(kempty + ks, kph ^ 1, gave_up, sa.polls)) break;
                mb_expect(kfull + ks, Sh::kTile);
#pragma unroll
                for (int x = 0; x < kStBoxes; ++x)
                    for (int c = 0; c < Sh::kBlocks; ++c) tma_load_3d(sK + ks * Sh::kTile + c * Sh::kKBlock + x * kStBox * 128, &tmK, 64 * c, at[x], row[x], kfull + ks);
                if (!tc_wait(vempty + vs, vph ^ 1, gave_up, sa.polls)) break;
                mb_expect(vfull + vs, Sh::kTile);
#pragma unroll
                for (int x = 0; x < kStBoxes; ++x)
                    for (int c = 0; c < Sh::kBlocks; ++c) tma_load_3d(sV + vs * Sh::kTile + c * Sh::kKBlock + x * kStBox * 128, &tmV, 64 * c, at[x], row[x], vfull + vs);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (elect_one()) {   // ===== MMA issuer =====
            constexpr uint32_t idesc_s = umma_idesc_bf16(kStRows, kStKeys), idesc_o = umma_idesc_bf16(kStRows, HD) | (1u << 16);      // B MN-major
            const uint64_t q_desc = umma_desc_sw128(sQ), k_desc = umma_desc_sw128(sK), v_desc = umma_desc_mn_sw128(sV, Sh::kKBlock);  // + bytes / 16: another place
            auto scores = [&](int i) {
                const uint64_t k = k_desc + (was + i) % KS * (Sh::kTile / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    tc_mma_bf16(tmem, q_desc + (uint32_t)((ks / 4) * (Sh::kQBlock / 16) + 2 * (ks % 4)), k + (uint32_t)((ks / 4) * (Sh::kKBlock / 16) + 2 * (ks % 4)), idesc_s, ks != 0);
                tc_commit(sfull);
                tc_commit(kempty + (was + i) % KS);
            };
            bool ok = n > 0 && tc_wait(qready, turn & 1, gave_up, sa.polls) && tc_wait(kfull + was % KS, was / KS & 1, gave_up, sa.polls);
            if (ok) {
                tc_fence_after();
                scores(0);
            }
            for (int i = 0; ok && i < n; ++i) {
                const uint32_t at = was + i;
                if (i + 1 < n) {        // the next scores, as soon as these have been read
                    ok = tc_wait(kfull + (at + 1) % KS, (at + 1) / KS & 1, gave_up, sa.polls) && tc_wait(sread, at & 1, gave_up, sa.polls);
                    if (!ok) break;
                    tc_fence_after();
                    scores(i + 1);
                }
                ok = tc_wait(vready + at % VS, at / VS & 1, gave_up, sa.polls) && tc_wait(pready, at & 1, gave_up, sa.polls);
                if (!ok) break;
                tc_fence_after();
                const uint64_t v = v_desc + at % VS * (Sh::kTile / 16);
#pragma unroll
                for (int ks = 0; ks < 3 * kStKeys / 16; ++ks)                    // first terms, then second ones, then third ones, against the same values
                    tc_mma_bf16_ts(tmem + 128, tmem + kStTerms + 8 * ks, v + (uint32_t)((ks % (kStKeys / 16)) * 128), idesc_o, (i % kStFlush | ks) != 0);
                tc_commit(odone);
                tc_commit(vempty + at % VS);
            }
        }
        __syncwarp();
    } else if (warp >= 6) {   // ===== values that are not the share's, or no numbers =====
        for (int i = 0; i < n; ++i) {
            const uint32_t s = (was + i) % VS;
            const int j0 = tiles.tile_of(i) * kStKeys, from = max(0, it.key0 - j0), to = min(kStKeys, key1 - j0);
            if (!tc_wait_warp(vfull + s, (was + i) / VS & 1, gave_up, sa.polls)) break;
            constexpr int kLoads = kStKeys * 8 * Sh::kBlocks / 64;                       // 16 bytes each, all on their way before the first is looked at
            uint4* const at = reinterpret_cast<uint4*>(sV + s * Sh::kTile) + (warp - 6) * 32 + lane;      // (the rows of a block of 64 columns lie one behind the other)
            uint4 v[kLoads];
            uint32_t sum[4] = {};
#pragma unroll
            for (int x = 0; x < kLoads; ++x) v[x] = at[64 * x];
#pragma unroll
            for (int x = 0; x < kLoads; ++x) st_times_zero(sum[x % 4], v[x]);
            bool odd = st_odd(sum[0]) || st_odd(sum[1]) || st_odd(sum[2]) || st_odd(sum[3]);
            if (from > 0 || to < kStKeys || __any_sync(0xffffffffu, odd)) {
                odd = false;
#pragma unroll
                for (int x = 0; x < kLoads; ++x) {
                    const int r = (x * 64 + (warp - 6) * 32 + lane) / 8 % kStKeys;
                    uint32_t one = 0;
                    st_times_zero(one, v[x]);
                    if (r < from || r >= to) {
                        at[64 * x] = make_uint4(0u, 0u, 0u, 0u);
                    } else if (st_odd(one)) {
                        at[64 * x] = st_without(v[x]);
                        odd = true;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            if (odd) *taken = 1;
            __syncwarp();
            if (lane == 0) mb_arrive(vready + s);
        }
    }
    bool ok = true;
    float ref = -INFINITY, l = 0.0f;         // what the weights are relative to; their sum
    float* place = sh_record(p, it.tok0 + qi, h, it.which) + kShHead;
    if (warp < 4) {   // ===== softmax: row = warp * 32 + lane = token * hpc + head =====
        const int qpos = live ? st_pos(sa, it, qi) : -1;
        const uint32_t s_tmem = tmem + ((uint32_t)(warp * 32) << 16), o_tmem = s_tmem + 128;
        const float slope = kOpts && p.slopes && live ? p.slopes[h] : 0.0f;
        const bool plain = !kOpts;           // weights are 2^(score * mul - ref): one rounding between a score and its exponential. Without caps or charges mul holds the scale, too
        const float mul = plain ? p.scale * kStLog2e : kStLog2e;
        float flushed = -INFINITY, lw = 0.0f;        // the reference of what has been flushed; the weights' sum since then
        float4* const flush = reinterpret_cast<float4*>(p.flush) + (size_t)blockIdx.x * (kStRows * HD / 4) + row;      // [columns / 4][rows]: a warp reads and writes whole lines
        auto add_flushed = [&](uint32_t* o, int c) {        // thirty-two columns, carried over to the present reference
            const float f = flushed == ref ? 1.0f : tc_exp2(flushed - ref);
            float4 w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __ldcg(flush + (size_t)(c / 4 + e) * kStRows);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o[4 * e] = __float_as_uint(fmaf(w[e].x, f, __uint_as_float(o[4 * e])));
                o[4 * e + 1] = __float_as_uint(fmaf(w[e].y, f, __uint_as_float(o[4 * e + 1])));
                o[4 * e + 2] = __float_as_uint(fmaf(w[e].z, f, __uint_as_float(o[4 * e + 2])));
                o[4 * e + 3] = __float_as_uint(fmaf(w[e].w, f, __uint_as_float(o[4 * e + 3])));
            }
        };
        constexpr uint64_t kAll = (1ull << kStKeys) - 1;
        // what the block table has for a tile's first key and its last (pages are a multiple of 32 positions: two of them at most), a tile ahead and not looked at before then: a lookup that is looked at holds everything up until it has arrived
        auto entry = [&](int pos) {
            int in_page;
            const int at = page_of(pos, p.b.page_len, p.page_magic, in_page);
            return it.slot >= 0 && at < p.b.max_pages ? p.b.block_table[(size_t)it.slot * p.b.max_pages + at] : -1;
        };
        int next0 = -1, next1 = -1;
        if (n > 0) {
            const int j0 = tiles.tile_of(0) * kStKeys;
            next0 = entry(j0);
            next1 = entry(min(j0 + kStKeys, key1) - 1);
        }
        for (int i = 0; i < n; ++i) {
            const int j0 = tiles.tile_of(i) * kStKeys;
            ok = tc_wait_warp(sfull, (was + i) & 1, gave_up, sa.polls);
            if (!ok) break;
            tc_fence_after();
            if (i % kStFlush == 0 && i > 0) {
                ok = tc_wait_warp(odone, (was + i - 1) & 1, gave_up, sa.polls);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tc_ld32_async(o_tmem + c, o);
                    tc_arrived(o);
                    if (i > kStFlush) add_flushed(o, c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) __stcg(flush + (size_t)(c / 4 + e) * kStRows, make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3])));
                }
                l += lw;
                lw = 0.0f;
                flushed = ref;
            }
            const bool page0 = (unsigned)next0 < (unsigned)p.n_pages, page1 = (unsigned)next1 < (unsigned)p.n_pages;
            if (i + 1 < n) {
                const int j1 = tiles.tile_of(i + 1) * kStKeys;
                next0 = entry(j1);
                next1 = entry(min(j1 + kStKeys, key1) - 1);
            }
            uint32_t s[kStKeys];
            tc_ld32_async(s_tmem, s);
            st_ld16_async(s_tmem + 32, s + 32);
            tc_arrived(s);
#pragma unroll
            for (int e = 32; e < kStKeys; ++e) asm volatile("" : "+r"(s[e]));
            tc_fence_before();
            mb_arrive(sread);
            // whether every row of the tile sees every key: as a rule the positions of the rows say so at once
            uint64_t have = kAll;
            bool all = j0 >= it.key0 && j0 + kStKeys <= key1 && page0 && page1 && j0 + kStKeys - 1 <= it.low && (it.high - j0 < p.window || j0 + kStKeys <= p.keep_first);
            if (!all) {          // keys of the tile that are in the share and in a page
                const int from = max(0, it.key0 - j0), to = min(kStKeys, key1 - j0);
                int in_page;
                page_of(j0, p.b.page_len, p.page_magic, in_page);
                const uint64_t first = (1ull << min(kStKeys, p.b.page_len - in_page)) - 1;
                have = ((1ull << to) - 1) & ~((1ull << from) - 1) & ((page0 ? first : 0ull) | (page1 ? ~first : 0ull));
                all = have == kAll && __all_sync(0xffffffffu, !live || (j0 + kStKeys - 1 <= qpos && (qpos - j0 < p.window || j0 + kStKeys <= p.keep_first)));
            }
            if (kOpts && p.softcap > 0.0f) {
                const float inv = p.scale / p.softcap;
                const uint64_t inv2 = tc_two(__float_as_uint(inv), __float_as_uint(inv));
                float top0 = 0.0f, top1 = 0.0f;
#pragma unroll
                for (int e = 0; e < kStKeys; e += 2) {
                    float x, y;
                    tc_split(tc_mul2(tc_two(s[e], s[e + 1]), inv2), x, y);
                    s[e] = __float_as_uint(x);
                    s[e + 1] = __float_as_uint(y);
                    if (e & 2) top1 = tc_max3(top1, fabsf(x), fabsf(y));
                    else top0 = tc_max3(top0, fabsf(x), fabsf(y));
                }
                // scores within a quarter of the cap, as nearly all are: the series that tc_tanh takes for them, two at a time
                if (__any_sync(0xffffffffu, fmaxf(top0, top1) >= 0.25f)) {
#pragma unroll
                    for (int e = 0; e < kStKeys; ++e) s[e] = __float_as_uint(p.softcap * tc_tanh(__uint_as_float(s[e])));
                } else {
                    auto both = [](float v) { return tc_two(__float_as_uint(v), __float_as_uint(v)); };
                    const uint64_t c4 = both(62.0f / 2835.0f), c3 = both(-17.0f / 315.0f), c2 = both(2.0f / 15.0f), c1 = both(-1.0f / 3.0f), c0 = both(1.0f), cap2 = both(p.softcap);
#pragma unroll
                    for (int e = 0; e < kStKeys; e += 2) {
                        const uint64_t x = tc_two(s[e], s[e + 1]), x2 = tc_mul2(x, x);
                        float a, c;
                        tc_split(tc_mul2(cap2, tc_mul2(x, tc_fma2(x2, tc_fma2(x2, tc_fma2(x2, tc_fma2(x2, c4, c3), c2), c1), c0))), a, c);
                        s[e] = __float_as_uint(a);
                        s[e + 1] = __float_as_uint(c);
                    }
                }
            } else if (!plain) {
#pragma unroll
                for (int e = 0; e < kStKeys; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * p.scale);
            }
            if (kOpts && p.slopes) {
                const float d0 = (float)(qpos - j0);
#pragma unroll
                for (int e = 0; e < kStKeys; ++e) s[e] = __float_as_uint(fmaf(-slope, d0 - (float)e, __uint_as_float(s[e])));
            }
            if (!all) {          // the keys of the tile that this row sees, a bit each: up to its own position, and from the window's oldest on or among the first
                auto below = [&](int key) { return key <= j0 ? 0ull : key >= j0 + kStKeys ? ~0ull : (1ull << (key - j0)) - 1; };
                const uint64_t sees = have & below(qpos + 1) & (~below(p.window > qpos ? 0 : qpos - p.window + 1) | below(p.keep_first));
                const uint32_t seen[2] = {(uint32_t)sees, (uint32_t)(sees >> 32)};
#pragma unroll
                for (int e = 0; e < kStKeys; ++e)
                    if (!(seen[e / 32] >> (e % 32) & 1)) s[e] = 0xff800000u;       // -inf
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < kStKeys; e += 2) m[(e / 2) & 3] = tc_max3(m[(e / 2) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
            const float mx = tc_max3(fmaxf(m[0], m[1]), m[2], m[3]) * mul;
            if (i == 0) {
                ref = mx;
            } else if (__any_sync(0xffffffffu, mx > ref + 8.0f)) {
                ok = tc_wait_warp(odone, (was + i - 1) & 1, gave_up, sa.polls);
                if (!ok) break;
                tc_fence_after();
                const float nr = mx > ref + 8.0f ? mx : ref, f = nr == ref ? 1.0f : tc_exp2(ref - nr);      // (each row by what it sees itself: no other row's keys show in its bits)
                l *= f;
                lw *= f;
                ref = nr;
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                    uint32_t o[16];
                    st_ld16(o_tmem + c, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tc_st16(o_tmem + c, o);
                }
            }
            const float base = ref == -INFINITY ? 0.0f : ref;                   // nothing seen yet: every weight is exp(-inf) = 0
            const uint64_t mul2 = tc_two(__float_as_uint(mul), __float_as_uint(mul)), base2 = tc_two(__float_as_uint(-base), __float_as_uint(-base));
            const uint64_t less = tc_two(__float_as_uint(-1.0f), __float_as_uint(-1.0f));
            auto terms = [](uint32_t w) { return tc_two(w << 16, w & 0xffff0000u); };
            uint64_t sum[kStKeys / 16] = {};                                    // of a product's sixteen keys each
#pragma unroll
            for (int part = 0; part < kStKeys / 16; ++part) {
                uint32_t hi[8], mid[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x, y;
                    tc_split(tc_fma2(tc_two(s[part * 16 + 2 * e], s[part * 16 + 2 * e + 1]), mul2, base2), x, y);
                    x = tc_exp2(x);
                    y = tc_exp2(y);
                    const uint64_t w = tc_two(__float_as_uint(x), __float_as_uint(y));
                    sum[part] = tc_add2(sum[part], w);
                    hi[e] = tc_pack(x, y);
                    const uint64_t r = tc_fma2(terms(hi[e]), less, w);          // what the first terms leave: exact
                    tc_split(r, x, y);
                    mid[e] = tc_pack(x, y);
                    tc_split(tc_fma2(terms(mid[e]), less, r), x, y);
                    lo[e] = tc_pack(x, y);
                }
                if (part == 0 && i > 0) {            // the product before this one still reads where the weights go
                    ok = tc_wait_warp(odone, (was + i - 1) & 1, gave_up, sa.polls);
                    if (!ok) break;
                    tc_fence_after();
                }
                st_st8(s_tmem + kStTerms + part * 8, hi);
                st_st8(s_tmem + kStTerms + kStKeys / 2 + part * 8, mid);
                st_st8(s_tmem + kStTerms + kStKeys + part * 8, lo);
            }
            if (!ok) break;
            tc_wait_st();
            tc_fence_before();
            mb_arrive(pready);
            // The tensor core truncates as it adds: each of a tile's nine products (three of first terms, three of second, three of third ones) loses half a unit of O's last place on average. The
            // weights' sum is added up in the same nine steps, truncated too, so that the quotient keeps a fraction of the loss only: with plain additions it was 2e-7 too small a tile.
            constexpr float k9 = 1.0f / 512, k18 = k9 * k9;                     // what is left of a weight behind its first term, behind its second: at most, to which the steps' sizes need not be exact
            float steps[kStKeys / 16];
#pragma unroll
            for (int k = 0; k < kStKeys / 16; ++k) {
                float a, b;
                tc_split(sum[k], a, b);
                steps[k] = a + b;
            }
#pragma unroll
            for (int k = 0; k < 3 * kStKeys / 16; ++k) lw = __fadd_rz(lw, steps[k % (kStKeys / 16)] * (k < kStKeys / 16 ? 1.0f - k9 : k < kStKeys / 8 ? k9 - k18 : k18));
        }
        l += lw;
        if (ok && n > 0) ok = tc_wait_warp(odone, (was + n - 1) & 1, gave_up, sa.polls);
        tc_fence_after();
        if (ok && live) {
            place[-kShHead] = ref;
            place[1 - kShHead] = l;
        }
        // A pair of lanes writes the even lane's row first, then the odd one's, 32 bytes each time: 16 bytes into each of 32 rows would be half sectors, and through shared memory, whole lines, it took
        // 7000 clocks.
        const bool odd = lane & 1, peer = __shfl_xor_sync(0xffffffffu, live, 1);
        float* other = reinterpret_cast<float*>(__shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(place), 1));
        float *even_row = (odd ? other : place) + (odd ? 4 : 0), *odd_row = (odd ? place : other) + (odd ? 4 : 0);
        const bool even_live = odd ? peer : live, odd_live = odd ? live : peer;
#pragma unroll 1
        for (int c = 0; ok && c < HD; c += 32) {
            uint32_t o[32];
            if (n > 0) {
                tc_ld32_async(o_tmem + c, o);
                tc_arrived(o);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
            if (n > kStFlush) add_flushed(o, c);
            __syncwarp();
            uint32_t got[16];        // (all of them before the first store: behind a store each shuffle waited)
#pragma unroll
            for (int e = 0; e < 16; ++e) got[e] = __shfl_xor_sync(0xffffffffu, odd ? o[(e & ~3) * 2 + (e & 3)] : o[(e & ~3) * 2 + 4 + (e & 3)], 1);
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                const uint4 g = make_uint4(got[e / 2], got[e / 2 + 1], got[e / 2 + 2], got[e / 2 + 3]);
                if (even_live) *reinterpret_cast<uint4*>(even_row + c + e) = odd ? g : make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                if (odd_live) *reinterpret_cast<uint4*>(odd_row + c + e) = odd ? make_uint4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]) : g;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*taken && warp < 4 && live) {     // infinities and NaN that were taken out of the values: back to the rows that see them (columns of this row alone, written behind the barrier)
        const int qpos = st_pos(sa, it, qi);
        for (int i = 0; i < n; ++i) {
            const int j0 = tiles.tile_of(i) * kStKeys;
            for (int key = max(j0, it.key0); key < min(j0 + kStKeys, key1); ++key) {
                int in_page;
                const int page = sh_page(p, it.slot, key, in_page);
                if (page < 0 || !seq_sees(qpos, key, p.window, p.keep_first)) continue;
                const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v_pool) + seq_pool_row(page, p.kv_heads, it.g, p.b.page_len, in_page, HD);
                for (int c = 0; c < HD; ++c) {
                    const float x = seq_ld(v, c);
                    if (!(fabsf(x) <= FLT_MAX)) place[c] += x;
                }
            }
        }
    }
}

// Keys of a share of the shared positions: by what all groups have (row tiles x key tiles), such that the shares are a round of the grid or a few, their beginnings and ends counted
// as kStEnds key tiles. Thirty-two lengths about the even one are tried, a lane each. group(g, tiles, keys): row tiles and key tiles of a group. By one warp.
template <class F>
__device__ __forceinline__ int st_least(const SharedArgs& p, int all_sets, F group) {
    const int lane = threadIdx.x & 31;
    const float inv = 1.0f / (float)gridDim.x;       // (these are estimates: whole-number divisions of 64 bits took 1000 clocks)
    float units = 0.0f, items = 0.0f, longest = 0.0f;
    for (int g = lane; g < p.n_groups; g += 32) {
        int tiles, keys;
        group(g, tiles, keys);
        units += (float)tiles * (float)keys;
    }
    const float even = ceilf(warp_sum(units) * (float)all_sets * inv);
    const int length = (int)fmaxf(4.0f, fminf(1048576.0f, even * (float)(4 + lane) * (1.0f / 16.0f)));
    const float per = 1.0f / (float)length;
    for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
        int tiles = 0, keys = 0;
        if (g0 + lane < p.n_groups) group(g0 + lane, tiles, keys);
        for (unsigned rest = __ballot_sync(0xffffffffu, tiles > 0 && keys > 0); rest; rest &= rest - 1) {
            const int who = __ffs(rest) - 1;
            const float k = (float)__shfl_sync(0xffffffffu, keys, who), cuts = fminf((float)p.shares, ceilf(k * per));
            items += (float)__shfl_sync(0xffffffffu, tiles, who) * cuts;
            longest = fmaxf(longest, ceilf(__fdividef(k, cuts)));
        }
    }
    const float cost = ceilf(items * (float)all_sets * inv) * (longest + (float)kStEnds), least = -warp_max(-cost);
    return __shfl_sync(0xffffffffu, length, __ffs(__ballot_sync(0xffffffffu, cost == least)) - 1) * kStKeys;
}

// x / d for numbers below 2^24, the estimate put right
__device__ __forceinline__ uint32_t st_div(uint32_t x, uint32_t d) {
    uint32_t q = (uint32_t)__fdividef((float)x, (float)d);
    if (q * d > x) --q;
    else if (x - q * d >= d) ++q;
    return q;
}

template <int HD, bool kOpts>
__global__ void __launch_bounds__(kStThreads, 2) seq_attention_shared_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const StArgs sa) {
    after_previous();        // in front of the allocation of TMEM: a CTA that waits for another kernel must not hold what that kernel's CTAs may be waiting for
    extern __shared__ uint8_t st_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(st_raw) + 1023) & ~(uintptr_t)1023);
    StPlan& plan = *reinterpret_cast<StPlan*>(smem + StShape<HD>::kPlan);
    volatile int* gave_up = st_gave_up<HD>(smem);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(st_gave_up<HD>(smem) + 7);
    const SharedArgs& p = sa.a;
    const int all_sets = p.kv_heads * sa.sets, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = p.heads / p.kv_heads;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        st_barriers<HD>(smem);
        *gave_up = sa.polls == 0;
        st_gave_up<HD>(smem)[1] = 0;             // of the first item; each makes that of the next one ready
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) tc_alloc(tmem_slot, kStTmem);
    uint32_t done = 0, turn = 0;             // key tiles and items of the first kind so far
    long long mine = blockIdx.x;             // the next item of this CTA, counted from the present entries' first
    bool stop = sa.polls == 0;               // a wait was given up
    const int entries = p.n_groups + p.b.n_qtiles;
    for (int e0 = 0; e0 < entries; e0 += kStEntries) {
        {   // an entry a thread
            const int e = e0 + threadIdx.x, i = threadIdx.x;
            int tok0 = 0, n = 0, slot = -1, from = 0, end = 0, cuts = 0, tiles = 0, seg = -1, shared = 0;
            if (e < p.n_groups) {
                sh_group_tokens(p, e, tok0, n);
                end = sh_group_len(p, e);
                tiles = (n + sa.queries - 1) / sa.queries;
                if (n > 0) slot = p.b.seg_slot[p.group_start[e]];
                plan.n[i] = n; plan.end[i] = end; plan.tiles[i] = tiles; plan.from[i] = p.group_start[e]; plan.low[i] = INT_MAX; plan.high[i] = -1;
            } else if (e < entries) {
                const int off = p.b.qt_off[e - p.n_groups];
                seg = p.b.qt_seg[e - p.n_groups];
                n = min(kBQ, p.b.seg_len[seg] - off);
                end = p.b.seg_pos0[seg] + off + n;
                tok0 = p.b.seg_start[seg] + off;
                slot = p.b.seg_slot[seg];
                tiles = n * sa.hpc <= kStFew ? 1 : (n + sa.queries - 1) / sa.queries;
            }
            tc_fence_before();
            __syncthreads();
            const bool all = p.n_groups <= kStEntries;           // of the first entries: every group is at hand
            if (e0 == 0 && warp == kStWarps - 1) {               // (as a rule without an entry: the others look their groups up meanwhile)
                const int least = all ? st_least(p, all_sets, [&](int g, int& t, int& k) { t = plan.tiles[g]; k = (plan.end[g] + kStKeys - 1) / kStKeys; })
                                      : st_least(p, all_sets, [&](int g, int& t, int& k) {
                                            int first, m;
                                            sh_group_tokens(p, g, first, m);
                                            t = (m + sa.queries - 1) / sa.queries;
                                            k = (sh_group_len(p, g) + kStKeys - 1) / kStKeys;
                                        });
                if (lane == 0) plan.least = least;
            }
            if (seg >= 0) {
                int lo = 0, hi = p.n_groups;                     // group_start[lo] <= seg < group_start[hi]
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if ((all && e0 == 0 ? plan.from[mid] : p.group_start[mid]) <= seg) lo = mid; else hi = mid;
                }
                shared = all && e0 == 0 ? plan.end[lo] : sh_group_len(p, lo);
                from = min(shared, end);
                cuts = sh_cuts(end - from, p.own_least, p.own);
                if (all && e0 == 0) {
                    atomicMin(&plan.low[lo], end - n);
                    atomicMax(&plan.high[lo], end - 1);
                }
            }
            __syncthreads();
            if (e < p.n_groups) cuts = sh_cuts(end, plan.least, p.shares);
            else if (blockIdx.x == 0 && seg >= 0) p.plan[e - p.n_groups] = sh_cuts(shared, plan.least, p.shares) | cuts << 16;
            if (e < p.n_groups && entries > kStEntries) { plan.low[i] = 0; plan.high[i] = INT_MAX - 1; }      // not all of its tiles are here
            plan.tok0[i] = tok0; plan.n[i] = n; plan.slot[i] = slot; plan.from[i] = from; plan.end[i] = end; plan.cuts[i] = cuts; plan.tiles[i] = tiles;
            const bool few = seg >= 0 && n * sa.hpc <= kStFew;
            int upto = few ? (cuts * all_sets + kStTeams - 1) / kStTeams : tiles * cuts * all_sets;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            if (lane == 31) plan.warp[warp] = upto;
            __syncthreads();
            for (int w = 0; w < warp; ++w) upto += plan.warp[w];
            plan.upto[i] = upto;
            __syncthreads();
        }
        tc_fence_after();                    // (the allocation, at the first turn)
        const uint32_t tmem = *tmem_slot;
        const int total = plan.upto[kStEntries - 1];
        for (; mine < total && !stop; mine += gridDim.x) {
            int e = 0;                       // the first entry that reaches beyond it
            for (int w = kStEntries / 2; w > 0; w /= 2)
                if (plan.upto[e + w - 1] <= (int)mine) e += w;
            int x = (int)mine - (e ? plan.upto[e - 1] : 0);
            const bool group = e0 + e < p.n_groups;
            const uint32_t tiles = plan.tiles[e], cuts = plan.cuts[e];
            const int n = plan.n[e], from = plan.from[e], end = plan.end[e], t0 = from / kStKeys, span = (end + kStKeys - 1) / kStKeys - t0;
            const bool few = !group && n * sa.hpc <= kStFew;
            if (few) x = kStTeams * x + threadIdx.x / (32 * kStTeam);
            // (item numbers may be larger than st_div takes; what is left of them by then is not)
            const uint32_t y = tiles == 1 ? (uint32_t)x : (uint32_t)x < 1u << 24 ? st_div(x, tiles) : (uint32_t)x / tiles, tile = x - y * tiles;
            const uint32_t z = y < 1u << 24 ? st_div(y, all_sets) : y / (uint32_t)all_sets, set = y - z * all_sets;
            StItem it;
            it.g = sa.sets == 1 ? set : set / (uint32_t)sa.sets;
            it.tok0 = plan.tok0[e] + tile * sa.queries;
            it.nq = min(sa.queries, n - (int)tile * sa.queries);
            it.slot = plan.slot[e];
            it.pos0 = group ? -1 : end - n + (int)tile * sa.queries;
            it.h0 = it.g * per + (set - it.g * sa.sets) * sa.hpc;
            auto cut = [&](uint32_t k) { return cuts == 1 ? span * k : span * k < 1u << 24 ? st_div(span * k, cuts) : span * k / cuts; };      // (2^25 key tiles at most, 32 shares)
            it.key0 = max(from, (int)(t0 + cut(z)) * kStKeys);
            it.key1 = min(end, (int)(t0 + cut(z + 1)) * kStKeys);
            it.which = (group ? 0 : p.shares) + z;
            it.low = group ? plan.low[e] : it.pos0;
            it.high = group ? plan.high[e] : it.pos0 + it.nq - 1;
            if (few) {
                if (z < cuts) st_few<HD>(sa, it, smem);
            } else {
                st_many<HD, kOpts>(tmK, tmV, sa, it, smem, tmem, done, turn++);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the next item's copies may land where this one has written
            stop = *gave_up;                 // (what this item's waits set it to lies behind a barrier, what the next one's do behind the one that follows: all threads see the same)
            __syncthreads();
        }
        mine -= total;
        __syncthreads();                     // the entries have been read
        if (stop && blockIdx.x > 0) break;   // (the first CTA leaves the plan of every tile, whatever became of the items: the last kernel goes by it)
    }
    if (stop) tc_gave_up(sa.status);
    if (warp == 5) {
        tc_fence_after();
        tc_dealloc(*tmem_slot, kStTmem);
    }
}

template <int HD, bool kOpts>
static int st_launch(const SharedArgs& p, cudaStream_t st) {
    using Sh = StShape<HD>;
    static_assert(Sh::kBars >= kStWarps * 64 * HD && 64 * HD >= (8 * HD + 16) * 4, "the warps' areas");
    auto* kernel = seq_attention_shared_tc_kernel<HD, kOpts>;
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
            return SLLM_OK;
        }))
        return rc;
    StArgs a{};
    a.a = p;
    const int per = p.heads / p.kv_heads;
    for (a.hpc = std::min(per, 16); per % a.hpc; --a.hpc) {}
    a.sets = per / a.hpc;
    a.queries = kStRows / a.hpc;
    a.hpc_magic = (65536u + a.hpc - 1) / a.hpc;
    if (int rc = status_word(&a.status)) return rc;
    a.polls = (unsigned)g_tune_tc_polls;
    a.vec_q = p.ldq % 4 == 0 && ((uintptr_t)p.q % 16) == 0;
    CUtensorMap tmK, tmV;
    const cuuint64_t dims[3] = {HD, (cuuint64_t)p.b.page_len, (cuuint64_t)p.n_pages * p.kv_heads};
    const cuuint64_t strides[2] = {HD * 2, (cuuint64_t)p.b.page_len * HD * 2};
    const cuuint32_t box[3] = {64, kStBox, 1};
    if (int rc = tc_encode_bf16(&tmK, p.k_pool, 3, dims, strides, box)) return rc;
    if (int rc = tc_encode_bf16(&tmV, p.v_pool, 3, dims, strides, box)) return rc;
    const long long row_tiles = (p.b.T + a.queries - 1) / a.queries + p.n_groups, all_sets = (long long)p.kv_heads * a.sets;
    SLLM_REQUIRE((row_tiles * p.shares + ((long long)p.b.n_qtiles + row_tiles) * p.own) * all_sets <= 0x7fffffffLL, SLLM_ENOTSUP, "seq_attention_shared: too many tokens or heads");
    const long long most = (row_tiles * p.shares + (long long)p.b.n_qtiles * ((kBQ + a.queries - 1) / a.queries) * p.own) * all_sets;
    overlapping(kernel)<<<(unsigned)std::min<long long>(most, 2 * sm_count()), kStThreads, Sh::kSmem, st>>>(tmK, tmV, a);
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

int64_t attention_shared_tc_flush_floats(int dk, int dv) { return dk == dv && (dk == 64 || dk == 128) ? 2LL * sm_count() * kStRows * dv : 0; }

int launch_attention_shared_tc(const SharedArgs& p, cudaStream_t st) {
    const bool opts = p.softcap > 0.0f || p.slopes;
    if (p.dk == 128) return opts ? st_launch<128, true>(p, st) : st_launch<128, false>(p, st);
    return opts ? st_launch<64, true>(p, st) : st_launch<64, false>(p, st);
}

}  // namespace sllm
