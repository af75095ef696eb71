// csrc/seq_linear8.cu — products of 8-bit integers with a scale for every token and every output channel, and the rows of codes they read.
//
//   s_t = max(max_k |x_tk| / 127, 2^-126),  a_tk = round(x_tk / s_t);   C_tn = (sum_k a_tk w_nk) * s_t * v_n + bias_n
// Sums of codes are exact in 32 bits (127 * 127 * 131072 < 2^31; with codes of -128, which no row here gets, 2^14 * 131071 < 2^31), so a result is three roundings of fp32 away from the formula and does not depend on how a product is cut.
#include <type_traits>

#include "seq_common.cuh"
#include "tcgen05.cuh"

namespace sllm {

// ---- rows to codes --------------------------------------------------------------------------------------------------------------------------------------------------------------------
// A row belongs to a team of warps, which keeps it in registers as it was loaded, up to eight loads of 16 bytes a thread (longer rows are read a second time); a CTA has several teams. The largest
// magnitude is taken over the values' bits, in whose order infinity and NaN come last: a row that has one gets the scale NaN and zeros.
// The quotient has to be the IEEE one, but a division costs some ten instructions: x times the inverse of the scale is off by less than two units of the last place (2^-16 at 127), so only where one
// of a load's quotients is within 2^-14 of a border between two whole numbers are they divided out. Bound: instructions, some five a value, and then what comes in (14336 rows of 4096 in bf16 33 us,
// 5.3 TB/s; 36 with one value an instruction).
constexpr int kQzLoads = 8, kQzFewLoads = 2, kQzThreads = 256, kQzWide = 1024;
constexpr float kQzLeast = 1.17549435e-38f;      // 2^-126
constexpr float kQzMagic = 12582912.0f;          // 1.5 * 2^23: a sum with it is rounded to a whole number, which the low bits hold

struct QuantiseArgs {
    const void* x;
    int8_t* codes;
    float* scales;
    int64_t ldx, ldc;
    int T, K;
};

__device__ __forceinline__ uint32_t qz_pack(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <int N>
__device__ __forceinline__ void qz_codes(const float (&x)[N], float inv, float scale, int (&q)[N]) {
    float near = 0.0f;
    if constexpr (N == 1) {
        const float r = x[0] * inv, whole = r + kQzMagic;
        near = fabsf(r - (whole - kQzMagic));
        q[0] = __float_as_int(whole);
    } else {                                 // two at a time: the instructions are what bounds a matrix of rows
        auto both = [](float v) { return tc_two(__float_as_uint(v), __float_as_uint(v)); };
        const uint64_t inv2 = both(inv), magic = both(kQzMagic), less = both(-kQzMagic), minus = both(-1.0f);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const uint64_t r = tc_mul2(tc_two(__float_as_uint(x[e]), __float_as_uint(x[e + 1])), inv2), whole = tc_add2(r, magic);
            float a, b;
            tc_split(tc_fma2(tc_add2(whole, less), minus, r), a, b);
            near = tc_max3(near, fabsf(a), fabsf(b));
            tc_split(whole, a, b);
            q[e] = __float_as_int(a);
            q[e + 1] = __float_as_int(b);
        }
    }
    if (near > 0.5f - 6.103515625e-05f) {
#pragma unroll
        for (int e = 0; e < N; ++e) q[e] = __float_as_int(__fdiv_rn(x[e], scale) + kQzMagic);
    }
}
// the floats of a load: eight bf16 or four fp32 values
__device__ __forceinline__ void qz_floats(const uint4& v, float (&x)[8]) {
    x[0] = bf16_lo(v.x); x[1] = bf16_hi(v.x); x[2] = bf16_lo(v.y); x[3] = bf16_hi(v.y); x[4] = bf16_lo(v.z); x[5] = bf16_hi(v.z); x[6] = bf16_lo(v.w); x[7] = bf16_hi(v.w);
}
__device__ __forceinline__ void qz_floats(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}

// blockDim.x threads a row, blockDim.y rows. kVec: rows start at multiples of 16 bytes and are a number of whole loads; else a "load" is one value
template <bool kBf16, bool kVec, int kMost, int kLoads>
__global__ void __launch_bounds__(kMost) quantise_rows_kernel(QuantiseArgs p) {
    after_previous();
    __shared__ uint32_t s_top[kMost / 32];
    constexpr int kRun = !kVec ? 1 : kBf16 ? 8 : 4;
    const int row = blockIdx.x * blockDim.y + threadIdx.y, i = threadIdx.x, n = blockDim.x, per = n * kLoads * kRun;
    const bool live = row < p.T;
    const size_t from = (size_t)(live ? row : p.T - 1) * p.ldx;
    uint4 v[kLoads];
    auto load = [&](int base) {              // every address is inside the row, so that nothing is asked before a load; what is behind the end counts as the value that is there
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const size_t c = from + min(base + (j * n + i) * kRun, p.K - kRun);
            if constexpr (kVec) v[j] = kBf16 ? ld_stream(reinterpret_cast<const uint16_t*>(p.x) + c) : ld_stream(reinterpret_cast<const float*>(p.x) + c);
            else v[j].x = kBf16 ? (uint32_t)reinterpret_cast<const uint16_t*>(p.x)[c] << 16 : __float_as_uint(reinterpret_cast<const float*>(p.x)[c]);
        }
    };
    uint32_t top = 0;
    for (int base = 0; base < p.K; base += per) {
        load(base);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if constexpr (!kVec) {
                top = max(top, v[j].x & 0x7fffffffu);
            } else {
                const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) top = kBf16 ? __vmaxu2(top, w[e] & 0x7fff7fffu) : max(top, w[e] & 0x7fffffffu);
            }
        }
    }
    if (kVec && kBf16) top = max(top << 16, top & 0xffff0000u);              // two values' bits beside one another until here
    top = __reduce_max_sync(0xffffffffu, top);
    if (n > 32) {                            // the row's warps, by a barrier of their own where the CTA has several rows
        const int warp = (threadIdx.y * n + i) >> 5, first = threadIdx.y * n >> 5;
        if ((i & 31) == 0) s_top[warp] = top;
        if (blockDim.y == 1) __syncthreads();
        else asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(n) : "memory");
        for (int w = 0; w < n / 32; ++w) top = max(top, s_top[first + w]);
    }
    if (!live) return;
    const bool finite = top < 0x7f800000u;
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), kQzLeast), inv = finite ? 1.0f / scale : 0.0f;
    if (i == 0) p.scales[row] = finite ? scale : NAN;
    int8_t* to = p.codes + (size_t)row * p.ldc;
    for (int base = 0; base < p.K; base += per) {
        if (p.K > per) load(base);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int c = base + (j * n + i) * kRun;
            if (c >= p.K) break;
            float x[kRun];
            int q[kRun] = {};
            if constexpr (kVec) qz_floats(v[j], x);
            else x[0] = __uint_as_float(v[j].x);
            if (finite) qz_codes(x, inv, scale, q);
            if constexpr (kRun == 8) *reinterpret_cast<uint2*>(to + c) = make_uint2(qz_pack(q[0], q[1], q[2], q[3]), qz_pack(q[4], q[5], q[6], q[7]));
            else if constexpr (kRun == 4) *reinterpret_cast<uint32_t*>(to + c) = qz_pack(q[0], q[1], q[2], q[3]);
            else to[c] = (int8_t)q[0];
        }
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------------------------------------------------------------------
struct Linear8Args {
    const int8_t *a, *w;
    const float *a_scale, *w_scale, *bias;
    float* out;
    int64_t lda, ldw, ldc;
    int T, N, K, accumulate;
};

// every rounding by itself: a result does not depend on where a compiler contracts, so not on which kernel it comes from
__device__ __forceinline__ float l8_value(int sum, float s, float w, float bias) { return __fadd_rn(__fmul_rn(__fmul_rn((float)sum, s), w), bias); }
__device__ __forceinline__ void l8_store(const Linear8Args& p, int t, int n, int sum) {
    const float v = l8_value(sum, p.a_scale[t], p.w_scale[n], p.bias ? p.bias[n] : 0.0f);
    float* to = p.out + (size_t)t * p.ldc + n;
    *to = p.accumulate ? __fadd_rn(*to, v) : v;
}

// One or two tokens: a warp takes kRows rows of W, sixteen codes a load, four products an instruction, eight loads of W on their way. Bound: what those bring in. us, N x K:
//   one token, 1 | 2 | 4 rows a warp, tcgen05: 4096 x 4096 5.7 | 6.4 | 8.7, 7.1; 6144 x 4096 6.6 | 7.2 | 9.1, 8.7; 8192 x 4096 10.0 | 8.1 | 9.6, 9.7; 11008 x 4096 10.6 | 9.8 | 10.8, 11.1;
//     14336 x 4096 14.2 | 13.7 | 12.2, 12.9; 28672 x 4096 24.5 | 21.3 | 22.6, 22.7; 4096 x 14336 14.8 | 17.7 | 24.3, 13.7; 8192 x 14336 28.7 | 22.7 | 26.8, 22.5
//   two, 1 | 2 rows, tcgen05: 4096 x 4096 6.5 | 6.7, 7.2; 6144 x 4096 11.3 | 7.4, 8.7; 8192 x 4096 11.6 | 8.3, 9.8; 14336 x 4096 16.8 | 13.8, 12.8; 28672 x 4096 29.2 | 25.9, 23.2; 4096 x 14336 17.1 | 18.2, 13.7
// One row a warp below kL8Wide rows, else four for one token and two for two, is right to a tenth in most places, not in all: two tokens through 6144 rows would be 7.4 with two rows a warp, and long
// rows are faster on tcgen05 even for one token. Four tokens here took 19.5, where tcgen05 takes 13.6.
constexpr int kL8Warps = 8, kL8Few = 2, kL8Wide = 8192;
template <int kT, int kRows>
__global__ void __launch_bounds__(kL8Warps * 32) linear8_few_kernel(Linear8Args p) {
    after_previous();
    const int lane = threadIdx.x & 31, n0 = (blockIdx.x * kL8Warps + (threadIdx.x >> 5)) * kRows;
    if (n0 >= p.N) return;
    int sum[kRows][kT] = {};
    const int8_t *w[kRows], *a[kT];
#pragma unroll
    for (int r = 0; r < kRows; ++r) w[r] = p.w + (size_t)min(n0 + r, p.N - 1) * p.ldw;
#pragma unroll
    for (int t = 0; t < kT; ++t) a[t] = p.a + (size_t)min(t, p.T - 1) * p.lda;
    auto products = [&](const uint4 (&x)[kRows], int c) {
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const uint4 y = *reinterpret_cast<const uint4*>(a[t] + c);
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                sum[r][t] = __dp4a((int)x[r].w, (int)y.w, __dp4a((int)x[r].z, (int)y.z, __dp4a((int)x[r].y, (int)y.y, __dp4a((int)x[r].x, (int)y.x, sum[r][t]))));
        }
    };
    const int whole = p.K & ~511;                // up to there every lane has sixteen codes
#pragma unroll 8 / kRows
    for (int c = lane * 16; c < whole; c += 512) {
        uint4 x[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) x[r] = ld_stream(w[r] + c);
        products(x, c);
    }
    if (const int c = whole + lane * 16; c < p.K) {
        uint4 x[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) x[r] = ld_stream(w[r] + c);
        // columns behind the last one: whatever the rows hold there does not count
        const int have = p.K - c;
        auto keep = [&](uint32_t v, int first) { return have >= first + 4 ? v : have <= first ? 0u : v & ((1u << 8 * (have - first)) - 1); };
#pragma unroll
        for (int r = 0; r < kRows; ++r) x[r] = make_uint4(keep(x[r].x, 0), keep(x[r].y, 4), keep(x[r].z, 8), keep(x[r].w, 12));
        products(x, c);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const int v = __reduce_add_sync(0xffffffffu, sum[r][t]);
            if (lane == 0 && n0 + r < p.N && t < p.T) l8_store(p, t, n0 + r, v);
        }
}

// Above kL8Few tokens: tcgen05, products of 8-bit integers with sums in TMEM. The rows of W are the rows of a tile and the tokens its columns, however few there are: a tile is 128 rows of W by up
// to 256 tokens, and the results of a token, neighbours in memory, lie in neighbouring lanes of a warp.
//   warp 0 (one lane)  TMA producer: 128 bytes of K of the rows and of the tokens a stage (zeros behind the last of either);
//   warp 1 (one lane)  MMA issuer, four products of 32 values of K a stage;
//   warps 2-5          the sums out of TMEM, scales and bias, rows out, while the issuer fills the second accumulator.
// Where there are many tiles (kPair), the two SMs of a pair share one of 256 rows by up to 256 tokens, each with 128 rows and half of the tokens: what a stage brings in from L2 is what bounds
// one SM (48 KB for the 512 clocks of its products; 32 KB like this).
// Where rows and tokens make fewer tiles than the machine has SMs, a cluster shares a tile: its CTAs take a part of K each, leave their sums in shared memory and add up a part of the tokens each
// (whole numbers: the order does not matter).
constexpr int kL8TcThreads = 192, kL8Block = 128, kL8Stages = 12;
constexpr uint32_t kL8RowBytes = 128 * kL8Block;
constexpr int kL8Ring = 192 * 1024, kL8Smem = 1024 + kL8Ring + 512 + 4 * 256 * 4;      // operands, barriers, the tokens' scales for each of the four warps that store

struct Linear8Tc {
    Linear8Args a;
    int bn, t_tiles, units, blocks, stages, split, cols;      // tokens of a tile; tiles of tokens and in all; blocks of K; CTAs of a tile; TMEM columns of an accumulator
    int32_t* status;
    long long wait_clocks;
};

__device__ __forceinline__ int l8_peer(const void* local, uint32_t cta) {      // a word of another CTA of the cluster
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(local, cta)) : "memory");
    return v;
}

template <bool kPair>
__global__ void __launch_bounds__(kL8TcThreads, 1) linear8_tc_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const Linear8Tc p) {
    after_previous();        // in front of the allocation of TMEM: a CTA that waits for another kernel must not hold what that kernel's CTAs may be waiting for
    extern __shared__ uint8_t l8_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(l8_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kRows = kPair ? 256 : 128;
    const int a_rows = kPair ? p.bn / 2 : p.bn;              // tokens that this CTA brings in
    const uint32_t stage_bytes = kL8RowBytes + (uint32_t)a_rows * kL8Block;
    const int ST = p.stages;
    uint64_t *full = reinterpret_cast<uint64_t*>(smem + kL8Ring), *empty = full + kL8Stages, *tfull = empty + kL8Stages, *tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;    // 0 issues the pair's products
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmA);
        for (int i = 0; i < ST; ++i) { mb_init(full + i, 1); mb_init(empty + i, 1); }
        for (int i = 0; i < 2; ++i) { mb_init(tfull + i, 1); mb_init(tempty + i, kPair ? 8 : 4); }
        *gave_up = p.wait_clocks == 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (kPair) cluster_sync_all();       // the pair's forms of alloc and dealloc act on both CTAs: whoever issues one has to know that the peer runs (and, at the end, that it is still there)
    if (warp == 1) { if (kPair) tc_alloc_pair(tmem_slot, 2 * p.cols); else tc_alloc(tmem_slot, 2 * p.cols); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int group = kPair ? 2 : p.split, part = kPair ? 0 : (int)blockIdx.x % p.split, first = (int)blockIdx.x / group, step = (int)gridDim.x / group;
    const int k0 = p.blocks * part / p.split, k1 = p.blocks * (part + 1) / p.split;
    if (warp == 0) {
        if (elect_one()) {
            const uint32_t full_at = kPair ? mapa_u32(full, 0) : s_addr(full), ring = s_addr(smem);      // pair: both CTAs' bytes are counted on the first one's barriers
            int stage = 0;
            uint32_t phase = 0;
            bool ok = p.wait_clocks != 0;
            for (int unit = first; ok && unit < p.units; unit += step) {
                const int n0 = unit / p.t_tiles * kRows + (int)rank * 128, t0 = unit % p.t_tiles * p.bn + (int)rank * a_rows;
                for (int k = k0; k < k1; ++k) {
                    ok = pf_wait<kPair>(empty + stage, phase ^ 1, gave_up, p.wait_clocks);
                    if (!ok) break;
                    const uint32_t at = ring + (uint32_t)stage * stage_bytes, bar = full_at + 8 * stage;
                    if (!kPair) mb_expect(full + stage, stage_bytes);
                    else if (rank == 0) mb_expect(full + stage, 2 * stage_bytes);
                    pf_load_2d<kPair>(at, &tmW, k * kL8Block, n0, bar);
                    pf_load_2d<kPair>(at + kL8RowBytes, &tmA, k * kL8Block, t0, bar);
                    if (++stage == ST) { stage = 0; phase ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = umma_idesc_i8(kRows, p.bn);
            const uint64_t w_desc = umma_desc_sw128(smem), a_desc = umma_desc_sw128(smem + kL8RowBytes);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = p.wait_clocks != 0;
            for (int unit = first; ok && unit < p.units; unit += step) {
                ok = pf_wait<kPair>(tempty + acc, acc_phase ^ 1, gave_up, p.wait_clocks);
                if (!ok) break;
                tc_fence_after();
                for (int k = k0; k < k1; ++k) {
                    ok = pf_wait<kPair>(full + stage, phase, gave_up, p.wait_clocks);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t off = (uint64_t)((uint32_t)stage * (stage_bytes >> 4));
#pragma unroll
                    for (int i = 0; i < kL8Block / 32; ++i) {
                        if (kPair) tc_mma_i8_pair(tmem + (uint32_t)(acc * p.cols), w_desc + off + 2 * i, a_desc + off + 2 * i, idesc, k > k0 || i);
                        else tc_mma_i8(tmem + (uint32_t)(acc * p.cols), w_desc + off + 2 * i, a_desc + off + 2 * i, idesc, k > k0 || i);
                    }
                    if (kPair) tc_commit_pair(empty + stage); else tc_commit(empty + stage);
                    if (++stage == ST) { stage = 0; phase ^= 1; }
                }
                if (!ok) break;
                if (kPair) tc_commit_pair(tfull + acc); else tc_commit(tfull + acc);
                if (++acc == 2) { acc = 0; acc_phase ^= 1; }
            }
        }
        __syncwarp();
    } else {
        const int quad = warp & 3;
        const uint32_t drained[2] = {kPair ? mapa_u32(tempty, 0) : 0u, kPair ? mapa_u32(tempty + 1, 0) : 0u};
        int acc = 0;
        uint32_t acc_phase = 0;
        float* scales = reinterpret_cast<float*>(smem + kL8Ring + 512) + quad * 256;
        for (int unit = first; p.wait_clocks != 0 && unit < p.units; unit += step) {
            const int t0 = unit % p.t_tiles * p.bn;
            __syncwarp();
            for (int i = lane; i < p.bn; i += 32) scales[i] = p.a.a_scale[min(t0 + i, p.a.T - 1)];
            __syncwarp();
            if (!__all_sync(0xffffffffu, pf_wait<kPair>(tfull + acc, acc_phase, gave_up, p.wait_clocks))) break;
            tc_fence_after();
            const int n = unit / p.t_tiles * kRows + (int)rank * 128 + quad * 32 + lane;
            const bool live = n < p.a.N;
            const float ws = live ? p.a.w_scale[n] : 0.0f, bias = live && p.a.bias ? p.a.bias[n] : 0.0f;
            const uint32_t src = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * p.cols);
#pragma unroll 1
            for (int c = 0; c < p.bn; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tc_ld32(src + (uint32_t)c, v);
                if (c + 32 >= p.bn) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { if (kPair) mb_arrive_cluster(drained[acc]); else mb_arrive(tempty + acc); }
                }
                if (p.split > 1) {               // (every stage has been read: the ring is free)
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c + j < p.bn) reinterpret_cast<int*>(smem)[(c + j) * 128 + quad * 32 + lane] = (int)v[j];
                } else {
                    // (no shuffles between the stores: behind each of them the next one waited, 2000 clocks for the 32)
                    const int have = live ? min(32, min(p.bn - c, p.a.T - t0 - c)) : 0;
                    float* to = p.a.out + (size_t)(t0 + c) * p.a.ldc + n;
                    float y[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 s = *reinterpret_cast<const float4*>(scales + c + j);
                        const float t[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[j + e] = l8_value((int)v[j + e], t[e], ws, bias);
                    }
                    if (p.a.accumulate) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j < have) y[j] = __fadd_rn(to[(size_t)j * p.a.ldc], y[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (j < have) to[(size_t)j * p.a.ldc] = y[j];
                }
            }
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
        __syncwarp();
    }
    if (!kPair && p.split > 1) {                 // one tile a cluster
        cluster_sync_all();
        const int n = first / p.t_tiles * 128 + (warp & 3) * 32 + lane, t0 = first % p.t_tiles * p.bn;
        if (warp >= 2 && n < p.a.N) {
            const int* mine = reinterpret_cast<int*>(smem) + (warp & 3) * 32 + lane;
            const int have = min(p.bn, p.a.T - t0);
            const float ws = p.a.w_scale[n], bias = p.a.bias ? p.a.bias[n] : 0.0f;
            auto join = [&](auto ctas) {         // of four tokens at a time all parts are on their way before the first is added
                constexpr int S = ctas.value;
                for (int j0 = part; j0 < have; j0 += 4 * S) {
                    int v[4][S];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int r = 0; r < S; ++r) v[e][r] = l8_peer(mine + min(j0 + e * S, have - 1) * 128, (uint32_t)r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int sum = 0;
#pragma unroll
                        for (int r = 0; r < S; ++r) sum += v[e][r];
                        const int t = t0 + j0 + e * S;
                        if (j0 + e * S >= have) break;
                        float* to = p.a.out + (size_t)t * p.a.ldc + n;
                        const float y = l8_value(sum, p.a.a_scale[t], ws, bias);
                        *to = p.a.accumulate ? __fadd_rn(*to, y) : y;
                    }
                }
            };
            if (p.split == 2) join(std::integral_constant<int, 2>{});
            else if (p.split == 4) join(std::integral_constant<int, 4>{});
            else join(std::integral_constant<int, 8>{});
        }
        cluster_sync_all();                      // nobody leaves while its sums are being read
    }
    tc_fence_before();
    if (kPair) cluster_sync_all(); else __syncthreads();      // pair: nobody leaves while the peer may still signal its barriers or read its operands
    if (*gave_up) tc_gave_up(p.status);
    if (warp == 1) {
        tc_fence_after();
        if (kPair) tc_dealloc_pair(tmem, 2 * p.cols); else tc_dealloc(tmem, 2 * p.cols);
    }
    if (kPair) cluster_sync_all();
}

// Tokens of a tile, SMs (or CTAs of K) that share one: the cheapest of all, a stage reckoned at what its products or its bytes take (clocks), a wave of tiles at its beginning and end beside its
// stages. us without and with pairs, the rows' quantisation aside: 2000 x 4096 x 14336 87 | 78, 2000 x 14336 x 4096 95 | 85, 512 x 4096 x 4096 13.4 | 14.5.
struct Linear8Plan { int bn, split, pair; };
static Linear8Plan l8_plan(int T, int N, int K) {
    const int sms = sm_count(), blocks = (K + kL8Block - 1) / kL8Block, most = std::min(256, (T + 15) / 16 * 16);
    Linear8Plan best{16, 1, 0};
    double least = 1e30;
    for (int pair = 0; pair < 2; ++pair)
        for (int bn = pair ? 32 : 16; bn <= (pair ? std::min(256, (T + 31) / 32 * 32) : most); bn += pair ? 32 : 16)
            for (int split = 1; split <= (pair ? 1 : 8) && split <= blocks; split *= 2) {
                if (split > 1 && bn > 128) break;
                const long long units = (long long)((N + (pair ? 255 : 127)) / (pair ? 256 : 128)) * ((T + bn - 1) / bn) * split, workers = pair ? sms / 2 : sms;
                const double stage = std::max(2.0 * bn, (kL8RowBytes + (pair ? bn / 2 : bn) * kL8Block) / 60.0);
                const double cost = (double)((units + workers - 1) / workers) * (((blocks + split - 1) / split) * stage + (split > 1 ? 4000.0 : (pair ? 3500.0 : 1500.0) + 4.0 * bn));
                if (cost < least - 1e-9) { least = cost; best = {bn, split, pair}; }
            }
    return best;
}

static int l8_tc(const Linear8Args& a, cudaStream_t st) {
    static OncePerDevice ready;
    if (int rc = ready([&] {
            SLLM_CUDA(cudaFuncSetAttribute(linear8_tc_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kL8Smem));
            SLLM_CUDA(cudaFuncSetAttribute(linear8_tc_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kL8Smem));
            return SLLM_OK;
        }))
        return rc;
    const Linear8Plan pl = l8_plan(a.T, a.N, a.K);
    const int rows = pl.pair ? 256 : 128, a_rows = pl.pair ? pl.bn / 2 : pl.bn;
    Linear8Tc p{};
    p.a = a;
    p.bn = pl.bn;
    p.split = pl.split;
    p.t_tiles = (a.T + pl.bn - 1) / pl.bn;
    const long long units = (long long)((a.N + rows - 1) / rows) * p.t_tiles;
    SLLM_REQUIRE(units * pl.split <= 0x7fffffffLL, SLLM_ENOTSUP, "seq_linear8: %d rows for %d tokens", a.N, a.T);
    p.units = (int)units;
    p.blocks = (a.K + kL8Block - 1) / kL8Block;
    p.stages = std::min(kL8Stages, kL8Ring / ((int)kL8RowBytes + a_rows * kL8Block));
    p.cols = 32;
    while (p.cols < pl.bn) p.cols *= 2;
    if (int rc = status_check()) return rc;
    if (int rc = status_word(&p.status)) return rc;
    p.wait_clocks = kPollClocks * g_tune_tc_polls;
    CUtensorMap tmW, tmA;
    if (int rc = tc_encode_rows(&tmW, a.w, (uint64_t)a.N, a.K, a.ldw, 128)) return rc;
    if (int rc = tc_encode_rows(&tmA, a.a, (uint64_t)a.T, a.K, a.lda, a_rows)) return rc;
    const int workers = pl.pair ? std::max(1, sm_count() / 2) : sm_count(), cluster = pl.pair ? 2 : pl.split;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)cluster * (pl.split > 1 ? p.units : std::min(p.units, workers)));
    cfg.blockDim = dim3(kL8TcThreads);
    cfg.dynamicSmemBytes = kL8Smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (pl.pair) SLLM_CUDA(cudaLaunchKernelEx(&cfg, overlapping(linear8_tc_kernel<true>), tmW, tmA, p));
    else SLLM_CUDA(cudaLaunchKernelEx(&cfg, overlapping(linear8_tc_kernel<false>), tmW, tmA, p));
    ++g_launches;
    SLLM_LAUNCH_CHECK_ONLY();
    return SLLM_OK;
}

}  // namespace sllm

using namespace sllm;

extern "C" {

int sllm_seq_quantise_rows(const void* x, int32_t x_bf16, int64_t ldx, void* codes, int64_t ldc, float* scales, int32_t T, int32_t K, sllm_stream_t stream) {
    SLLM_REQUIRE(x && codes && scales && T > 0 && K > 0, SLLM_EINVAL, "seq_quantise_rows: null pointer, no rows or no columns");
    SLLM_REQUIRE(T <= 1 << 30 && K <= 1 << 30, SLLM_ENOTSUP, "seq_quantise_rows: %d rows of %d columns", T, K);
    SLLM_REQUIRE(ldx >= K && ldc >= K, SLLM_EINVAL, "seq_quantise_rows: rows of %d values lie %lld and %lld apart", K, (long long)ldx, (long long)ldc);
    const int size = x_bf16 ? 2 : 4, run = x_bf16 ? 8 : 4;
    SLLM_REQUIRE((uintptr_t)x % size == 0, SLLM_EINVAL, "seq_quantise_rows: values are not aligned");
    const bool vec = K % run == 0 && ldx % run == 0 && ((uintptr_t)x % 16) == 0 && ldc % run == 0 && ((uintptr_t)codes % run) == 0;
    QuantiseArgs p{x, (int8_t*)codes, scales, ldx, ldc, T, K};
    // threads of a row: where there are rows enough, as few as keep it in registers, so that each has eight loads on their way; else four times as many. us, few | many: 14336 rows of 4096 in bf16
    // 33 | 54, one row of 4096 in fp32 2.2 | 2.1
    const int loads = vec ? K / run : K;
    const bool many = (long long)T * loads >= 4096LL * sm_count();
    const int each = many ? kQzLoads : kQzFewLoads, threads = (std::min(kQzWide, (loads + each - 1) / each) + 31) / 32 * 32, rows = threads >= kQzThreads ? 1 : kQzThreads / threads;
    const dim3 grid((T + rows - 1) / rows), block(threads, rows);
    cudaStream_t st = as_stream(stream);
    auto launch = [&](auto bf16, auto whole) {
        if (!many) overlapping(quantise_rows_kernel<bf16.value, whole.value, kQzWide, kQzFewLoads>)<<<grid, block, 0, st>>>(p);
        else if (threads > kQzThreads) overlapping(quantise_rows_kernel<bf16.value, whole.value, kQzWide, kQzLoads>)<<<grid, block, 0, st>>>(p);
        else overlapping(quantise_rows_kernel<bf16.value, whole.value, kQzThreads, kQzLoads>)<<<grid, block, 0, st>>>(p);
    };
    using yes = std::true_type;
    using no = std::false_type;
    if (x_bf16 && vec) launch(yes{}, yes{});
    else if (x_bf16) launch(yes{}, no{});
    else if (vec) launch(no{}, yes{});
    else launch(no{}, no{});
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}

int sllm_seq_linear8(const void* a, int64_t lda, const float* a_scale, const void* w, int64_t ldw, const float* w_scale, const float* bias, float* C, int64_t ldc, int32_t T, int32_t N, int32_t K,
                     int32_t accumulate, sllm_stream_t stream) {
    SLLM_REQUIRE(a && a_scale && w && w_scale && C && T > 0 && N > 0 && K > 0, SLLM_EINVAL, "seq_linear8: null pointer or empty product");
    SLLM_REQUIRE(K <= 131072, SLLM_ENOTSUP, "seq_linear8: sums over %d products do not fit 32 bits", K);
    SLLM_REQUIRE(T <= 1 << 30 && N <= 1 << 30, SLLM_ENOTSUP, "seq_linear8: %d rows for %d tokens", N, T);
    SLLM_REQUIRE(lda >= K && ldw >= K && ldc >= N, SLLM_EINVAL, "seq_linear8: a row is shorter than its values");
    SLLM_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && (((uintptr_t)a | (uintptr_t)w) % 16) == 0, SLLM_EINVAL, "seq_linear8: rows of codes have to start at multiples of 16 bytes");
    Linear8Args p{(const int8_t*)a, (const int8_t*)w, a_scale, w_scale, bias, C, lda, ldw, ldc, T, N, K, accumulate != 0};
    cudaStream_t st = as_stream(stream);
    if (T > kL8Few) return l8_tc(p, st);
    const int rows = N < kL8Wide ? 1 : T == 1 ? 4 : 2;       // of a warp
    LaunchCfg lc(dim3((N + kL8Warps * rows - 1) / (kL8Warps * rows)), dim3(kL8Warps * 32), 0, st, true);
    if (rows == 1) SLLM_CUDA(T == 1 ? cudaLaunchKernelEx(&lc.cfg, overlapping(linear8_few_kernel<1, 1>), p) : cudaLaunchKernelEx(&lc.cfg, overlapping(linear8_few_kernel<2, 1>), p));
    else SLLM_CUDA(T == 1 ? cudaLaunchKernelEx(&lc.cfg, overlapping(linear8_few_kernel<1, 4>), p) : cudaLaunchKernelEx(&lc.cfg, overlapping(linear8_few_kernel<2, 2>), p));
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}

}  // extern "C"
