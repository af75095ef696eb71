// csrc/seq_linear8.cu — products of 8-bit integers with a scale for every token and every output channel, and the rows of codes they read.
//
//   s_t = max(max_k |x_tk| / 127, 2^-126),  a_tk = round(x_tk / s_t);   C_tn = (sum_k a_tk w_nk) * s_t * v_n + bias_n
// Sums of codes are exact in 32 bits (127 * 127 * 131072 < 2^31), so a result is three roundings of fp32 away from the formula and does not depend on how a product is cut.
#include "seq_common.cuh"

namespace sllm {

// ---- rows to codes --------------------------------------------------------------------------------------------------------------------------------------------------------------------
// A row belongs to blockDim.x threads, which keep kQzValues of its values each in registers (longer rows are read a second time). The largest magnitude is taken over the values' bits, in
// whose order infinity and NaN come last: a row that has one gets the scale NaN and zeros.
// The quotient has to be the IEEE one, but a division costs some ten instructions: x times the inverse of the scale is off by less than two units of the last place (2^-16 at 127), so only quotients
// within 2^-14 of a border between two whole numbers are divided out.
constexpr int kQzValues = 16, kQzThreads = 1024;
constexpr float kQzLeast = 1.17549435e-38f;      // 2^-126

struct QuantiseArgs {
    const void* x;
    int8_t* codes;
    float* scales;
    int64_t ldx, ldc;
    int T, K;
};

__device__ __forceinline__ int qz_code(float x, float inv, float scale) {
    constexpr float magic = 12582912.0f;         // 1.5 * 2^23: a sum with it is rounded to a whole number, which the low bits hold
    const float r = x * inv, whole = r + magic, rest = fabsf(r - (whole - magic));
    if (rest > 0.5f - 6.103515625e-05f) return __float_as_int(__fdiv_rn(x, scale) + magic);
    return __float_as_int(whole);
}
__device__ __forceinline__ uint32_t qz_pack(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// value j of thread i of a row: eight neighbours (bf16) or four (fp32) to a load where rows allow that (kVec), else every blockDim.x-th value
template <bool kBf16, bool kVec>
__global__ void __launch_bounds__(kQzThreads) quantise_rows_kernel(QuantiseArgs p) {
    after_previous();
    __shared__ uint32_t s_top[kQzThreads / 32];
    constexpr int kRun = !kVec ? 1 : kBf16 ? 8 : 4;
    const int row = blockIdx.x * blockDim.y + threadIdx.y, i = threadIdx.x, n = blockDim.x, per = n * kQzValues;
    const bool live = row < p.T;
    const size_t from = (size_t)(live ? row : 0) * p.ldx;
    float v[kQzValues];
    auto column = [&](int base, int j) { return base + (j / kRun * n + i) * kRun + j % kRun; };
    auto load = [&](int base) {
#pragma unroll
        for (int j = 0; j < kQzValues; j += kRun) {
            const int c = column(base, j);
            const bool take = live && c < p.K;
            if constexpr (kRun == 8) {
                const uint4 q = take ? ld_stream(reinterpret_cast<const uint16_t*>(p.x) + from + c) : make_uint4(0u, 0u, 0u, 0u);
                v[j] = bf16_lo(q.x); v[j + 1] = bf16_hi(q.x); v[j + 2] = bf16_lo(q.y); v[j + 3] = bf16_hi(q.y);
                v[j + 4] = bf16_lo(q.z); v[j + 5] = bf16_hi(q.z); v[j + 6] = bf16_lo(q.w); v[j + 7] = bf16_hi(q.w);
            } else if constexpr (kRun == 4) {
                const uint4 q = take ? ld_stream(reinterpret_cast<const float*>(p.x) + from + c) : make_uint4(0u, 0u, 0u, 0u);
                v[j] = __uint_as_float(q.x); v[j + 1] = __uint_as_float(q.y); v[j + 2] = __uint_as_float(q.z); v[j + 3] = __uint_as_float(q.w);
            } else if constexpr (kBf16) {
                v[j] = take ? seq_ld(reinterpret_cast<const uint16_t*>(p.x), from + c) : 0.0f;
            } else {
                v[j] = take ? reinterpret_cast<const float*>(p.x)[from + c] : 0.0f;
            }
        }
    };
    uint32_t top = 0;
    for (int base = 0; base < p.K; base += per) {
        load(base);
#pragma unroll
        for (int j = 0; j < kQzValues; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (n > 32) {
        const int warp = (threadIdx.y * n + i) >> 5, first = threadIdx.y * n >> 5;
        if ((i & 31) == 0) s_top[warp] = top;
        __syncthreads();
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
        for (int j = 0; j < kQzValues; j += kRun) {
            const int c = column(base, j);
            if (c >= p.K) continue;
            int q[kRun];
#pragma unroll
            for (int e = 0; e < kRun; ++e) q[e] = finite ? qz_code(v[j + e], inv, scale) : 0;
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

__device__ __forceinline__ void l8_store(const Linear8Args& p, int t, int n, int sum) {
    float v = (float)sum * p.a_scale[t] * p.w_scale[n];
    if (p.bias) v += p.bias[n];
    float* to = p.out + (size_t)t * p.ldc + n;
    *to = p.accumulate ? *to + v : v;
}

// A warp takes two rows of W and kT tokens: sixteen codes a load, four products an instruction.
constexpr int kL8Warps = 8, kL8Rows = 2;
template <int kT>
__global__ void __launch_bounds__(kL8Warps * 32) linear8_few_kernel(Linear8Args p) {
    after_previous();
    const int lane = threadIdx.x & 31, n0 = (blockIdx.x * kL8Warps + (threadIdx.x >> 5)) * kL8Rows, t0 = blockIdx.y * kT;
    if (n0 >= p.N) return;
    int sum[kL8Rows][kT] = {};
    const int8_t *w[kL8Rows], *a[kT];
#pragma unroll
    for (int r = 0; r < kL8Rows; ++r) w[r] = p.w + (size_t)min(n0 + r, p.N - 1) * p.ldw;
#pragma unroll
    for (int t = 0; t < kT; ++t) a[t] = p.a + (size_t)min(t0 + t, p.T - 1) * p.lda;
#pragma unroll 4
    for (int c = lane * 16; c < p.K; c += 512) {
        uint4 x[kL8Rows];
#pragma unroll
        for (int r = 0; r < kL8Rows; ++r) x[r] = ld_stream(w[r] + c);
        if (c + 16 > p.K) {                      // columns behind the last one: whatever the rows hold there does not count
            const int have = p.K - c;
            auto keep = [&](uint32_t v, int first) { return have >= first + 4 ? v : have <= first ? 0u : v & ((1u << 8 * (have - first)) - 1); };
#pragma unroll
            for (int r = 0; r < kL8Rows; ++r) x[r] = make_uint4(keep(x[r].x, 0), keep(x[r].y, 4), keep(x[r].z, 8), keep(x[r].w, 12));
        }
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const uint4 y = *reinterpret_cast<const uint4*>(a[t] + c);
#pragma unroll
            for (int r = 0; r < kL8Rows; ++r)
                sum[r][t] = __dp4a((int)x[r].w, (int)y.w, __dp4a((int)x[r].z, (int)y.z, __dp4a((int)x[r].y, (int)y.y, __dp4a((int)x[r].x, (int)y.x, sum[r][t]))));
        }
    }
#pragma unroll
    for (int r = 0; r < kL8Rows; ++r)
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const int v = __reduce_add_sync(0xffffffffu, sum[r][t]);
            if (lane == 0 && n0 + r < p.N && t0 + t < p.T) l8_store(p, t0 + t, n0 + r, v);
        }
}

}  // namespace sllm

using namespace sllm;

extern "C" {

int sllm_seq_quantise_rows(const void* x, int32_t x_bf16, int64_t ldx, void* codes, int64_t ldc, float* scales, int32_t T, int32_t K, sllm_stream_t stream) {
    SLLM_REQUIRE(x && codes && scales && T > 0 && K > 0, SLLM_EINVAL, "seq_quantise_rows: null pointer, no rows or no columns");
    SLLM_REQUIRE(ldx >= K && ldc >= K, SLLM_EINVAL, "seq_quantise_rows: rows of %d values lie %lld and %lld apart", K, (long long)ldx, (long long)ldc);
    const int size = x_bf16 ? 2 : 4, run = x_bf16 ? 8 : 4;
    SLLM_REQUIRE((uintptr_t)x % size == 0, SLLM_EINVAL, "seq_quantise_rows: values are not aligned");
    const bool vec = K % run == 0 && ldx % run == 0 && ((uintptr_t)x % 16) == 0 && ldc % run == 0 && ((uintptr_t)codes % run) == 0;
    QuantiseArgs p{x, (int8_t*)codes, scales, ldx, ldc, T, K};
    // threads of a row: enough to keep it in registers; short rows share a CTA
    const int threads = std::min(kQzThreads, std::max(32, (K + kQzValues - 1) / kQzValues + 31) / 32 * 32), rows = std::max(1, 128 / threads);
    const dim3 grid((T + rows - 1) / rows), block(threads, rows);
    cudaStream_t st = as_stream(stream);
    if (x_bf16 && vec) overlapping(quantise_rows_kernel<true, true>)<<<grid, block, 0, st>>>(p);
    else if (x_bf16) overlapping(quantise_rows_kernel<true, false>)<<<grid, block, 0, st>>>(p);
    else if (vec) overlapping(quantise_rows_kernel<false, true>)<<<grid, block, 0, st>>>(p);
    else overlapping(quantise_rows_kernel<false, false>)<<<grid, block, 0, st>>>(p);
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}

int sllm_seq_linear8(const void* a, int64_t lda, const float* a_scale, const void* w, int64_t ldw, const float* w_scale, const float* bias, float* C, int64_t ldc, int32_t T, int32_t N, int32_t K,
                     int32_t accumulate, sllm_stream_t stream) {
    SLLM_REQUIRE(a && a_scale && w && w_scale && C && T > 0 && N > 0 && K > 0, SLLM_EINVAL, "seq_linear8: null pointer or empty product");
    SLLM_REQUIRE(K <= 131072, SLLM_ENOTSUP, "seq_linear8: sums over %d products do not fit 32 bits", K);
    SLLM_REQUIRE(lda >= K && ldw >= K && ldc >= N, SLLM_EINVAL, "seq_linear8: a row is shorter than its values");
    SLLM_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && (((uintptr_t)a | (uintptr_t)w) % 16) == 0, SLLM_EINVAL, "seq_linear8: rows of codes have to start at multiples of 16 bytes");
    Linear8Args p{(const int8_t*)a, (const int8_t*)w, a_scale, w_scale, bias, C, lda, ldw, ldc, T, N, K, accumulate != 0};
    cudaStream_t st = as_stream(stream);
    const int wide = (N + kL8Warps * kL8Rows - 1) / (kL8Warps * kL8Rows), per = T > 2 ? 4 : T;
    SLLM_REQUIRE((T + per - 1) / per <= 65535, SLLM_ENOTSUP, "seq_linear8: %d tokens", T);
    const dim3 grid(wide, (T + per - 1) / per);
    if (per == 1) overlapping(linear8_few_kernel<1>)<<<grid, kL8Warps * 32, 0, st>>>(p);
    else if (per == 2) overlapping(linear8_few_kernel<2>)<<<grid, kL8Warps * 32, 0, st>>>(p);
    else overlapping(linear8_few_kernel<4>)<<<grid, kL8Warps * 32, 0, st>>>(p);
    ++g_launches;
    SLLM_LAUNCH_CHECK();
    return SLLM_OK;
}

}  // extern "C"
