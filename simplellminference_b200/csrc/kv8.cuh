// csrc/kv8.cuh — the 8-bit key/value cache: what appending (seq_kv8.cu) and attention (seq_attn8.cu) agree on.
//
// Pools [pages][kv_heads][page_len][width] of e4m3 codes, scales [pages][kv_heads][page_len / 32] of fp32: a value is code * scale. The scale is a power of two, the smallest
// (2^-100 at least) under which the block's largest finite magnitude is at most 448, e4m3's largest number. e4m3 is a floating format: a scale between two powers of two would
// not make a code more exact, only the range 2^15 below the largest value longer by less than one bit. What the power of two buys: dividing by it is exact, so that a code is one
// rounding away from the value (2^-4 of it at most), and a block whose scale grows keeps its older codes' values (the exponent moves; only codes that become subnormal are rounded again).
#pragma once
#include <cuda_fp16.h>

#include "seq_common.cuh"

namespace sllm {

constexpr int kKv8Block = 32;              // positions that share a scale (SLLM_KV8_BLOCK)
constexpr int kKv8LeastExp = -100;         // both the scale and its reciprocal stay normal fp32 numbers

#ifdef __CUDACC__

// exponent of the scale for a largest magnitude (finite): the least e with amax <= 448 * 2^e = 1.75 * 2^(8 + e)
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), kKv8LeastExp);
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // -126 <= e <= 127
// two values as e4m3 codes, `lo` in the low byte; NaN stays NaN
__device__ __forceinline__ uint32_t kv8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) { return kv8_pack2(a, b) | (kv8_pack2(c, d) << 16); }
// two codes (the low half of v) as fp16 values: exact, fp16 holds every e4m3 number
__device__ __forceinline__ uint32_t kv8_half2(uint32_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
    return r;
}
__device__ __forceinline__ float2 kv8_float2(uint32_t v) {
    const uint32_t h = kv8_half2(v);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// page of position `pos` of the sequence in `slot`, or -1 where the table has none that exists
__device__ __forceinline__ int kv8_page(const sllm_seq_batch& b, int n_pages, int slot, int pos) {
    const int i = pos / b.page_len;
    if (slot < 0 || pos < 0 || i >= b.max_pages) return -1;
    const int page = b.block_table[(size_t)slot * b.max_pages + i];
    return page >= 0 && page < n_pages ? page : -1;
}
__device__ __forceinline__ size_t kv8_scale_at(int page, int kv_heads, int g, int page_len, int in_page) {
    return ((size_t)page * kv_heads + g) * (page_len / kKv8Block) + in_page / kKv8Block;
}

#endif

}  // namespace sllm
