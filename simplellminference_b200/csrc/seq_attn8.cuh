// csrc/seq_attn8.cuh — what the attention kernels over the 8-bit cache share (seq_attn8.cu).
#pragma once
#include "kv8.cuh"
#include "seq_attn.cuh"

namespace sllm {

struct Attn8Args {
    sllm_seq_batch b;
    const float* q;
    int ldq, heads, kv_heads, dk, dv;
    float scale;
    const uint8_t *k_pool, *v_pool;
    const float *k_scale, *v_scale;
    int n_pages, window, keep_first, chunk;
    float softcap;
    const float* slopes;
    float* out;
    int ldo;
    uint16_t* out16;
};

#ifdef __CUDACC__

// a score after its scale: capped, then charged for its distance
__device__ __forceinline__ float attn8_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}

#endif

}  // namespace sllm
