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

// The workspace: counters that every call leaves zero, then what CTAs that share an item leave for the one that is done last. Its layout is the same for every step.
constexpr int kA8Workers = 512;                                        // CTAs of a launch at most
constexpr int kA8MaxHeads = 8;                                         // query heads of an item at most
constexpr int kA8Record = kA8MaxHeads * (128 + 4);                     // floats: sums of a column each, then reference, sum, exponent of a head
constexpr size_t kA8Ws = kA8Workers * sizeof(int) + (size_t)kA8Workers * 2 * kA8Record * sizeof(float);

// single tokens, heads of up to 128 columns (seq_attn8_decode.cu); tiles of more than one query are passed over, and reported when this launch is the step's only one
int launch_attention8_decode(const Attn8Args& p, bool only, void* ws, cudaStream_t st);

#ifdef __CUDACC__

// a score after its scale: capped, then charged for its distance
__device__ __forceinline__ float attn8_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}

#endif

}  // namespace sllm
