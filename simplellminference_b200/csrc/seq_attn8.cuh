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
// of the kernel for portions (seq_attn8_tc.cu): its CTAs, floats of what one leaves of an item, and the plan of a step
constexpr int kA8TcWorkers = 160, kA8Part = 2 * 128 * 130, kA8Runs = 8192, kA8Segs = 4096;
struct A8Plan {
    int runs, pad[3];
    int seg[kA8Runs], first[kA8Runs], before[kA8Runs + 4];      // of a run of neighbouring queries: its segment, its first query there, key tiles (and beginnings) of the runs before it
    uint32_t mask[kA8Runs][8];                                  // which of its queries are in listed tiles
};
constexpr size_t kA8PlanAt = (size_t)2 * kA8Workers * sizeof(int), kA8RecordsAt = kA8PlanAt + sizeof(A8Plan),
                 kA8PartsAt = kA8RecordsAt + (size_t)kA8Workers * 2 * kA8Record * sizeof(float), kA8Ws = kA8PartsAt + (size_t)kA8TcWorkers * 2 * kA8Part * sizeof(float);
static_assert(sizeof(A8Plan) % 16 == 0, "alignment of what lies behind the plan");

// single tokens, heads of up to 128 columns (seq_attn8_decode.cu); tiles of more than one query are passed over, and reported when this launch is the step's only one
int launch_attention8_decode(const Attn8Args& p, bool only, void* ws, cudaStream_t st);
// tiles of more than one query, on tcgen05 (seq_attn8_tc.cu), and whether it takes a step like this
bool attention8_tc_takes(const Attn8Args& p);
int launch_attention8_tc(const Attn8Args& p, void* ws, cudaStream_t st);

#ifdef __CUDACC__

// a score after its scale: capped, then charged for its distance
__device__ __forceinline__ float attn8_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}

#endif

}  // namespace sllm
