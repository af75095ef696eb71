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

// Softmax weights are the sum of two fp16 numbers, whose steps end at 2^-24: they are multiplied by 2^14 first (2 of them fit fp16 then), so that a weight is off by 2^-39 of the power of two above
// the largest at most, or by 2^-22 of itself. As they are they would be off by 2^-25: a key 14 nats below the largest kept five bits of its weight, one 18 nats below none.
constexpr int kA8Lift = 14;

// The workspace: counters that every call leaves zero, then what CTAs that share an item leave of it. Its layout is the same for every step.
constexpr int kA8Workers = 512;                                        // CTAs of a launch at most
constexpr int kA8MaxHeads = 8;                                         // query heads of an item at most
constexpr int kA8Record = kA8MaxHeads * (128 + 4);                     // floats: sums of a column each, then reference, sum, exponent of a head
// of the kernel for portions (seq_attn8_tc.cu): its CTAs, floats of what one leaves of an item, bytes that say which item, and the plan of a step
constexpr int kA8TcWorkers = 160, kA8Part = 2 * 128 * 130, kA8Runs = 8192, kA8Segs = 4096, kA8Cut = 128;
constexpr int kA8Keys = 64, kA8Extra = 4;                              // keys of a tile; key tiles that an item's beginning and end count for
constexpr int kA8PlanFew = 640, kA8PlanSmem = (kA8Segs + 32 + kA8PlanFew * 10) * 4;      // runs whose masks fit shared memory; bytes
struct A8Plan {
    int runs, pad[3];
    int seg[kA8Runs], first[kA8Runs], before[kA8Runs + 4];      // of a run of neighbouring queries: its segment, its first query there, key tiles (and beginnings) of the runs before it
    uint32_t mask[kA8Runs][8];                                  // which of its queries are in listed tiles
};
constexpr size_t kA8PlanAt = (size_t)kA8Workers * sizeof(int), kA8CutsAt = kA8PlanAt + sizeof(A8Plan), kA8RecordsAt = kA8CutsAt + (size_t)kA8TcWorkers * kA8Cut,
                 kA8PartsAt = kA8RecordsAt + (size_t)kA8Workers * 2 * kA8Record * sizeof(float), kA8Ws = kA8PartsAt + (size_t)kA8TcWorkers * 2 * kA8Part * sizeof(float);
static_assert(sizeof(A8Plan) % 16 == 0, "alignment of what lies behind the plan");

// single tokens, heads of up to 128 columns (seq_attn8_decode.cu); tiles of more than one query are passed over, and reported when this launch is the step's only one.
// plan_width: the plan for runs of so many queries is made on the way (0: none)
int launch_attention8_decode(const Attn8Args& p, bool only, int plan_width, void* ws, cudaStream_t st);
// tiles of more than one query, on tcgen05 (seq_attn8_tc.cu), and whether it takes a step like this
bool attention8_tc_takes(const Attn8Args& p);
int attention8_tc_width(const Attn8Args& p);                           // queries of a run of its plan
int launch_attention8_tc(const Attn8Args& p, void* ws, cudaStream_t st);

#ifdef __CUDACC__

// The plan of the kernel for portions: which runs of `width` neighbouring queries have listed tiles, and how many key tiles each. Tiles of one query are not its. One CTA of the kernel for single
// tokens makes it (kThreads, kA8PlanSmem bytes of its shared memory), beside the others' work: a kernel of its own took 8 us in front of every step with a prompt.
template <int kThreads>
__device__ __noinline__ void a8_plan(const Attn8Args& p, int width, A8Plan* plan, void* smem) {
    const sllm_seq_batch& b = p.b;
    constexpr int kFew = kA8PlanFew;
    int* s_base = static_cast<int*>(smem);
    int *s_warp = s_base + kA8Segs, *s_seg = s_warp + 32, *s_first = s_seg + kFew;
    uint32_t* s_mask = reinterpret_cast<uint32_t*>(s_first + kFew);
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
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += s_warp[w];
            total += s_warp[w];
        }
        return before + upto - v;
    };
    int runs = 0;
    for (int s0 = 0; s0 < b.nseg; s0 += kThreads) {
        const int s = s0 + threadIdx.x, len = s < b.nseg ? b.seg_len[s] : 0;
        int total;
        const int at = scan(len > 1 ? (len + width - 1) / width : 0, total);
        if (s < b.nseg) s_base[s] = runs + at;
        runs += total;
    }
    runs = min(runs, kA8Runs);                   // (the host has made sure)
    const bool few = runs <= kFew;               // their masks fit shared memory
    for (int i = threadIdx.x; i < runs * 8; i += kThreads) {
        if (few) s_mask[i] = 0; else plan->mask[i / 8][i % 8] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < b.nseg; i += kThreads) {
        const int len = b.seg_len[i], n = len > 1 ? (len + width - 1) / width : 0;
        for (int r = 0; r < n && s_base[i] + r < runs; ++r) {
            const int at = s_base[i] + r;
            if (few) { s_seg[at] = i; s_first[at] = r * width; } else { plan->seg[at] = i; plan->first[at] = r * width; }
        }
    }
    for (int i = threadIdx.x; i < b.n_qtiles; i += kThreads) {
        const int seg = b.qt_seg[i], off = b.qt_off[i], n = min(kBQ, b.seg_len[seg] - off);
        if (n <= 1 || off < 0) continue;
        for (int q = off; q < off + n;) {        // a word of a run's mask at a time
            const int run = s_base[seg] + q / width, bit = q % width, count = min(off + n - q, 32 - bit % 32);
            if (run < runs) atomicOr(few ? &s_mask[run * 8 + bit / 32] : &plan->mask[run][bit / 32], (count == 32 ? 0xffffffffu : (1u << count) - 1) << (bit % 32));
            q += count;
        }
    }
    __syncthreads();
    __threadfence_block();
    int all = 0, kept = 0;
    for (int r0 = 0; r0 < runs; r0 += kThreads) {
        const int r = r0 + threadIdx.x;
        int units = 0, seg = 0, first = 0;
        uint32_t m[8];
        if (r < runs) {
            int lo = -1, hi = -1;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                m[w] = few ? s_mask[r * 8 + w] : *reinterpret_cast<volatile uint32_t*>(&plan->mask[r][w]);
                if (!m[w]) continue;
                if (lo < 0) lo = 32 * w + __ffs(m[w]) - 1;
                hi = 32 * w + 31 - __clz(m[w]);
            }
            seg = few ? s_seg[r] : plan->seg[r];
            first = few ? s_first[r] : plan->first[r];
            const int pos0 = b.seg_pos0[seg] + first;
            if (lo >= 0 && pos0 >= 0) units = TileList(pos0 + lo, pos0 + hi, seq_row_window(pos0 + lo, p.window, p.chunk), p.keep_first, kA8Keys).n + kA8Extra;
        }
        int total, kept_here;
        const int at = scan(units, total), to = kept + scan(units > 0, kept_here);      // (behind its barriers every run of this turn has been read)
        if (units > 0) {                         // a run without listed tiles is left out
            plan->before[to] = all + at;
            plan->seg[to] = seg;
            plan->first[to] = first;
#pragma unroll
            for (int w = 0; w < 8; ++w) plan->mask[to][w] = m[w];
        }
        all += total;
        kept += kept_here;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        plan->before[kept] = all;
        plan->runs = kept;
    }
}

// a score after its scale: capped, then charged for its distance
__device__ __forceinline__ float attn8_score(float s, float softcap, float slope, int pos, int key) {
    if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
    return fmaf(-slope, (float)(pos - key), s);
}

#endif

}  // namespace sllm
