// oxide_attn_q8.cuh -- what the two kernels of int8-cache decode attention
// share: arguments, the tile division and the form of their partial results.
//
// Partials.  Worker c of W takes tiles [c T / W, (c + 1) T / W) of the
// flattened tile space and so a run of consecutive pairs.  Its partial for
// pair g goes to part c + g: both numbers only grow along the tiles, and one
// of them grows from each partial to the next, so the parts are distinct and
// a pair's parts are consecutive; (W + pairs) parts hold them all.
#pragma once

#include "oxide_q8.cuh"
#include "oxide_tiles.cuh"

namespace oxide {

constexpr uint32_t Q8A_MAX_BATCH = 4096;   // the tile prefix of one call fits shared memory
constexpr uint32_t Q8A_MAX_D = 256;
constexpr uint32_t Q8A_PARTS = 2560;       // parts beyond two for each pair that the workspace holds

struct Q8AttnArgs {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    const void* q;             // f32 or bf16 (q_bf16)
    const int32_t* lens;       // NULL: max_seq
    float* part_ml;            // [part][nr][2]: base-2 maximum, sum
    float* part_o;             // [part][nr][q8a_dims(head_dim)], relative to the maximum
    uint32_t* err;             // set when a bounded wait ran out
    uint32_t* pre_out;         // [batch + 1] tile prefix, for the combine kernel
    uint64_t max_seq;
    uint32_t batch, q_heads, kv_heads, head_dim;
    uint32_t rep, chunks, nr;  // query heads a kv head; pieces of at most nr of them
    uint32_t nblk, shift;      // scale blocks a head, log2 of their tokens
    uint32_t workers, halves;  // halves (1 or 2): a worker's tiles go in turn to so many, each with a part of its own
    uint32_t half_dims;        // dims of a tile's half (k_attention_q8_tc.cu)
    double inv_workers;        // 1 / workers
    FastDiv by_q_heads, by_rep, by_nr, by_chunks;
    uint32_t q_bf16;
    float c1;                  // scale * log2(e)
};

// Floats a row of part_o has: whole 16-byte vectors.
__host__ __device__ __forceinline__ uint32_t q8a_dims(uint32_t head_dim) { return (head_dim + 3) & ~3u; }

__device__ __forceinline__ uint32_t q8a_len(const Q8AttnArgs& p, uint32_t b) {
    if (!p.lens) return (uint32_t)p.max_seq;
    const int32_t l = p.lens[b];
    return l <= 0 ? 0u : ((uint64_t)l < p.max_seq ? (uint32_t)l : (uint32_t)p.max_seq);
}

// floor(c T / workers), where worker c's tiles begin (c <= workers, T < 2^31): the
// f64 product is within one of it, the remainder says which.  (64-bit divisions
// took most of the combine kernel's instructions.)
__device__ __forceinline__ uint32_t q8a_start(const Q8AttnArgs& p, uint32_t c, uint32_t T) {
    const uint64_t n = (uint64_t)c * T;
    uint32_t q = (uint32_t)((double)n * p.inv_workers);
    const int64_t r = (int64_t)(n - (uint64_t)q * p.workers);
    if (r < 0) --q;
    else if (r >= (int64_t)p.workers) ++q;
    return q;
}
// The worker that has tile t: the largest c with q8a_start(c) <= t, that is
// floor(((t + 1) workers - 1) / T) -- at most 12 bits, so an f32 quotient is
// within one of it.
__device__ __forceinline__ uint32_t q8a_owner(const Q8AttnArgs& p, uint32_t t, uint32_t T) {
    const uint64_t n = ((uint64_t)t + 1) * p.workers - 1;
    uint32_t q = (uint32_t)__fdividef((float)n, (float)T);
    const int64_t r = (int64_t)(n - (uint64_t)q * T);
    if (r < 0) --q;
    else if (r >= (int64_t)T) ++q;
    return q;
}

// The key scale to use: a key whose block has a scale that is NaN, infinite or
// negative, in k or in v, has the score NaN, in both kernels alike.
__device__ __forceinline__ float q8a_key_scale(float k, float v) {
    return k >= 0.0f && k < INFINITY && v >= 0.0f && v < INFINITY ? k : q8_nan();
}

// One warp: the prefix of the batches' tile counts into shared memory, pre[0 .. batch].
__device__ __forceinline__ void q8a_prefix(const Q8AttnArgs& p, uint32_t tile, uint32_t* pre, bool store) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t carry = 0;
    for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
        const uint32_t b = b0 + lane;
        uint32_t v = b < p.batch ? (q8a_len(p, b) + tile - 1) / tile : 0u;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= (uint32_t)off) v += u;
        }
        if (b < p.batch) pre[b + 1] = carry + v;
        carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
    __syncwarp();
    if (store)
        for (uint32_t i = lane; i <= p.batch; i += 32) p.pre_out[i] = pre[i];
}

// Largest value over the warp, NaN ignored unless every lane has one.
__device__ __forceinline__ float warp_fmax(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The tcgen05 kernel (sets a.workers and a.halves); *used is false where
// shapes or device do not allow it.
cudaError_t decode_attention_q8_tc(Q8AttnArgs& a, bool withhold, cudaStream_t st, bool* used);
int decode_path();  // oxide_debug_decode_attention_path's choice

}  // namespace oxide
