// oxide_tiles.cuh -- work division of the decode-attention kernels: the
// (batch, kv head) pairs' key tiles laid end to end (pair order batch-major)
// and cut into equal ranges, one for each worker.
#pragma once

#include "oxide_common.cuh"

namespace oxide {

// Walks the flattened tile space in order: pair (b, kvh), tile lt of tb.
struct TileWalk {
    const uint32_t* pre;  // pre[b] = tiles per kv head of batches < b; pre[B] = total
    uint32_t nb, hkv;
    uint32_t b, kvh, lt, tb;
    __device__ void seek(uint32_t t) {
        // the batch holding global tile t: pre[b] * hkv <= t < pre[b + 1] * hkv
        uint32_t lo = 0, hi = nb;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (pre[mid] * hkv <= t) lo = mid;
            else hi = mid;
        }
        b = lo;
        while (b + 1 < nb && pre[b + 1] * hkv <= t) ++b;  // skip batches without tiles
        tb = pre[b + 1] - pre[b];
        const uint32_t r = t - pre[b] * hkv;
        kvh = tb ? r / tb : 0;
        lt = tb ? r % tb : 0;
    }
    __device__ void next() {
        if (++lt < tb) return;
        lt = 0;
        if (++kvh < hkv) return;
        kvh = 0;
        do {
            ++b;
            tb = b < nb ? pre[b + 1] - pre[b] : 0;
        } while (b < nb && tb == 0);
    }
};

// The CTA (of G) whose tile range holds global tile t: the largest c with
// floor(c T / G) <= t.
__device__ __forceinline__ uint32_t tc_owner(uint32_t t, uint32_t T, uint32_t G) {
    return (uint32_t)((((uint64_t)t + 1) * G - 1) / T);
}

}  // namespace oxide
