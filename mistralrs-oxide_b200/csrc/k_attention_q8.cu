// k_attention_q8.cu -- one-token (decode) attention over int8 KV caches with a
// scale for each block of tokens and head (the caches of k_kvcache_q8.cu).
//
// Reference: the attention of src/ops/attention.rs:41-87 for q_len = 1, with
// the head map of repeat_kv (:161-201); the 8-bit cache is an addition.
// With codes c, d and scales ks, vs of key j's block:
//     s_j = (q . c_j) ks scale,  p = softmax(s),  out = sum_j p_j vs d_j:
// the scales factor out of both products, so codes enter them as they are.
//
// Two kernels write partial results in one form (oxide_attn_q8.cuh) and
// decode_attn_q8_combine_kernel merges them:
//   k_attention_q8_tc.cu   head_dim a multiple of 16: both products in int8 on
//                          tcgen05;
//   here, any other shape  (head_dim up to 256, any group, more than 1024
//                          sequences): a warp is a worker and streams 32-key
//                          tiles.  Scores: lane = key, its row read in words of
//                          16 or 4 bytes against the group's query heads in
//                          shared memory; P V: lane = four dims, each key's
//                          weights broadcast by shuffles.  f32 throughout.
// Bound by HBM bytes, 2 head_dim a key and kv head; the kernel here by its
// instructions, some 1200 for 32 keys and four heads: 8 sequences of 16384 keys,
// 32 heads over 8, head_dim 37, take 139 us (214 with a load a byte and a dim a
// lane), 0.56 TB/s; 32 of 4096 keys, head_dim 20, 60 us (96 with one key at a time).
#include "oxide_attn_q8.cuh"

namespace oxide {

constexpr int QW_WARPS = 8;
constexpr uint32_t QW_TK = 32;  // keys a tile

// The four bytes at `a`, which need not lie on a word: from the aligned words
// around them, neither of them behind `last`, the word of the array's last byte
// (bytes behind it are anything: they are nobody's dims).
__device__ __forceinline__ uint32_t qw_word(const int8_t* a, const uint32_t* last) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(a);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(u & ~(uintptr_t)3);
    const uint32_t lo = __ldg(w), hi = __ldg(w < last ? w + 1 : last);
    return __funnelshift_r(lo, hi, 8u * (uint32_t)(u & 3));
}

// A lane owns four dims of every 128 (NG of them) in P V; head_dim up to 64 and
// 32 leaves half of the lanes and more without dims, so KG = 2 and 4 keys are
// taken at once.  WORDS: rows start on words (head_dim a multiple of 4, aligned
// caches); else words are put together from two.
template <int NR, int NG, int KG, bool WORDS>
__global__ void __launch_bounds__(QW_WARPS * 32, 2) decode_attn_q8_warp_kernel(Q8AttnArgs p) {
    pdl_begin();
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int W = 4, LANES = 32 / KG;  // dims a lane and group; lanes a key
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kg = lane / LANES, dl = lane % LANES;
    const uint32_t D = p.head_dim, DP = (D + 3) & ~3u;
    float* qs = reinterpret_cast<float*>(smem) + (size_t)warp * NR * DP;  // this warp's query heads [NR][DP]
    uint32_t* pre = reinterpret_cast<uint32_t*>(smem + (size_t)QW_WARPS * NR * DP * 4);
    if (warp == 0) q8a_prefix(p, QW_TK, pre, blockIdx.x == 0);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0u;
    __syncthreads();
    const uint32_t heads = p.kv_heads * p.chunks;
    const uint32_t T = pre[p.batch] * heads, G = p.workers;
    const uint32_t c = blockIdx.x * QW_WARPS + warp;
    if (c >= G) return;
    const uint32_t t0 = q8a_start(p, c, T), t1 = q8a_start(p, c + 1, T);
    if (t0 >= t1) return;
    TileWalk w{pre, p.batch, heads, 0, 0, 0, 0};
    w.seek(t0);
    float m[NR], l[NR], acc[NR][NG * W];
    uint32_t nh = 0, len = 0;
    const int8_t *kh = nullptr, *vh = nullptr;
    const float *ksh = nullptr, *vsh = nullptr;
    const uint64_t bytes = (uint64_t)p.batch * p.kv_heads * p.max_seq * D;
    auto last_word = [&](const int8_t* c) {
        return reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(c + bytes - 1) & ~(uintptr_t)3);
    };
    const uint32_t *klast = last_word(p.kc), *vlast = last_word(p.vc);
    for (uint32_t t = t0; t < t1; ++t, w.next()) {
        if (t == t0 || w.lt == 0) {  // a new pair: its query heads and caches
            const uint32_t kvh = p.by_chunks.div(w.kvh), h0 = (w.kvh - kvh * p.chunks) * NR;
            nh = min(p.rep - h0, (uint32_t)NR);
            len = q8a_len(p, w.b);
            const uint64_t bh = (uint64_t)w.b * p.kv_heads + kvh, row = (uint64_t)w.b * p.q_heads + kvh * p.rep + h0;
            kh = p.kc + bh * p.max_seq * D;
            vh = p.vc + bh * p.max_seq * D;
            ksh = p.ks + bh * p.nblk;
            vsh = p.vs + bh * p.nblk;
            __syncwarp();
            for (uint32_t i = lane; i < NR * DP; i += 32) {
                const uint32_t h = i / DP, d = i - h * DP;
                float v = 0.0f;
                if (h < nh && d < D) {
                    const uint64_t at = (row + h) * D + d;
                    v = p.q_bf16 ? Vec<bf16_t>::load1(static_cast<const bf16_t*>(p.q) + at)
                                 : Vec<float>::load1(static_cast<const float*>(p.q) + at);
                }
                qs[i] = v;
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                m[h] = -INFINITY;
                l[h] = 0.0f;
#pragma unroll
                for (int e = 0; e < NG * W; ++e) acc[h][e] = 0.0f;
            }
        }
        const uint32_t key0 = w.lt * QW_TK, nk = min(len - key0, QW_TK);
        const bool on = (uint32_t)lane < nk;
        float dot[NR], ks = 0.0f, vs = 0.0f;
#pragma unroll
        for (int h = 0; h < NR; ++h) dot[h] = 0.0f;
        if (on) {
            const uint32_t key = key0 + lane;
            vs = __ldg(vsh + (key >> p.shift));
            ks = q8a_key_scale(__ldg(ksh + (key >> p.shift)), vs);
            const int8_t* row = kh + (uint64_t)key * D;
            if (WORDS && D % 16 == 0) {
#pragma unroll 4
                for (uint32_t i = 0; i < D; i += 16) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + i));
                    const uint32_t wd[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float f[4];
                        q8_unpack4(wd[e], f);
#pragma unroll
                        for (int h = 0; h < NR; ++h) {
                            const float4 qv = *reinterpret_cast<const float4*>(qs + h * DP + i + 4 * e);
                            dot[h] = __fmaf_rn(f[0], qv.x, dot[h]);
                            dot[h] = __fmaf_rn(f[1], qv.y, dot[h]);
                            dot[h] = __fmaf_rn(f[2], qv.z, dot[h]);
                            dot[h] = __fmaf_rn(f[3], qv.w, dot[h]);
                        }
                    }
                }
            } else {
#pragma unroll 4
                for (uint32_t i = 0; i < D; i += 4) {  // (qs is zero past head_dim)
                    float f[4];
                    q8_unpack4(WORDS ? __ldg(reinterpret_cast<const unsigned int*>(row + i)) : qw_word(row + i, klast), f);
#pragma unroll
                    for (int h = 0; h < NR; ++h) {
                        const float4 qv = *reinterpret_cast<const float4*>(qs + h * DP + i);
                        dot[h] = __fmaf_rn(f[0], qv.x, dot[h]);
                        dot[h] = __fmaf_rn(f[1], qv.y, dot[h]);
                        dot[h] = __fmaf_rn(f[2], qv.z, dot[h]);
                        dot[h] = __fmaf_rn(f[3], qv.w, dot[h]);
                    }
                }
            }
        }
        float pv[NR];
        const float kf = fmul(ks, p.c1);
#pragma unroll
        for (int h = 0; h < NR; ++h) {
            const float s = on ? fmul(dot[h], kf) : -INFINITY;
            const float mn = fmaxf(m[h], warp_fmax(s));
            const float cr = m[h] == -INFINITY ? 0.0f : ex2_approx(fsub(m[h], mn));
            const float pr = s == -INFINITY ? 0.0f : ex2_approx(fsub(s, mn));  // a NaN score stays NaN
            m[h] = mn;
            l[h] = __fmaf_rn(l[h], cr, pr);
            pv[h] = on ? fmul(pr, vs) : 0.0f;
#pragma unroll
            for (int e = 0; e < NG * W; ++e) acc[h][e] = fmul(acc[h][e], cr);
        }
        const int8_t* vrow = vh + (uint64_t)key0 * D;
#pragma unroll 8
        for (uint32_t j0 = 0; j0 < nk; j0 += KG) {
            const uint32_t j = j0 + kg;  // (keys past nk: their weight is zero)
            float f[NG][W];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t d = W * (dl + 32 * g);
                const int8_t* at = vrow + (uint64_t)j * D + d;
                uint32_t x = 0u;
                if (d < D && (KG == 1 || j < nk))
                    x = WORDS ? __ldg(reinterpret_cast<const unsigned int*>(at)) : qw_word(at, vlast);
                q8_unpack4(x, f[g]);
            }
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                const float x = __shfl_sync(0xffffffffu, pv[h], j);
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[h][g * W + e] = __fmaf_rn(x, f[g][e], acc[h][g * W + e]);
            }
        }
        if (t + 1 == t1 || w.lt + 1 == w.tb) {  // this worker's last tile of the pair
            const uint64_t part = (uint64_t)c + (uint64_t)w.b * heads + w.kvh;
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                const float ls = warp_sum(l[h]);
#pragma unroll
                for (int o = LANES; o < 32; o *= 2)  // the keys taken at once
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[h][e] = fadd(acc[h][e], __shfl_xor_sync(0xffffffffu, acc[h][e], o));
                if ((uint32_t)h >= nh) continue;
                const uint64_t slot = part * NR + h;
                if (lane == 0) {
                    p.part_ml[slot * 2] = m[h];
                    p.part_ml[slot * 2 + 1] = ls;
                }
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const uint32_t d = W * (dl + 32 * g) + e;
                        if (kg == 0 && d < D) p.part_o[slot * DP + d] = acc[h][g * W + e];
                    }
            }
        }
    }
}

// Merge the parts of one (batch, query head): with NW warps, warp w takes every
// NW-th part of the pair, the loads of QC_UNROLL of them in flight at once (the
// parts' places follow from the tile division alone), lane = four dims (DV of
// them 128 apart), and the NW states are joined through shared memory.  A part
// whose scores are all -infinity has sum 0.  A pair without keys gives zeros; one
// with keys and no weight (every score -infinity) gives NaN, as 0 / 0 in the
// definition, and so does everything if a wait of the main kernel ran out.
// NW: 8 warps while there are fewer CTAs than SMs -- a CTA then merges many
// parts (one sequence of 131072 keys, 37 parts a head: the whole call 51.0 us
// against 53.0 with 4) -- else 4, so that more CTAs are resident at once (8
// sequences of 1024 to 32768, 256 CTAs: 54.7 us against 55.9 with 8).  With as
// many pairs as workers have parts, a head has four parts or fewer on average,
// which one warp loads at once: EACH gives a head to each of a CTA's four warps
// (2048 pairs 51.2 us against 57.5 without, 512 pairs 22.4 against 22.7; but 150
// pairs 43.1 against 41.7).  A long sequence among short ones, whose heads then have
// hundreds of parts, gains nothing from four warps that take a CTA's heads in turn
// (65536 keys beside 399 sequences of 60, 296 parts: 87 us against 82).
constexpr int QC_UNROLL = 5;
struct Q8Parts {  // the parts of a head: workers c0 .. that had tiles tfirst .. tend - 1 of its pair
    uint32_t pair, h, tfirst, tend, c0, n;
};
__device__ __forceinline__ Q8Parts q8_parts(const Q8AttnArgs& p, uint32_t bh, uint32_t heads, uint32_t all) {
    const uint32_t b = p.by_q_heads.div(bh), qh = bh - b * p.q_heads;
    const uint32_t kvh = p.by_rep.div(qh), r = qh - kvh * p.rep, chunk = p.by_nr.div(r);
    const uint32_t before = p.pre_out[b], tb = p.pre_out[b + 1] - before;
    Q8Parts x{b * heads + kvh * p.chunks + chunk, r - chunk * p.nr, 0, 0, 0, 0};
    if (tb) {
        x.tfirst = before * heads + (x.pair - b * heads) * tb;
        x.tend = x.tfirst + tb;
        x.c0 = q8a_owner(p, x.tfirst, all);
        x.n = (q8a_owner(p, x.tend - 1, all) - x.c0 + 1) * p.halves;
    }
    return x;
}
template <int DV>
struct Q8State {
    float M, L;
    float4 acc[DV];
};
// The parts first, first + step, ... of a head.
template <int DV>
__device__ __forceinline__ Q8State<DV> q8_merge(const Q8AttnArgs& p, const Q8Parts& x, uint32_t all, uint32_t first,
                                                uint32_t step, uint32_t lane) {
    const uint32_t DP = q8a_dims(p.head_dim);
    Q8State<DV> s;
    s.M = -INFINITY;
    s.L = 0.0f;
#pragma unroll
    for (int k = 0; k < DV; ++k) s.acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = first; i0 < x.n; i0 += step * QC_UNROLL) {
        float ms[QC_UNROLL], ls[QC_UNROLL];
        float4 o[QC_UNROLL][DV];
#pragma unroll
        for (int u = 0; u < QC_UNROLL; ++u) {
            const uint32_t i = i0 + u * step, c = x.c0 + (i >> (p.halves - 1)), half = i & (p.halves - 1);
            ms[u] = -INFINITY;
            ls[u] = 0.0f;
#pragma unroll
            for (int k = 0; k < DV; ++k) o[u][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i >= x.n) continue;
            const uint32_t f0 = q8a_start(p, c, all), f1 = q8a_start(p, c + 1, all);
            const uint32_t a = max(f0, x.tfirst), e = min(f1, x.tend);
            if (a >= e || (e - a < p.halves && ((a - f0) ^ half) & 1)) continue;  // no tile, or the other half's one tile
            const uint64_t slot = (((uint64_t)c + x.pair) * p.halves + half) * p.nr + x.h;
            ms[u] = p.part_ml[slot * 2];
            ls[u] = p.part_ml[slot * 2 + 1];
#pragma unroll
            for (int k = 0; k < DV; ++k) {
                const uint32_t d = 4 * (lane + 32 * k);
                if (d < DP) o[u][k] = *reinterpret_cast<const float4*>(p.part_o + slot * DP + d);
            }
        }
#pragma unroll
        for (int u = 0; u < QC_UNROLL; ++u) {
            if (ls[u] == 0.0f) continue;
            const float mn = fmaxf(s.M, ms[u]);
            const float cr = s.M == -INFINITY ? 0.0f : ex2_approx(fsub(s.M, mn)), w = ex2_approx(fsub(ms[u], mn));
            s.L = __fmaf_rn(ls[u], w, fmul(s.L, cr));
#pragma unroll
            for (int k = 0; k < DV; ++k) {
                s.acc[k].x = __fmaf_rn(o[u][k].x, w, fmul(s.acc[k].x, cr));
                s.acc[k].y = __fmaf_rn(o[u][k].y, w, fmul(s.acc[k].y, cr));
                s.acc[k].z = __fmaf_rn(o[u][k].z, w, fmul(s.acc[k].z, cr));
                s.acc[k].w = __fmaf_rn(o[u][k].w, w, fmul(s.acc[k].w, cr));
            }
            s.M = mn;
        }
    }
    return s;
}

template <typename T, int DV, int NW, bool EACH>
__global__ void __launch_bounds__(NW * 32) decode_attn_q8_combine_kernel(T* out, Q8AttnArgs p) {
    pdl_begin();
    __shared__ float wm[NW], wl[NW];
    __shared__ float4 wo[NW][32 * DV];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t heads = p.kv_heads * p.chunks, D = p.head_dim, all = p.pre_out[p.batch] * heads;
    const uint32_t failed = *p.err, bh = EACH ? blockIdx.x * NW + warp : blockIdx.x;
    if (EACH && bh >= p.batch * p.q_heads) return;
    const Q8Parts x = q8_parts(p, bh, heads, all);
    const Q8State<DV> s = q8_merge<DV>(p, x, all, EACH ? 0 : warp, EACH ? 1 : NW, lane);
    const float none = x.n == 0 ? 0.0f : q8_nan();
    if constexpr (EACH) {
#pragma unroll
        for (int k = 0; k < DV; ++k) {
            const float o[4] = {s.acc[k].x, s.acc[k].y, s.acc[k].z, s.acc[k].w};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const uint32_t d = 4 * (lane + 32 * k) + e;
                const float y = failed ? q8_nan() : (s.L == 0.0f ? none : fdiv(o[e], s.L));
                if (d < D) Vec<T>::store1(out + (uint64_t)bh * D + d, y);
            }
        }
    } else {
        if (lane == 0) {
            wm[warp] = s.M;
            wl[warp] = s.L;
        }
#pragma unroll
        for (int k = 0; k < DV; ++k) wo[warp][lane + 32 * k] = s.acc[k];
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < D; d += NW * 32) {
            float mx = -INFINITY, ls = 0.0f, o = 0.0f;
#pragma unroll
            for (int i = 0; i < NW; ++i) mx = fmaxf(mx, wm[i]);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (wl[i] == 0.0f) continue;
                const float f = ex2_approx(fsub(wm[i], mx));
                ls = __fmaf_rn(wl[i], f, ls);
                o = __fmaf_rn(reinterpret_cast<const float*>(wo[i])[d], f, o);
            }
            float y = ls == 0.0f ? none : fdiv(o, ls);
            if (failed) y = q8_nan();
            Vec<T>::store1(out + (uint64_t)bh * D + d, y);
        }
    }
}

int q8_block_shift(uint64_t block);
int q8_cache_check(const char* name, uint64_t batch, uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim,
                   uint64_t block);

template <int NR, int NG, int KG, bool WORDS>
static cudaError_t launch_warp(Q8AttnArgs& a, cudaStream_t st) {
    auto kern = decode_attn_q8_warp_kernel<NR, NG, KG, WORDS>;
    const size_t smem = (size_t)QW_WARPS * NR * ((a.head_dim + 3) & ~3u) * 4 + (a.batch + 1) * 4;
    if (!ensure_dyn_smem(reinterpret_cast<const void*>(kern), smem)) return cudaErrorInvalidConfiguration;
    // one worker a resident warp, as many as the workspace has parts for
    uint64_t ctas = (uint64_t)resident_blocks(reinterpret_cast<const void*>(kern), QW_WARPS * 32, smem);
    if (ctas > Q8A_PARTS / QW_WARPS) ctas = Q8A_PARTS / QW_WARPS;
    const uint64_t tiles = (uint64_t)a.batch * a.kv_heads * a.chunks * ((a.max_seq + QW_TK - 1) / QW_TK);
    if (ctas > (tiles + QW_WARPS - 1) / QW_WARPS) ctas = (tiles + QW_WARPS - 1) / QW_WARPS;
    a.workers = (uint32_t)ctas * QW_WARPS;
    a.inv_workers = 1.0 / a.workers;
    return launch_k(kern, (unsigned)ctas, QW_WARPS * 32, smem, st, a);
}
template <int NR, bool WORDS>
static cudaError_t launch_warp_d(Q8AttnArgs& a, cudaStream_t st) {
    if (a.head_dim > 128) return launch_warp<NR, 2, 1, WORDS>(a, st);
    if (a.head_dim > 64) return launch_warp<NR, 1, 1, WORDS>(a, st);
    return a.head_dim > 32 ? launch_warp<NR, 1, 2, WORDS>(a, st) : launch_warp<NR, 1, 4, WORDS>(a, st);
}
template <bool WORDS>
static cudaError_t launch_warp_nr(Q8AttnArgs& a, cudaStream_t st) {
    switch (a.nr) {
        case 1: return launch_warp_d<1, WORDS>(a, st);
        case 2: return launch_warp_d<2, WORDS>(a, st);
        case 4: return launch_warp_d<4, WORDS>(a, st);
        default: return launch_warp_d<8, WORDS>(a, st);
    }
}

template <typename T, int DV>
static cudaError_t launch_combine(T* out, const Q8AttnArgs& a, cudaStream_t st) {
    const unsigned grid = a.batch * a.q_heads;
    if ((uint64_t)a.batch * a.kv_heads * a.chunks >= (uint64_t)a.halves * a.workers)
        return launch_k(decode_attn_q8_combine_kernel<T, DV, 4, true>, (grid + 3) / 4, 128, 0, st, out, a);
    return grid < (unsigned)sm_count() ? launch_k(decode_attn_q8_combine_kernel<T, DV, 8, false>, grid, 256, 0, st, out, a)
                                       : launch_k(decode_attn_q8_combine_kernel<T, DV, 4, false>, grid, 128, 0, st, out, a);
}

static uint64_t attn_q8_parts(uint64_t batch, uint64_t q_heads, uint64_t kv_heads) {
    // pairs: pieces of up to 8 query heads of each kv head; workers * halves <= Q8A_PARTS
    const uint64_t rep = kv_heads ? q_heads / kv_heads : 0, chunks = (rep + 7) / 8;
    return 2 * batch * kv_heads * chunks + Q8A_PARTS;
}
static uint64_t attn_q8_nr(uint64_t q_heads, uint64_t kv_heads) {
    const uint64_t rep = kv_heads ? q_heads / kv_heads : 0;
    return rep <= 1 ? 1 : (rep <= 2 ? 2 : (rep <= 4 ? 4 : 8));
}

template <typename T>
static int attn_q8_entry(const char* name, const T* q, const int8_t* kc, const int8_t* vc, const float* ks,
                         const float* vs, const int32_t* lens, T* out, uint64_t batch, uint64_t q_heads,
                         uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim, uint64_t block, float scale, void* ws,
                         uint64_t ws_bytes, cudaStream_t st) {
    OXIDE_INJECT(name);
    if (int rc = q8_cache_check(name, batch, kv_heads, max_seq, head_dim, block)) return rc;
    if (batch == 0 || q_heads == 0) return OXIDE_OK;
    OXIDE_REQUIRE(q && kc && vc && ks && vs && out, name, "null pointer");
    OXIDE_REQUIRE(kv_heads >= 1 && q_heads % kv_heads == 0, name, "q_heads must be a multiple of kv_heads");
    OXIDE_REQUIRE(head_dim >= 1 && head_dim <= Q8A_MAX_D, name, "head_dim must be in [1, 256]");
    OXIDE_REQUIRE(q_heads < (1u << 20) && max_seq >= 1, name, "q_heads must be < 2^20 and max_seq >= 1");
    OXIDE_REQUIRE(batch <= Q8A_MAX_BATCH && batch * q_heads < (1ull << 31), name,
                  "batch must be <= 4096 and batch * q_heads < 2^31");
    OXIDE_REQUIRE(out != q, name, "out must not alias q");
    const uint64_t rep = q_heads / kv_heads, nr = attn_q8_nr(q_heads, kv_heads), chunks = (rep + 7) / 8;
    // the flattened tile index is 32 bits wide (tiles of at least 32 keys)
    OXIDE_REQUIRE(batch * kv_heads * chunks * ((max_seq + QW_TK - 1) / QW_TK) < (1ull << 31), name,
                  "too many keys for one call: batch * kv_heads * max_seq must be < 2^36 (for up to 8 query heads a kv head)");
    const uint64_t need = oxide_decode_attention_q8_workspace_bytes(batch, q_heads, kv_heads, head_dim);
    if (!ws || ws_bytes < need || !aligned16(ws))
        return set_error(OXIDE_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned and >= %llu bytes", name,
                         (unsigned long long)need);
    const uint64_t parts = attn_q8_parts(batch, q_heads, kv_heads);
    Q8AttnArgs a{};
    a.kc = kc;
    a.vc = vc;
    a.ks = ks;
    a.vs = vs;
    a.q = q;
    a.lens = lens;
    a.part_o = static_cast<float*>(ws);
    a.part_ml = a.part_o + parts * nr * q8a_dims((uint32_t)head_dim);
    a.err = reinterpret_cast<uint32_t*>(a.part_ml + parts * nr * 2);
    a.pre_out = a.err + 4;
    a.max_seq = max_seq;
    a.batch = (uint32_t)batch;
    a.q_heads = (uint32_t)q_heads;
    a.kv_heads = (uint32_t)kv_heads;
    a.head_dim = (uint32_t)head_dim;
    a.rep = (uint32_t)rep;
    a.chunks = (uint32_t)chunks;
    a.nr = (uint32_t)nr;
    a.shift = (uint32_t)q8_block_shift(block);
    a.nblk = (uint32_t)((max_seq + block - 1) / block);
    a.halves = 1;
    a.by_q_heads = FastDiv(a.q_heads);
    a.by_rep = FastDiv(a.rep);
    a.by_nr = FastDiv(a.nr);
    a.by_chunks = FastDiv(a.chunks);
    a.q_bf16 = sizeof(T) == 2;
    a.c1 = scale * 1.4426950408889634f;
    const int path = decode_path();
    bool done = false;  // the tcgen05 kernel ran
    cudaError_t e = path == 1 ? cudaSuccess : decode_attention_q8_tc(a, path == 2, st, &done);
    const uint64_t word = head_dim % 16 == 0 ? 16 : 4;
    const bool words = head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(kc) & (word - 1)) == 0 &&
                       (reinterpret_cast<uintptr_t>(vc) & 3) == 0;
    if (e == cudaSuccess && !done) e = words ? launch_warp_nr<true>(a, st) : launch_warp_nr<false>(a, st);
    if (e == cudaSuccess) e = head_dim <= 128 ? launch_combine<T, 1>(out, a, st) : launch_combine<T, 2>(out, a, st);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(OXIDE_ERR_LAUNCH, "%s: launch failed: %s", name, cudaGetErrorString(e));
    }
    return check_launch(name);
}

}  // namespace oxide

using oxide::bf16_t;

extern "C" {

uint64_t oxide_decode_attention_q8_workspace_bytes(uint64_t batch, uint64_t q_heads, uint64_t kv_heads,
                                                   uint64_t head_dim) {
    const uint64_t parts = oxide::attn_q8_parts(batch, q_heads, kv_heads);
    return parts * oxide::attn_q8_nr(q_heads, kv_heads) * ((head_dim + 3) / 4 * 4 + 2) * 4 + 16 + (batch + 4) / 4 * 16;
}
int oxide_decode_attention_q8_f32(const float* q, const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                  const float* v_scale, const int32_t* lens, float* out, uint64_t batch,
                                  uint64_t q_heads, uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim,
                                  uint64_t block, float scale, void* workspace, uint64_t workspace_bytes,
                                  oxide_stream_t stream) {
    return oxide::attn_q8_entry<float>("oxide_decode_attention_q8_f32", q, k_cache, v_cache, k_scale, v_scale, lens,
                                       out, batch, q_heads, kv_heads, max_seq, head_dim, block, scale, workspace,
                                       workspace_bytes, stream);
}
int oxide_decode_attention_q8_bf16(const oxide_bf16* q, const int8_t* k_cache, const int8_t* v_cache,
                                   const float* k_scale, const float* v_scale, const int32_t* lens, oxide_bf16* out,
                                   uint64_t batch, uint64_t q_heads, uint64_t kv_heads, uint64_t max_seq,
                                   uint64_t head_dim, uint64_t block, float scale, void* workspace,
                                   uint64_t workspace_bytes, oxide_stream_t stream) {
    return oxide::attn_q8_entry<bf16_t>("oxide_decode_attention_q8_bf16", q, k_cache, v_cache, k_scale, v_scale,
                                        lens, out, batch, q_heads, kv_heads, max_seq, head_dim, block, scale,
                                        workspace, workspace_bytes, stream);
}

}  // extern "C"
