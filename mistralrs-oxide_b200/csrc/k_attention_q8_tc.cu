// k_attention_q8_tc.cu -- decode attention over int8 KV caches with both
// products in int8 on the 5th-generation tensor cores.
//
// Mathematics.  The cache's codes c, d are int8 as they lie in memory, so the
// other operand of each product is written in int8 digits as well and the
// products are exact integer sums:
//   q of a head = x u with integers |x| below 2^31 and u a power of two, and
//   x = x0 + 256 x1 + 65536 x2 + 2^24 x3 in balanced digits (-128 .. 127), so
//   q . c = (x0 . c + 256 x1 . c + ...) u: the four digit rows are four columns
//   of one product, each sum at most 2^22 and exact.  bf16 elements are exact so
//   far, those below 2^-23 of the head's largest rounded to 2^-31 of it; f32
//   elements take four digits more, for what the first ones leave (2^-61).  So
//   a strong channel over small codes costs the others nothing (with three
//   digits, an element of 1e4 beside others of 1 left scores off by 1e-3);
//   p_j vs_j (the softmax weight times the value block's scale) likewise, in
//   eight digits: an integer in units of 2^-30 of the largest of the tile, and
//   what that leaves in units of 2^-61.  The largest is found in the log2 domain
//   (t_j + log2 vs_j), so neither a far maximum in another tile nor blocks
//   with very different scales cost a weight its digits.  A weight down to 2^-37 of
//   its tile's largest keeps f32's 24 bits: where one key holds the weight and its
//   values are zero or cancel, the others make up the output (with three digits
//   it was off by 1 % where that key's score was 12 to 14 above theirs).
// The N side of a product, which is 16 wide at least, carries the digits: the
// tensor cores read the cache once for up to eight query heads of a kv head.
//
// Work division as in k_attention_tc.cu (tiles of 128 keys laid end to end,
// one CTA per SM, equal ranges); partials as in oxide_attn_q8.cuh, two halves
// a CTA.  head_dim a multiple of 16, in one piece up to 128 and in two halves
// above (half_dims each, rounded up to 16): a box is as wide as its piece and its
// rows are 128 bytes apart in shared memory, whose rest is anything -- it meets
// digits that are zero, or dims that nobody reads.  (Boxes of 128 bytes, filled
// with zeros past head_dim, took 63.6 us instead of 38.8 at 8 sequences of 16384
// keys, head_dim 80, and 47.2 instead of 37.6 at 8192 keys, head_dim 144.)
//
// CTA of 13 warps:
//   warp 0      TMA producer: K and V tiles [128 keys x 128 bytes],
//               128-byte swizzle, a ring of up to 192 KB: 6 stages of 32 KB, or
//               3 of 64 KB with two halves (5 and 2 with eight heads, whose
//               operands take the room);
//   warp 1      TMEM owner and issuer of the scores' products,
//                 S[128 keys x N] = K . X^T   (A = K, K-major; B = digits of q);
//   warp 12     issuer of the outputs' products,
//                 O[128 dims x N] = V^T . Y^T (A = V read MN-major; B = digits
//                                              of the weights, N-major: a
//                                              key's digits are 8 to 64 bytes
//                                              in a row, one to four stores of
//                                              its thread),
//               N = digits times heads, in steps of 16.  One thread issuing
//               both spent 2100 cycles a tile on waits and issue, twice what
//               the loads allow;
//   warp 2      the query heads' digits, one pair ahead, from raw bits loaded two
//               pairs ahead.  (A second such warp gained nothing, nor did asking
//               L2 for the queries four pairs early, when it was tried: 59.2 and
//               71.2 us where this took 59.1, at 256 sequences of 200 keys.)
//   warp 3      the tile prefix; then each tile's scales, ready for the softmax
//               threads (the key scale, log2 of the value scale, masks), loaded
//               two tiles ahead.  One scale for a lane's four keys wherever
//               blocks allow it: with one for every key this warp alone took
//               1400 cycles a tile, 200 more than the loads;
//   warps 4-7 and 8-11  two softmax groups that take the tiles in turn, each
//               with its own S and O in TMEM, weights buffer and online state:
//               one group's barriers and latencies hide behind the other's
//               work.  Thread i = key i of S and dim i of each half of O.
// Measured (bf16 queries, 32 heads over 8, blocks of 64; time, and the codes'
// rate of 6540 GB/s): 8 sequences of 1024 to 32768 keys 52 us (81 %), one of
// 131072 keys 48.4 us (85 %); 8 of 8192 keys, head_dim 256, 48.7 us (84 %); 64
// heads over 8 at 8 of 8192 keys 35.4 us (58 %), f32 queries 38.8; 256 of 200 keys
// 48.5 us; starting, joining the parts and the last tiles' way through the roles
// take 7 to 8 us whatever the lengths (one sequence of 100 keys: 7.2 us).
// A group's buffers need few barriers: its O of tile k is read before its
// weights of tile k + 1 are handed over, so that hand-over also says that O and
// the weights buffer are free.
// Every wait is bounded, as in k_attention_tc.cu: a wait that runs out raises
// the CTA's abort flag, all roles stop at points their barriers agree on,
// copies and products in flight are waited for, TMEM is freed, and the error
// word makes the combine kernel write NaN.
#include <stdlib.h>

#include "oxide_attn_q8.cuh"
#include "oxide_tc.cuh"

namespace oxide {

constexpr uint32_t QT_TK = 128, QT_DB = 128;  // keys a tile, bytes a row of a tile half
constexpr int QT_THREADS = 416;
constexpr uint32_t QT_MAX_BATCH = 1024;
// Maxima start here, not at -infinity: differences stay numbers, and a masked
// score (-infinity) is a zero weight without being asked about.  No finite
// score is lower.
constexpr float QT_LOW = -3.402823466e38f;
constexpr uint32_t QT_TILE = QT_TK * QT_DB;  // 16 KB
constexpr uint32_t QT_SMEM = 227 * 1024;     // what a CTA can have
constexpr int QT_PD = 8;                     // digits of a weight

// Rows of a B operand, and columns of its product: `digits` of NR query heads
// (M = 128 takes N in steps of 16).
constexpr uint32_t qt_n(int nr, int digits) { return (uint32_t)(nr * digits + 15) / 16 * 16; }

// Places of the kernel for NR query heads of QD digits and DH halves of 128 bytes a
// row (head_dim up to 128, 256).
template <int NR, int DH, int QD>
struct QtMap {
    static constexpr uint32_t NS = qt_n(NR, QD), NO = qt_n(NR, QT_PD);  // columns of S, of O
    static constexpr uint32_t STAGE_BYTES = 2 * DH * QT_TILE;           // K, V
    static constexpr uint32_t Q_HALF = NS * QT_DB, Q_BYTES = DH * Q_HALF, P_BYTES = NO * QT_DB;
    // as many stages as fit, at most 192 KB
    static constexpr uint32_t FIXED = 2 * Q_BYTES + 2 * P_BYTES + (QT_MAX_BATCH + 8) * 4 + 2048 + 1024;
    static constexpr int FIT = (int)((QT_SMEM - FIXED) / (STAGE_BYTES + QT_TK * 8));
    static constexpr int STAGES = FIT < 6 / DH ? FIT : 6 / DH;
    // TMEM columns: S of group g at SW g, its O (half x) at O + OW (DH g + x)
    static constexpr uint32_t SW = NS < 32 ? 32 : NS, OW = NO < 32 ? 32 : NO, O = 2 * SW;
    static constexpr uint32_t TMEM_USED = O + 2 * DH * OW;
    static constexpr uint32_t TMEM_COLS = TMEM_USED <= 128 ? 128 : (TMEM_USED <= 256 ? 256 : 512);
    // shared memory (offsets from a 1024-byte aligned base)
    static constexpr uint32_t OFF_Q = STAGES * STAGE_BYTES;                  // 2 slots
    static constexpr uint32_t OFF_P = OFF_Q + 2 * Q_BYTES;                   // 2 groups
    static constexpr uint32_t OFF_PRE = OFF_P + 2 * P_BYTES;
    static constexpr uint32_t OFF_SC = OFF_PRE + (QT_MAX_BATCH + 8) * 4;     // a stage's keys: float2 [128]
    static constexpr uint32_t OFF_SQ = OFF_SC + STAGES * QT_TK * 8;          // [2][8] factors of the scores
    static constexpr uint32_t OFF_RED = OFF_SQ + 2 * 8 * 4;                  // [2][4][16] each warp's tile maxima
    static constexpr uint32_t OFF_SUM = OFF_RED + 2 * 4 * 16 * 4;            // [2][5][8] each warp's sums; the maxima
    static constexpr uint32_t OFF_BAR = OFF_SUM + 2 * 5 * 8 * 4;
    enum : int {
        FULL = 0,                 // [stages] loaded (TMA bytes)
        EMPTY = FULL + STAGES,    // [stages] consumed (MMA commit)
        CFULL = EMPTY + STAGES,   // [stages] the tile's scales written (warp 3)
        QFULL = CFULL + STAGES,   // [2] digits of a pair's query heads written (warp 2)
        QEMPTY = QFULL + 2,       // [2] read: MMA commit and the eight softmax warps
        SFULL = QEMPTY + 2,       // [2] scores in TMEM (MMA commit)
        SEMPTY = SFULL + 2,       // [2] scores read (4 warps)
        PFULL = SEMPTY + 2,       // [2] weights written, O free (1 thread)
        OFULL = PFULL + 2,        // [2] tile output in TMEM, weights read (MMA commit)
        DONE = OFULL + 2,         // every product issued has completed
        COUNT = DONE + 1
    };
    static constexpr uint32_t OFF_MISC = OFF_BAR + ((COUNT + 1) & ~1) * 8;
    static constexpr size_t SMEM = OFF_MISC + 48 + 1024;  // + alignment slack
};
static_assert(2 * 1024 <= Q8A_PARTS, "two parts a CTA fit the workspace");

__device__ unsigned int g_device_status_q8;  // sticky failure flags, read by oxide_device_status

// C columns of TMEM (8, 16 or 32).
template <int C>
__device__ __forceinline__ void qt_load(uint32_t taddr, uint32_t (&v)[C]) {
    if constexpr (C == 32) tmem_ld32(taddr, v);
    else if constexpr (C == 16) tmem_ld16(taddr, v);
    else tmem_ld8(taddr, v);
    tmem_wait_ld();
}
// The number that the sums of four digits spell.  Each sum is at most 2^22 in
// magnitude, so two of them join in 32 bits; the upper two are a whole number
// that f32 holds, or else far above the lower ones.
__device__ __forceinline__ float qt_spell(uint32_t d0, uint32_t d1, uint32_t d2, uint32_t d3) {
    return __fmaf_rn((float)((int)d3 * 256 + (int)d2), 65536.0f, (float)((int)d1 * 256 + (int)d0));
}
// Balanced digits of an integer, |x| <= 0x7f7f7f7f, in bytes 0 .. 3.
__device__ __forceinline__ uint32_t qt_digits(int x) { return ((uint32_t)x + 0x80808080u) ^ 0x80808080u; }
// Byte j of word i becomes byte i of word j: digit rows from the digits of four
// dims.  (A shift and a pack a byte made this warp the bound of short sequences:
// 256 of 200 keys 51.4 us instead of 48.5, f32 queries 58.3 instead of 55.0.)
__device__ __forceinline__ void qt_transpose(uint32_t (&d)[4]) {
    const uint32_t a = __byte_perm(d[0], d[1], 0x5140), b = __byte_perm(d[2], d[3], 0x5140);
    const uint32_t c = __byte_perm(d[0], d[1], 0x7362), e = __byte_perm(d[2], d[3], 0x7362);
    d[0] = __byte_perm(a, b, 0x5410);
    d[1] = __byte_perm(a, b, 0x7632);
    d[2] = __byte_perm(c, e, 0x5410);
    d[3] = __byte_perm(c, e, 0x7632);
}
// Scores: digit i of head h is column i NR + h.  Of eight digits the upper four
// come first; the lower ones count units of 2^-31 of theirs.
template <int NR, int QD>
__device__ __forceinline__ void qt_scores(uint32_t taddr, float (&x)[NR]) {
    uint32_t v[(4 * NR + 7) / 8 * 8];
    qt_load(taddr, v);
#pragma unroll
    for (int h = 0; h < NR; ++h) x[h] = qt_spell(v[h], v[NR + h], v[2 * NR + h], v[3 * NR + h]);
    if constexpr (QD == 8) {
        qt_load(taddr + 4 * NR, v);
#pragma unroll
        for (int h = 0; h < NR; ++h)
            x[h] = __fmaf_rn(qt_spell(v[h], v[NR + h], v[2 * NR + h], v[3 * NR + h]), 0x1p-31f, x[h]);
    }
}
// Outputs: digit i of head h is column 8 h + i, the upper four first.
template <int NR>
__device__ __forceinline__ void qt_outputs(uint32_t taddr, float (&x)[NR]) {
    constexpr int H = NR < 2 ? NR : 2;  // heads at once
#pragma unroll
    for (int h0 = 0; h0 < NR; h0 += H) {
        uint32_t v[8 * H];
        qt_load(taddr + 8 * h0, v);
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint32_t* d = v + 8 * h;
            x[h0 + h] = __fmaf_rn(qt_spell(d[4], d[5], d[6], d[7]), 0x1p-31f, qt_spell(d[0], d[1], d[2], d[3]));
        }
    }
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory");
}

// Weights and rescaling factors: off by at most 2^-22 of the result, as ex2_approx
// everywhere in these kernels; results below 2^-126 are zero.
__device__ __forceinline__ float qt_ex2(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}

// 96 registers: CTAs of the combine kernel, which is launched early, then fit beside
// this one and wait there (with 104, one quarter of the register file is short of
// two of their warps: 1.5 us a call).  Eight heads or two halves need more.
// QD: digits of a query element, 4 for bf16 and 8 for f32.
template <int NR, int DH, int QD>
__global__ void __launch_bounds__(QT_THREADS, 1) __maxnreg__(NR < 8 && DH == 1 ? 96 : 128)
    decode_attn_q8_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                             Q8AttnArgs p, uint32_t withhold) {
    pdl_trigger();
    typedef QtMap<NR, DH, QD> M;
    constexpr bool BF16 = QD == 4;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t* pre = reinterpret_cast<uint32_t*>(smem + M::OFF_PRE);
    float* sq = reinterpret_cast<float*>(smem + M::OFF_SQ);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + M::OFF_MISC);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + M::OFF_MISC + 4);
    volatile int* consumed = reinterpret_cast<volatile int*>(smem + M::OFF_MISC + 8);  // stages warp 1 waited for
    uint32_t* begin = reinterpret_cast<uint32_t*>(smem + M::OFF_MISC + 16);  // where this CTA's tiles begin: b, kvh, lt, tb
    auto bar = [&](int i) { return sbase + M::OFF_BAR + 8u * (uint32_t)i; };

    if (tid == 0) {
        *abort = 0;
        *consumed = 0;
        for (int i = 0; i < M::STAGES; ++i) {
            mbar_init(bar(M::FULL + i), 1);
            mbar_init(bar(M::EMPTY + i), 1);
            mbar_init(bar(M::CFULL + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(M::QFULL + i), 1);
            mbar_init(bar(M::QEMPTY + i), 9);
            mbar_init(bar(M::SFULL + i), 1);
            mbar_init(bar(M::SEMPTY + i), 4);
            mbar_init(bar(M::PFULL + i), 1);
            mbar_init(bar(M::OFULL + i), 1);
        }
        mbar_init(bar(M::DONE), 2);
        mbar_init_fence();
        tma_prefetch_map(&tmk);
        tma_prefetch_map(&tmv);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), M::TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait();  // the previous kernel's writes (lengths, caches, queries) are visible
    const uint32_t heads = p.kv_heads * p.chunks;
    if (warp == 3) {  // the tile prefix and this CTA's first tile
        q8a_prefix(p, QT_TK, pre, blockIdx.x == 0);
        const uint32_t all = pre[p.batch] * heads;
        if (all) {
            TileWalk at{pre, p.batch, heads, 0, 0, 0, 0};
            at.seek(q8a_start(p, blockIdx.x, all));
            if (lane == 0) {
                begin[0] = at.b;
                begin[1] = at.kvh;
                begin[2] = at.lt;
                begin[3] = at.tb;
            }
            // The first pair's query heads and scales go ahead of the ring's 192 KB
            // a CTA: asked for behind them they came 3 us later.
            const uint32_t kvh = p.by_chunks.div(at.kvh), h0 = (at.kvh - kvh * p.chunks) * NR;
            const uint32_t es = BF16 ? 2 : 4, bytes = min(p.rep - h0, (uint32_t)NR) * p.head_dim * es;
            if (lane * 128u < bytes)
                prefetch_l2(static_cast<const char*>(p.q) +
                            ((uint64_t)at.b * p.q_heads + kvh * p.rep + h0) * p.head_dim * es + lane * 128u);
            const uint64_t sc = ((uint64_t)at.b * p.kv_heads + kvh) * p.nblk + ((at.lt * QT_TK) >> p.shift);
            if (lane < 2) prefetch_l2((lane ? p.vs : p.ks) + sc);
        }
    }
    if (tid == 0 && blockIdx.x == 0) *p.err = 0u;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot, hd = p.half_dims;
    const uint32_t T = pre[p.batch] * heads;
    const uint32_t nt = q8a_start(p, blockIdx.x + 1, T) - q8a_start(p, blockIdx.x, T);  // this CTA's tiles, n = 0 .. nt - 1
    TileWalk w{pre, p.batch, heads, begin[0], begin[1], begin[2], begin[3]};  // (unset, and unused, without tiles)

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const bool leader = elect_one();
        uint32_t n = 0, s = 0, ph = 1;  // the stage and its phase
        if (!withhold) {
            for (; n < nt && !*abort; ++n) {
                if (!warp_wait_all(bar(M::EMPTY + s), ph, abort)) break;
                const int z = (int)(w.b * p.kv_heads + (p.by_chunks.div(w.kvh)));
                const int y = (int)(w.lt * QT_TK);
                const uint32_t sd = sbase + s * M::STAGE_BYTES;
                if (leader) {
                    mbar_arrive_expect_tx(bar(M::FULL + s), 2 * DH * QT_TK * hd);
#pragma unroll
                    for (int x = 0; x < DH; ++x) tma_load_3d(sd + x * QT_TILE, &tmk, bar(M::FULL + s), x * (int)hd, y, z);
#pragma unroll
                    for (int x = 0; x < DH; ++x)
                        tma_load_3d(sd + (DH + x) * QT_TILE, &tmv, bar(M::FULL + s), x * (int)hd, y, z);
                }
                __syncwarp();
                w.next();
                if (++s == M::STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        // Drain (after an abort): copies issued but never waited for by warp 1
        // land before the CTA exits.
        if (leader && *abort) {
            for (uint32_t i = (uint32_t)*consumed; i < n; ++i)
                tc_wait_drain(bar(M::FULL + i % M::STAGES), (i / M::STAGES) & 1u);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- issuer of the scores ----------------
        constexpr uint32_t IDESC_S = umma_idesc_s8(128, M::NS, false, false);
        const bool leader = elect_one();
        const uint64_t kd = umma_desc(sbase, 16, 1024, UMMA_SWIZZLE_128B);
        const uint64_t qd = umma_desc(sbase + M::OFF_Q, 16, 1024, UMMA_SWIZZLE_128B);
        uint32_t left = 0, q = 0, s = 0, ph = 0;  // tiles left of the pair, its number, the stage and its phase
        for (uint32_t n = 0; n < nt; ++n) {
            const uint32_t g = n & 1u;
            if (left == 0) {
                left = min(w.tb - w.lt, nt - n);
                w.lt += left - 1;
                w.next();
                if (!warp_wait_all(bar(M::QFULL + (q & 1u)), (q >> 1) & 1u, abort)) break;
            }
            if (!warp_wait_all(bar(M::FULL + s), ph, abort)) break;
            if (leader) *consumed = (int)n + 1;
            if (!warp_wait_all(bar(M::SEMPTY + g), ((n >> 1) & 1u) ^ 1u, abort)) break;
            tc_fence_after();
            const uint64_t ka = kd + s * (M::STAGE_BYTES >> 4), qa = qd + (q & 1u) * (M::Q_BYTES >> 4);
            --left;
            if (leader) {
#pragma unroll
                for (uint32_t kk = 0; kk < 4 * DH; ++kk)  // 32 dims (32 bytes) a product, four products a half
                    umma_s8(tmem + g * M::SW, ka + (kk >> 2) * (QT_TILE >> 4) + (kk & 3) * 2,
                            qa + (kk >> 2) * (M::Q_HALF >> 4) + (kk & 3) * 2, IDESC_S, kk > 0);
                umma_commit(bar(M::SFULL + g));
                if (left == 0) umma_commit(bar(M::QEMPTY + (q & 1u)));  // the pair's last product that reads its digits
            }
            __syncwarp();
            if (left == 0) ++q;
            if (++s == M::STAGES) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (leader) umma_commit(bar(M::DONE));
        __syncwarp();
    } else if (warp == 12) {
        // ---------------- issuer of the outputs ----------------
        constexpr uint32_t IDESC_O = umma_idesc_s8(128, M::NO, true, true);
        const bool leader = elect_one();
        const uint64_t vd = umma_desc(sbase + DH * QT_TILE, 16, 1024, UMMA_SWIZZLE_128B);
        const uint64_t pd = umma_desc(sbase + M::OFF_P, 128, QT_TK * 16, UMMA_SWIZZLE_NONE);
        uint32_t s = 0;
        for (uint32_t n = 0; n < nt; ++n) {
            const uint32_t g = n & 1u;
            if (!warp_wait_all(bar(M::PFULL + g), (n >> 1) & 1u, abort)) break;
            tc_fence_after();
            const uint64_t va = vd + s * (M::STAGE_BYTES >> 4), pa = pd + g * (M::P_BYTES >> 4);
            if (leader) {
#pragma unroll
                for (uint32_t kk = 0; kk < 4 * DH; ++kk)  // 32 keys a product: 4096 bytes of a V half, 512 of the weights
                    umma_s8(tmem + M::O + (g * DH + (kk >> 2)) * M::OW, va + (kk >> 2) * (QT_TILE >> 4) + (kk & 3) * 256,
                            pa + (kk & 3) * 32, IDESC_O, (kk & 3) > 0);
                umma_commit(bar(M::OFULL + g));
                umma_commit(bar(M::EMPTY + s));
            }
            __syncwarp();
            if (++s == M::STAGES) s = 0;
        }
        if (leader) {  // every product issued has completed before TMEM is freed
            umma_commit(bar(M::DONE));
            if (!tc_wait_drain(bar(M::DONE), 0)) *abort = 1;
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------- digits of the query heads ----------------
        // Dims 4 lane .. 4 lane + 3 (of each half); as a head is done, the next
        // pair's is loaded, and stays as it lies in memory until its turn: a
        // conversion beside the load made the warp wait for each head, some 5000
        // cycles while HBM is busy (53.9 instead of 51.7 us at 8 sequences of 1024
        // to 32768 keys, 72 instead of 59 at 256 of 200).
        uint2 x[NR][2 * DH];
        uint64_t row = 0;  // of the pair loaded next, and its heads (0: no more pairs)
        uint32_t nh = 0;
        auto place = [&](bool more) {
            const uint32_t kvh = p.by_chunks.div(w.kvh), h0 = (w.kvh - kvh * p.chunks) * NR;
            row = (uint64_t)w.b * p.q_heads + kvh * p.rep + h0;
            nh = more ? p.rep - h0 : 0;
        };
        auto load = [&](uint32_t h, uint2 (&v)[2 * DH]) {
#pragma unroll
            for (int half = 0; half < DH; ++half) {
                const uint32_t d = 4u * lane + hd * half;
                const bool there = h < nh && 4u * lane < hd && d < p.head_dim;
                const uint2* at = reinterpret_cast<const uint2*>(static_cast<const char*>(p.q) +
                                                                 ((row + h) * p.head_dim + d) * (BF16 ? 2 : 4));
                v[2 * half] = v[2 * half + 1] = make_uint2(0, 0);
                if (there) v[2 * half] = __ldg(at);
                if (there && !BF16) v[2 * half + 1] = __ldg(at + 1);
            }
        };
        auto value = [&](const uint2 (&v)[2 * DH], int i) {  // element i of the lane's four (of each half)
            const uint2 lo = v[i >> 2 << 1], hi = v[(i >> 2 << 1) + 1];
            const uint32_t b = (i & 2) ? lo.y : lo.x, f = (i & 2) ? ((i & 1) ? hi.y : hi.x) : ((i & 1) ? lo.y : lo.x);
            return BF16 ? ((i & 1) ? bf16_hi(b) : bf16_lo(b)) : __uint_as_float(f);
        };
        uint32_t n = 0;
        auto step = [&]() {
            if (n >= nt) return;
            const uint32_t cnt = min(w.tb - w.lt, nt - n);
            n += cnt;
            w.lt += cnt - 1;
            w.next();
        };
        place(n < nt);
#pragma unroll
        for (int h = 0; h < NR; ++h) load(h, x[h]);
        for (uint32_t q = 0; n < nt; ++q) {
            const uint32_t slot = q & 1u;
            step();
            if (!warp_wait_all(bar(M::QEMPTY + slot), (~q >> 1) & 1u, abort)) break;
            unsigned char* out = smem + M::OFF_Q + slot * M::Q_BYTES;
            place(n < nt);
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                uint32_t a = 0;
                float u[4 * DH];
#pragma unroll
                for (int e = 0; e < 4 * DH; ++e) {
                    u[e] = value(x[h], e);
                    a = max(a, q8_abs_bits(u[e]));
                }
                a = q8_warp_max(a);
                // The unit is a power of two: 2^30 of them (2^29 where the
                // largest element would pass four digits) reach from 2^e to
                // the largest element, 2^e <= amax < 2^(e + 1).  Elements below
                // 2^-60 are brought up first.
                const bool bad = a >= Q8_INF, tiny = a < 0x21800000u;  // not finite; below 2^-60
                const float up = tiny ? 0x1p80f : 1.0f, amax = fmul(__uint_as_float(a), up);
                const uint32_t e = __float_as_uint(amax) & 0x7f800000u;
                const uint32_t k = amax <= fmul(__uint_as_float(e), 1.992f) ? 30u : 29u;
                const float inv = bad || a == 0 ? 0.0f : __uint_as_float(((254u + k) << 23) - e);
                if (lane == 0)
                    sq[slot * 8 + h] = bad ? q8_nan()
                                           : (a == 0 ? 0.0f : fmul(fmul(__uint_as_float(e - (k << 23)), p.c1), tiny ? 0x1p-80f : 1.0f));
#pragma unroll
                for (int half = 0; half < DH; ++half) {
                    float y[4];  // in units
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = bad ? 0.0f : fmul(fmul(u[4 * half + i], up), inv);
#pragma unroll
                    for (int g0 = 0; g0 < QD; g0 += 4) {  // the upper four digits, then those of the rest
                        uint32_t d[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int n = __float2int_rn(y[i]);
                            d[i] = qt_digits(n);
                            y[i] = fmul(fsub(y[i], (float)n), 0x1p31f);  // exact
                        }
                        qt_transpose(d);
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const uint32_t r = (g0 + g) * NR + h;
                            *reinterpret_cast<uint32_t*>(out + half * M::Q_HALF + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                                         ((lane & 3) << 2)) = d[g];
                        }
                    }
                }
                load(h, x[h]);
            }
            fence_async_smem();  // the digits are visible to the tensor core
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(M::QFULL + slot));
        }
    } else if (warp == 3) {
        // ---------------- scales of the tiles: keys 4 lane .. 4 lane + 3 ----------------
        struct Keys {
            float k[4], v[4];
            uint32_t live;  // how many of the tile's keys the sequence has
        };
        const bool shared = p.shift >= 2;  // the lane's four keys share a scale
        uint32_t len = 0, ahead = 0, s = 0, ph = 1;  // ahead: the tile loaded next; the stage and its phase
        const float *ks = p.ks, *vs = p.vs;          // the head's scales
        auto load = [&](Keys& x) {
            if (ahead >= nt) return;
            if (ahead == 0 || w.lt == 0) {  // a new pair
                len = q8a_len(p, w.b);
                const uint64_t bh = (uint64_t)w.b * p.kv_heads + (p.by_chunks.div(w.kvh));
                ks = p.ks + bh * p.nblk;
                vs = p.vs + bh * p.nblk;
            }
            const uint32_t key0 = w.lt * QT_TK, key = key0 + 4 * lane;
            x.live = len - key0;
            if (shared) {
                x.k[0] = x.v[0] = 1.0f;
                if (key < len) {
                    x.k[0] = __ldg(ks + (key >> p.shift));
                    x.v[0] = __ldg(vs + (key >> p.shift));
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    x.k[i] = x.v[i] = 1.0f;
                    if (key + i < len) {
                        x.k[i] = __ldg(ks + ((key + i) >> p.shift));
                        x.v[i] = __ldg(vs + ((key + i) >> p.shift));
                    }
                }
            }
            ++ahead;
            w.next();
        };
        // What a softmax thread needs of its key: the key scale (NaN where the scales
        // are not sound) and log2 of the value scale; +infinity as the log2 marks a
        // masked key.
        auto ready = [&](float k, float v) -> float2 {
            return make_float2(q8a_key_scale(k, v), v >= 0.0f && v < INFINITY ? lg2_approx(v) : 0.0f);
        };
        auto put = [&](const Keys& x) -> bool {
            float2 r[4];
            r[0] = ready(x.k[0], x.v[0]);
            if (shared) {
                r[1] = r[2] = r[3] = r[0];
            } else {
#pragma unroll
                for (int i = 1; i < 4; ++i) r[i] = ready(x.k[i], x.v[i]);
            }
            if (x.live < QT_TK) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (4 * lane + i >= x.live) r[i] = make_float2(0.0f, INFINITY);
            }
            // the output product of the stage's last tile came after its scales were read
            if (!warp_wait_all(bar(M::EMPTY + s), ph, abort)) return false;
            float4* out = reinterpret_cast<float4*>(smem + M::OFF_SC) + (s * QT_TK + 4 * lane) / 2;
            out[0] = make_float4(r[0].x, r[0].y, r[1].x, r[1].y);
            out[1] = make_float4(r[2].x, r[2].y, r[3].x, r[3].y);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(M::CFULL + s));
            if (++s == M::STAGES) {
                s = 0;
                ph ^= 1u;
            }
            return true;
        };
        Keys a, b;  // tiles n and n + 1 in turn
        load(a);
        load(b);
        for (uint32_t n = 0; n < nt; n += 2) {
            if (!put(a)) break;
            load(a);
            if (n + 1 >= nt || !put(b)) break;
            load(b);
        }
    } else if (warp < 12) {
        // ---------------- softmax and epilogue: group g takes tiles n = g mod 2 ----------------
        const uint32_t g = (uint32_t)(warp >> 2) - 1, q4 = (uint32_t)(warp & 3);
        const uint32_t L = q4 * 32 + (uint32_t)lane;  // key of the S tile, dim of the O tile
        const uint32_t s_tmem = tmem + ((q4 * 32u) << 16) + g * M::SW, o_tmem = tmem + ((q4 * 32u) << 16) + M::O + g * DH * M::OW;
        const int nbar = 1 + (int)g;
        float* red = reinterpret_cast<float*>(smem + M::OFF_RED) + g * 64;   // [4][16]
        float* lsum = reinterpret_cast<float*>(smem + M::OFF_SUM) + g * 40;  // [4][8] sums of a finished pair, [8] its maxima
        unsigned char* pt = smem + M::OFF_P + g * M::P_BYTES;
        // m, l: online softmax of the scores; wm (relative to m), acc: the same for
        // the weights times scales (acc in units of 2^-30); corr, tf: factors of
        // the output not yet read
        float m[NR], l[NR], wm[NR], acc[DH][NR], corr[NR], tf[NR];
        bool fail = false;
#pragma unroll
        for (int h = 0; h < NR; ++h) corr[h] = tf[h] = 0.0f;

        const float2* scales = reinterpret_cast<const float2*>(smem + M::OFF_SC) + L;
        uint32_t st = g, ph = 0, k = 0;  // the stage and its phase, and the number, of this group's next tile
        auto epilogue = [&](uint32_t k) {  // add the output of this group's tile k
            const bool ok = warp_wait_all(bar(M::OFULL + g), k & 1u, abort);
            fail |= !ok;
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < DH; ++x) {
                float o[NR];
                qt_outputs<NR>(o_tmem + M::OW * x, o);
#pragma unroll
                for (int h = 0; h < NR; ++h) acc[x][h] = __fmaf_rn(acc[x][h], corr[h], fmul(o[h], tf[h]));
            }
            tc_fence_before();
        };
        bool dead = false;
        for (uint32_t n = 0, q = 0; n < nt && !dead; ++q) {
            const uint32_t cnt = min(w.tb - w.lt, nt - n), j0 = (n ^ g) & 1u;
            // every warp waits for the digits, also of a pair without a tile
            // for it: its arrival below then belongs to this use of the slot
            fail |= !warp_wait_all(bar(M::QFULL + (q & 1u)), (q >> 1) & 1u, abort);
            float f[NR];
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                f[h] = sq[(q & 1u) * 8 + h];
                m[h] = wm[h] = QT_LOW;
                l[h] = 0.0f;
#pragma unroll
                for (int x = 0; x < DH; ++x) acc[x][h] = 0.0f;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(M::QEMPTY + (q & 1u)));
            for (uint32_t j = j0; j < cnt; j += 2) {
                float t[NR];
                bool ok = warp_wait_all(bar(M::CFULL + st), ph, abort);
                const float2 sc = scales[st * QT_TK];  // key scale; log2 of the value scale, or the mark of a masked key
                const float mask = sc.y == INFINITY ? -INFINITY : 0.0f, lv = sc.y == INFINITY ? 0.0f : sc.y;
                ok = warp_wait_all(bar(M::SFULL + g), k & 1u, abort) && ok;
                fail |= !ok;
                if (ok) {
                    tc_fence_after();
                    float v[NR];
                    qt_scores<NR, QD>(s_tmem, v);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(M::SEMPTY + g));
#pragma unroll
                    for (int h = 0; h < NR; ++h) {
                        t[h] = __fmaf_rn(v[h], fmul(sc.x, f[h]), mask);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < NR; ++h) t[h] = -INFINITY;
                }
#pragma unroll
                for (int h = 0; h < NR; ++h) {
                    const float a = warp_fmax(t[h]), b = warp_fmax(fadd(t[h], lv));
                    if (lane == 0) {
                        red[q4 * 16 + h] = a;
                        red[q4 * 16 + 8 + h] = b;
                    }
                }
                if (j != j0) epilogue(k - 1);  // its product has run meanwhile; the weights buffer and O are free after it
                nbar_sync128(nbar);            // the four warps' maxima are in red
                // The largest weight of the tile, wt, and of the tiles so far, wm, are
                // log2 of it relative to the largest score: differences of near
                // numbers, so scores of some hundred (whose sum with log2 of a
                // scale is off by 1e-5) cost the outputs nothing.
                float mn[NR], wt[NR], wn[NR];
                bool moved = false;
#pragma unroll
                for (int h = 0; h < NR; ++h) {
                    const float* r = red + h;
                    mn[h] = fmaxf(fmaxf(fmaxf(r[0], r[16]), fmaxf(r[32], r[48])), m[h]);
                    wt[h] = fmaxf(fsub(fmaxf(fmaxf(r[8], r[24]), fmaxf(r[40], r[56])), mn[h]), QT_LOW);
                    wn[h] = fmaxf(wt[h], fadd(wm[h], fsub(m[h], mn[h])));
                    moved |= mn[h] != m[h] || wn[h] != wm[h];
                    corr[h] = 1.0f;
                }
                if (moved) {  // the same for every thread of the group
#pragma unroll
                    for (int h = 0; h < NR; ++h) {
                        const float dm = fsub(m[h], mn[h]);
                        l[h] = fmul(l[h], qt_ex2(dm));
                        corr[h] = qt_ex2(fsub(fadd(wm[h], dm), wn[h]));
                        m[h] = mn[h];
                        wm[h] = wn[h];
                    }
                }
                uint32_t d[2 * NR];
#pragma unroll
                for (int h = 0; h < NR; ++h) {
                    const float dt = fsub(t[h], m[h]);
                    l[h] = fadd(l[h], qt_ex2(dt));
                    tf[h] = qt_ex2(fsub(wt[h], wm[h]));
                    // the weight in units of 2^-30 of the tile's largest, and what that
                    // leaves in units of 2^-61
                    const float y = fmul(qt_ex2(fsub(fadd(dt, lv), wt[h])), 0x1p30f);
                    const int n = __float2int_rn(y);
                    d[2 * h] = qt_digits(n);
                    d[2 * h + 1] = qt_digits(__float2int_rn(fmul(fsub(y, (float)n), 0x1p31f)));
                }
                // the B operand, N-major: 16 columns (two heads) of every key, key by key
                if constexpr (NR == 1) *reinterpret_cast<uint2*>(pt + L * 16) = make_uint2(d[0], d[1]);
                else
#pragma unroll
                    for (int c = 0; c < NR / 2; ++c)
                        *reinterpret_cast<uint4*>(pt + c * QT_TK * 16 + L * 16) =
                            make_uint4(d[4 * c], d[4 * c + 1], d[4 * c + 2], d[4 * c + 3]);
                fence_async_smem();  // the weights are visible to the tensor core
                tc_fence_before();
                if (nbar_or128(fail, nbar)) {
                    dead = true;
                    break;
                }
                if ((tid & 127) == 0) mbar_arrive(bar(M::PFULL + g));  // every thread has written its weights and read O
                ++k;
                st += 2;
                if (st >= M::STAGES) {
                    st -= M::STAGES;
                    ph ^= 1u;
                }
            }
            if (dead) break;
            // the pair is complete here; what its partial does not wait for comes
            // while its last output product runs
            const uint64_t part = ((uint64_t)blockIdx.x + (uint64_t)w.b * heads + w.kvh) * 2 + g;
            const uint32_t nh = min(p.rep - (w.kvh - p.by_chunks.div(w.kvh) * p.chunks) * NR, (uint32_t)NR);
            n += cnt;
            w.lt += cnt - 1;
            w.next();
            if (j0 >= cnt) continue;
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                const float x = warp_sum(l[h]);
                if (lane == 0) lsum[q4 * 8 + h] = x;
                if (L == 0) lsum[32 + h] = m[h];
                f[h] = ex2_approx(wm[h]);
            }
            epilogue(k - 1);
#pragma unroll
            for (int h = 0; h < NR; ++h)
#pragma unroll
                for (int x = 0; x < DH; ++x)
                    if ((uint32_t)h < nh && L < hd && L + hd * x < p.head_dim)
                        p.part_o[(part * NR + h) * p.head_dim + L + hd * x] = fmul(fmul(acc[x][h], 0x1p-30f), f[h]);
            if (nbar_or128(fail, nbar)) {
                dead = true;
                break;
            }
            if (L < nh) {
                p.part_ml[(part * NR + L) * 2] = lsum[32 + L];
                p.part_ml[(part * NR + L) * 2 + 1] = fadd(fadd(lsum[L], lsum[8 + L]), fadd(lsum[16 + L], lsum[24 + L]));
            }
            // lsum is written again behind the next tile's barriers
        }
        if (fail || dead) *abort = 1;
    }
    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, M::TMEM_COLS);
    if (tid == 0 && *abort) {
        atomicOr(p.err, 1u);
        atomicOr(&g_device_status_q8, OXIDE_DEVICE_WAIT_TIMEOUT);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A cache [heads, max_seq, head_dim] of bytes as a TMA map with boxes of 128
// positions by `width` bytes, 128-byte swizzle; bytes past head_dim and positions
// past max_seq are filled with zeros.  False if the driver refuses it.
static bool qt_map(CUtensorMap* m, const void* base, uint64_t heads, uint64_t max_seq, uint64_t head_dim,
                   uint32_t width) {
    static EncodeTiledFn enc = reinterpret_cast<EncodeTiledFn>(driver_fn("cuTensorMapEncodeTiled"));
    if (!enc) return false;
    const cuuint64_t dims[3] = {head_dim, max_seq, heads};
    const cuuint64_t strides[2] = {head_dim, max_seq * head_dim};
    const cuuint32_t box[3] = {width, QT_TK, 1};
    const cuuint32_t es[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tc_enabled();  // an sm_100 device, and not switched off (k_attention_tc.cu)

template <int NR, int DH, int QD>
static cudaError_t qt_launch(const CUtensorMap& mk, const CUtensorMap& mv, const Q8AttnArgs& a, bool withhold,
                             cudaStream_t st) {
    auto kern = decode_attn_q8_tc_kernel<NR, DH, QD>;
    constexpr size_t smem = QtMap<NR, DH, QD>::SMEM;
    static_assert(smem <= QT_SMEM && QtMap<NR, DH, QD>::STAGES >= 2 && QtMap<NR, DH, QD>::TMEM_USED <= 512, "fits an SM");
    // one half: room is left beside the CTA for one of the combine kernel (4.1 KB)
    static_assert(DH == 2 || smem <= 221 * 1024, "the combine kernel waits beside the CTA");
    if (!ensure_dyn_smem(reinterpret_cast<const void*>(kern), smem)) return cudaErrorInvalidConfiguration;
    return launch_k(kern, a.workers, QT_THREADS, smem, st, mk, mv, a, withhold ? 1u : 0u);
}

template <int DH, int QD>
static cudaError_t qt_launch_nr(const CUtensorMap& mk, const CUtensorMap& mv, const Q8AttnArgs& a, bool withhold,
                                cudaStream_t st) {
    switch (a.nr) {
        case 1: return qt_launch<1, DH, QD>(mk, mv, a, withhold, st);
        case 2: return qt_launch<2, DH, QD>(mk, mv, a, withhold, st);
        case 4: return qt_launch<4, DH, QD>(mk, mv, a, withhold, st);
        default: return qt_launch<8, DH, QD>(mk, mv, a, withhold, st);
    }
}

cudaError_t decode_attention_q8_tc(Q8AttnArgs& a, bool withhold, cudaStream_t st, bool* used) {
    *used = false;
    // head_dim: rows of whole 16-byte units (TMA strides), at most two 128-byte halves.
    if (!tc_enabled() || a.head_dim % 16 != 0 || a.head_dim > 2 * QT_DB || a.batch > QT_MAX_BATCH ||
        !aligned16(a.kc) || !aligned16(a.vc) || !aligned16(a.q))
        return cudaSuccess;
    const uint64_t pairs = (uint64_t)a.batch * a.kv_heads, tiles = pairs * a.chunks * ((a.max_seq + QT_TK - 1) / QT_TK);
    uint64_t G = (uint64_t)sm_count();
    if (G > tiles) G = tiles;
    if (2 * G > Q8A_PARTS) return cudaSuccess;
    a.half_dims = a.head_dim <= QT_DB ? a.head_dim : (a.head_dim / 2 + 15) / 16 * 16;
    CUtensorMap mk, mv;
    if (!qt_map(&mk, a.kc, pairs, a.max_seq, a.head_dim, a.half_dims) ||
        !qt_map(&mv, a.vc, pairs, a.max_seq, a.head_dim, a.half_dims))
        return cudaSuccess;
    a.workers = (uint32_t)G;
    a.inv_workers = 1.0 / a.workers;
    a.halves = 2;
    *used = true;
    if (a.q_bf16)
        return a.head_dim <= QT_DB ? qt_launch_nr<1, 4>(mk, mv, a, withhold, st) : qt_launch_nr<2, 4>(mk, mv, a, withhold, st);
    return a.head_dim <= QT_DB ? qt_launch_nr<1, 8>(mk, mv, a, withhold, st) : qt_launch_nr<2, 8>(mk, mv, a, withhold, st);
}

int device_status_q8(int reset, uint32_t* flags) {
    unsigned int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_device_status_q8, sizeof(v));
    if (e == cudaSuccess && reset) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_device_status_q8, &zero, sizeof(zero));
    }
    if (e != cudaSuccess) return set_error(OXIDE_ERR_CUDA, "oxide_device_status: %s", cudaGetErrorString(e));
    *flags |= v;
    return OXIDE_OK;
}

}  // namespace oxide
