// k_rmsnorm_q8.cu -- RMSNorm, and residual add + RMSNorm, whose output rows
// are int8 codes with one f32 scale a row.
//
// Reference: src/ops/norm.rs:33-47 (rms = sqrt(sum x*x / cols + eps),
// y = (x / rms) * w) and the residual add before it
// (src/layers/transformer.rs:64-67).  The 8-bit output has no counterpart
// there: it is what a caller's int8 projection reads next.
//
// Mathematics.  With p_j = h_j w_j, y_j = p_j / rms, so y_j / max|y| =
// p_j / max|p|: the row's rms decides only the scale, max|p| / (127 rms), and
// the codes are nearest(127 p_j / max|p|) whatever the rms.  One reduction
// therefore finds the sum of squares and max|p| together, where quantising
// a stored y would take a second one behind the first.
//
// bf16: p is exact in f32 (two 8-bit significands).  f32: p in f32 decides
// almost every code; the products of two floats are exact in f64, max|p| there
// is the largest of the elements whose f32 product is the f32 maximum (rounding
// is monotonic), and a code next to a half-integer is decided by the sign of
// 254 p - (2 n + 1) max|p|, taken without rounding (norm_nearest; the f64 quotient
// 127 p / max|p| is off by 2^-46 and missed half-integers).  Rows of vectors look
// for max|p| in f64 only where they have such a code, one in ten at 4096 columns.
//
// Layout.  A warp (rows of at most 128 vectors of 16 bytes) or a CTA owns a
// row and keeps it packed in registers, four vectors a thread, so each row
// crosses HBM once.  A thread meets the same columns in every row: its part of
// w stays in registers too, and CTAs take rows in turn (reading w twice a row
// through L1 instead left L1 the bound: 118 us at [16384, 4096] bf16 against
// 72 us of bytes).  Bound by HBM bytes: x, r and h in their type, one byte out.
// Measured: add + norm bf16 [16384, 4096] 78 us, 6.0 TB/s, without r 57 us; f32
// [2048, 4096] 14.3 us, 2.9 TB/s -- a row's chain of load, reduction and codes
// takes 3 us, four rows in turn to a CTA -- and [16384, 4096] 78 us, 4.3 TB/s;
// eight rows 2.5 us, launch latency.
// Rows that do not divide into aligned vectors are held element by element in
// the same way (up to 16 a thread); longer ones are read twice, the second
// time through L1 / L2.
#include "oxide_q8.cuh"

namespace oxide {

struct NormQ8Args {
    uint64_t rows;
    uint32_t cols;
    float eps;
};

// The larger of two magnitudes, NaN if one is.
__device__ __forceinline__ float norm_larger(float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
}
// |p| in f64 as an ordered number that carries NaN and infinities.
__device__ __forceinline__ unsigned long long norm_top_bits(float h, float w) {
    return (unsigned long long)__double_as_longlong((double)h * (double)w) & 0x7fffffffffffffffull;
}
// The f32 products neither overflowed nor lost bits below the normal range.
__device__ __forceinline__ bool norm_sure(float top) { return top >= 0x1p-90f && top <= 0x1p90f; }

// Where a CTA's threads meet: two sets, alternating from row to row (`turn`), so
// that a row's writes never meet the reads of the row before it.
struct NormShared {
    float2 red[2][32];
    unsigned long long top[2];
};
__device__ __forceinline__ NormShared& norm_shared() {
    __shared__ NormShared s;
    return s;
}

// Sum of squares and the largest |p| over a row's threads: a warp, or the
// whole CTA (one barrier).
template <bool WARP>
__device__ __forceinline__ void norm_q8_reduce(float& ss, float& top, int turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss = fadd(ss, __shfl_xor_sync(0xffffffffu, ss, o));
    top = __uint_as_float(q8_warp_max(__float_as_uint(top)));  // magnitudes: ordered as their bits, NaN last
    if (WARP) return;
    NormShared& sh = norm_shared();
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) sh.red[turn][warp] = make_float2(ss, top);
    if (threadIdx.x == 0) sh.top[turn] = 0;  // for norm_q8_refine
    __syncthreads();
    float2 v = sh.red[turn][0];
    ss = v.x;
    top = v.y;
    for (int i = 1; i < nw; ++i) {
        v = sh.red[turn][i];
        ss = fadd(ss, v.x);
        top = norm_larger(top, v.y);
    }
}
// Rare: a f64 sum and maximum over the row's threads (two barriers).
template <bool WARP>
__device__ __noinline__ double2 norm_q8_again(double ss, unsigned long long top) {
    ss = warp_sum_d(ss);
    top = warp_max_u64(top);
    if (!WARP) {
        __shared__ double rs[32];
        __shared__ unsigned long long rt[32];
        const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            rs[warp] = ss;
            rt[warp] = top;
        }
        __syncthreads();
        ss = rs[0];
        top = rt[0];
        for (int i = 1; i < nw; ++i) {
            ss += rs[i];
            top = rt[i] > top ? rt[i] : top;
        }
        __syncthreads();
    }
    return make_double2(ss, __longlong_as_double((long long)top));
}
// f32 rows: max|p| in f64 from the elements whose f32 product is the largest
// (one barrier).
template <bool WARP, typename VISIT>
__device__ __forceinline__ double norm_q8_refine(float top, int turn, VISIT visit) {
    unsigned long long t = 0;
    bool here = false;  // one branch for the few threads that hold the maximum
    visit([&](float h, float w) { here |= fabsf(fmul(h, w)) == top; });
    if (here) {
        visit([&](float h, float w) {
            const unsigned long long b = norm_top_bits(h, w);
            t = b > t ? b : t;
        });
    }
    if (WARP) return __longlong_as_double((long long)warp_max_u64(t));
    NormShared& sh = norm_shared();
    if (t) atomicMax(&sh.top[turn], t);
    __syncthreads();
    return __longlong_as_double((long long)sh.top[turn]);
}

// What a row's codes are decided by, and its scale.  visit(f) calls f(h, w) for
// each of the thread's elements, all threads of the row together.  Where the
// f32 sum of squares has left its range (values near 1e19, or all below 1e-18)
// or the f32 products have, both are taken in f64.
struct NormRow {
    double top;   // max|p|
    float scale;
    bool rounded;  // top is the f32 maximum of products that f32 rounds
};
template <typename T, bool WARP, typename VISIT>
__device__ __forceinline__ NormRow norm_q8_row(float ss, float top, const NormQ8Args& p, VISIT visit) {
    NormRow r;
    r.rounded = false;
    if (norm_sure(top) && ss >= 0x1p-80f && ss <= 0x1p100f) {
        r.top = (double)top;
        r.rounded = sizeof(T) == 4;
        const float rms = fsqrt(fadd(fdiv(ss, (float)p.cols), p.eps));
        r.scale = fdiv(top, fmul(127.0f, rms));
        return r;
    }
    double d = 0.0;
    unsigned long long t = 0;
    visit([&](float h, float w) {
        d = __fma_rn((double)h, (double)h, d);
        const unsigned long long b = norm_top_bits(h, w);
        t = b > t ? b : t;
    });
    const double2 again = norm_q8_again<WARP>(d, t);
    r.top = again.y;
    const double rms = sqrt(again.x / (double)p.cols + (double)p.eps);
    r.scale = (float)(r.top / (127.0 * rms));
    if (!(r.top <= 1.7976931348623157e308)) {  // a NaN or an infinity in the row (or in w): the whole row is NaN
        r.scale = q8_nan();
        r.top = 0.0;
    }
    return r;
}

// f32 rows: the exact max|p| (all threads of the row).
template <typename T, bool WARP, typename VISIT>
__device__ __forceinline__ void norm_q8_exact(NormRow& r, int turn, VISIT visit) {
    if (sizeof(T) == 4 && r.rounded) {
        r.top = norm_q8_refine<WARP>((float)r.top, turn, visit);
        r.rounded = false;
    }
}
// The same behind the row's codes, if one of its threads has codes to decide.
// In every row and before the codes it took 16.0 us instead of 14.6 at f32
// [2048, 4096], 98 instead of 85 at [16384, 4096]; rows held element by element
// are the faster for it, 20.9 instead of 22.6 us at [2047, 4097].
template <typename T, bool WARP, typename VISIT>
__device__ __forceinline__ void norm_q8_settle(NormRow& r, bool open, int turn, VISIT visit) {
    if constexpr (sizeof(T) == 4) {
        if (WARP ? __any_sync(0xffffffffu, open) : __syncthreads_or(open)) norm_q8_exact<T, WARP>(r, turn, visit);
    }
}

// nearest(127 p / top) for |p| <= top of at most 48 bits each, ties to even; 0
// where top is zero.  The f64 quotient, off by 2^-46, decides all but those next
// to a half-integer.  There 254 |p| = hi + lo exactly, and hi - (2 n + 1) top
// from one fused step is less than 2^16 units of the last place of either, so
// exact: the sum of the two has the sign of 254 |p| - (2 n + 1) top. 
static __device__ __forceinline__ int norm_nearest_here(double p, double top) {
    if (!(top > 0.0)) return 0;
    const double a = fabs(p), q = 127.0 * a / top, n = rint(q);
    int c = (int)n;
    if (fabs(q - n) > 0.5 - 0x1p-40) {
        const double hi = 254.0 * a, lo = __fma_rn(254.0, a, -hi);
        const double up = __fma_rn(-(2.0 * n + 1.0), top, hi) + lo, down = __fma_rn(-(2.0 * n - 1.0), top, hi) + lo;
        if (up > 0.0 || (up == 0.0 && (c & 1))) ++c;
        else if (down < 0.0 || (down == 0.0 && (c & 1))) --c;
    }
    return p < 0.0 ? -c : c;
}

// The same as a call, for kernels with many places of it.
static __device__ __noinline__ int norm_nearest(double p, double top) { return norm_nearest_here(p, top); }

// Codes nearest(127 p / top).
template <typename T>
struct NormCoder {
    double top;
    float ftop, inv;
    bool slow;
    Q8Bracket br;
    __device__ __forceinline__ explicit NormCoder(double t)
        : top(t),
          ftop((float)t),
          inv(norm_sure(ftop) ? fdiv(127.0f, ftop) : 0.0f),
          slow(!norm_sure(ftop)),
          br(inv) {}
    __device__ __forceinline__ int exact(float h, float w) const {
        if (sizeof(T) == 4 || slow) return norm_nearest((double)h * (double)w, top);
        const float p = fmul(h, w);  // 16 bits; 254 |p| and (2 n + 1) top are exact
        return q8_beside(p, 254.0f * fabsf(p), inv, ftop);
    }
};
// The codes of a packed vector by the definition.  (Without a call of norm_nearest
// inside, which cost the kernels 50 bytes of spills: f32 [16384, 4096] with r 140.6
// us against 144.1.)
template <typename T>
__device__ __noinline__ uint2 norm_decide(uint4 h, uint4 w, double top) {
    constexpr int V = Vec<T>::N;
    const NormCoder<T> c(top);
    float hv[V], wv[V];
    uint32_t q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    Vec<T>::unpack(h, hv);
    Vec<T>::unpack(w, wv);
#pragma unroll
    for (int e = 0; e < V; ++e)
        q[e] = (uint32_t)(sizeof(T) == 4 ? norm_nearest_here((double)hv[e] * (double)wv[e], top) : c.exact(hv[e], wv[e]));
    return make_uint2(q8_pack4(q[0], q[1], q[2], q[3]), q8_pack4(q[4], q[5], q[6], q[7]));
}

constexpr int NQ_VPT = 4;  // 16-byte vectors a thread holds

// WARP: eight rows per 256-thread CTA; else one row per CTA of up to MAXT threads.
// Three CTAs of 256 an SM at 80 registers, four for f32 without r at 64 (14.0 us
// against 14.6 with three, 77 against 85 when it was chosen; with r four were slower, 27.8 against
// 22.0).  All of these spill some: f32 about 100 bytes a thread, bf16 with r 40.
// Two CTAs, which spill nothing, were slower everywhere: bf16 [16384, 4096] with r
// 87.9 us against 82.0, f32 with r 158 against 141, f32 116 against 78.
template <typename T, bool ADD, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? (sizeof(T) == 4 && !ADD ? 4 : 3) : 1)
    rmsnorm_q8_vec_kernel(const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale, NormQ8Args p) {
    pdl_begin();
    constexpr int V = Vec<T>::N;
    constexpr bool KEEP = MAXT == 256;  // w in registers
    const uint32_t t = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
    const uint32_t nvec = p.cols / V;
    const uint64_t per = WARP ? 8 : 1;
    uint4 wraw[KEEP ? NQ_VPT : 1] = {};
    auto weight = [&](int k) -> uint4 {
        if (KEEP) return wraw[KEEP ? k : 0];
        return ld_keep(w + (uint64_t)(t + k * tpr) * V);
    };
    if (KEEP) {
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k)
            if (t + k * tpr < nvec) wraw[KEEP ? k : 0] = ld_keep(w + (uint64_t)(t + k * tpr) * V);
    }
    int turn = 0;
    for (uint64_t row = blockIdx.x * per + (WARP ? threadIdx.x >> 5 : 0); row < p.rows;
         row += gridDim.x * per, turn ^= 1) {
        const uint64_t off = row * p.cols;
        uint4 raw[NQ_VPT], rawr[ADD ? NQ_VPT : 1];
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k) {
            const uint32_t j = t + k * tpr;
            if (j < nvec) {
                raw[k] = ld_stream(x + off + (uint64_t)j * V);
                if (ADD) rawr[k] = ld_stream(r + off + (uint64_t)j * V);
            }
        }
        float2 acc = f2(0.0f, 0.0f);
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k) {
            const uint32_t j = t + k * tpr;
            if (j < nvec) {
                float v[V], wv[V];
                Vec<T>::unpack(raw[k], v);
                if (ADD) {
                    float rv[V], sv[V];
                    Vec<T>::unpack(rawr[ADD ? k : 0], rv);
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 u = fadd2(f2(v[e], v[e + 1]), f2(rv[e], rv[e + 1]));
                        sv[e] = u.x;
                        sv[e + 1] = u.y;
                    }
                    raw[k] = Vec<T>::pack(sv);  // h as stored
                    Vec<T>::unpack(raw[k], v);
                    st_stream(h + off + (uint64_t)j * V, raw[k]);
                }
                Vec<T>::unpack(weight(k), wv);
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 u = f2(v[e], v[e + 1]);
                    acc = __ffma2_rn(u, u, acc);
                    const float2 pr = fmul2(u, f2(wv[e], wv[e + 1]));
                    top = norm_larger(top, fabsf(pr.x));
                    top = norm_larger(top, fabsf(pr.y));
                }
            }
        }
        float ss = fadd(acc.x, acc.y);
        norm_q8_reduce<WARP>(ss, top, turn);
        auto visit = [&](auto f) {
#pragma unroll
            for (int k = 0; k < NQ_VPT; ++k) {
                if (t + k * tpr < nvec) {
                    float v[V], wv[V];
                    Vec<T>::unpack(raw[k], v);
                    Vec<T>::unpack(weight(k), wv);
#pragma unroll
                    for (int e = 0; e < V; ++e) f(v[e], wv[e]);
                }
            }
        };
        NormRow nr = norm_q8_row<T, WARP>(ss, top, p, visit);
        const NormCoder<T> coder(nr.top);
        uint32_t open = 0;  // vectors with codes that the definition has to decide
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k) {
            const uint32_t j = t + k * tpr;
            if (j < nvec) {
                float v[V], wv[V], pr[V];
                uint32_t c[V / 4];
                Vec<T>::unpack(raw[k], v);
                Vec<T>::unpack(weight(k), wv);
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 u = fmul2(f2(v[e], v[e + 1]), f2(wv[e], wv[e + 1]));
                    pr[e] = u.x;
                    pr[e + 1] = u.y;
                }
                open |= (q8_codes<V>(coder, pr, c) ? 1u : 0u) << k;
                q8_store(y + off + (uint64_t)j * V, c);
            }
        }
        norm_q8_settle<T, WARP>(nr, open != 0, turn, visit);
        if (open) {  // once more, behind the other stores
#pragma unroll
            for (int k = 0; k < NQ_VPT; ++k)
                if (open >> k & 1u) {
                    uint32_t c[V / 4];
                    q8_take(c, norm_decide<T>(raw[k], weight(k), nr.top));
                    q8_store(y + off + (uint64_t)(t + k * tpr) * V, c);
                }
        }
        if (t == 0) scale[row] = nr.scale;
    }
}

// Rows that are no whole aligned vectors, element by element in registers:
// thread t holds columns t + k blockDim.x, EPT of them, and its part of w.
// [2047, 4097] f32 19.3 us, 2.2 TB/s: loads of one element a thread.  (Aligned
// vectors shifted into place between neighbours took 24.6 us; all of a thread's
// codes decided by the definition where one of them has to be, 21.6.)
template <typename T, bool ADD, int EPT, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 320 ? 3 : (MAXT == 640 ? 2 : 1))
    rmsnorm_q8_odd_kernel(const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale, NormQ8Args p) {
    pdl_begin();
    float wv[EPT];
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
        const uint32_t i = threadIdx.x + k * blockDim.x;
        wv[k] = i < p.cols ? Vec<T>::load1(w + i) : 0.0f;
    }
    int turn = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const uint64_t off = row * p.cols;
        float v[EPT], rv[ADD ? EPT : 1];
#pragma unroll
        for (int k = 0; k < EPT; ++k) {
            const uint32_t i = threadIdx.x + k * blockDim.x;
            v[k] = i < p.cols ? Vec<T>::load1(x + off + i) : 0.0f;
            if (ADD) rv[ADD ? k : 0] = i < p.cols ? Vec<T>::load1(r + off + i) : 0.0f;
        }
        float ss = 0.0f, top = 0.0f;
#pragma unroll
        for (int k = 0; k < EPT; ++k) {
            const uint32_t i = threadIdx.x + k * blockDim.x;
            if (ADD) {
                v[k] = Vec<T>::rnd(fadd(v[k], rv[ADD ? k : 0]));
                if (i < p.cols) Vec<T>::store1(h + off + i, v[k]);
            }
            // places behind the row are zeros (0 + 0): they add nothing
            ss = __fmaf_rn(v[k], v[k], ss);
            top = norm_larger(top, fabsf(fmul(v[k], wv[k])));
        }
        norm_q8_reduce<false>(ss, top, turn);
        auto visit = [&](auto f) {
#pragma unroll
            for (int k = 0; k < EPT; ++k) f(v[k], wv[k]);
        };
        NormRow nr = norm_q8_row<T, false>(ss, top, p, visit);
        norm_q8_exact<T, false>(nr, turn, visit);
        const NormCoder<T> coder(nr.top);
        uint32_t c[EPT], open = 0;  // pairs with codes that the definition has to decide
#pragma unroll
        for (int k = 0; k < EPT; k += 2) {
            uint32_t diff = 0;
            const uint2 q = coder.br.two(fmul2(f2(v[k], v[k + 1]), f2(wv[k], wv[k + 1])), diff);
            c[k] = q.x;
            c[k + 1] = q.y;
            open |= (coder.slow || diff != 0 ? 1u : 0u) << k;
        }
        if (open) {
#pragma unroll
            for (int k = 0; k < EPT; ++k)
                if (open >> (k & ~1) & 1u) c[k] = (uint32_t)coder.exact(v[k], wv[k]);
        }
#pragma unroll
        for (int k = 0; k < EPT; ++k) {
            const uint32_t i = threadIdx.x + k * blockDim.x;
            if (i < p.cols) y[off + i] = (int8_t)(c[k] & 0xffu);
        }
        if (threadIdx.x == 0) scale[row] = nr.scale;
    }
}

// Any row length: one CTA per row, the row read twice (pass 2 re-reads x, or
// the stored h, with coherent loads, so x or r may be h).
template <typename T, bool ADD>
__global__ void __launch_bounds__(1024)
    rmsnorm_q8_long_kernel(const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale, NormQ8Args p) {
    pdl_begin();
    int turn = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const uint64_t off = row * p.cols;
        const T* src = (ADD ? h : x) + off;
        auto held = [&](uint32_t i) -> float {
            if (sizeof(T) == 4) return *reinterpret_cast<const volatile float*>(src + i);
            return bf16_to_f32(*reinterpret_cast<const volatile uint16_t*>(src + i));
        };
        float ss = 0.0f;
        float top = 0.0f;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            float v = Vec<T>::load1(x + off + i);
            if (ADD) {
                v = Vec<T>::rnd(fadd(v, Vec<T>::load1(r + off + i)));
                Vec<T>::store1(h + off + i, v);
            }
            ss = __fmaf_rn(v, v, ss);
            top = norm_larger(top, fabsf(fmul(v, Vec<T>::load1(w + i))));
        }
        norm_q8_reduce<false>(ss, top, turn);
        auto visit = [&](auto f) {
            for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) f(held(i), Vec<T>::load1(w + i));
        };
        NormRow nr = norm_q8_row<T, false>(ss, top, p, visit);
        norm_q8_exact<T, false>(nr, turn, visit);
        const NormCoder<T> coder(nr.top);
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            const float hv = held(i), wv = Vec<T>::load1(w + i);
            y[off + i] = (int8_t)q8_code(coder, fmul(hv, wv), [&] { return coder.exact(hv, wv); });
        }
        if (threadIdx.x == 0) scale[row] = nr.scale;
    }
}

template <typename T, bool ADD>
static int norm_q8_entry(const char* name, const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale,
                         uint64_t rows, uint64_t cols, float eps, cudaStream_t st) {
    OXIDE_INJECT(name);
    if (rows == 0) return OXIDE_OK;
    OXIDE_REQUIRE(x && w && y && scale && (!ADD || (r && h)), name, "null pointer");
    OXIDE_REQUIRE(cols >= 1 && cols < (1ull << 31), name, "cols must be in [1, 2^31)");
    OXIDE_REQUIRE(rows <= UINT64_MAX / 4 / cols, name, "rows * cols overflows");
    OXIDE_REQUIRE(static_cast<const void*>(y) != x && static_cast<const void*>(y) != r &&
                      static_cast<const void*>(y) != h, name, "the codes must not alias x, r or h");
    constexpr int V = Vec<T>::N;
    const NormQ8Args p{rows, (uint32_t)cols, eps};
    const bool vec = cols % V == 0 && aligned16(x) && aligned16(w) && (!ADD || (aligned16(r) && aligned16(h))) &&
                     (reinterpret_cast<uintptr_t>(y) & (V - 1)) == 0;
    const uint64_t nvec = cols / V, cap = 1ull << 30;
    // CTAs take rows in turn, one wave of them
    auto go = [&](auto kern, int threads, uint64_t per) {
        const uint64_t want = (rows + per - 1) / per;
        const uint64_t wave = (uint64_t)resident_blocks(reinterpret_cast<const void*>(kern), threads, 0);
        launch_k(kern, (unsigned)(want < wave ? want : wave), threads, 0, st, x, r, w, h, y, scale, p);
    };
    if (vec && nvec <= 32ull * NQ_VPT) {
        go(rmsnorm_q8_vec_kernel<T, ADD, true, 256>, 256, 8);
    } else if (vec && nvec <= 1024ull * NQ_VPT) {
        const int threads = (int)(((nvec + NQ_VPT - 1) / NQ_VPT + 31) / 32 * 32);
        if (threads <= 256) go(rmsnorm_q8_vec_kernel<T, ADD, false, 256>, threads, 1);
        else go(rmsnorm_q8_vec_kernel<T, ADD, false, 1024>, threads, 1);
    } else if (cols <= 1024ull * 16) {
        // Columns a thread holds: 16, or 8 where r and h are there as well ([2047,
        // 4097] bf16 31.0 us against 45.5 with 16, f32 30.2 against 33.0; without
        // them f32 23.0 against 21.5, and [30000, 300] bf16 28.1 against 25.4).
        constexpr uint64_t E = ADD ? 8 : 16;
        auto threads = [&](uint64_t e) { return (int)(((cols + e - 1) / e + 31) / 32 * 32); };
        if (cols <= 5120) go(rmsnorm_q8_odd_kernel<T, ADD, E, 5120 / E>, threads(E), 1);
        else if (cols <= 1024 * E) go(rmsnorm_q8_odd_kernel<T, ADD, E, 1024>, threads(E), 1);
        else go(rmsnorm_q8_odd_kernel<T, ADD, 16, 1024>, threads(16), 1);
    } else {
        launch_k(rmsnorm_q8_long_kernel<T, ADD>, (unsigned)(rows < cap ? rows : cap), 1024, 0, st, x, r, w, h, y, scale, p);
    }
    return check_launch(name);
}

}  // namespace oxide

using oxide::bf16_t;

extern "C" {

int oxide_rms_norm_q8_f32(const float* x, const float* w, int8_t* out, float* scale, uint64_t rows, uint64_t cols,
                          float eps, oxide_stream_t stream) {
    return oxide::norm_q8_entry<float, false>("oxide_rms_norm_q8_f32", x, nullptr, w, nullptr, out, scale, rows, cols,
                                              eps, stream);
}
int oxide_rms_norm_q8_bf16(const oxide_bf16* x, const oxide_bf16* w, int8_t* out, float* scale, uint64_t rows,
                           uint64_t cols, float eps, oxide_stream_t stream) {
    return oxide::norm_q8_entry<bf16_t, false>("oxide_rms_norm_q8_bf16", x, nullptr, w, nullptr, out, scale, rows,
                                               cols, eps, stream);
}
int oxide_add_rms_norm_q8_f32(const float* x, const float* r, const float* w, float* h, int8_t* out, float* scale,
                              uint64_t rows, uint64_t cols, float eps, oxide_stream_t stream) {
    return oxide::norm_q8_entry<float, true>("oxide_add_rms_norm_q8_f32", x, r, w, h, out, scale, rows, cols, eps,
                                             stream);
}
int oxide_add_rms_norm_q8_bf16(const oxide_bf16* x, const oxide_bf16* r, const oxide_bf16* w, oxide_bf16* h,
                               int8_t* out, float* scale, uint64_t rows, uint64_t cols, float eps,
                               oxide_stream_t stream) {
    return oxide::norm_q8_entry<bf16_t, true>("oxide_add_rms_norm_q8_bf16", x, r, w, h, out, scale, rows, cols, eps,
                                              stream);
}

}  // extern "C"
