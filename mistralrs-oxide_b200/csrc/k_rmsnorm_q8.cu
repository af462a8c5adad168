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
// almost every code; max|p| is found in f64 (the products of two floats are
// exact there), and a code next to a half-integer is decided from the f64
// product (oxide_q8.cuh).
//
// Layout.  A warp (rows of at most 128 vectors of 16 bytes) or a CTA owns a
// row and keeps it packed in registers, four vectors a thread, so each row
// crosses HBM once; w comes from L1 both times it is needed.  Bound by HBM
// bytes: x, r and h in their type, one byte out.  Odd or unaligned rows and
// rows over 4096 vectors take a two-pass kernel whose second read is served
// by L1 / L2.
#include "oxide_q8.cuh"

namespace oxide {

struct NormQ8Args {
    uint64_t rows;
    uint32_t cols;
    float eps;
};

// Sum of squares and the largest |p| over a row's threads: a warp, or the
// whole CTA (then through shared memory; contains __syncthreads()).
template <bool WARP, typename M>
__device__ __forceinline__ void norm_q8_reduce(float& ss, M& top) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ss = fadd(ss, __shfl_xor_sync(0xffffffffu, ss, o));
        const M t = __shfl_xor_sync(0xffffffffu, top, o);
        top = t > top ? t : top;
    }
    if (WARP) return;
    __shared__ float rs[32];
    __shared__ M rt[32];
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        rs[warp] = ss;
        rt[warp] = top;
    }
    __syncthreads();
    ss = rs[0];
    top = rt[0];
    for (int i = 1; i < nw; ++i) {
        ss = fadd(ss, rs[i]);
        top = rt[i] > top ? rt[i] : top;
    }
    __syncthreads();  // the arrays are written again for the next row
}
template <bool WARP>
__device__ __forceinline__ double norm_q8_sum(double v) {
    v = warp_sum_d(v);
    if (WARP) return v;
    __shared__ double rd[32];
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) rd[warp] = v;
    __syncthreads();
    v = rd[0];
    for (int i = 1; i < nw; ++i) v += rd[i];
    __syncthreads();
    return v;
}

// |p| of one product as an ordered number that carries NaN and infinities:
// bf16 products in f32 (exact), f32 products in f64 (exact).
template <typename T>
struct NormTop;
template <>
struct NormTop<bf16_t> {
    typedef uint32_t M;
    __device__ __forceinline__ static M of(float h, float w) { return q8_abs_bits(fmul(h, w)); }
    __device__ __forceinline__ static double value(M m) { return (double)__uint_as_float(m); }
    // the f32 products neither overflowed nor lost bits below the normal range
    __device__ __forceinline__ static bool sure(M m) { return m >= 0x0d800000u && m < 0x72000000u; }
};
template <>
struct NormTop<float> {
    typedef unsigned long long M;
    __device__ __forceinline__ static M of(float h, float w) {
        return (M)__double_as_longlong((double)h * (double)w) & 0x7fffffffffffffffull;
    }
    __device__ __forceinline__ static double value(M m) { return __longlong_as_double((long long)m); }
    __device__ __forceinline__ static bool sure(M m) {
        const double v = value(m);
        return v >= 0x1p-100 && v <= 0x1p100;
    }
};

// What a row's codes are decided by, and its scale.  `again(what)` recomputes
// a row statistic in f64 (every thread of the row calls it together): the f32
// sum of squares has left its range (values near 1e19, or all below 1e-18),
// or the bf16 products have.
struct NormRow {
    double top;   // max|p|
    float scale;
};
template <typename T, typename SS, typename TT>
__device__ __forceinline__ NormRow norm_q8_row(float ss, typename NormTop<T>::M m, const NormQ8Args& p, SS again_ss,
                                               TT again_top) {
    NormRow r;
    if (NormTop<T>::sure(m) && ss >= 0x1p-80f && ss <= 0x1p100f) {
        r.top = NormTop<T>::value(m);
        const float rms = fsqrt(fadd(fdiv(ss, (float)p.cols), p.eps));
        r.scale = fdiv((float)r.top, fmul(127.0f, rms));
        return r;
    }
    const double s = again_ss();
    r.top = again_top();
    const double rms = sqrt(s / (double)p.cols + (double)p.eps);
    r.scale = (float)(r.top / (127.0 * rms));
    if (!(r.top <= 1.7976931348623157e308)) {  // a NaN or an infinity in the row (or in w): the whole row is NaN
        r.scale = q8_nan();
        r.top = 0.0;
    }
    return r;
}

// Codes of N products h w, in f32 where that is certain, else in f64.
template <int N>
__device__ __forceinline__ void norm_q8_codes(const Q8Coder& c, const float (&h)[N], const float (&w)[N],
                                              uint32_t (&out)[N / 4]) {
    float near = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const float2 a = c.fast2(fmul2(f2(h[e], h[e + 1]), f2(w[e], w[e + 1])), near);
        const float2 b = c.fast2(fmul2(f2(h[e + 2], h[e + 3]), f2(w[e + 2], w[e + 3])), near);
        out[e / 4] = q8_pack4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    }
    if (c.slow || near > Q8_NEAR) {
#pragma unroll 1
        for (int e = 0; e < N; e += 4) {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = (uint32_t)c.exact((double)h[e + i] * (double)w[e + i]);
            out[e / 4] = q8_pack4(q[0], q[1], q[2], q[3]);
        }
    }
}

constexpr int NQ_VPT = 4;  // 16-byte vectors a thread holds

// WARP: eight rows per 256-thread CTA; else one row per CTA.
template <typename T, bool ADD, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
    rmsnorm_q8_vec_kernel(const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale, NormQ8Args p) {
    pdl_begin();
    constexpr int V = Vec<T>::N;
    typedef NormTop<T> Top;
    const uint32_t t = WARP ? threadIdx.x & 31 : threadIdx.x, tpr = WARP ? 32 : blockDim.x;
    const uint32_t nvec = p.cols / V;
    const uint64_t per = WARP ? 8 : 1;
    for (uint64_t row = blockIdx.x * per + (WARP ? threadIdx.x >> 5 : 0); row < p.rows; row += gridDim.x * per) {
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
        typename Top::M top = 0;
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k) {
            const uint32_t j = t + k * tpr;
            if (j < nvec) {
                float v[V], wv[V];
                Vec<T>::unpack(raw[k], v);
                Vec<T>::unpack(ld_keep(w + (uint64_t)j * V), wv);
                if (ADD) {
                    float rv[V];
                    Vec<T>::unpack(rawr[ADD ? k : 0], rv);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = Vec<T>::rnd(fadd(v[e], rv[e]));
                    raw[k] = Vec<T>::pack(v);  // exact: v already holds T values
                    st_stream(h + off + (uint64_t)j * V, raw[k]);
                }
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 u = f2(v[e], v[e + 1]);
                    acc = __ffma2_rn(u, u, acc);
                    const typename Top::M a = Top::of(v[e], wv[e]), b = Top::of(v[e + 1], wv[e + 1]);
                    const typename Top::M ab = a > b ? a : b;
                    top = ab > top ? ab : top;
                }
            }
        }
        float ss = fadd(acc.x, acc.y);
        norm_q8_reduce<WARP>(ss, top);
        auto again_ss = [&]() {
            double d = 0.0;
#pragma unroll
            for (int k = 0; k < NQ_VPT; ++k) {
                if (t + k * tpr < nvec) {
                    float v[V];
                    Vec<T>::unpack(raw[k], v);
#pragma unroll
                    for (int e = 0; e < V; ++e) d = __fma_rn((double)v[e], (double)v[e], d);
                }
            }
            return norm_q8_sum<WARP>(d);
        };
        auto again_top = [&]() {
            unsigned long long m = 0;
#pragma unroll
            for (int k = 0; k < NQ_VPT; ++k) {
                const uint32_t j = t + k * tpr;
                if (j < nvec) {
                    float v[V], wv[V];
                    Vec<T>::unpack(raw[k], v);
                    Vec<T>::unpack(ld_keep(w + (uint64_t)j * V), wv);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const unsigned long long a = NormTop<float>::of(v[e], wv[e]);
                        m = a > m ? a : m;
                    }
                }
            }
            float none = 0.0f;
            norm_q8_reduce<WARP>(none, m);
            return NormTop<float>::value(m);
        };
        const NormRow nr = norm_q8_row<T>(ss, top, p, again_ss, again_top);
        const Q8Coder coder(127.0, nr.top);
#pragma unroll
        for (int k = 0; k < NQ_VPT; ++k) {
            const uint32_t j = t + k * tpr;
            if (j < nvec) {
                float v[V], wv[V];
                uint32_t c[V / 4];
                Vec<T>::unpack(raw[k], v);
                Vec<T>::unpack(ld_keep(w + (uint64_t)j * V), wv);
                norm_q8_codes<V>(coder, v, wv, c);
                q8_store(y + off + (uint64_t)j * V, c);
            }
        }
        if (t == 0) scale[row] = nr.scale;
    }
}

// Any row length and alignment: one CTA per row, the row read twice (pass 2
// re-reads x, or the stored h, with coherent loads, so x or r may be h).
template <typename T, bool ADD>
__global__ void __launch_bounds__(256)
    rmsnorm_q8_scalar_kernel(const T* x, const T* r, const T* w, T* h, int8_t* y, float* scale, NormQ8Args p) {
    pdl_begin();
    typedef NormTop<T> Top;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const uint64_t off = row * p.cols;
        const T* src = (ADD ? h : x) + off;
        auto held = [&](uint32_t i) -> float {
            if (sizeof(T) == 4) return *reinterpret_cast<const volatile float*>(src + i);
            return bf16_to_f32(*reinterpret_cast<const volatile uint16_t*>(src + i));
        };
        float ss = 0.0f;
        typename Top::M top = 0;
        for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            float v = Vec<T>::load1(x + off + i);
            if (ADD) {
                v = Vec<T>::rnd(fadd(v, Vec<T>::load1(r + off + i)));
                Vec<T>::store1(h + off + i, v);
            }
            ss = __fmaf_rn(v, v, ss);
            const typename Top::M a = Top::of(v, Vec<T>::load1(w + i));
            top = a > top ? a : top;
        }
        norm_q8_reduce<false>(ss, top);
        auto again_ss = [&]() {
            double d = 0.0;
            for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) d = __fma_rn((double)held(i), (double)held(i), d);
            return norm_q8_sum<false>(d);
        };
        auto again_top = [&]() {
            unsigned long long m = 0;
            for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
                const unsigned long long a = NormTop<float>::of(held(i), Vec<T>::load1(w + i));
                m = a > m ? a : m;
            }
            float none = 0.0f;
            norm_q8_reduce<false>(none, m);
            return NormTop<float>::value(m);
        };
        const NormRow nr = norm_q8_row<T>(ss, top, p, again_ss, again_top);
        const Q8Coder coder(127.0, nr.top);
        for (uint32_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            const float v = held(i), wv = Vec<T>::load1(w + i);
            float near = 0.0f;
            const float2 q = coder.fast2(fmul2(f2(v, v), f2(wv, wv)), near);
            int c = (int)(int8_t)(__float_as_uint(q.x) & 0xffu);
            if (coder.slow || near > Q8_NEAR) c = coder.exact((double)v * (double)wv);
            y[off + i] = (int8_t)c;
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
    if (vec && nvec <= 32ull * NQ_VPT) {
        const uint64_t want = (rows + 7) / 8;
        launch_k(rmsnorm_q8_vec_kernel<T, ADD, true>, (unsigned)(want < cap ? want : cap), 256, 0, st, x, r, w, h, y,
                 scale, p);
    } else if (vec && nvec <= 1024ull * NQ_VPT) {
        const int threads = (int)(((nvec + NQ_VPT - 1) / NQ_VPT + 31) / 32 * 32);
        launch_k(rmsnorm_q8_vec_kernel<T, ADD, false>, (unsigned)(rows < cap ? rows : cap), threads, 0, st, x, r, w, h,
                 y, scale, p);
    } else {
        launch_k(rmsnorm_q8_scalar_kernel<T, ADD>, (unsigned)(rows < cap ? rows : cap), 256, 0, st, x, r, w, h, y,
                 scale, p);
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
