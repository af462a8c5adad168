// oxide_q8.cuh -- symmetric int8 codes: a code c stands for c * s, s the f32
// scale of its group (a row, or a block of tokens of one head), s = amax / 127.
//
// A code is the integer nearest to the real quotient x / s, ties to even, and
// is decided exactly.  The fast path brackets the quotient: x times a
// reciprocal made a little smaller and a little larger than 1 / s, each rounded
// to an integer in one fused step.  Rounding is monotonic, so where both agree
// the quotient's integer is theirs; where they differ (about 1 element in 10^5)
// the quotient lies next to a half-integer and is compared with it: the sign
// of x - (n + 1/2) s from one fused step is exact.  So codes do not depend on
// the order of any sum or on the rounding of a reciprocal, and a 64-bit
// evaluation of the definition gives the same ones (near a half-integer
// x - (n + 1/2) s is a multiple of ulp(s) / 4, so another quotient is at least
// 2^-26 away from it, far above f64's 2^-47).  The norms' quotients are of
// 48-bit products: theirs take another decision (k_rmsnorm_q8.cu).
#pragma once

#include "oxide_common.cuh"

namespace oxide {

constexpr uint32_t Q8_INF = 0x7f800000u;  // bits of +inf: |x| bits above or at it are not finite
constexpr float Q8_MAGIC = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer in the low bits
// Relative half-width of the bracket around a quotient: 8 units of 2^-24, where
// the reciprocal, its two copies and -- the norm's f32 products -- x and the
// divisor are off by at most 5.
constexpr float Q8_WIDTH = 0x1p-21f;

__device__ __forceinline__ float q8_nan() { return __uint_as_float(0x7fffffffu); }

// Bits of |x| as an unsigned number: ordered like |x|, infinities above every
// number and NaN above those, so an unsigned maximum carries them along.
__device__ __forceinline__ uint32_t q8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a group whose largest |x| has these bits: amax / 127, NaN if
// the group holds a NaN or an infinity (all of it then reads back as NaN).
__device__ __forceinline__ float q8_scale_of(uint32_t amax_bits) {
    return amax_bits >= Q8_INF ? q8_nan() : fdiv(__uint_as_float(amax_bits), 127.0f);
}

// Largest |x| of one 16-byte vector, as bits.
__device__ __forceinline__ uint32_t q8_vec_amax(uint4 v, uint32_t a, float) {
    a = max(a, v.x & 0x7fffffffu);
    a = max(a, v.y & 0x7fffffffu);
    a = max(a, v.z & 0x7fffffffu);
    return max(a, v.w & 0x7fffffffu);
}
// bf16: two 16-bit maxima at a time; the accumulator holds two halves, joined
// by q8_amax_join.
__device__ __forceinline__ uint32_t q8_vec_amax(uint4 v, uint32_t a, bf16_t) {
    a = __vmaxu2(a, v.x & 0x7fff7fffu);
    a = __vmaxu2(a, v.y & 0x7fff7fffu);
    a = __vmaxu2(a, v.z & 0x7fff7fffu);
    return __vmaxu2(a, v.w & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t q8_amax_join(uint32_t a, float) { return a; }
__device__ __forceinline__ uint32_t q8_amax_join(uint32_t a, bf16_t) { return max(a << 16, a & 0xffff0000u); }

// The bracket of x times a factor.
struct Q8Bracket {
    float lo, hi;
    __device__ __forceinline__ explicit Q8Bracket(float inv)
        : lo(fmul(inv, 1.0f - Q8_WIDTH)), hi(fmul(inv, 1.0f + Q8_WIDTH)) {}
    // Two codes, in the low bytes of the result's bits; `diff` stays zero
    // while both ends of every bracket agree.
    __device__ __forceinline__ uint2 two(float2 x, uint32_t& diff) const {
        const float2 m = f2(Q8_MAGIC, Q8_MAGIC);
        const float2 a = __ffma2_rn(x, f2(lo, lo), m), b = __ffma2_rn(x, f2(hi, hi), m);
        diff |= __float_as_uint(a.x) ^ __float_as_uint(b.x);
        diff |= __float_as_uint(a.y) ^ __float_as_uint(b.y);
        return make_uint2(__float_as_uint(a.x), __float_as_uint(a.y));
    }
};

// A code next to a half-integer: |x| against (n - 1/2) s and (n + 1/2) s for an
// n within one of |x| / s.  a = 2 |x| u and s = d u, both exact, for any unit u.
__device__ __forceinline__ int q8_beside(float x, float twice, float inv, float d) {
    const float n = rintf(fmul(fabsf(x), inv));
    const float up = __fmaf_rn(-(2.0f * n + 1.0f), d, twice), down = __fmaf_rn(-(2.0f * n - 1.0f), d, twice);
    int c = (int)n;
    if (up > 0.0f || (up == 0.0f && (c & 1))) ++c;
    else if (down < 0.0f || (down == 0.0f && (c & 1))) --c;
    return x < 0.0f ? -c : c;
}

// Codes of values of type T under a group's f32 scale.
//
// bf16 values under a bf16 maximum's scale meet half-integers all the time (half
// the maximum is 63.5 steps), so they get a factor that needs no bracket.  Let a
// be the bf16 value with s = RN(a / 127), X and A the 8-bit significands of x
// and a.  127 x / a is a half-integer or at least a 254 X-th part of itself away
// from one (its distance is a fraction over 2 A 2^k): more than 2^-16.  x / s is
// (1 + d) times it, |d| <= 2^-24, d of the sign of a - 127 s.  So a factor
// 127 / a made larger or smaller by 2^-20 in that direction puts every x on its
// side: away from half-integers it changes nothing, on them it goes where d
// does.  Where a = 127 s exactly, 127 / a is a power of two and the rounding
// itself takes the half-integers to even.
template <typename T>
struct Q8Coder {
    bool slow;  // zero, not finite, or so small or large that the fast path leaves the normal range
    Q8Bracket br;
    // amax: the largest |x| if the scale is RN(amax / 127), else negative.
    __device__ __forceinline__ Q8Coder(float scale, float amax)
        : slow(!(scale >= 0x1p-100f && scale <= 0x1p100f)), br(0.0f) {
        if (slow) return;
        if (sizeof(T) == 2) {
            float a = amax;
            if (amax < 0.0f) {  // an older scale: of some bf16 maximum, mostly
                a = round_bf16(fmul(127.0f, scale));
                if (fdiv(a, 127.0f) != scale) a = -1.0f;
            }
            if (a > 0.0f) {
                const float r = __fmaf_rn(-127.0f, scale, a);  // its sign is exact
                const float f = fdiv(127.0f, a);
                br.lo = br.hi = r == 0.0f ? f : __fmaf_rn(f, r > 0.0f ? 0x1p-20f : -0x1p-20f, f);
                return;
            }
        }
        br = Q8Bracket(fdiv(1.0f, scale));
    }
};
// One code under a scale by the definition; 0 under a scale that is zero or not
// finite.  Scales far from 1 are brought near it, with x, by a power of two
// (exact for every x that reaches half a step).  A quotient passes 127 only
// under a subnormal scale, whose own rounding is coarse: it is held to 127.
__device__ __forceinline__ int q8_definition(float x, float scale) {
    if (!(scale > 0.0f && scale < INFINITY)) return 0;
    const float k = scale < 0x1p-60f ? 0x1p80f : (scale > 0x1p60f ? 0x1p-80f : 1.0f);
    const float xs = fmul(x, k), s = fmul(scale, k);
    const int c = q8_beside(xs, 2.0f * fabsf(xs), fdiv(1.0f, s), s);
    return max(-127, min(127, c));
}
// The code nearest to i had / s (0 <= i <= 127, had <= s finite, s > 0): products
// of a float and a small integer are exact in f64.
__device__ __forceinline__ int q8_restated(int i, float had, float s) {
    const double twice = 2.0 * i * (double)had;
    int c = (int)rintf(fdiv(fmul((float)i, had), s));
    const double up = (2 * c + 1) * (double)s, down = (2 * c - 1) * (double)s;
    if (twice > up || (twice == up && (c & 1))) ++c;
    else if (twice < down || (twice == down && (c & 1))) --c;
    return c;
}

// The low bytes of four words, in order.
__device__ __forceinline__ uint32_t q8_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// N codes of N values (N = 4 or 8) as N / 4 words; true if some of them have to
// be decided by the definition (the caller does that from its packed vector).
template <int N, typename C>
__device__ __forceinline__ bool q8_codes(const C& c, const float (&x)[N], uint32_t (&out)[N / 4]) {
    uint32_t diff = 0;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const uint2 a = c.br.two(f2(x[e], x[e + 1]), diff), b = c.br.two(f2(x[e + 2], x[e + 3]), diff);
        out[e / 4] = q8_pack4(a.x, a.y, b.x, b.y);
    }
    return c.slow || diff != 0;
}
// The codes of a packed vector by the definition.
template <typename T>
__device__ __forceinline__ uint2 q8_decide(uint4 raw, float scale) {
    constexpr int V = Vec<T>::N;
    float x[V];
    uint32_t q[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    Vec<T>::unpack(raw, x);
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = (uint32_t)q8_definition(x[e], scale);
    return make_uint2(q8_pack4(q[0], q[1], q[2], q[3]), q8_pack4(q[4], q[5], q[6], q[7]));
}
__device__ __forceinline__ void q8_take(uint32_t (&c)[1], uint2 v) { c[0] = v.x; }
__device__ __forceinline__ void q8_take(uint32_t (&c)[2], uint2 v) {
    c[0] = v.x;
    c[1] = v.y;
}
// One code.
template <typename C, typename X>
__device__ __forceinline__ int q8_code(const C& c, float x, X exact) {
    uint32_t diff = 0;
    const int q = (int)(int8_t)(c.br.two(f2(x, x), diff).x & 0xffu);
    return c.slow || diff != 0 ? exact() : q;
}

// Four codes as floats: the biased byte becomes the low significand bits of
// 2^23 + (c + 128).
__device__ __forceinline__ void q8_unpack4(uint32_t w, float (&f)[4]) {
    const uint32_t b = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = fsub(__uint_as_float(__byte_perm(b, 0x4B000000u, 0x7440 + i)), 8388736.0f);
}

// Byte stores of 4 or 8 codes.
__device__ __forceinline__ void q8_store(int8_t* p, const uint32_t (&c)[1]) {
    asm volatile("st.global.cs.u32 [%0], %1;" ::"l"(p), "r"(c[0]) : "memory");
}
__device__ __forceinline__ void q8_store(int8_t* p, const uint32_t (&c)[2]) {
    asm volatile("st.global.cs.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(c[0]), "r"(c[1]) : "memory");
}

// Loads of 4, 8 or 16 codes, used once.
__device__ __forceinline__ void q8_load(const int8_t* p, uint32_t (&c)[1]) {
    c[0] = __ldcs(reinterpret_cast<const unsigned int*>(p));
}
__device__ __forceinline__ void q8_load(const int8_t* p, uint32_t (&c)[2]) {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
    c[0] = v.x;
    c[1] = v.y;
}
__device__ __forceinline__ void q8_load(const int8_t* p, uint32_t (&c)[4]) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    c[0] = v.x;
    c[1] = v.y;
    c[2] = v.z;
    c[3] = v.w;
}
// Stores of 16 or 32 bytes of values.
__device__ __forceinline__ void st_stream32(void* p, uint4 a, uint4 b) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                 "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}
template <typename T, int N>
__device__ __forceinline__ void q8_store_values(T* p, const float (&x)[N]) {
    constexpr int V = Vec<T>::N;
    static_assert(N == V || N == 2 * V, "one or two 16-byte vectors");
    if constexpr (N == V) st_stream(p, Vec<T>::pack(x));
    else st_stream32(p, Vec<T>::pack(x), Vec<T>::pack(x + V));
}

// Largest value over the warp (one instruction for unsigned numbers).
__device__ __forceinline__ uint32_t q8_warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

}  // namespace oxide
