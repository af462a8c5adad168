// oxide_q8.cuh -- symmetric int8 codes: a code c stands for c * s, s the f32
// scale of its group (a row, or a block of tokens of one head), s = amax / 127.
//
// A code is the integer nearest to the real quotient x / s, ties to even,
// decided exactly: the fast path multiplies by a rounded reciprocal and is
// certain unless the product lies within its error of a half-integer; such a
// vector (about 1 element in 10^4) is redone with the f64 quotient.  That is
// enough: x and s have 24-bit significands, so near a half-integer
// x - (n + 1/2) s is a multiple of ulp(s) / 4, and a quotient that is not a
// half-integer is at least 2^-26 away from it, far above f64's 2^-47.
// So codes do not depend on the order of any sum or on the rounding of a
// reciprocal, and a 64-bit evaluation of the definition gives the same ones.
#pragma once

#include "oxide_common.cuh"

namespace oxide {

constexpr uint32_t Q8_INF = 0x7f800000u;  // bits of +inf: |x| bits above or at it are not finite
constexpr float Q8_MAGIC = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer in the low bits
// |t - round(t)| above this may be on either side of the half-integer.  t is
// off by at most 127.5 * 3 * 2^-24 = 2.3e-5 (three roundings: the reciprocal,
// and -- the norm's f32 products -- x and its maximum).
constexpr float Q8_NEAR = 0.49996f;

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

// Codes of values x against a divisor: code = nearest(x * num / den).
//   num = 1, den = s: a group's f32 scale;  num = 127, den = amax: a row's codes
//   from its largest value, without the rounding of a scale.
struct Q8Coder {
    double num, den;
    float inv;    // RN(num / den)
    bool slow;    // den zero, not finite, or so small or large that the fast path leaves the normal range
    __device__ __forceinline__ Q8Coder(double n, double d) : num(n), den(d) {
        const float df = (float)d;
        slow = !(df >= 0x1p-100f && df <= 0x1p100f);
        inv = slow ? 0.0f : (float)(n / d);
    }
    // A group's f32 scale as the divisor: one f32 reciprocal.
    __device__ __forceinline__ explicit Q8Coder(float s) : num(1.0), den((double)s) {
        slow = !(s >= 0x1p-100f && s <= 0x1p100f);
        inv = slow ? 0.0f : __frcp_rn(s);
    }
    // The definition itself; 0 where the divisor is zero or not finite.  The
    // quotient passes 127 only against a subnormal scale, whose own rounding
    // is coarse: it is held to 127.
    __device__ __forceinline__ int exact(double x) const {
        if (!(den > 0.0 && den <= 1.7976931348623157e308)) return 0;
        const double q = rint(x * num / den);
        return (int)(q > 127.0 ? 127.0 : (q < -127.0 ? -127.0 : q));
    }
    // Two codes, in the low bytes of the results' bits; `near` collects the
    // largest distance from an integer.
    __device__ __forceinline__ float2 fast2(float2 x, float& near) const {
        const float2 i2 = f2(inv, inv);
        const float2 r = __ffma2_rn(x, i2, f2(Q8_MAGIC, Q8_MAGIC));
        const float2 q = fadd2(r, f2(-Q8_MAGIC, -Q8_MAGIC));
        const float2 d = __ffma2_rn(x, i2, make_float2(-q.x, -q.y));
        near = fmaxf(near, fmaxf(fabsf(d.x), fabsf(d.y)));
        return r;
    }
};

// The low bytes of four words, in order.
__device__ __forceinline__ uint32_t q8_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// N codes of N values (N = 4 or 8) as N / 4 words.
template <int N>
__device__ __forceinline__ void q8_codes(const Q8Coder& c, const float (&x)[N], uint32_t (&out)[N / 4]) {
    float near = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const float2 a = c.fast2(f2(x[e], x[e + 1]), near), b = c.fast2(f2(x[e + 2], x[e + 3]), near);
        out[e / 4] = q8_pack4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    }
    if (c.slow || near > Q8_NEAR) {
#pragma unroll 1
        for (int e = 0; e < N; e += 4)
            out[e / 4] = q8_pack4((uint32_t)c.exact(x[e]), (uint32_t)c.exact(x[e + 1]), (uint32_t)c.exact(x[e + 2]),
                                  (uint32_t)c.exact(x[e + 3]));
    }
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

// Largest value over the warp (one instruction for unsigned numbers).
__device__ __forceinline__ uint32_t q8_warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

}  // namespace oxide
