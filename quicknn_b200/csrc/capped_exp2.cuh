// Weights of attention on the 5th-generation tensor cores, taken on pairs of scores: exponentials to base 2, and exp(cap tanh(score / cap)) with part of
// the exponentials on the FMA pipe.
#pragma once
#include "common.cuh"
#include <float.h>
#include <math_constants.h>

namespace qnn {
namespace tc {

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two floats in a register pair: one instruction does both, each rounded like the single operation.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void one_by_one(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 2^x on the FMA and integer pipes, for |x| < 126: x = n + f with n the nearest integer (the sum with 1.5 * 2^23
// leaves n in the low mantissa bits), 2^f by a cubic on [-0.5, 0.5] (relative error 7.5e-5, a thirtieth of
// bfloat16's rounding), n added to the exponent field.  The special-function unit does 16 operations a clock per
// SM and a capped score needs two (tanh, 2^x): taking some of the exponentials here relieves it.  Prompt attention, measured with
// 0, 2, 4, 6, 8 of every 8 columns done this way, 8 heads of 256, one prompt: 2048 tokens 36.8 / 36.1 / 35.1 / 35.2 /
// 38.4 us, 8192 tokens 243 / 241 / 238 / 239 / 253 us; 32 heads of 128 at 8192: 831 / 815 / 796 / 800 / 869 us.
constexpr int POLY = 4;            // of every 8 columns of a row

// (a, b) <- exp(cap tanh(score / cap)) of two scores; `poly`: 2^x by the polynomial described at POLY.  There a score that is NaN
// comes out as FLT_MAX: the shifted bits of n = NaN wrap the exponent field.  `capped_sum` finds it.
__device__ __forceinline__ uint64_t capped_exp2(float& a, float& b, uint64_t k1, uint64_t k2, bool poly) {
    float x, y;
    one_by_one(mul2(two(a, b), k1), x, y);
    const uint64_t t = two(tanh_approx(x), tanh_approx(y));
    if (poly) {
        const uint64_t magic = two(12582912.f, 12582912.f), minus = two(-1.f, -1.f);
        const uint64_t xf = fma2(t, k2, magic);
        const uint64_t f = fma2(t, k2, fma2(xf, minus, magic));
        uint64_t q = fma2(f, two(0.055171407759189606f, 0.055171407759189606f), two(0.24261075258255005f, 0.24261075258255005f));
        q = fma2(q, f, two(0.6932609677314758f, 0.6932609677314758f));
        q = fma2(q, f, two(0.9999281167984009f, 0.9999281167984009f));
        float qa, qb, na, nb;
        one_by_one(q, qa, qb);
        one_by_one(xf, na, nb);
        a = __int_as_float(__float_as_int(qa) + (__float_as_int(na) << 23));
        b = __int_as_float(__float_as_int(qb) + (__float_as_int(nb) << 23));
    } else {
        one_by_one(mul2(t, k2), x, y);
        a = exp2_fast(x);
        b = exp2_fast(y);
    }
    return two(a, b);
}
// The sum of up to 64 such weights from the sums of their columns c % 4.  Weights are positive and at most e^70, so a sum that reaches FLT_MAX holds one
// of a NaN: it becomes a NaN, and with it everything that is divided by the row's sum.
__device__ __forceinline__ float capped_sum(uint64_t s01, uint64_t s23) {
    float a, b, c, d;
    one_by_one(s01, a, b);
    one_by_one(s23, c, d);
    const float s = (a + b) + (c + d);
    return s < FLT_MAX ? s : CUDART_NAN_F;
}

}  // namespace tc
}  // namespace qnn
