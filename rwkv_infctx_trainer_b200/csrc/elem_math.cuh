// Exponentials, sigmoids and softplus on the special function unit, with what their approximations lack made good: shared by the selective scan and
// the gated recurrence.
#pragma once
#include "wkv_common.cuh"

namespace wkv {

// (log2(e) as the sum of two floats)
constexpr float LOG2E = 1.4426950408889634f, LOG2E_LOW = 1.9259629911266175e-8f, LN2 = 0.6931471805599453f, EX2_MEAN = 1.8e-8f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ f2 ex2(f2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// e^x for x from -126 to 0: the rounding of the exponent x log2(e), up to 2^-24 of it, is made good, and so is the mean error of ex2,
// -5e-8 over exponents below -1 (above them it is -2e-8 and less: 3e-8 too much is added there, half a rounding)
__device__ __forceinline__ float exp_near(float x) {
    const float e = LOG2E * x, lo = fmaf(LOG2E, x, -e) + LOG2E_LOW * x, t = ex2(e);
    return fmaf(t, fmaf(lo, LN2, 5e-8f), t);
}
__device__ __forceinline__ float sigm(float x) { return rcp(1.f + ex2(-LOG2E * x)); }

// softplus(x) = max(x, 0) + log(1 + t), t = e^-|x|, and with SIG its derivative sigmoid(x), for any x: no term overflows.
// log(1 + t) = 2 artanh(s), s = t / (2 + t) <= 1/3: its power series up to s^13 is short of it by less than 2 s^15 / (15 (1 - s^2)), at
// most 1.05e-8 or a relative 1.5e-8, and keeps the digits of small steps (log of a rounded 1 + t does not).
template <bool SIG>
__device__ __forceinline__ float softplus(float x, float &sig) {
    float ax = -fabsf(x), s;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(ax) : "f"(-126.f));        // (infinities; a NaN stays)
    const float t = exp_near(ax);
    if (SIG) {
        const float w = rcp((1.f + t) * (2.f + t)), r = (2.f + t) * w;       // r = 1 / (1 + t)
        s = t * (1.f + t) * w;
        sig = x >= 0.f ? r : t * r;
    } else {
        s = t * rcp(2.f + t);
    }
    const float s2 = s * s;
    float p = 1.f / 13.f;
    p = p * s2 + 1.f / 11.f;
    p = p * s2 + 1.f / 9.f;
    p = p * s2 + 1.f / 7.f;
    p = p * s2 + 1.f / 5.f;
    p = p * s2 + 1.f / 3.f;
    p = p * s2 + 1.f;
    // (fmaxf drops a NaN, s brings it back)
    return fmaxf(x, 0.f) + 2.f * s * p;
}

}  // namespace wkv
