// The gated dense block's activations (gated.hip, gemm_x3.hip).
#pragma once
#include "common.h"

namespace geogcn {

// Every epilogue element pays for these, so they are written with the hardware's exponential and reciprocal (1 ulp each); what is held is the
// absolute error, about 2e-7 of the larger of 1 and |x| -- that of the pre-activation itself.
__device__ __forceinline__ float exp_neg(float y) { return __builtin_amdgcn_exp2f(-1.44269504f * y); }       // e^-y, y >= 0 (its relative error grows as 1e-7 y: harmless, the value shrinks faster)

// tanh: odd polynomial where 1 - e^-2|x| would cancel (|x| < 0.3; the Taylor series to x^9, next term 6e-8 x at most), else (1 - e) / (1 + e)
__device__ __forceinline__ float tanh_fast(float x) {
    const float a = fabsf(x), e = exp_neg(2.f * a), s = x * x;
    const float t = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
    const float p = fmaf(s, fmaf(s, fmaf(s, fmaf(s, 0.021869489f, -0.053968254f), 0.13333333f), -0.33333333f), 1.f) * x;
    return a < 0.3f ? p : copysignf(t, x);
}
// the normal distribution at x: e = exp(-x^2 / 2), cdf = Phi(x) = e * R(t) / 2 for x < 0 (1 - that for x > 0), t = 1 / (1 + 0.3 |x|), where R is a
// polynomial fitted here to exp(z^2) erfc(z), z = |x| / sqrt 2, over t in (0, 1] (ten terms t .. t^10, largest error 1.8e-8, at t = 0.97)
__device__ __forceinline__ void normal_fast(float x, float& cdf, float& e) {
    const float a = fabsf(x), t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
    e = exp_neg(0.5f * x * x);
    constexpr float k[10] = {0.239366293f, 0.239314735f, 0.218773827f, 0.165909439f, 0.162710696f, -0.098400034f, 0.305306107f, -0.394102961f, 0.197030291f, -0.035908401f};
    float r = k[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) r = fmaf(r, t, k[i]);
    const float q = 0.5f * e * r * t;
    cdf = x < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float gate_value(int act, float x) {
    switch (act) {
        case GEOGCN_ACT_SILU: return x * apply_act<GEOGCN_ACT_SIGMOID>(x);
        case GEOGCN_ACT_GELU: {
            float c, e;
            normal_fast(x, c, e);
            return x * c;
        }
        case GEOGCN_ACT_SIGMOID: return apply_act<GEOGCN_ACT_SIGMOID>(x);
        case GEOGCN_ACT_TANH: return tanh_fast(x);
        case GEOGCN_ACT_RELU: return x > 0.f ? x : (x == x ? 0.f : x);
        default: return x;
    }
}
__device__ __forceinline__ void gate_value_grad(int act, float x, float& v, float& d) {
    switch (act) {
        case GEOGCN_ACT_SILU: {
            const float s = apply_act<GEOGCN_ACT_SIGMOID>(x);
            v = x * s;
            d = s * fmaf(x, 1.f - s, 1.f);
            return;
        }
        case GEOGCN_ACT_GELU: {
            float c, e;
            normal_fast(x, c, e);
            v = x * c;
            d = fmaf(x * 0.39894228f, e, c);
            return;
        }
        case GEOGCN_ACT_SIGMOID: {
            v = apply_act<GEOGCN_ACT_SIGMOID>(x);
            d = v * (1.f - v);
            return;
        }
        case GEOGCN_ACT_TANH: {
            v = tanh_fast(x);
            d = fmaf(-v, v, 1.f);
            return;
        }
        case GEOGCN_ACT_RELU: {
            v = x > 0.f ? x : (x == x ? 0.f : x);
            d = x > 0.f ? 1.f : 0.f;
            return;
        }
        default: v = x; d = 1.f;
    }
}

}  // namespace geogcn
