// gelu.hpp — GELU and its slope on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vector16.hpp"

namespace ttp {
namespace {

constexpr float kSqrt2OverPi = 0.79788456080286535588f;
constexpr float kCubic = 0.044715f;

// The normal distribution function and its density at x.  With z = |x| / sqrt 2 and
// t = 1 / (1 + 0.46 z), erfc(z) = t poly(t) exp(-z^2), whose exponential is the density's.  poly is
// of the sixth degree, fitted here by least maximum error to exp(z^2) erfc(z) / t over z = 0 to 25,
// weighted by t max(exp(-z^2), 1e-4).  With its coefficients in fp32 erfc is 4.5e-8 off at 0 (2.2e-8
// of the distribution, whose fp32 unit there is 6e-8), 1.2e-8 from |x| = 0.7 and 6e-9 from 2 on, and
// 6e-5 of itself at x = -6; in fp32 arithmetic the distribution is 2e-7 off at most.
struct Normal {
    float cdf, pdf;
};
__device__ __forceinline__ Normal normal(float x) {
    const float z = fabsf(x) * 0.70710678118654752440f;
    const float e = exp2_fast(-z * z * kLog2e);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.46f, z, 1.0f));
    float poly = __builtin_fmaf(t, 0.0879725963f, -0.443790019f);
    poly = __builtin_fmaf(t, poly, 0.700208485f);
    poly = __builtin_fmaf(t, poly, -0.212298155f);
    poly = __builtin_fmaf(t, poly, 0.373866349f);
    poly = __builtin_fmaf(t, poly, 0.232440144f);
    poly = __builtin_fmaf(t, poly, 0.261600554f);
    const float upper = 0.5f * poly * t * e;  // beyond |x|
    return {x < 0.0f ? upper : 1.0f - upper, 0.39894228040143267794f * e};
}

template <bool kTanh>
__device__ __forceinline__ float gelu(float x) {
    if constexpr (kTanh) {
        // x / 2 (1 + tanh u) = x / (1 + exp(-2 u)); the exponential may be infinite
        const float u2 = 2.0f * kSqrt2OverPi * kLog2e * (x * __builtin_fmaf(kCubic * x, x, 1.0f));
        return x * __builtin_amdgcn_rcpf(1.0f + exp2_fast(-u2));
    } else {
        return x * normal(x).cdf;
    }
}
// gelu'(x); beyond 30 it is 0 or 1 in either form, and x^3 would overflow (NaN stays NaN)
template <bool kTanh>
__device__ __forceinline__ float gelu_slope(float x) {
    x = x < -30.0f ? -30.0f : x > 30.0f ? 30.0f : x;
    if constexpr (kTanh) {
        const float u2 = 2.0f * kSqrt2OverPi * kLog2e * (x * __builtin_fmaf(kCubic * x, x, 1.0f));
        // s = sigmoid(2 u), t = 1 - s; an infinite e leaves s = 0, and nothing but s
        const float e = exp2_fast(-u2), s = __builtin_amdgcn_rcpf(1.0f + e);
        const float t = fminf(e, 3.4e38f) * s;
        const float du2 = 2.0f * kSqrt2OverPi * __builtin_fmaf(3.0f * kCubic * x, x, 1.0f);
        return __builtin_fmaf(x * s * t, du2, s);
    } else {
        const Normal n = normal(x);
        return __builtin_fmaf(x, n.pdf, n.cdf);
    }
}

}  // namespace
}  // namespace ttp
