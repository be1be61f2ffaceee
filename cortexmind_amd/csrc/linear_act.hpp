// Activations of the layer products and their slopes from the saved
// pre-activation z.  The branch on the code is the same in every lane.
#pragma once

#include "ops.hpp"

namespace cxm {
namespace {

// Phi(z), the normal distribution, and exp(-z^2 / 2) beside it.  With
// a = |z| and t = 1 / (1 + c a): Phi(-a) exp(a^2 / 2) = t p(t), p fitted
// (iteratively reweighted least squares toward minimax in the relative error)
// over all a >= 0; Phi(a) = 1 - Phi(-a).  Relative error of t p(t): 7.5e-6
// with degree 6 (FINE = false, for 16-bit results, whose half step is 4.9e-4),
// 2.4e-7 with degree 9.  No branch, and the negative tail keeps its digits
// where 1 + erf loses them.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float z, float *bell) {
    const float a = fabsf(z);
    float p, t;
    if constexpr (FINE) {
        const float d = fmaf(a, 0.25f, 1.0f), r0 = __builtin_amdgcn_rcpf(d);
        t = d < FLT_MAX ? fmaf(fmaf(-d, r0, 1.0f), r0, r0) : 0.0f;
        p = 0x1.441b8ep-6f;
        p = fmaf(p, t, -0x1.4b45cap-4f);
        p = fmaf(p, t, 0x1.879068p-4f);
        p = fmaf(p, t, -0x1.03d3b0p-5f);
        p = fmaf(p, t, 0x1.04e924p-4f);
        p = fmaf(p, t, 0x1.e32000p-5f);
        p = fmaf(p, t, 0x1.4e3f0cp-4f);
        p = fmaf(p, t, 0x1.7ed694p-4f);
        p = fmaf(p, t, 0x1.98853ap-4f);
        p = fmaf(p, t, 0x1.988452p-4f);
    } else {
        t = __builtin_amdgcn_rcpf(fmaf(a, 0.4f, 1.0f));
        p = 0x1.982524p-5f;
        p = fmaf(p, t, -0x1.1df79ep-3f);
        p = fmaf(p, t, 0x1.e6effep-5f);
        p = fmaf(p, t, 0x1.3c3a50p-4f);
        p = fmaf(p, t, 0x1.12593ap-3f);
        p = fmaf(p, t, 0x1.46ee38p-3f);
        p = fmaf(p, t, 0x1.46cfa6p-3f);
    }
    const float u = z * -0x1.715476p-1f;  // -log2(e) / 2
    const float e = FINE ? exp2f(u * z) : __builtin_amdgcn_exp2f(u * z);
    *bell = e;
    const float low = p * t * e;
    return z > 0.0f ? 1.0f - low : low;
}

template <bool FINE>
__device__ __forceinline__ float sigmoid_of(float z) {
    if constexpr (FINE) {
        return act<CXM_ACT_SIGMOID>(z);
    } else {
        // 1 / (1 + 2^(-z log2 e)); the infinity of a large -z gives 0
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -0x1.715476p+0f));
    }
}

template <bool FINE, int N>
__device__ __forceinline__ void act_apply(int code, float (&z)[N]) {
    float b;
    switch (code) {
        case CXM_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = act<CXM_ACT_RELU>(z[e]);
            break;
        case CXM_ACT_SIGMOID:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = sigmoid_of<FINE>(z[e]);
            break;
        case CXM_ACT_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = act<CXM_ACT_TANH>(z[e]);
            break;
        case CXM_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] *= normal_cdf<FINE>(z[e], &b);
            break;
        case CXM_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] *= sigmoid_of<FINE>(z[e]);
            break;
        default: break;
    }
}

// act'(z).  tanh' is 4 s (1 - s) with s = sigmoid(2 z): 1 - tanh^2 loses its
// digits where tanh nears 1.
template <bool FINE, int N>
__device__ __forceinline__ void act_slope(int code, const float (&z)[N], float (&d)[N]) {
    switch (code) {
        case CXM_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) d[e] = z[e] > 0.0f ? 1.0f : 0.0f;
            break;
        case CXM_ACT_SIGMOID:
        case CXM_ACT_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float x = code == CXM_ACT_TANH ? 2.0f * z[e] : z[e];
                const float s = sigmoid_of<FINE>(-fabsf(x));  // the smaller of s and 1 - s
                const float t = s * (1.0f - s);
                d[e] = code == CXM_ACT_TANH ? 4.0f * t : t;
            }
            break;
        case CXM_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float b;
                const float c = normal_cdf<FINE>(z[e], &b);
                d[e] = fmaf(z[e] * 0x1.988454p-2f, b, c);  // Phi + z phi, phi = bell / sqrt(2 pi)
            }
            break;
        case CXM_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float s = sigmoid_of<FINE>(z[e]), q = sigmoid_of<FINE>(-z[e]);
                d[e] = s * fmaf(z[e], q, 1.0f);
            }
            break;
        default:
#pragma unroll
            for (int e = 0; e < N; ++e) d[e] = 1.0f;
            break;
    }
}

}  // namespace
}  // namespace cxm
