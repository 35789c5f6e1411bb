// Activations of the linear layers and their slopes, in fp32.
#pragma once
#include <type_traits>

#include "mq_api_internal.hpp"
#include "mq_common.hpp"

namespace mq {

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// exp(-z^2 / 2) and Phi(z), the normal distribution's share below z.  The smaller side is exp(-z^2 / 2) r(|z| / sqrt 2), r(x) =
// erfc(x) exp(x^2) / 2, and r a polynomial in t = 1 / (1 + 0.415 x) without a constant, for r falls like 1 / x.  Its six coefficients
// come from a linear program over 0 <= x <= 9.7 that makes the larger of the error of r over 3e-5 r and that of the share over 7e-8 as
// small as can be.  In fp32 the share is off by at most 2.5e-7, and below -3 by at most 5e-5 of itself, a tenth of half a step of an
// fp16 result, down to where a bf16 one is subnormal (-13).  (Five coefficients do not do: 16 times those bounds.)
__device__ __forceinline__ void normal_share(float z, float& bell, float& share) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.29344931419f, __builtin_fabsf(z), 1.0f));          // (0.415 / sqrt 2)
    float p = __builtin_fmaf(t, -0.0853783410f, 0.2613799623f);
    p = __builtin_fmaf(t, p, -0.0655398461f);
    p = __builtin_fmaf(t, p, 0.1658386323f);
    p = __builtin_fmaf(t, p, 0.1057916691f);
    p = __builtin_fmaf(t, p, 0.1179078515f);
    bell = __builtin_amdgcn_exp2f(z * z * -0.7213475204444817f);
    const float tail = t * p * bell;
    share = z < 0.0f ? tail : 1.0f - tail;
}
// (0 from -87.4 down, where the reciprocal would be subnormal: what SiLU and tanh GELU lose there is below 1.1e-36)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == MQ_ACT_RELU) return z < 0.0f ? 0.0f : z;          // (a NaN stays)
    if (ACT == MQ_ACT_SILU) return z * sigmoid(z);
    if (ACT == MQ_ACT_GELU) {
        float bell, share;
        normal_share(z, bell, share);
        return z * share;
    }
    // 0.5 z (1 + tanh(u)) = z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
    if (ACT == MQ_ACT_GELU_TANH) return z * sigmoid(1.5957691216057308f * z * __builtin_fmaf(0.044715f, z * z, 1.0f));
    return z;
}
// The slope of the activation at z.  From 128 on it is 0 or 1 in fp32, and there it is taken: a larger z, or its cube, would be an
// infinity times 0 (z is finite, or an infinity that an 8-bit copy made of a value next to the largest).  A NaN stays.
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if (ACT == MQ_ACT_RELU) return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    const float c = __builtin_fabsf(z) > 128.0f ? __builtin_copysignf(128.0f, z) : z;
    if (ACT == MQ_ACT_SILU) {
        const float s = sigmoid(c);
        return s * __builtin_fmaf(c, 1.0f - s, 1.0f);
    }
    if (ACT == MQ_ACT_GELU) {
        float bell, share;
        normal_share(c, bell, share);
        return __builtin_fmaf(c * 0.3989422804014327f, bell, share);
    }
    if (ACT == MQ_ACT_GELU_TANH) {
        const float s = sigmoid(1.5957691216057308f * c * __builtin_fmaf(0.044715f, c * c, 1.0f));
        return s * __builtin_fmaf(1.5957691216057308f * c * __builtin_fmaf(0.134145f, c * c, 1.0f), 1.0f - s, 1.0f);
    }
    return 1.0f;
}

// the activation as a template argument
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
    if (act == MQ_ACT_GELU) f(std::integral_constant<int, MQ_ACT_GELU>{});
    else if (act == MQ_ACT_SILU) f(std::integral_constant<int, MQ_ACT_SILU>{});
    else if (act == MQ_ACT_RELU) f(std::integral_constant<int, MQ_ACT_RELU>{});
    else if (act == MQ_ACT_GELU_TANH) f(std::integral_constant<int, MQ_ACT_GELU_TANH>{});
    else f(std::integral_constant<int, MQ_ACT_NONE>{});
}

}  // namespace mq
