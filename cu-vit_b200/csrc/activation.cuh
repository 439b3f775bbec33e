// The activations of cuvit_linear in FP32.
#pragma once

#include "cuvit_b200.h"
#include "ptx.cuh"

namespace cuvit::dev {

// x Phi(x) = x erfc(-x / sqrt 2) / 2, which keeps its relative accuracy where 1 + erf cancels.
__device__ __forceinline__ float gelu_exact(float x) {
    return 0.5F * x * erfcf(-0.7071067811865475F * x);
}

// x (1 + tanh u) / 2 = x / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3).
__device__ __forceinline__ float gelu_tanh_exact(float x) {
    const float u2 = 1.5957691216057308F * fmaf(0.044715F * x * x, x, x);
    return x / (1.0F + expf(-u2));
}

__device__ __forceinline__ float silu_exact(float x) { return x / (1.0F + expf(-x)); }

__device__ __forceinline__ float activate_exact(int activation, float x) {
    switch (activation) {
    case CUVIT_ACTIVATION_GELU:
        return gelu_exact(x);
    case CUVIT_ACTIVATION_GELU_TANH:
        return gelu_tanh_exact(x);
    case CUVIT_ACTIVATION_SILU:
        return silu_exact(x);
    default:
        return x;
    }
}

} // namespace cuvit::dev
