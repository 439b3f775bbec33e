// The activations of cuvit_linear in FP32: forms for float outputs (within 6e-7 relative, from the
// hardware's exponential and reciprocal with their roundings corrected), and cheaper ones for bfloat16
// outputs. Where the exponential leaves the normal floats (the erf form at -13, tanh GELU at -10, SiLU
// at -87, values below 1e-36) they give zero.
#pragma once

#include "cuvit_b200.h"
#include "ptx.cuh"

namespace cuvit::dev {

// 2^(t + low) where low carries what rounding the exponent t cost it: for -100 that alone would be
// 2^-18 of the result. The hardware exponential is within 2^-22.
__device__ __forceinline__ float exp2_sum(float t, float low) {
    const float e = ex2_approx(t);
    return fmaf(e * 0.6931471806F, low, e);
}

// 1 / d for d >= 1: the hardware's reciprocal and one Newton step. (NaN for an infinite d.)
__device__ __forceinline__ float reciprocal(float d) {
    const float r = rcp_approx(d);
    return fmaf(r, fmaf(-d, r, 1.0F), r);
}

// x Phi(x) = max(x, 0) - |x| Q(|x|), Q(z) = erfc(z / sqrt 2) / 2 = exp(-z^2 / 2) t P(t) with
// t = 1 / (1 + 0.3 z) and P of degree 7, fitted here for minimax relative error on [0, 13.5]
// (1.3e-7; 5.1e-7 as evaluated in FP32; beyond, Q is below the smallest float). It keeps its
// relative accuracy in the negative tail, where 1 + erf cancels.
__device__ __forceinline__ float gelu_exact(float x) {
    const float z = fabsf(x);
    const float t = reciprocal(fmaf(0.3F, z, 1.0F));
    float p = fmaf(t, 0.03593173250555992F, -0.15827599167823792F);
    p = fmaf(t, p, 0.20820657908916473F);
    p = fmaf(t, p, -0.055393826216459274F);
    p = fmaf(t, p, 0.12946918606758118F);
    p = fmaf(t, p, 0.09963749349117279F);
    p = fmaf(t, p, 0.12079835683107376F);
    p = fmaf(t, p, 0.11962638795375824F);
    constexpr float kHalf = -0.7213475204F;  // -log2(e) / 2
    constexpr float kHalfLow = -9.629815e-9F; // what the float leaves of it
    const float square = __fmul_rn(x, x);
    const float exponent = __fmul_rn(square, kHalf);
    const float low = fmaf(square, kHalfLow,
                           fmaf(fmaf(x, x, -square), kHalf, fmaf(square, kHalf, -exponent)));
    const float tail = exp2_sum(exponent, low);
    // Beyond: x, or a zero of its sign and, for minus infinity, NaN, as in the formula.
    return z > 14.0F ? (x > 0.0F ? x : x * 0.0F) : fmaf(-z * t * p, tail, fmaxf(x, 0.0F));
}

// x / (1 + 2^(t + low)), within 3e-7: with s = 2^-|t + low|, x / (1 + s) or x s / (1 + s). Far from
// zero (where low may be infinite or NaN) x itself, or a zero of its sign and, for minus infinity, NaN.
__device__ __forceinline__ float logistic_times(float x, float t, float low) {
    const bool negative = t > 0.0F; // x is
    const float s = exp2_sum(-fabsf(t), negative ? -low : low);
    const float factor = (negative ? s : 1.0F) * reciprocal(1.0F + s);
    return x * (fabsf(t) < 190.0F ? factor : (negative ? 0.0F : 1.0F));
}

__device__ __forceinline__ float silu_exact(float x) {
    constexpr float kRate = -1.4426950409F;   // -log2(e)
    constexpr float kRateLow = -1.925963e-8F; // what the float leaves of it
    const float t = kRate * x;
    return logistic_times(x, t, fmaf(kRateLow, x, fmaf(kRate, x, -t)));
}

// x (1 + tanh u) / 2 = x / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3). The exponent
// t = x (a + b x^2) is formed with the roundings of its square, products and sum carried along (without
// them the result was off by 2e-6 at -5 and 1e-5 at -9).
__device__ __forceinline__ float gelu_tanh_exact(float x) {
    constexpr float kA = -2.3022081985F;                        // -2 sqrt(2/pi) log2(e)
    constexpr float kB = -0.1029432397F, kBLow = 2.0161983e-9F; // 0.044715 times that
    const float square = __fmul_rn(x, x);
    const float product = __fmul_rn(kB, square);
    const float sum = __fadd_rn(kA, product);
    // What the sum lost: of two numbers of one sign, the smaller less what it added to the larger.
    const float lost =
        __fadd_rn(fmaxf(kA, product), -__fadd_rn(sum, -fminf(kA, product)));
    float rest = fmaf(kB, square, -product);
    rest = fmaf(kB, fmaf(x, x, -square), rest);
    rest = fmaf(kBLow, square, rest);
    const float t = __fmul_rn(x, sum);
    return logistic_times(x, t, fmaf(x, lost + rest, fmaf(x, sum, -t)));
}

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

// ---- for bfloat16 outputs: errors far below the store's 2^-8 -------------------------------

// 1 / (1 + 2^t) with the hardware's exponential and reciprocal (2^-21 relative).
__device__ __forceinline__ float logistic_of_exp2(float t) {
    return rcp_approx(1.0F + ex2_approx(t));
}

__device__ __forceinline__ float silu_fast(float x) {
    return x * logistic_of_exp2(-1.4426950408889634F * x);
}

__device__ __forceinline__ float gelu_tanh_fast(float x) {
    // exp(-2u) with 2 sqrt(2/pi) log2(e) folded into the cubic.
    const float x2 = x * x;
    return x * logistic_of_exp2(x * fmaf(-0.1029432397F, x2, -2.3022081985F));
}

// x Phi(x) = max(x, 0) - |x| Q(|x|), Q(z) = erfc(z / sqrt 2) / 2 = exp(-z^2 / 2) t P(t) with
// t = 1 / (1 + 0.375 z) and P of degree 4, fitted here for minimax relative error on [0, 13.5]
// (2.9e-5 in FP32; beyond, Q is below the smallest float). Two values, the multiply-adds packed.
__device__ __forceinline__ float2 gelu_fast2(float x0, float x1) {
    // Bounded above: for a positive infinity |x| times t = 0 would be NaN. A negative one has NaN, as
    // in the formula.
    const float m0 = fabsf(fminf(x0, 1.0e18F));
    const float m1 = fabsf(fminf(x1, 1.0e18F));
    const uint64_t m = f32x2(m0, m1);
    const float2 den = f32x2_split(fma_f32x2(f32x2(0.375F, 0.375F), m, f32x2(1.0F, 1.0F)));
    const uint64_t t = f32x2(rcp_approx(den.x), rcp_approx(den.y));
    // The polynomial's negative, so that its product is added to max(x, 0).
    uint64_t poly = fma_f32x2(t, f32x2(0.0909852013F, 0.0909852013F),
                              f32x2(-0.201043248F, -0.201043248F));
    poly = fma_f32x2(t, poly, f32x2(-0.0829740912F, -0.0829740912F));
    poly = fma_f32x2(t, poly, f32x2(-0.157920063F, -0.157920063F));
    poly = fma_f32x2(t, poly, f32x2(-0.149041131F, -0.149041131F));
    poly = mul_f32x2(poly, mul_f32x2(m, t));
    const uint64_t x = f32x2(x0, x1);
    constexpr float kHalfLog2e = -0.5F * 1.4426950408889634F;
    const float2 arg = f32x2_split(mul_f32x2(x, mul_f32x2(x, f32x2(kHalfLog2e, kHalfLog2e))));
    const uint64_t tail = f32x2(ex2_approx(arg.x), ex2_approx(arg.y));
    return f32x2_split(fma_f32x2(poly, tail, f32x2(fmaxf(x0, 0.0F), fmaxf(x1, 0.0F))));
}

// The activation on N values: the forms above (Fast), or the exact ones.
template <bool Fast, int N>
__device__ __forceinline__ void activate(int activation, float (&v)[N]) {
    if (activation == CUVIT_ACTIVATION_NONE) {
        return;
    }
    if constexpr (Fast) {
        if (activation == CUVIT_ACTIVATION_SILU) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[j] = silu_fast(v[j]);
            }
        } else if (activation == CUVIT_ACTIVATION_GELU) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 g = gelu_fast2(v[j], v[j + 1]);
                v[j] = g.x;
                v[j + 1] = g.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[j] = gelu_tanh_fast(v[j]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = activate_exact(activation, v[j]);
        }
    }
}

} // namespace cuvit::dev
