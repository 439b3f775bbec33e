// FP32 products on TF32 tensor cores: x = hi + lo + e with hi = rn_tf32(x) and lo = x - hi, of which
// the tensor core cuts off its 12th bit at most: |e| <= 2^-23 |x|. Then
//   x w = lo_x hi_w + hi_x lo_w + hi_x hi_w  (+ lo_x lo_w, 2^-22 at most)
// with each product exact in the accumulator. An accumulator cuts off instead of rounding, so a long
// sum kept there drifts towards zero; kernels hand partial sums of 64 products to registers.
#pragma once

#include "ptx.cuh"

#include <cstdint>

namespace cuvit::dev {

// Four values: hi, and lo in their place. Adding half a step and masking rounds to nearest, x - hi
// is exact. An infinity, a NaN or an x that rounds to infinity leaves a rest that is not finite and
// turns `check`, otherwise zero, into a NaN; the warp that meets one takes the checked form.
__device__ __forceinline__ void split4(float (&x)[4], float (&hi)[4], uint64_t& check) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hi[j] = __uint_as_float((__float_as_uint(x[j]) + 0x1000u) & 0xFFFFE000u);
    }
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const uint64_t rest = sub_f32x2(f32x2(x[j], x[j + 1]), f32x2(hi[j], hi[j + 1]));
        check = fma_f32x2(rest, f32x2(0.0F, 0.0F), check);
        const float2 both = f32x2_split(rest);
        x[j] = both.x;
        x[j + 1] = both.y;
    }
}

__device__ __forceinline__ bool any_special(uint64_t check) {
    const float2 both = f32x2_split(check);
    return __any_sync(0xFFFFFFFFu, !(both.x + both.y == 0.0F));
}

__device__ __forceinline__ void split4_checked(const float (&x)[4], float (&hi)[4],
                                               float (&lo)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool special = (__float_as_uint(x[j]) & 0x7F800000u) == 0x7F800000u;
        // The tensor core takes the upper 19 bits: a NaN whose payload lies below them would be an
        // infinity there. A sum gives the NaN whose bits are all set.
        hi[j] = special ? x[j] + x[j] : round_to_tf32(x[j]);
        lo[j] = special ? 0.0F : x[j] - hi[j];
    }
}

// 16 values into as many tensor-memory columns of this warp's lanes.
__device__ __forceinline__ void tmem_store_floats(uint32_t to, const float (&v)[4][4]) {
    uint32_t words[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        words[j] = __float_as_uint(v[j / 4][j % 4]);
    }
    tmem_store_16(to, words);
}

} // namespace cuvit::dev
