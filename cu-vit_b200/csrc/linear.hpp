// Linear layers: the checked problem its kernels share.
#pragma once

#include "cuvit_b200.h"
#include "gemm.hpp"
#include "linear_tc.cuh"
#include "runtime.hpp"

#include <cuda_runtime.h>

namespace cuvit::linear {

// Pointers and row distances in elements, defaults resolved.
struct Params {
    const void* x;
    const void* w;
    const float* bias;
    const float* scale;
    const void* residual;
    void* out;
    int m, n, k;
    int out_kind; // cuvit_dtype
    int activation;
    int gated;
    long long ldx, ldw, ldr, ldo;
};

// out[row][col] from the sums of its gate (or only) column and its upper column.
__device__ __forceinline__ void finish(const Params& p, int row, int col, float gate, float up) {
    float value = p.bias != nullptr ? gate + p.bias[col] : gate;
    value = dev::activate_exact(p.activation, value);
    if (p.gated) {
        value *= p.bias != nullptr ? up + p.bias[p.n + col] : up;
    }
    if (p.scale != nullptr) {
        value *= p.scale[col];
    }
    if (p.out_kind == CUVIT_DTYPE_BF16) {
        if (p.residual != nullptr) {
            value += __bfloat162float(
                static_cast<const __nv_bfloat16*>(p.residual)[row * p.ldr + col]);
        }
        static_cast<__nv_bfloat16*>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(value);
    } else {
        if (p.residual != nullptr) {
            value += static_cast<const float*>(p.residual)[row * p.ldr + col];
        }
        static_cast<float*>(p.out)[row * p.ldo + col] =
            p.out_kind == CUVIT_DTYPE_TF32 ? dev::round_to_tf32(value) : value;
    }
}

// Outputs written a few neighbours at a time.
struct OutRows {
    Params p;
    int out_vector;      // bytes per access of out's rows
    int residual_vector; // of the residual's
};

// Four neighbouring outputs of a row, `valid` of them inside it: adds the residual, rounds and
// stores.
__device__ __forceinline__ void write_four(const OutRows& s, long long row, int col,
                                           const float (&sums)[4], int valid) {
    const Params& p = s.p;
    float v[4] = {sums[0], sums[1], sums[2], sums[3]};
    if (p.out_kind == CUVIT_DTYPE_BF16) {
        const __nv_bfloat16* const res = static_cast<const __nv_bfloat16*>(p.residual);
        __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + col;
        if (res != nullptr) {
            const __nv_bfloat16* const from = res + row * p.ldr + col;
            if (valid == 4 && s.residual_vector >= 8) {
                const uint2 old = *reinterpret_cast<const uint2*>(from);
                v[0] += __uint_as_float(old.x << 16);
                v[1] += __uint_as_float(old.x & 0xFFFF0000u);
                v[2] += __uint_as_float(old.y << 16);
                v[3] += __uint_as_float(old.y & 0xFFFF0000u);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j < valid) {
                        v[j] += __bfloat162float(from[j]);
                    }
                }
            }
        }
        if (valid == 4 && s.out_vector >= 8) {
            *reinterpret_cast<uint2*>(out) =
                make_uint2(dev::pack_bf16x2(v[0], v[1]), dev::pack_bf16x2(v[2], v[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < valid) {
                    out[j] = __float2bfloat16_rn(v[j]);
                }
            }
        }
    } else {
        const float* const res = static_cast<const float*>(p.residual);
        float* const out = static_cast<float*>(p.out) + row * p.ldo + col;
        if (res != nullptr) {
            const float* const from = res + row * p.ldr + col;
            if (valid == 4 && s.residual_vector >= 16) {
                const float4 old = *reinterpret_cast<const float4*>(from);
                v[0] += old.x;
                v[1] += old.y;
                v[2] += old.z;
                v[3] += old.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j < valid) {
                        v[j] += from[j];
                    }
                }
            }
        }
        if (p.out_kind == CUVIT_DTYPE_TF32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = dev::round_to_tf32(v[j]);
            }
        }
        if (valid == 4 && s.out_vector >= 16) {
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < valid) {
                    out[j] = v[j];
                }
            }
        }
    }
}

// A few rows (linear_rows.cu).
constexpr int kMaxRows = 8;
bool rows_kernel_takes(const Params& p, bool bf16);
int launch_rows(const Params& p, bool bf16, int sm_count, cudaStream_t stream);

// Bytes per access that every row of a matrix allows, from 16 down to an element.
int access_bytes(const void* base, long long pitch_bytes);

// A row-major matrix as a TMA tensor of boxes of box_rows rows of 128 bytes.
bool describe(const void* base, bool bf16, long long columns, long long rows, long long pitch,
              int box_rows, CUtensorMap* map);

// FP32 math on the tensor cores (linear_split.cu). False where TMA cannot describe x or the
// weight, or k is 0; else *result is the launch's status.
bool launch_split(const Params& p, const host::DeviceContext& context, cudaStream_t stream,
                  int* result);

// BF16 math for too few output tiles to fill the GPU: k is divided among the CTAs of a cluster
// (linear_slices.cu). False where that does not apply; else *result is the launch's status.
bool launch_slices(const Params& p, const host::DeviceContext& context, cudaStream_t stream,
                   int* result);

// A prepared launch on the tensor-core kernels of one product.
struct TcPlan {
    CUtensorMap map_x{};
    CUtensorMap map_w{};
    CUtensorMap map_out{};
    gemm::LinearParams params{};
    int block_n = 128;
    bool pair = false;
    int grid = 0;
};

// Pairs of CTAs of the pair kernel that the current device holds at once.
int pair_resident(int* pairs);

int launch_tc_bf16(const TcPlan& plan, cudaStream_t stream);
int launch_tc_tf32(const TcPlan& plan, cudaStream_t stream);

} // namespace cuvit::linear
