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
