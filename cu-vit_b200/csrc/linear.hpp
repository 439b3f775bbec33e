// Linear layers: the checked problem its kernels share.
#pragma once

#include "cuvit_b200.h"
#include "gemm.hpp"
#include "linear_tc.cuh"
#include "runtime.hpp"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

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

// ---- slices of k: a cluster's CTAs share a tile and add up their sums ------------------------

__device__ __forceinline__ void store_remote(uint32_t at, const float (&v)[4]) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v[0]), "f"(v[1]),
                 "f"(v[2]), "f"(v[3])
                 : "memory");
}

// Four columns' sums of every slice, `distance` floats apart, in the order of k.
__device__ __forceinline__ void sum_slices(const float* from, int slices, int distance,
                                           float (&v)[4]) {
    v[0] = v[1] = v[2] = v[3] = 0.0F;
    for (int r = 0; r < slices; ++r) {
        const float4 slice = *reinterpret_cast<const float4*>(from + r * distance);
        v[0] += slice.x;
        v[1] += slice.y;
        v[2] += slice.z;
        v[3] += slice.w;
    }
}

// Four neighbouring outputs from their sums: sum(at, v) gives the four of (gate) column `at` of the
// tile, `up_at` the ones that multiply them.
template <class Sum>
__device__ __forceinline__ void finish_four(const OutRows& s, long long row, int col, int at,
                                            int up_at, Sum&& sum) {
    const Params& p = s.p;
    const int valid = min(4, p.n - col);
    if (valid <= 0) {
        return;
    }
    const auto add_columns = [&](float(&v)[4], const float* vector) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] += j < valid ? __ldg(vector + col + j) : 0.0F;
        }
    };
    float v[4];
    sum(at, v);
    if (p.bias != nullptr) {
        add_columns(v, p.bias);
    }
    if (p.out_kind == CUVIT_DTYPE_BF16) {
        dev::activate<true>(p.activation, v);
    } else {
        dev::activate<false>(p.activation, v);
    }
    if (p.gated) {
        float up[4];
        sum(up_at, up);
        if (p.bias != nullptr) {
            add_columns(up, p.bias + p.n);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] *= up[j];
        }
    }
    if (p.scale != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] *= j < valid ? __ldg(p.scale + col + j) : 0.0F;
        }
    }
    write_four(s, row, col, v, valid);
}

// How many clusters of 1, 2, 4 and 8 CTAs of a kernel the current device holds at once (clusters do
// not span its processor clusters, so less than the SMs would: 15 of 8, 33 of 4 on B200). Zeros where
// that cannot be told.
struct ClusterLimits {
    int of[4] = {};
};

template <auto Kernel>
ClusterLimits cluster_limits(int threads, size_t smem) {
    constexpr auto* kernel = Kernel;
    constexpr int kMaxDevices = 64;
    static ClusterLimits limits[kMaxDevices];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) {
        return {};
    }
    const cudaError_t error = host::once_per_device(
        reinterpret_cast<const void*>(kernel), [&](int current) {
            cudaError_t status = cudaFuncSetAttribute(
                kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            for (int i = 0; i < 4 && status == cudaSuccess; ++i) {
                cudaLaunchAttribute attribute{};
                attribute.id = cudaLaunchAttributeClusterDimension;
                attribute.val.clusterDim.x = 1u << i;
                attribute.val.clusterDim.y = 1;
                attribute.val.clusterDim.z = 1;
                cudaLaunchConfig_t probe{};
                probe.gridDim = dim3(1u << i);
                probe.blockDim = dim3(static_cast<unsigned>(threads));
                probe.dynamicSmemBytes = smem;
                probe.attrs = &attribute;
                probe.numAttrs = 1;
                status = cudaOccupancyMaxActiveClusters(&limits[current].of[i], kernel, &probe);
            }
            return status;
        });
    return error == cudaSuccess ? limits[device] : ClusterLimits{};
}

// A launch in clusters of `size` CTAs (1: without).
template <class... KernelArgs, class... Args>
void launch_cluster(void (*kernel)(KernelArgs...), int size, unsigned blocks, int threads,
                    size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    int count = 0;
    if (size > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = static_cast<unsigned>(size);
        attributes[count].val.clusterDim.y = 1;
        attributes[count].val.clusterDim.z = 1;
        ++count;
    }
    if (host::pdl_enabled()) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    config.attrs = attributes;
    config.numAttrs = static_cast<unsigned>(count);
    cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
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

// BF16 math: the accumulator columns of a tile with one CTA to each, and where a cluster of CTAs to
// each, k divided among them, takes less time, theirs (slices 1: it does not).
struct TileChoice {
    int block_n;
    int slices;
    int slice_n;
};
TileChoice choose_tiles(const Params& p, const host::DeviceContext& context);

// k divided among the CTAs of a cluster (linear_slices.cu). False where TMA cannot describe x or the
// weight; else *result is the launch's status.
bool launch_slices(const Params& p, const TileChoice& choice, const host::DeviceContext& context,
                   cudaStream_t stream, int* result);

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
