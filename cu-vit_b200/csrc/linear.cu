// Linear layers: out = residual + scale * act(x W^T + b), or with a gate act(x Wg^T + bg) *
// (x Wu^T + bu). Argument checks, choice of kernel, and the FP32 kernel for operands TMA cannot
// describe.
#include "activation.cuh"
#include "cuvit_b200.h"
#include "ptx.cuh"
#include "runtime.hpp"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::linear {
namespace {

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

constexpr int kTile = 64;
constexpr int kTileK = 16;
constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float load_value(const T* p) {
    if constexpr (sizeof(T) == 2) {
        return __bfloat162float(*p);
    } else {
        return *p;
    }
}

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

// Any alignment and any k: 64 x 64 outputs per block, 4 x 4 per thread, FP32 products.
template <typename T, bool Gated>
__global__ void __launch_bounds__(kThreads) linear_simt_kernel(const Params p) {
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    constexpr int kParts = Gated ? 2 : 1;
    __shared__ float xs[kTileK][kTile + 4];
    __shared__ float ws[kParts][kTileK][kTile + 4];
    const int tx = threadIdx.x % 16;
    const int ty = threadIdx.x / 16;
    const int col_tiles = (p.n + kTile - 1) / kTile;
    const int row0 = static_cast<int>(blockIdx.x / col_tiles) * kTile;
    const int col0 = static_cast<int>(blockIdx.x % col_tiles) * kTile;
    const T* const x = static_cast<const T*>(p.x);
    const T* const w = static_cast<const T*>(p.w);
    float acc[kParts][4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += kTileK) {
        for (int i = threadIdx.x; i < kTile * kTileK; i += kThreads) {
            const int r = i / kTileK;
            const int kk = i % kTileK;
            const bool in_k = k0 + kk < p.k;
            xs[kk][r] = row0 + r < p.m && in_k ? load_value(x + (row0 + r) * p.ldx + k0 + kk) : 0.0F;
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
                const long long col = static_cast<long long>(h) * p.n + col0 + r;
                ws[h][kk][r] =
                    col0 + r < p.n && in_k ? load_value(w + col * p.ldw + k0 + kk) : 0.0F;
            }
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kTileK; ++kk) {
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        acc[h][i][j] =
                            fmaf(xs[kk][ty * 4 + i], ws[h][kk][tx * 4 + j], acc[h][i][j]);
                    }
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col0 + tx * 4 + j;
            if (row < p.m && col < p.n) {
                finish(p, row, col, acc[0][i][j], acc[kParts - 1][i][j]);
            }
        }
    }
}

template <typename T>
int launch_simt(const Params& p, cudaStream_t stream) {
    const long long blocks = static_cast<long long>((p.m + kTile - 1) / kTile) *
                             ((p.n + kTile - 1) / kTile);
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "linear launch exceeds the CUDA grid limit");
    }
    host::pdl_launch(p.gated ? linear_simt_kernel<T, true> : linear_simt_kernel<T, false>,
                     dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, p);
    return host::after_launch("linear_simt_kernel");
}

int run(const void* x, const void* weight, const float* bias, const float* scale,
        const void* residual, void* out, const cuvit_linear_problem* problem,
        cudaStream_t stream) {
    if (problem == nullptr) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "linear problem cannot be null");
    }
    const cuvit_linear_problem& c = *problem;
    if (c.m < 0 || c.n < 0 || c.k < 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "linear dimensions cannot be negative");
    }
    if (c.math != CUVIT_MATH_FP32 && c.math != CUVIT_MATH_TF32 && c.math != CUVIT_MATH_BF16) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "unknown linear math mode");
    }
    if (c.out_dtype != CUVIT_DTYPE_F32 && c.out_dtype != CUVIT_DTYPE_BF16 &&
        c.out_dtype != CUVIT_DTYPE_TF32) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "unknown output data type");
    }
    if (c.activation < CUVIT_ACTIVATION_NONE || c.activation > CUVIT_ACTIVATION_SILU) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "unknown activation");
    }
    if (c.m == 0 || c.n == 0) {
        return CUVIT_OK;
    }
    if (out == nullptr || (c.k > 0 && (x == nullptr || weight == nullptr))) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "linear operands cannot be null");
    }
    constexpr int kMaxExtent = 0x7FFFFFFF - 4096; // tile ends past the last row stay in int
    if (c.m > kMaxExtent || c.n > kMaxExtent / 2 || c.k > kMaxExtent) {
        return host::fail(CUVIT_LENGTH_ERROR, "linear dimensions are too large");
    }
    Params p{};
    p.x = x;
    p.w = weight;
    p.bias = bias;
    p.scale = scale;
    p.residual = residual;
    p.out = out;
    p.m = c.m;
    p.n = c.n;
    p.k = c.k;
    p.out_kind = c.out_dtype;
    p.activation = c.activation;
    p.gated = c.gated ? 1 : 0;
    p.ldx = c.ldx != 0 ? c.ldx : c.k;
    p.ldw = c.ldw != 0 ? c.ldw : c.k;
    p.ldr = c.ldr != 0 ? c.ldr : c.n;
    p.ldo = c.ldo != 0 ? c.ldo : c.n;
    if (p.ldx < c.k || p.ldw < c.k || p.ldr < c.n || p.ldo < c.n) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "a linear row distance is smaller than its row");
    }
    const long long limit = 1LL << 58; // byte distances stay within 64 bits
    if (p.ldx > limit / c.m || p.ldr > limit / c.m || p.ldo > limit / c.m ||
        p.ldw > limit / (2LL * c.n)) {
        return host::fail(CUVIT_LENGTH_ERROR, "a linear row distance is too large");
    }
    const int in_bytes = c.math == CUVIT_MATH_BF16 ? 2 : 4;
    const int out_bytes = c.out_dtype == CUVIT_DTYPE_BF16 ? 2 : 4;
    const auto aligned = [](const void* pointer, int bytes) {
        return reinterpret_cast<uintptr_t>(pointer) % bytes == 0;
    };
    if (!aligned(x, in_bytes) || !aligned(weight, in_bytes) || !aligned(bias, 4) ||
        !aligned(scale, 4) || !aligned(residual, out_bytes) || !aligned(out, out_bytes)) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "linear operands must be aligned to their type");
    }
    const int64_t weight_rows = static_cast<int64_t>(c.n) * (c.gated ? 2 : 1);
    const int64_t row_bytes = static_cast<int64_t>(c.n) * out_bytes;
    const host::RowSpan out_span{out, c.m, row_bytes, p.ldo * out_bytes};
    const host::RowSpan res_span{residual, residual != nullptr ? c.m : 0, row_bytes,
                                 p.ldr * out_bytes};
    const bool in_place = residual == out && p.ldr == p.ldo;
    if ((!in_place && host::rows_overlap(out_span, res_span)) ||
        host::rows_overlap(out_span, {x, c.m, static_cast<int64_t>(c.k) * in_bytes,
                                      p.ldx * in_bytes}) ||
        host::rows_overlap(out_span, {weight, weight_rows, static_cast<int64_t>(c.k) * in_bytes,
                                      p.ldw * in_bytes}) ||
        host::rows_overlap(out_span, {bias, bias != nullptr ? 1 : 0, weight_rows * 4,
                                      weight_rows * 4}) ||
        host::rows_overlap(out_span, {scale, scale != nullptr ? 1 : 0, c.n * int64_t{4},
                                      c.n * int64_t{4}})) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "the linear output overlaps an operand");
    }
    const host::DeviceContext* context = nullptr;
    CUVIT_TRY(host::current_context(&context));
    CUVIT_TRY(host::check_operands({x, weight, bias, scale, residual, out}));
    return c.math == CUVIT_MATH_BF16 ? launch_simt<__nv_bfloat16>(p, stream)
                                     : launch_simt<float>(p, stream);
}

} // namespace
} // namespace cuvit::linear

extern "C" int cuvit_linear(const void* x, const void* weight, const float* bias,
                            const float* scale, const void* residual, void* out,
                            const cuvit_linear_problem* problem, cuvit_stream_t stream) {
    return cuvit::host::guarded([&]() {
        return cuvit::linear::run(x, weight, bias, scale, residual, out, problem,
                                  reinterpret_cast<cudaStream_t>(stream));
    });
}
