// Linear layers of a few rows (one token, a pooled row per image): bound by reading the weight
// once, so each weight element is multiplied with every row as it arrives, in FP32.
//
// A warp has four columns (gated: two gate columns and the two they multiply) and its lanes
// consecutive 16-byte pieces of their rows; x is small and comes from L1. Where the columns alone
// would not fill the GPU, several warps of a block share the columns and add up their parts of k
// in shared memory, in a fixed order.
#include "linear.hpp"
#include "ptx.cuh"

#include <cuda_bf16.h>

namespace cuvit::linear {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kColumns = 4;

template <typename T>
struct Piece {
    static constexpr int kElems = 16 / sizeof(T);

    static __device__ __forceinline__ void unpack(const uint4& raw, float (&out)[kElems]) {
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) {
                out[2 * i] = __uint_as_float(words[i] << 16);
                out[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
            } else {
                out[i] = __uint_as_float(words[i]);
            }
        }
    }
};

template <typename T, int Rows>
__global__ void __launch_bounds__(kThreads)
    linear_rows_kernel(const Params p, int warps_per_columns) {
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    constexpr int kElems = Piece<T>::kElems;
    __shared__ float parts[kWarps][Rows * kColumns];
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int part = warp % warps_per_columns;
    const int outputs = p.gated ? kColumns / 2 : kColumns; // output columns of a warp
    const int col0 = (static_cast<int>(blockIdx.x) * (kWarps / warps_per_columns) +
                      warp / warps_per_columns) *
                     outputs;
    const T* w[kColumns];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
        // Columns past the end read the last one and are not stored.
        const int col = min(p.gated ? col0 + c / 2 : col0 + c, p.n - 1);
        const long long row = col + (p.gated && (c & 1) ? static_cast<long long>(p.n) : 0LL);
        w[c] = static_cast<const T*>(p.w) + row * p.ldw;
    }
    const T* const x = static_cast<const T*>(p.x);
    float acc[Rows][kColumns] = {};
    const int step = warps_per_columns * 32 * kElems;
    // kPieces pieces of every column are loaded before the first is used.
    constexpr int kPieces = Rows <= 2 ? 4 : (Rows <= 4 ? 2 : 1);
    for (int k0 = (part * 32 + lane) * kElems; k0 < p.k; k0 += kPieces * step) {
        uint4 raw[kPieces][kColumns];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int k = k0 + i * step;
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                raw[i][c] = k < p.k ? __ldg(reinterpret_cast<const uint4*>(w[c] + k))
                                    : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int k = k0 + i * step;
            if (k < p.k) { // x may hold anything past its rows' ends
                float wf[kColumns][kElems];
#pragma unroll
                for (int c = 0; c < kColumns; ++c) {
                    Piece<T>::unpack(raw[i][c], wf[c]);
                }
#pragma unroll
                for (int r = 0; r < Rows; ++r) {
                    const int row = min(r, p.m - 1); // rows past the end are not stored
                    float xf[kElems];
                    Piece<T>::unpack(__ldg(reinterpret_cast<const uint4*>(x + row * p.ldx + k)),
                                     xf);
#pragma unroll
                    for (int c = 0; c < kColumns; ++c) {
#pragma unroll
                        for (int j = 0; j < kElems; ++j) {
                            acc[r][c] = fmaf(xf[j], wf[c][j], acc[r][c]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
#pragma unroll
            for (int offset = 16; offset > 0; offset /= 2) {
                acc[r][c] += __shfl_xor_sync(0xFFFFFFFFu, acc[r][c], offset);
            }
            if (lane == (r * kColumns + c) % 32) {
                parts[warp][r * kColumns + c] = acc[r][c];
            }
        }
    }
    __syncthreads();
    // The first warp of a column group finishes its outputs, one per lane.
    if (part == 0 && lane < Rows * kColumns && lane < p.m * outputs) {
        const int r = lane / outputs;
        const int c = lane - r * outputs;
        const int col = col0 + c;
        if (col < p.n) {
            const int at = r * kColumns + (p.gated ? 2 * c : c);
            float value = 0.0F;
            float up = 0.0F;
            for (int i = 0; i < warps_per_columns; ++i) {
                value += parts[warp + i][at];
                up += p.gated ? parts[warp + i][at + 1] : 0.0F;
            }
            finish(p, r, col, value, up);
        }
    }
}

template <typename T, int Rows>
int launch_count(const Params& p, int sm_count, cudaStream_t stream) {
    const int outputs = p.gated ? kColumns / 2 : kColumns;
    const long long groups = (static_cast<long long>(p.n) + outputs - 1) / outputs;
    // Share columns between warps until there are 16 warps for every SM or a lane would be left
    // with less than two pieces of a row.
    int share = 1;
    while (share < kWarps && groups * share < 16LL * sm_count &&
           p.k >= 4 * share * 32 * Piece<T>::kElems) {
        share *= 2;
    }
    const long long blocks = (groups + kWarps / share - 1) / (kWarps / share);
    host::pdl_launch(linear_rows_kernel<T, Rows>, dim3(static_cast<unsigned>(blocks)),
                     dim3(kThreads), 0, stream, p, share);
    return host::after_launch("linear_rows_kernel");
}

template <typename T>
int launch_typed(const Params& p, int sm_count, cudaStream_t stream) {
    if (p.m <= 1) {
        return launch_count<T, 1>(p, sm_count, stream);
    }
    if (p.m <= 2) {
        return launch_count<T, 2>(p, sm_count, stream);
    }
    return p.m <= 4 ? launch_count<T, 4>(p, sm_count, stream)
                    : launch_count<T, 8>(p, sm_count, stream);
}

} // namespace

bool rows_kernel_takes(const Params& p, bool bf16) {
    const int size = bf16 ? 2 : 4;
    const auto fits = [size](const void* base, long long pitch) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && pitch * size % 16 == 0;
    };
    return p.m <= kMaxRows && p.k > 0 && p.k * size % 16 == 0 && fits(p.x, p.ldx) &&
           fits(p.w, p.ldw);
}

int launch_rows(const Params& p, bool bf16, int sm_count, cudaStream_t stream) {
    return bf16 ? launch_typed<__nv_bfloat16>(p, sm_count, stream)
                : launch_typed<float>(p, sm_count, stream);
}

} // namespace cuvit::linear
