// Linear layers: out = residual + scale * act(x W^T + b), or with a gate act(x Wg^T + bg) *
// (x Wu^T + bu). Argument checks, choice of kernel, and the FP32 kernel for operands TMA cannot
// describe.
#include "linear.hpp"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::linear {

int access_bytes(const void* base, long long pitch_bytes) {
    int bytes = 16;
    while (reinterpret_cast<uintptr_t>(base) % bytes != 0 || pitch_bytes % bytes != 0) {
        bytes /= 2;
    }
    return bytes;
}

bool describe(const void* base, bool bf16, long long columns, long long rows, long long pitch,
              int box_rows, CUtensorMap* map) {
    host::TmaTensor t;
    t.base = base;
    t.type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    t.element_bytes = bf16 ? 2 : 4;
    t.rank = 2;
    t.dims[0] = static_cast<uint64_t>(columns);
    t.dims[1] = static_cast<uint64_t>(rows);
    t.strides_bytes[0] = static_cast<uint64_t>(pitch) * t.element_bytes;
    t.box[0] = static_cast<uint32_t>(gemm::kSwizzleBytes / t.element_bytes);
    t.box[1] = static_cast<uint32_t>(box_rows);
    if (!host::tma_describable(t) || host::encode_tma(t, map) != CUVIT_OK) {
        host::clear_error(); // another path serves what TMA cannot
        return false;
    }
    return true;
}

namespace {

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

// Plans a tensor-core launch, bfloat16 math in tiles of block_n accumulator columns; false where TMA
// cannot describe x or the weight, or k is 0.
bool prepare(const Params& p, int math, int block_n, const host::DeviceContext& context,
             TcPlan* plan) {
    if (!host::is_blackwell(context) || p.k == 0) {
        return false;
    }
    const bool bf16 = math == CUVIT_MATH_BF16;
    const long long row_blocks = (p.m + gemm::kBlockM - 1LL) / gemm::kBlockM;
    const long long weight_rows = static_cast<long long>(p.n) * (p.gated ? 2 : 1);
    int bn = bf16 ? block_n
                  : gemm::choose_block_n(row_blocks, static_cast<int>(weight_rows), false, false,
                                         context.sm_count);
    if (p.gated && bn < 128) {
        bn = 128; // a half tile's columns of one operand stay a whole 32-column step
    }
    const int columns = p.gated ? bn / 2 : bn; // output columns of a tile
    const long long n_tiles = (p.n + columns - 1) / columns;
    const long long pair_rows = (p.m + 2LL * gemm::kBlockM - 1) / (2 * gemm::kBlockM);
    plan->pair = bf16 && bn == 256 && gemm::pairs_enabled() &&
                 pair_rows * n_tiles >= context.sm_count;
    const long long m_tiles = plan->pair ? pair_rows : row_blocks;
    const long long total = m_tiles * n_tiles;
    const int b_rows = plan->pair || p.gated ? bn / 2 : bn;
    if (total > 0x7FFFFFFFLL ||
        !describe(p.x, bf16, p.k, p.m, p.ldx, gemm::kBlockM, &plan->map_x) ||
        !describe(p.w, bf16, p.k, weight_rows, p.ldw, b_rows, &plan->map_w)) {
        return false;
    }
    const auto aligned16 = [](const void* pointer) {
        return reinterpret_cast<uintptr_t>(pointer) % 16 == 0 ? 1 : 0;
    };
    gemm::LinearParams& q = plan->params;
    const int element = bf16 ? 2 : 4;
    q.m = p.m;
    q.n = p.n;
    q.k = p.k;
    q.m_tiles = static_cast<int>(m_tiles);
    q.n_tiles = static_cast<int>(n_tiles);
    q.k_blocks = (p.k + gemm::kSwizzleBytes / element - 1) / (gemm::kSwizzleBytes / element);
    q.total_tiles = static_cast<int>(total);
    q.count = 1;
    q.a_rank = q.b_rank = q.c_rank = 2;
    q.alpha = 1.0F;
    q.bias = p.bias;
    q.bias_vector_ok = aligned16(p.bias);
    q.up_vector_ok = p.bias != nullptr ? aligned16(p.bias + p.n) : 0;
    q.scale = p.scale;
    q.scale_vector_ok = aligned16(p.scale);
    q.c = p.out;
    q.ldc = p.ldo;
    q.c_kind = p.out_kind;
    q.reverse = host::reverse_sweep() ? 1 : 0;
    q.status = context.status;
    q.activation = p.activation;
    q.gated = p.gated;
    q.residual = p.residual;
    q.ldr = p.ldr;
    // Whole slab rows (128 bytes: 64 bfloat16 or 32 float columns) go by TMA.
    const bool out_bf16 = p.out_kind == CUVIT_DTYPE_BF16;
    const int out_bytes = out_bf16 ? 2 : 4;
    const bool whole = !out_bf16 || columns / 2 >= 64;
    q.c_tma = whole && describe(p.out, out_bf16, p.n, p.m, p.ldo, 32, &plan->map_out) ? 1 : 0;
    q.residual_tma = p.residual != nullptr && whole &&
                             describe(p.residual, out_bf16, p.n, p.m, p.ldr, 32, &q.map_residual)
                         ? 1
                         : 0;
    q.out_vector = access_bytes(p.out, p.ldo * out_bytes);
    q.residual_vector = p.residual != nullptr ? access_bytes(p.residual, p.ldr * out_bytes) : 16;
    plan->block_n = bn;
    plan->grid = static_cast<int>(total < context.sm_count ? total : context.sm_count);
    if (plan->pair) {
        int resident = 0;
        if (pair_resident(&resident) != CUVIT_OK) {
            return false;
        }
        plan->grid = 2 * static_cast<int>(total < resident ? total : resident);
    }
    return true;
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
    // Tile ends past the last row stay in int, and the steps past the end of k that the kernels
    // count (at most 8192 further: linear_rows.cu).
    constexpr int kMaxExtent = 0x7FFFFFFF - 65536;
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
    const bool bf16 = c.math == CUVIT_MATH_BF16;
    if (rows_kernel_takes(p, bf16)) {
        return launch_rows(p, bf16, context->sm_count, stream);
    }
    int result = CUVIT_OK;
    if (c.math == CUVIT_MATH_FP32 && launch_split(p, *context, stream, &result)) {
        return result;
    }
    const TileChoice choice =
        bf16 && p.k > 0 ? choose_tiles(p, *context) : TileChoice{256, 1, 0};
    if (choice.slices > 1 && launch_slices(p, choice, *context, stream, &result)) {
        return result;
    }
    TcPlan plan;
    if (c.math != CUVIT_MATH_FP32 && prepare(p, c.math, choice.block_n, *context, &plan)) {
        return bf16 ? launch_tc_bf16(plan, stream) : launch_tc_tf32(plan, stream);
    }
    return bf16 ? launch_simt<__nv_bfloat16>(p, stream) : launch_simt<float>(p, stream);
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
