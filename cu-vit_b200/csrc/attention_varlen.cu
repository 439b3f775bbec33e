// Attention over packed sequences of any length: argument checks, choice of kernel, and the
// FP32 kernel for bfloat16 operands that TMA cannot describe.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(scale log2(e) q_i . k_j - m_i)
//
// in one pass over the keys: m_i is the maximum so far, and sums and outputs so far are
// multiplied by 2^(old m - new m) when it rises. A row that sees no key keeps a sum of zero and
// is written as zeros.
#include "attention_varlen.hpp"
#include "ptx.cuh"
#include "varlen.cuh"

#include <cuda_bf16.h>

#include <cmath>
#include <cstdint>

namespace cuvit::attn {
namespace {

constexpr int kSimtRows = 128;
constexpr int kSimtKeys = 64;
constexpr int kRowPitch = kSimtRows + 4; // floats; consecutive keys' rows start 4 banks apart
constexpr int kKeyPitch = kSimtKeys + 4;

// Elements e .. e + 3 of a row of d, zeros past its end.
__device__ __forceinline__ float4 load_four(const __nv_bfloat16* row, int e, int d) {
    return make_float4(e < d ? __bfloat162float(row[e]) : 0.0F,
                       e + 1 < d ? __bfloat162float(row[e + 1]) : 0.0F,
                       e + 2 < d ? __bfloat162float(row[e + 2]) : 0.0F,
                       e + 3 < d ? __bfloat162float(row[e + 3]) : 0.0F);
}

// Threads along the keys and elements of a tile (kX); each has 8 of its elements, and 8 or 4 of its
// keys, for 8 rows.
template <int DPad>
struct SimtShape {
    static constexpr int kX = DPad / 8;
    static constexpr int kCols = DPad / kX / 4; // element groups of four
    static constexpr int kThreads = 16 * kX;
    static constexpr int kKeyGroups = kSimtKeys / kX / 4; // of four keys
    static constexpr int kSmemBytes =
        4 * (DPad * (kRowPitch + kKeyPitch) + kSimtKeys * DPad + kSimtKeys * kRowPitch);
};

// acc[r][j] += a[r] * b[j] for 8 rows, contiguous in shared memory.
__device__ __forceinline__ void outer(const float* rows, const float4& b, float (&acc)[8][4]) {
    const float4 low = reinterpret_cast<const float4*>(rows)[0];
    const float4 high = reinterpret_cast<const float4*>(rows)[1];
    const float a[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
    const float c[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[r][j] = fmaf(a[r], c[j], acc[r][j]);
        }
    }
}

// 128 query rows of one head per block, keys in tiles of 64. Thread (ty, tx) of 16 x kX has rows
// 8 ty .. + 7 and, of the scores, the keys tx + kX m, of the output, elements 4 tx .. + 3 of every
// 4 kX. Operands come from shared memory as whole vectors (Q and P with rows contiguous): for heads
// up to 64, 64 multiply-adds share four loads, and two blocks fit an SM and load under each other's
// arithmetic. 4096 tokens, 8 heads whose base lies an element off a vector: heads of 64 1.20 ms,
// 29 TFLOP/s of the FP32 pipe's 74, heads of 128 2.62 ms. What keeps it from more are the loads of
// single elements, converted one by one: operands of floats, which attention_split.cu takes, took
// 0.95 ms (and 8 x 4 products a thread on twice the threads 0.99, shared memory then taking as many
// cycles as the arithmetic; packed multiply-adds on pairs of rows 1.05, since doubling the other
// operand takes moves on the same pipe). Heads up to 128 use 8 x 4 for the scores: the outputs take the
// registers. A tile's keys lie in the order the threads read them, kX apart, which also lets a warp
// write its weights without bank conflicts.
template <int DPad>
__global__ void __launch_bounds__(SimtShape<DPad>::kThreads, DPad == 64 ? 2 : 1)
    attention_varlen_simt(const VarlenParams p) {
    using T = __nv_bfloat16;
    using Shape = SimtShape<DPad>;
    constexpr int kX = Shape::kX;
    constexpr int kThreads = Shape::kThreads;
    constexpr int kGroups = Shape::kKeyGroups;
    constexpr int kCols = Shape::kCols;
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    extern __shared__ __align__(16) float smem[];
    float* const qs = smem;                  // [DPad][row pitch], element-major
    float* const ks = qs + DPad * kRowPitch; // [DPad][key pitch], element-major
    float* const vs = ks + DPad * kKeyPitch; // [keys][DPad]
    float* const ps = vs + kSimtKeys * DPad; // [keys][row pitch]

    const int item = static_cast<int>(blockIdx.x) / p.splits;
    const int split = static_cast<int>(blockIdx.x) - item * p.splits;
    const int block = item / p.q_heads;
    const int head = item - block * p.q_heads;
    const Sequence s = find_block(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                  block, kSimtRows);
    if (s.index < 0) {
        return;
    }
    const int rows = min(kSimtRows, s.q_end - s.q_first);
    const int keys = s.kv_end - s.kv_begin;
    // Query row r of this block sees keys j <= r + reach.
    const long long reach =
        static_cast<long long>(s.q_first - s.q_begin) + keys - (s.q_end - s.q_begin);
    int first_key, last_key;
    split_keys(keys, split, p.splits, first_key, last_key);
    if (p.causal) {
        last_key = static_cast<int>(min(static_cast<long long>(last_key), max(0LL, reach + rows)));
    }
    const int d = p.head_dim;
    const T* const q = static_cast<const T*>(p.q) + s.q_first * p.q_stride +
                       static_cast<long long>(head) * d;
    const T* const k = static_cast<const T*>(p.k) + s.kv_begin * p.k_stride +
                       static_cast<long long>(head / p.group) * d;
    const T* const v = static_cast<const T*>(p.v) + s.kv_begin * p.v_stride +
                       static_cast<long long>(head / p.group) * d;
    const auto zeros = []() { return make_float4(0.0F, 0.0F, 0.0F, 0.0F); };

    for (int i = threadIdx.x; i < kSimtRows * DPad / 4; i += kThreads) {
        const int r = i % kSimtRows;
        const int e = i / kSimtRows * 4;
        const float4 x = r < rows ? load_four(q + r * p.q_stride, e, d) : zeros();
        qs[e * kRowPitch + r] = x.x;
        qs[(e + 1) * kRowPitch + r] = x.y;
        qs[(e + 2) * kRowPitch + r] = x.z;
        qs[(e + 3) * kRowPitch + r] = x.w;
    }
    const int tx = threadIdx.x % kX;
    const int ty = threadIdx.x / kX;
    float o[kCols][8][4] = {}; // element group, row, element
    float maximum[8], sum[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        maximum[r] = -INFINITY;
        sum[r] = 0.0F;
    }
    for (int first = first_key; first < last_key; first += kSimtKeys) {
        __syncthreads(); // the previous tile has been used
        const int live = min(kSimtKeys, last_key - first);
        for (int i = threadIdx.x; i < kSimtKeys * DPad / 4; i += kThreads) {
            const int j = i % kSimtKeys;
            const int e = i / kSimtKeys * 4;
            const long long row = static_cast<long long>(first) + j;
            const float4 x = j < live ? load_four(k + row * p.k_stride, e, d) : zeros();
            const int m = j / kX;
            const int at = m / 4 * (4 * kX) + j % kX * 4 + m % 4;
            ks[e * kKeyPitch + at] = x.x;
            ks[(e + 1) * kKeyPitch + at] = x.y;
            ks[(e + 2) * kKeyPitch + at] = x.z;
            ks[(e + 3) * kKeyPitch + at] = x.w;
        }
        for (int i = threadIdx.x; i < kSimtKeys * DPad / 4; i += kThreads) {
            const int j = i / (DPad / 4);
            const int e = i % (DPad / 4) * 4;
            const long long row = static_cast<long long>(first) + j;
            *reinterpret_cast<float4*>(vs + j * DPad + e) =
                j < live ? load_four(v + row * p.v_stride, e, d) : zeros();
        }
        __syncthreads();
        float score[kGroups][8][4] = {}; // key group, row, key
#pragma unroll 4
        for (int e = 0; e < d; ++e) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                outer(qs + e * kRowPitch + 8 * ty,
                      *reinterpret_cast<const float4*>(ks + e * kKeyPitch + 4 * kX * g + 4 * tx),
                      score[g]);
            }
        }
        float factor[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int limit = static_cast<int>(
                p.causal ? min(static_cast<long long>(live), reach + 8 * ty + r + 1 - first)
                         : static_cast<long long>(live));
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4 * kGroups; ++j) {
                float& value = score[j / 4][r][j % 4];
                value = tx + kX * j < limit ? value * p.scale_log2 : -INFINITY;
                top = fmaxf(top, value);
            }
#pragma unroll
            for (int offset = kX / 2; offset > 0; offset /= 2) {
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
            }
            const float raised = fmaxf(maximum[r], top);
            // A row without a key so far: any finite stand-in keeps 2^(-inf - m) at zero.
            const float stand = raised == -INFINITY ? 0.0F : raised;
            factor[r] = exp2f(maximum[r] - stand);
            maximum[r] = raised;
            sum[r] *= factor[r];
#pragma unroll
            for (int j = 0; j < 4 * kGroups; ++j) {
                score[j / 4][r][j % 4] = exp2f(score[j / 4][r][j % 4] - stand);
                sum[r] += score[j / 4][r][j % 4];
            }
        }
#pragma unroll
        for (int j = 0; j < 4 * kGroups; ++j) {
            float4* const at =
                reinterpret_cast<float4*>(ps + (tx + kX * j) * kRowPitch + 8 * ty);
            const float(&s8)[8][4] = score[j / 4];
            const int c = j % 4;
            at[0] = make_float4(s8[0][c], s8[1][c], s8[2][c], s8[3][c]);
            at[1] = make_float4(s8[4][c], s8[5][c], s8[6][c], s8[7][c]);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[c][r][j] *= factor[r];
                }
            }
        }
        __syncwarp(); // the threads of a row are in one warp
#pragma unroll 4
        for (int j = 0; j < live; ++j) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                outer(ps + j * kRowPitch + 8 * ty,
                      *reinterpret_cast<const float4*>(vs + j * DPad + 4 * kX * c + 4 * tx), o[c]);
            }
        }
    }
    T* const out = static_cast<T*>(p.out) + s.q_first * p.out_stride +
                   static_cast<long long>(head) * d;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
        for (int offset = kX / 2; offset > 0; offset /= 2) {
            sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], offset);
        }
        const float inverse = sum[r] == 0.0F ? 0.0F : 1.0F / sum[r];
        const int row = 8 * ty + r;
        const long long at =
            (static_cast<long long>(split) * p.q_tokens + s.q_first + row) * p.q_heads + head;
        if (row < rows && p.splits > 1 && tx == 0) {
            p.part_stats[at] = make_float2(maximum[r], sum[r]);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = 4 * kX * c + 4 * tx + j;
                const float value = o[c][r][j];
                if (row < rows && e < d) {
                    if (p.splits > 1) {
                        p.part_out[at * d + e] = value;
                    } else {
                        out[row * p.out_stride + e] = __float2bfloat16_rn(value * inverse);
                    }
                }
            }
        }
    }
}

long long simt_items(const VarlenParams& p) {
    return (static_cast<long long>(p.q_tokens) / kSimtRows + p.batch) * p.q_heads;
}

template <int DPad>
int launch_simt(const VarlenParams& p, cudaStream_t stream) {
    auto* kernel = &attention_varlen_simt<DPad>;
    constexpr int kBytes = SimtShape<DPad>::kSmemBytes;
    CUVIT_TRY_CUDA(host::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kBytes));
    const long long blocks = simt_items(p) * p.splits;
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "attention launch exceeds the CUDA grid limit");
    }
    host::pdl_launch(kernel, dim3(static_cast<unsigned>(blocks)), dim3(SimtShape<DPad>::kThreads),
                     kBytes, stream, p);
    return host::after_launch("attention_varlen_simt");
}

// Checks a problem's numbers and resolves its defaults; pointers stay null.
int resolve(const cuvit_attention_problem* problem, VarlenParams* out, bool* empty) {
    if (problem == nullptr) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "attention problem cannot be null");
    }
    const cuvit_attention_problem& c = *problem;
    if (c.batch < 0 || c.q_tokens < 0 || c.kv_tokens < 0 || c.q_heads < 0 || c.kv_heads < 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "attention dimensions cannot be negative");
    }
    if (c.head_dim < 1 || c.head_dim > 128) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "attention head_dim must be from 1 to 128");
    }
    if (c.dtype != CUVIT_DTYPE_F32 && c.dtype != CUVIT_DTYPE_BF16) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "packed attention operands must be F32 or BF16");
    }
    // The kernels work with scale * log2(e), which has to be a float too.
    constexpr float kLog2e = 1.4426950408889634F;
    if (!(c.scale > 0.0F) || !std::isfinite(c.scale * kLog2e)) {
        return host::fail(CUVIT_INVALID_ARGUMENT,
                          "the attention scale must be positive and finite, also times log2(e)");
    }
    constexpr int kMaxTokens = 0x7FFFFFFF - 4096; // tile ends past the last row stay in int
    if (c.q_tokens > kMaxTokens || c.kv_tokens > kMaxTokens) {
        return host::fail(CUVIT_LENGTH_ERROR, "too many packed attention rows");
    }
    *empty = c.batch == 0 || c.q_tokens == 0 || c.q_heads == 0;
    if (*empty) {
        return CUVIT_OK;
    }
    if (c.kv_heads == 0 || c.q_heads % c.kv_heads != 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "kv_heads must divide q_heads");
    }
    VarlenParams p{};
    p.batch = c.batch;
    p.q_tokens = c.q_tokens;
    p.kv_tokens = c.kv_tokens;
    p.q_heads = c.q_heads;
    p.kv_heads = c.kv_heads;
    p.group = c.q_heads / c.kv_heads;
    p.head_dim = c.head_dim;
    p.causal = c.causal ? 1 : 0;
    p.bf16 = c.dtype == CUVIT_DTYPE_BF16 ? 1 : 0;
    p.splits = 1;
    p.scale_log2 = c.scale * kLog2e;
    const int64_t q_width = static_cast<int64_t>(c.q_heads) * c.head_dim;
    const int64_t kv_width = static_cast<int64_t>(c.kv_heads) * c.head_dim;
    p.q_stride = c.q_stride != 0 ? c.q_stride : q_width;
    p.k_stride = c.k_stride != 0 ? c.k_stride : kv_width;
    p.v_stride = c.v_stride != 0 ? c.v_stride : kv_width;
    p.out_stride = c.out_stride != 0 ? c.out_stride : q_width;
    if (p.q_stride < q_width || p.out_stride < q_width || p.k_stride < kv_width ||
        p.v_stride < kv_width) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "an attention row stride is smaller than its row");
    }
    const int64_t q_limit = (int64_t{1} << 58) / c.q_tokens;
    const int64_t kv_limit = (int64_t{1} << 58) / (c.kv_tokens > 0 ? c.kv_tokens : 1);
    if (p.q_stride > q_limit || p.out_stride > q_limit || p.k_stride > kv_limit ||
        p.v_stride > kv_limit) {
        return host::fail(CUVIT_LENGTH_ERROR, "an attention row stride is too large");
    }
    *out = p;
    return CUVIT_OK;
}

// Splits of the keys that give every SM `per_sm` blocks when the query rows alone do not, each
// split with at least min_keys of an average sequence's keys.
int choose_splits(const VarlenParams& p, long long items, int per_sm, int min_keys, int sm_count) {
    const long long wanted = (static_cast<long long>(sm_count) * per_sm) / (items > 0 ? items : 1);
    const long long most = p.kv_tokens / static_cast<long long>(p.batch) / min_keys;
    const long long splits = wanted < most ? wanted : most;
    return static_cast<int>(splits < 1 ? 1 : (splits > kMaxSplits ? kMaxSplits : splits));
}

enum class Kernel { kSimt, kRows, kTiles, kSplit };

// The splits of a call through each kernel, were a workspace given.
int splits_of(Kernel kernel, const VarlenParams& p, int sm_count) {
    switch (kernel) {
    case Kernel::kRows:
        // About half of the launch's bound on blocks have rows (varlen.cuh).
        return choose_splits(p, rows_kernel_items(p) / 2, 4, 128, sm_count);
    case Kernel::kTiles:
        return choose_splits(p, tiles_kernel_items(p), 1, 512, sm_count);
    case Kernel::kSplit:
        return choose_splits(p, split_kernel_items(p), 1, 512, sm_count);
    default:
        return choose_splits(p, simt_items(p), 2, 256, sm_count);
    }
}

Kernel choose(const VarlenParams& p) {
    if (rows_kernel_takes(p)) {
        return Kernel::kRows;
    }
    if (!p.bf16) {
        return Kernel::kSplit;
    }
    return tiles_kernel_takes(p) ? Kernel::kTiles : Kernel::kSimt;
}

// The parts' outputs, rounded up to whole 16-byte vectors, then their statistics.
size_t part_rows(const VarlenParams& p) {
    return static_cast<size_t>(p.splits) * static_cast<size_t>(p.q_tokens) *
           static_cast<size_t>(p.q_heads);
}

size_t part_out_bytes(const VarlenParams& p) {
    return (part_rows(p) * static_cast<size_t>(p.head_dim) * sizeof(float) + 15) / 16 * 16;
}

size_t workspace_bytes_of(const VarlenParams& p) {
    return p.splits <= 1 ? 0 : part_out_bytes(p) + part_rows(p) * sizeof(float2);
}

// Enough for every kernel the operands' alignments may select.
size_t workspace_bytes_at_most(VarlenParams p, int sm_count) {
    size_t most = 0;
    for (const Kernel kernel : {Kernel::kSimt, Kernel::kRows, Kernel::kTiles, Kernel::kSplit}) {
        p.splits = splits_of(kernel, p, sm_count);
        const size_t bytes = workspace_bytes_of(p);
        most = bytes > most ? bytes : most;
    }
    return most;
}

int run(const void* q, const void* k, const void* v, void* out, const int32_t* q_offsets,
        const int32_t* kv_offsets, const cuvit_attention_problem* problem, void* workspace,
        size_t workspace_bytes, cudaStream_t stream) {
    VarlenParams p{};
    bool empty = false;
    CUVIT_TRY(resolve(problem, &p, &empty));
    if (empty) {
        return CUVIT_OK;
    }
    if (q == nullptr || out == nullptr || q_offsets == nullptr ||
        (p.kv_tokens > 0 && (k == nullptr || v == nullptr))) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "attention operands cannot be null");
    }
    if (kv_offsets == nullptr) {
        if (p.kv_tokens != p.q_tokens) {
            return host::fail(CUVIT_INVALID_ARGUMENT,
                              "without key offsets there are as many keys as queries");
        }
        kv_offsets = q_offsets;
    }
    const bool bf16 = problem->dtype == CUVIT_DTYPE_BF16;
    const int element = bf16 ? 2 : 4;
    for (const void* operand : {q, k, v, static_cast<const void*>(out)}) {
        if (reinterpret_cast<uintptr_t>(operand) % element != 0) {
            return host::fail(CUVIT_INVALID_ARGUMENT,
                              "attention operands must be aligned to their type");
        }
    }
    if (reinterpret_cast<uintptr_t>(q_offsets) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(kv_offsets) % 4 != 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "offsets must be aligned to their type");
    }
    const int64_t q_width = static_cast<int64_t>(p.q_heads) * p.head_dim * element;
    const int64_t kv_width = static_cast<int64_t>(p.kv_heads) * p.head_dim * element;
    const host::RowSpan out_span{out, p.q_tokens, q_width, p.out_stride * element};
    const int64_t offset_bytes = (static_cast<int64_t>(p.batch) + 1) * 4;
    const host::RowSpan q_offset_span{q_offsets, 1, offset_bytes, offset_bytes};
    const host::RowSpan kv_offset_span{kv_offsets, 1, offset_bytes, offset_bytes};
    if (host::rows_overlap(out_span, {q, p.q_tokens, q_width, p.q_stride * element}) ||
        host::rows_overlap(out_span, {k, p.kv_tokens, kv_width, p.k_stride * element}) ||
        host::rows_overlap(out_span, {v, p.kv_tokens, kv_width, p.v_stride * element}) ||
        host::rows_overlap(out_span, q_offset_span) || host::rows_overlap(out_span, kv_offset_span)) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "the attention output overlaps an operand");
    }
    p.q = q;
    p.k = k;
    p.v = v;
    p.out = out;
    p.q_offsets = q_offsets;
    p.kv_offsets = kv_offsets;
    const host::DeviceContext* context = nullptr;
    CUVIT_TRY(host::current_context(&context));
    CUVIT_TRY(host::check_operands({q, k, v, out, q_offsets, kv_offsets}));
    const Kernel kernel = choose(p);
    p.splits = workspace != nullptr ? splits_of(kernel, p, context->sm_count) : 1;
    if (p.splits > 1) {
        const size_t needed = workspace_bytes_of(p);
        if (workspace_bytes < needed || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
            return host::fail(CUVIT_INVALID_ARGUMENT,
                              "the attention workspace is too small or not 16-byte aligned");
        }
        const int64_t area = static_cast<int64_t>(needed);
        const host::RowSpan span{workspace, 1, area, area};
        if (host::rows_overlap(span, {q, p.q_tokens, q_width, p.q_stride * element}) ||
            host::rows_overlap(span, {k, p.kv_tokens, kv_width, p.k_stride * element}) ||
            host::rows_overlap(span, {v, p.kv_tokens, kv_width, p.v_stride * element}) ||
            host::rows_overlap(span, q_offset_span) || host::rows_overlap(span, kv_offset_span) ||
            host::rows_overlap(span, out_span)) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "the attention workspace overlaps an operand");
        }
        CUVIT_TRY(host::check_operands({workspace}));
        p.part_out = static_cast<float*>(workspace);
        p.part_stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + part_out_bytes(p));
    }
    int status = CUVIT_OK;
    if (kernel == Kernel::kRows) {
        status = launch_rows(p, stream);
    } else if (kernel == Kernel::kTiles) {
        status = launch_tiles(p, stream);
    } else if (kernel == Kernel::kSplit) {
        status = launch_split(p, context->status, stream);
    } else {
        status = p.head_dim <= 64 ? launch_simt<64>(p, stream) : launch_simt<128>(p, stream);
    }
    if (status == CUVIT_OK && p.splits > 1) {
        status = launch_join(p, stream);
    }
    return status;
}

} // namespace
} // namespace cuvit::attn

extern "C" {

int cuvit_attention_varlen(const void* q, const void* k, const void* v, void* out,
                           const int32_t* q_offsets, const int32_t* kv_offsets,
                           const cuvit_attention_problem* problem, void* workspace,
                           size_t workspace_bytes, cuvit_stream_t stream) {
    return cuvit::host::guarded([&]() {
        return cuvit::attn::run(q, k, v, out, q_offsets, kv_offsets, problem, workspace,
                                workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
    });
}

int cuvit_attention_varlen_workspace(const cuvit_attention_problem* problem, size_t* bytes) {
    return cuvit::host::guarded([&]() {
        if (bytes == nullptr) {
            return cuvit::host::fail(CUVIT_INVALID_ARGUMENT, "workspace size cannot be null");
        }
        *bytes = 0;
        cuvit::attn::VarlenParams p{};
        bool empty = false;
        CUVIT_TRY(cuvit::attn::resolve(problem, &p, &empty));
        if (empty) {
            return static_cast<int>(CUVIT_OK);
        }
        const cuvit::host::DeviceContext* context = nullptr;
        CUVIT_TRY(cuvit::host::current_context(&context));
        *bytes = cuvit::attn::workspace_bytes_at_most(p, context->sm_count);
        return static_cast<int>(CUVIT_OK);
    });
}

} // extern "C"
