// Attention of a few bfloat16 query rows per sequence over many keys: pooling by one query, one new
// token of each sequence.
//
// Bound by HBM: every key and value is used for at most eight rows (queries times the heads that
// share a key head). Warp matrix instructions with the keys as the long side waste nothing on the
// few rows: per 16 keys, S^T = K Q^T is one m16n8k16 product per 16 elements and O^T += V^T P^T one
// as well, fed by ldmatrix from shared memory; the weights change from accumulator to operand by a
// transposing move. That is about 8 instructions a key and warp (dot products by lanes took 40,
// more than half of the time that the bytes take). tcgen05 has no shape for it: 128 rows are its
// least.
//
// Each warp of a block of two goes through every second group of 16 keys with a ring of its own
// (asynchronous copies, no barrier in the loop) and its own maximum, sum and output; warps and splits
// are merged at the end. Outputs are rescaled only when a maximum has risen by more than 2^8.
//
// One query of 16 heads over 4 key heads of 128, 16001 + 9000 keys (51 MB): 15.7 us (dot products
// 23.5), where the copy rate would allow 7.8; then the join. 256 queries over 197 keys each, 12 heads
// of 64: 36 us of 24. Half of the rest is a block's start (offsets, then its first keys) and end.
// Blocks of two warps: 4 take a tenth longer (fewer blocks start beside each other's ends), and so do
// 4 or 6 stages.
#include "attention_varlen.hpp"
#include "ptx.cuh"
#include "varlen.cuh"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::attn {
namespace {

constexpr int kWarps = 2;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = 16; // of a warp's step
constexpr int kStages = 3;
constexpr int kRows = kMaxRows;
static_assert(kRows == 8, "the products' short side");

// Steps: 16-element steps of a head.
template <int Steps>
struct Shape {
    static constexpr int kChunks = 2 * Steps;        // 16-byte chunks of a row
    static constexpr int kPitch = 16 * kChunks + 16; // an odd number of chunks: no bank conflicts
    static constexpr int kTileBytes = kKeys * kPitch;
    static constexpr int kRingBytes = kStages * 2 * kTileBytes; // of a warp
    static constexpr int kOutPitch = 16 * Steps + 4;            // floats
    static constexpr int kPartBytes = kRows * (kOutPitch * 4 + 8);
    static constexpr int kSmemBytes =
        kWarps * (kRingBytes > kPartBytes ? kRingBytes : kPartBytes);
};

__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from),
                 "r"(live ? 16 : 0)
                 : "memory");
}

__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&m)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
                 : "r"(at)
                 : "memory");
}

__device__ __forceinline__ void load_matrices_transposed(uint32_t at, uint32_t (&m)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
                 : "r"(at)
                 : "memory");
}

__device__ __forceinline__ uint32_t transpose_matrix(uint32_t m) {
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(m));
    return t;
}

// c += a (16 x 16) b (16 x 8), bfloat16 with FP32 sums.
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int Steps>
__global__ void __launch_bounds__(kThreads)
    attention_few_kernel(const VarlenParams p, int queries_per_block, int head_chunks) {
    using S = Shape<Steps>;
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    extern __shared__ __align__(16) uint8_t smem[];

    // Item: block of queries, split, key head (its rows lie next to the next head's), chunk of the
    // key head's query heads.
    long long item = blockIdx.x;
    const int chunk = static_cast<int>(item % head_chunks);
    item /= head_chunks;
    const int kv_head = static_cast<int>(item % p.kv_heads);
    item /= p.kv_heads;
    const int split = static_cast<int>(item % p.splits);
    item /= p.splits;
    const Sequence s = find_block_warp(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                       item, queries_per_block);
    if (s.index < 0) {
        return; // the whole block
    }
    const int per_query = kRows / queries_per_block;
    const int heads = min(per_query, p.group - chunk * per_query);
    const int head0 = kv_head * p.group + chunk * per_query;
    const int queries = min(queries_per_block, s.q_end - s.q_first);
    const int rows = heads * queries; // row r: query r / heads, head r % heads
    const int keys = s.kv_end - s.kv_begin;
    int first_key, end_key;
    split_keys(keys, split, p.splits, first_key, end_key);

    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const __nv_bfloat16* const k = static_cast<const __nv_bfloat16*>(p.k) +
                                   s.kv_begin * p.k_stride +
                                   static_cast<long long>(kv_head) * p.head_dim;
    const __nv_bfloat16* const v = static_cast<const __nv_bfloat16*>(p.v) +
                                   s.kv_begin * p.v_stride +
                                   static_cast<long long>(kv_head) * p.head_dim;
    const uint32_t ring = dev::smem_u32(smem) + warp * S::kRingBytes;
    const int k_stride = static_cast<int>(p.k_stride); // (host: 16 rows stay in 31 bits)
    const int v_stride = static_cast<int>(p.v_stride);
    const auto fetch = [&](int stage, int first) {
        const uint32_t to = ring + stage * 2 * S::kTileBytes;
        const __nv_bfloat16* const k_at = k + first * p.k_stride;
        const __nv_bfloat16* const v_at = v + first * p.v_stride;
#pragma unroll
        for (int i = 0; i < Steps; ++i) {
            const int row = (lane + 32 * i) / S::kChunks;
            const int c = (lane + 32 * i) % S::kChunks;
            const bool live = first + row < end_key && 8 * c < p.head_dim;
            const uint32_t here = to + row * S::kPitch + 16 * c;
            copy_async(here, live ? k_at + (row * k_stride + 8 * c) : k, live);
            copy_async(here + S::kTileBytes, live ? v_at + (row * v_stride + 8 * c) : k, live);
        }
    };
    const int own = first_key + warp * kKeys; // this warp's first keys
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (own + i * kWarps * kKeys < end_key) {
            fetch(i, own + i * kWarps * kKeys);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // The queries as the products' second operand: row lane / 4, elements 2 (lane % 4) and the next
    // of every eight.
    uint32_t q[Steps][2];
    {
        const int row = lane / 4;
        const int query = row / heads;
        const __nv_bfloat16* const from =
            static_cast<const __nv_bfloat16*>(p.q) + (s.q_first + query) * p.q_stride +
            static_cast<long long>(head0 + row - query * heads) * p.head_dim;
#pragma unroll
        for (int i = 0; i < 2 * Steps; ++i) {
            const int e = 8 * i + 2 * (lane % 4);
            q[i / 2][i % 2] = row < rows && e < p.head_dim
                                  ? __ldg(reinterpret_cast<const uint32_t*>(from + e))
                                  : 0u;
        }
    }
    // Of the scores and outputs a lane has rows 2 (lane % 4) and the next.
    int limit[2]; // keys the row sees
    float top[2]; // its maximum, at most 2^8 below the true one; the same in all its lanes
    float sum[2]; // its weights, of this lane's keys
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = 2 * (lane % 4) + h;
        const long long last = static_cast<long long>(s.q_first - s.q_begin) + r / heads + 1 + keys -
                               (s.q_end - s.q_begin);
        limit[h] = p.causal ? static_cast<int>(max(0LL, min(static_cast<long long>(end_key), last)))
                            : end_key;
        limit[h] = r < rows ? limit[h] : 0;
        top[h] = -INFINITY;
        sum[h] = 0.0F;
    }
    float o[Steps][4];
#pragma unroll
    for (int i = 0; i < Steps; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[i][j] = 0.0F;
        }
    }
    // Where this lane's rows of the 8 x 8 matrices are: keys by elements, and for values the same
    // matrices taken transposed.
    const uint32_t k_lane = ((lane & 7) + (lane & 8)) * S::kPitch + (lane >> 4) * 16;
    const uint32_t v_lane =
        S::kTileBytes + ((lane & 7) + (lane >> 4) * 8) * S::kPitch + (lane & 8) * 2;
    int stage = 0;
    for (int first = own; first < end_key; first += kWarps * kKeys) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp(); // the other lanes' copies
        const uint32_t tile = ring + stage * 2 * S::kTileBytes;
        float even[4] = {}, odd[4] = {}; // two chains of products
#pragma unroll
        for (int i = 0; i < Steps; ++i) {
            uint32_t a[4];
            load_matrices(tile + k_lane + 32 * i, a);
            multiply(i % 2 == 0 ? even : odd, a, q[i][0], q[i][1]);
        }
        float score[2][2]; // row, key lane / 4 and the one 8 on
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // Rounded before the maximum is taken off, so that huge scores lose what it loses.
                const float both = __fmul_rn(even[2 * j + h] + odd[2 * j + h], p.scale_log2);
                score[h][j] = first + 8 * j + lane / 4 < limit[h] ? both : -INFINITY;
            }
        }
        float high[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            high[h] = fmaxf(score[h][0], score[h][1]);
        }
        if (__any_sync(0xFFFFFFFFu, high[0] > top[0] + 8.0F || high[1] > top[1] + 8.0F)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int offset = 4; offset < 32; offset *= 2) {
                    high[h] = fmaxf(high[h], __shfl_xor_sync(0xFFFFFFFFu, high[h], offset));
                }
                // Without a key so far, any finite stand-in keeps 2^(-inf - m) at zero.
                const float raised = fmaxf(top[h], high[h]);
                const float factor = exp2f(top[h] - (raised == -INFINITY ? 0.0F : raised));
                top[h] = raised;
                sum[h] *= factor;
#pragma unroll
                for (int i = 0; i < Steps; ++i) {
                    o[i][h] *= factor;
                    o[i][2 + h] *= factor;
                }
            }
        }
        float weight[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float stand = top[h] == -INFINITY ? 0.0F : top[h];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                weight[h][j] = dev::ex2_approx(score[h][j] - stand);
            }
        }
        // Rounded to bfloat16 for the products; the sum takes the rounded weights, so that they
        // still add up to one.
        const uint32_t low = dev::pack_bf16x2(weight[0][0], weight[1][0]);
        const uint32_t up = dev::pack_bf16x2(weight[0][1], weight[1][1]);
        sum[0] += __uint_as_float(low << 16) + __uint_as_float(up << 16);
        sum[1] += __uint_as_float(low & 0xFFFF0000u) + __uint_as_float(up & 0xFFFF0000u);
        const uint32_t b0 = transpose_matrix(low);
        const uint32_t b1 = transpose_matrix(up);
#pragma unroll
        for (int i = 0; i < Steps; ++i) {
            uint32_t a[4];
            load_matrices_transposed(tile + v_lane + 32 * i, a);
            multiply(o[i], a, b0, b1);
        }
        __syncwarp(); // every lane has read the stage that is filled next but one
        const int next = first + (kStages - 1) * kWarps * kKeys;
        if (next < end_key) {
            fetch(stage == 0 ? kStages - 1 : stage - 1, next);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads(); // the rings become the warps' parts

    float* const parts = reinterpret_cast<float*>(smem); // [warp][row][kOutPitch]
    float2* const stats = reinterpret_cast<float2*>(parts + kWarps * kRows * S::kOutPitch);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int offset = 4; offset < 32; offset *= 2) {
            sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], offset);
        }
        const int r = 2 * (lane % 4) + h;
        if (lane < 4) {
            stats[warp * kRows + r] = make_float2(top[h], sum[h]);
        }
#pragma unroll
        for (int i = 0; i < Steps; ++i) {
            float* const at = parts + (warp * kRows + r) * S::kOutPitch + 16 * i + lane / 4;
            at[0] = o[i][h];
            at[8] = o[i][2 + h];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * p.head_dim; i += kThreads) {
        const int r = i / p.head_dim;
        const int e = i - r * p.head_dim;
        float raised = stats[r].x;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            raised = fmaxf(raised, stats[w * kRows + r].x);
        }
        const float stand = raised == -INFINITY ? 0.0F : raised;
        float total = 0.0F, value = 0.0F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 stat = stats[w * kRows + r];
            const float factor = exp2f(stat.x - stand);
            total = fmaf(factor, stat.y, total);
            value = fmaf(factor, parts[(w * kRows + r) * S::kOutPitch + e], value);
        }
        const int query = r / heads;
        const int head = head0 + r - query * heads;
        const long long row = s.q_first + query;
        if (p.splits > 1) {
            const long long at =
                (static_cast<long long>(split) * p.q_tokens + row) * p.q_heads + head;
            p.part_out[at * p.head_dim + e] = value;
            if (e == 0) {
                p.part_stats[at] = make_float2(raised, total);
            }
        } else {
            static_cast<__nv_bfloat16*>(p.out)[row * p.out_stride +
                                               static_cast<long long>(head) * p.head_dim + e] =
                __float2bfloat16_rn(total == 0.0F ? 0.0F : value / total);
        }
    }
}

template <int Steps>
int launch_steps(const VarlenParams& p, int queries, int chunks, unsigned blocks,
                 cudaStream_t stream) {
    auto* kernel = &attention_few_kernel<Steps>;
    constexpr int kBytes = Shape<Steps>::kSmemBytes;
    CUVIT_TRY_CUDA(host::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kBytes));
    host::pdl_launch(kernel, dim3(blocks), dim3(kThreads), kBytes, stream, p, queries, chunks);
    return host::after_launch("attention_few_kernel");
}

} // namespace

int launch_few(const VarlenParams& p, int queries_per_block, int head_chunks, unsigned blocks,
               cudaStream_t stream) {
    const auto start = [&](auto* launch) {
        return launch(p, queries_per_block, head_chunks, blocks, stream);
    };
    switch ((p.head_dim + 15) / 16) {
    case 1:
    case 2:
        return start(&launch_steps<2>);
    case 3:
    case 4:
        return start(&launch_steps<4>);
    case 5:
        return start(&launch_steps<5>);
    case 6:
        return start(&launch_steps<6>);
    default:
        return start(&launch_steps<8>);
    }
}

} // namespace cuvit::attn
