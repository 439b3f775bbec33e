// Attention of a few float query rows per sequence over many keys (pooling by one query, one new
// token of each sequence), and the kernel that joins the parts of calls that split their keys.
//
// Bound by HBM: every key and value is used for a handful of multiply-adds per byte. A group of
// lanes takes a few keys at a time, 16 bytes of each a lane (the query rows' same elements stay in
// registers), and keeps its own running maximum, sum and output for its share of the keys; groups,
// warps and splits are merged at the end. Rows that share a key head (grouped heads, several
// queries) are taken together, so keys are read once for them.
//
// What is left to spend is issue slots: 4 rows over heads of 128 at 24 bytes a cycle and SM leave
// about 40 instructions a key and warp. So the lanes' partial scores of all (row, key) pairs are
// summed by halving, each step leaving a lane with half the pairs (15 shuffles for 16 sums over 16
// lanes, where a butterfly for each takes 64), every weight is computed once, by the lane that ends
// up with its score, and handed back by one shuffle, products run as packed pairs, and outputs are
// rescaled only when a maximum has risen by more than 2^8 (weights stay below 2^8; the quotient
// does not change).
#include "attention_varlen.hpp"
#include "ptx.cuh"
#include "varlen.cuh"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::attn {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kStages = 3; // of keys and values in flight: 48 KB a block, four blocks an SM
// Keys a lane group has in flight (registers bound it: 8 rows hold 64 of queries and 64 of output).
template <int Rows>
constexpr int kUnrollOf = Rows >= 8 ? 2 : 4;

// One lane's 16 bytes of a row.
constexpr int kElems = 4;
constexpr int kPairs = kElems / 2;

__device__ __forceinline__ void unpack(const uint4& raw, uint64_t (&out)[kPairs]) {
    out[0] = dev::f32x2(__uint_as_float(raw.x), __uint_as_float(raw.y));
    out[1] = dev::f32x2(__uint_as_float(raw.z), __uint_as_float(raw.w));
}

// Copies 16 bytes to shared memory asynchronously, or zeros.
__device__ __forceinline__ void copy_async(uint4* to, const float* p, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dev::smem_u32(to)), "l"(p),
                 "r"(live ? 16 : 0)
                 : "memory");
}

__host__ __device__ constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// Which of a group's N = Rows * Unroll sums (sum r * Unroll + u is row r's of key u) a lane ends up
// with after halving: kHeld consecutive ones, from kHeld * (lane / kCopies) on.
template <int Lanes, int Rows, int Unroll>
struct Halving {
    static constexpr int kSums = Rows * Unroll;
    static constexpr int kSteps =
        log2_of(kSums) < log2_of(Lanes) ? log2_of(kSums) : log2_of(Lanes);
    static constexpr int kHeld = kSums >> kSteps;
    static constexpr int kCopies = Lanes >> kSteps; // lanes with the same sums
    static constexpr int kHeldRows = kHeld > Unroll ? kHeld / Unroll : 1;
    static constexpr int kHeldKeys = kHeld > Unroll ? Unroll : kHeld;

    // The lane of a group that holds sum i, and where.
    static __host__ __device__ constexpr int lane_of(int i) { return i / kHeld * kCopies; }
    static __host__ __device__ constexpr int place_of(int i) { return i % kHeld; }

    static __device__ __forceinline__ void reduce(float (&v)[kSums], int lane) {
#pragma unroll
        for (int step = 0; step < log2_of(Lanes); ++step) {
            const int offset = Lanes >> (step + 1);
            if (step < kSteps) {
                const int n = kSums >> (step + 1);
                const bool upper = (lane & offset) != 0;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const float send = upper ? v[i] : v[i + n];
                    const float keep = upper ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, offset);
                }
            } else {
                v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], offset);
            }
        }
    }
};

// Merges (m, l, o) with another part's; a part without a key has m = -inf and l = 0.
__device__ __forceinline__ void merge_factors(float m, float other, float& top, float& mine,
                                              float& theirs) {
    top = fmaxf(m, other);
    const float base = top == -INFINITY ? 0.0F : top;
    mine = exp2f(m - base);
    theirs = exp2f(other - base);
}

template <int Lanes, int Rows>
__global__ void __launch_bounds__(kThreads)
    attention_rows_kernel(const VarlenParams p, int queries_per_block, int head_chunks) {
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    constexpr int kUnroll = kUnrollOf<Rows>;
    using Halves = Halving<Lanes, Rows, kUnroll>;
    constexpr int kGroups = kThreads / Lanes; // key streams of the block
    // Keys and values in flight; each lane reads back only what it copied itself, so the ring
    // needs no barrier. Afterwards the warps' parts.
    struct Parts {
        float out[kWarps][Rows][Lanes * kElems];
        float2 stats[kWarps][Rows];
    };
    __shared__ union {
        uint4 ring[kStages][kUnroll][2][kThreads];
        Parts parts;
    } shared;
    auto& merged_out = shared.parts.out;
    auto& merged_stats = shared.parts.stats;

    // Item: block of queries, key head, chunk of its query heads, split (fastest: the splits of
    // one range run together).
    long long item = blockIdx.x;
    const int split = static_cast<int>(item % p.splits);
    item /= p.splits;
    const int chunk = static_cast<int>(item % head_chunks);
    item /= head_chunks;
    const int kv_head = static_cast<int>(item % p.kv_heads);
    const Sequence s = find_block(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                  item / p.kv_heads, queries_per_block);
    if (s.index < 0) {
        return;
    }
    const int heads = min(Rows / queries_per_block, p.group - chunk * (Rows / queries_per_block));
    const int head0 = kv_head * p.group + chunk * (Rows / queries_per_block);
    const int queries = min(queries_per_block, s.q_end - s.q_first);
    const int rows = heads * queries; // row r: query r / heads, head r % heads
    const int keys = s.kv_end - s.kv_begin;
    int first_key, end_key;
    split_keys(keys, split, p.splits, first_key, end_key);

    const int lane = threadIdx.x % Lanes;
    const int group = threadIdx.x / Lanes;
    const int element = lane * kElems;
    const bool in_row = element < p.head_dim;

    uint64_t q[Rows][kPairs];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int query = r / heads;
        const int head = head0 + r - query * heads;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            q[r][j] = 0u;
        }
        if (r < rows && in_row) {
            const float* const from = static_cast<const float*>(p.q) +
                                      (s.q_first + query) * p.q_stride +
                                      static_cast<long long>(head) * p.head_dim + element;
            unpack(__ldg(reinterpret_cast<const uint4*>(from)), q[r]);
            const uint64_t scale = dev::f32x2(p.scale_log2, p.scale_log2);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                q[r][j] = dev::mul_f32x2(q[r][j], scale);
            }
        }
    }
    // What this lane holds of the group's scores: rows from held_row on, keys from held_key on.
    const int held = lane / Halves::kCopies * Halves::kHeld;
    const int held_row = held / kUnroll;
    const int held_key = held % kUnroll;
    int limit[Halves::kHeldRows]; // keys a held row sees
    float top[Halves::kHeldRows]; // its maximum, at most 2^8 below the true one
    float sum[Halves::kHeldRows]; // its weights, of the keys held here
#pragma unroll
    for (int h = 0; h < Halves::kHeldRows; ++h) {
        const int r = held_row + h;
        const long long last = static_cast<long long>(s.q_first - s.q_begin) + r / heads + 1 +
                               keys - (s.q_end - s.q_begin);
        limit[h] = p.causal ? static_cast<int>(max(0LL, min(static_cast<long long>(end_key), last)))
                            : end_key;
        limit[h] = r < rows ? limit[h] : 0;
        top[h] = -INFINITY;
        sum[h] = 0.0F;
    }
    const float* const k0 = static_cast<const float*>(p.q); // never read: copies of no bytes name it
    const float* const k = static_cast<const float*>(p.k) + s.kv_begin * p.k_stride +
                       static_cast<long long>(kv_head) * p.head_dim + element;
    const float* const v = static_cast<const float*>(p.v) + s.kv_begin * p.v_stride +
                       static_cast<long long>(kv_head) * p.head_dim + element;

    uint64_t o[Rows][kPairs];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            o[r][j] = 0u;
        }
    }
    const int group_lane0 = threadIdx.x % 32 / Lanes * Lanes;
    const auto from_lane = [&](float value, int lane_of_group) {
        return __shfl_sync(0xFFFFFFFFu, value, group_lane0 + lane_of_group);
    };
    // Whole warps go round together (the sums need every lane).
    const int warp_group0 = (threadIdx.x / 32) * (32 / Lanes);
    const int step = kGroups * kUnroll;
    const auto fetch = [&](int stage, int base) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int key = base + u * kGroups + group;
            const bool live = key < end_key && in_row;
            const long long row = live ? key : 0;
            copy_async(&shared.ring[stage][u][0][threadIdx.x], live ? k + row * p.k_stride : k0,
                       live);
            copy_async(&shared.ring[stage][u][1][threadIdx.x], live ? v + row * p.v_stride : k0,
                       live);
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (first_key + i * step + warp_group0 < end_key) {
            fetch(i, first_key + i * step);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int stage = 0;
    for (int base = first_key; base + warp_group0 < end_key; base += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        float score[Halves::kSums];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            uint64_t kf[kPairs];
            unpack(shared.ring[stage][u][0][threadIdx.x], kf);
#pragma unroll
            for (int r = 0; r < Rows; ++r) {
                uint64_t dot = dev::mul_f32x2(q[r][0], kf[0]);
#pragma unroll
                for (int j = 1; j < kPairs; ++j) {
                    dot = dev::fma_f32x2(q[r][j], kf[j], dot);
                }
                const float2 both = dev::f32x2_split(dot);
                score[r * kUnroll + u] = both.x + both.y;
            }
        }
        Halves::reduce(score, lane);
        // The held scores' weights.
        bool raise = false;
        float high[Halves::kHeldRows];
#pragma unroll
        for (int h = 0; h < Halves::kHeldRows; ++h) {
            high[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < Halves::kHeldKeys; ++i) {
                float& value = score[h * Halves::kHeldKeys + i];
                const int key = base + (held_key + i) * kGroups + group;
                value = key < limit[h] ? value : -INFINITY;
                high[h] = fmaxf(high[h], value);
            }
            // Over the lanes that hold the row's other keys.
#pragma unroll
            for (int keys_held = Halves::kHeldKeys; keys_held < kUnroll; keys_held *= 2) {
                high[h] = fmaxf(high[h],
                                __shfl_xor_sync(0xFFFFFFFFu, high[h],
                                                keys_held / Halves::kHeld * Halves::kCopies));
            }
            raise = raise || high[h] > top[h] + 8.0F;
        }
        if (__any_sync(0xFFFFFFFFu, raise)) {
            float factor[Halves::kHeldRows];
#pragma unroll
            for (int h = 0; h < Halves::kHeldRows; ++h) {
                // Without a key so far, any finite stand-in keeps 2^(-inf - m) at zero.
                const float raised = fmaxf(top[h], high[h]);
                factor[h] = exp2f(top[h] - (raised == -INFINITY ? 0.0F : raised));
                top[h] = raised;
                sum[h] *= factor[h];
            }
#pragma unroll
            for (int r = 0; r < Rows; ++r) {
                const float f = from_lane(factor[Halves::place_of(r * kUnroll) / kUnroll],
                                          Halves::lane_of(r * kUnroll));
                const uint64_t f2 = dev::f32x2(f, f);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    o[r][j] = dev::mul_f32x2(o[r][j], f2);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < Halves::kHeldRows; ++h) {
            const float stand = top[h] == -INFINITY ? 0.0F : top[h];
#pragma unroll
            for (int i = 0; i < Halves::kHeldKeys; ++i) {
                float& value = score[h * Halves::kHeldKeys + i];
                value = dev::ex2_approx(value - stand);
                sum[h] += value;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            uint64_t vf[kPairs];
            unpack(shared.ring[stage][u][1][threadIdx.x], vf);
#pragma unroll
            for (int r = 0; r < Rows; ++r) {
                const float weight = from_lane(score[Halves::place_of(r * kUnroll + u)],
                                               Halves::lane_of(r * kUnroll + u));
                const uint64_t weight2 = dev::f32x2(weight, weight);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    o[r][j] = dev::fma_f32x2(weight2, vf[j], o[r][j]);
                }
            }
        }
        // Into the stage read in the previous round: its values have been used by now.
        const int ahead = stage == 0 ? kStages - 1 : stage - 1;
        const int next = base + (kStages - 1) * step;
        if (next + warp_group0 < end_key) {
            fetch(ahead, next);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads(); // the ring becomes the parts

    // Every lane gets its group's maxima and sums, then lane groups of a warp and the warps are
    // merged, in a fixed order.
    float row_top[Rows], row_sum[Rows];
    float part[Rows][kElems];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int slot = Halves::place_of(r * kUnroll) / kUnroll;
        row_top[r] = from_lane(top[slot], Halves::lane_of(r * kUnroll));
        row_sum[r] = 0.0F;
#pragma unroll
        for (int u = 0; u < kUnroll; u += Halves::kHeldKeys) {
            row_sum[r] += from_lane(sum[slot], Halves::lane_of(r * kUnroll + u));
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const float2 pair = dev::f32x2_split(o[r][j]);
            part[r][2 * j] = pair.x;
            part[r][2 * j + 1] = pair.y;
        }
    }
#pragma unroll
    for (int offset = Lanes; offset < 32; offset *= 2) {
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            const float other = __shfl_xor_sync(0xFFFFFFFFu, row_top[r], offset);
            const float other_sum = __shfl_xor_sync(0xFFFFFFFFu, row_sum[r], offset);
            float raised, mine, theirs;
            merge_factors(row_top[r], other, raised, mine, theirs);
            row_top[r] = raised;
            row_sum[r] = row_sum[r] * mine + other_sum * theirs;
#pragma unroll
            for (int j = 0; j < kElems; ++j) {
                const float other_o = __shfl_xor_sync(0xFFFFFFFFu, part[r][j], offset);
                part[r][j] = part[r][j] * mine + other_o * theirs;
            }
        }
    }
    const int warp = threadIdx.x / 32;
    if (threadIdx.x % 32 < Lanes) {
#pragma unroll
        for (int r = 0; r < Rows; ++r) {
            if (lane == 0) {
                merged_stats[warp][r] = make_float2(row_top[r], row_sum[r]);
            }
#pragma unroll
            for (int j = 0; j < kElems; ++j) {
                merged_out[warp][r][element + j] = part[r][j];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * p.head_dim; i += kThreads) {
        const int r = i / p.head_dim;
        const int e = i - r * p.head_dim;
        float raised = merged_stats[0][r].x;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            raised = fmaxf(raised, merged_stats[w][r].x);
        }
        const float stand = raised == -INFINITY ? 0.0F : raised;
        float total = 0.0F, value = 0.0F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float factor = exp2f(merged_stats[w][r].x - stand);
            total = fmaf(factor, merged_stats[w][r].y, total);
            value = fmaf(factor, merged_out[w][r][e], value);
        }
        const int query = r / heads;
        const int head = head0 + r - query * heads;
        const long long row = s.q_first + query;
        if (p.splits > 1) {
            const long long at = (static_cast<long long>(split) * p.q_tokens + row) * p.q_heads +
                                 head;
            p.part_out[at * p.head_dim + e] = value;
            if (e == 0) {
                p.part_stats[at] = make_float2(raised, total);
            }
        } else {
            value = total == 0.0F ? 0.0F : value / total;
            static_cast<float*>(p.out)[row * p.out_stride +
                                       static_cast<long long>(head) * p.head_dim + e] = value;
        }
    }
}

// One block per (query row, head): its warps take every fourth split, lanes every 32nd element,
// and the warps' sums are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const VarlenParams p) {
    __shared__ float sums[kWarps][128];
    dev::grid_dependency_wait(); // the parts
    dev::grid_launch_dependents();
    const long long row = blockIdx.x / p.q_heads;
    const int head = static_cast<int>(blockIdx.x - row * p.q_heads);
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    // Rows outside every sequence stay as they were.
    if (row < clamped_offset(p.q_offsets, 0, p.q_tokens) ||
        row >= clamped_offset(p.q_offsets, p.batch, p.q_tokens)) {
        return; // the whole block
    }
    const long long pitch = static_cast<long long>(p.q_tokens) * p.q_heads;
    const float2* const stats = p.part_stats + row * p.q_heads + head;
    constexpr int kEach = kMaxSplits / 32; // splits' statistics per lane
    static_assert(kMaxSplits % 32 == 0, "whole statistics per lane");
    __shared__ float factors[kWarps][kMaxSplits];
    float2 stat[kEach];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = lane + 32 * i;
        stat[i] = at < p.splits ? stats[at * pitch] : make_float2(-INFINITY, 0.0F);
        top = fmaxf(top, stat[i].x);
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, offset));
    }
    const float stand = top == -INFINITY ? 0.0F : top;
    float total = 0.0F;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const float factor = exp2f(stat[i].x - stand);
        total = fmaf(factor, stat[i].y, total);
        factors[warp][lane + 32 * i] = factor;
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, offset);
    }
    __syncwarp();
    // Lane's elements: 4 lane .. + 3 as one vector, or lane, lane + 32, ... where rows are not whole
    // vectors. Eight splits' loads are in flight at a time.
    const float* const parts = p.part_out + (row * p.q_heads + head) * p.head_dim;
    const bool vector = p.head_dim % 4 == 0;
    constexpr int kBatch = 8;
    float value[4] = {};
#pragma unroll 1
    for (int first = 0; first < p.splits; first += kBatch * kWarps) {
        float4 loaded[kBatch];
        float weight[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = first + warp + kWarps * i;
            weight[i] = at < p.splits ? factors[warp][at] : 0.0F;
            loaded[i] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
            if (at < p.splits) {
                const float* const from = parts + at * pitch * p.head_dim;
                if (vector) {
                    if (4 * lane < p.head_dim) {
                        loaded[i] = reinterpret_cast<const float4*>(from)[lane];
                    }
                } else {
                    loaded[i].x = lane < p.head_dim ? from[lane] : 0.0F;
                    loaded[i].y = lane + 32 < p.head_dim ? from[lane + 32] : 0.0F;
                    loaded[i].z = lane + 64 < p.head_dim ? from[lane + 64] : 0.0F;
                    loaded[i].w = lane + 96 < p.head_dim ? from[lane + 96] : 0.0F;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (first + warp + kWarps * i < p.splits) { // a weight past the end is a NaN's at worst
                value[0] = fmaf(weight[i], loaded[i].x, value[0]);
                value[1] = fmaf(weight[i], loaded[i].y, value[1]);
                value[2] = fmaf(weight[i], loaded[i].z, value[2]);
                value[3] = fmaf(weight[i], loaded[i].w, value[3]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = vector ? 4 * lane + j : lane + 32 * j;
        sums[warp][e] = value[j];
    }
    __syncthreads();
    const int e = threadIdx.x;
    if (e < p.head_dim) {
        float sum = sums[0][e];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            sum += sums[w][e];
        }
        sum = total == 0.0F ? 0.0F : sum / total;
        T* const out = static_cast<T*>(p.out) + row * p.out_stride +
                       static_cast<long long>(head) * p.head_dim + e;
        if constexpr (sizeof(T) == 2) {
            *out = __float2bfloat16_rn(sum);
        } else {
            *out = sum;
        }
    }
}

int queries_per_block(const VarlenParams& p) {
    const int rows = rows_kernel_rows(p);
    return rows > p.group ? rows / p.group : 1;
}

int head_chunks(const VarlenParams& p) {
    const int heads = rows_kernel_rows(p) / queries_per_block(p);
    return (p.group + heads - 1) / heads;
}

template <int Lanes>
int launch_lanes(const VarlenParams& p, unsigned blocks, cudaStream_t stream) {
    const auto start = [&](auto* kernel) {
        host::pdl_launch(kernel, dim3(blocks), dim3(kThreads), 0, stream, p, queries_per_block(p),
                         head_chunks(p));
        return host::after_launch("attention_rows_kernel");
    };
    switch (rows_kernel_rows(p)) {
    case 1:
        return start(&attention_rows_kernel<Lanes, 1>);
    case 2:
        return start(&attention_rows_kernel<Lanes, 2>);
    case 4:
        return start(&attention_rows_kernel<Lanes, 4>);
    default:
        return start(&attention_rows_kernel<Lanes, 8>);
    }
}

} // namespace

// Rows of one key head taken together: for floats as many as an average sequence has, up to
// kMaxRows; the bfloat16 kernel's products have place for eight.
int rows_kernel_rows(const VarlenParams& p) {
    const long long queries = (p.q_tokens + static_cast<long long>(p.batch) - 1) / p.batch;
    int rows = p.bf16 ? kMaxRows : 1;
    while (rows < kMaxRows && rows < queries * p.group) {
        rows *= 2;
    }
    return rows;
}

long long rows_kernel_items(const VarlenParams& p) {
    return (p.q_tokens / queries_per_block(p) + static_cast<long long>(p.batch)) * p.kv_heads *
           head_chunks(p);
}

// 16-byte rows of q, k and v heads, at distances whose 16-fold fits 31 bits, and on average no more
// rows than the kernels take at once, or one query a sequence, whose heads are then taken eight at a
// time. The kernels for many rows read the keys once for each query head, these once for eight rows:
// 16 sequences of 2000 keys, one query, heads of 128, bfloat16 (float): 16 heads over 2 key heads 16 us
// (28) against 59 (325), over one 16 (28) against 60 (325); 256 of 197 keys, 12 heads of 64, 8 queries
// 40 (119) against 101 (293). With 16 queries the former take 102.
bool rows_kernel_takes(const VarlenParams& p) {
    const int size = p.bf16 ? 2 : 4;
    const auto fits = [size](const void* base, long long stride) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride * size % 16 == 0 &&
               stride < (1LL << 26);
    };
    const bool few = p.q_tokens <= p.batch ||
                     static_cast<long long>(p.q_tokens) * p.group <=
                         static_cast<long long>(kMaxRows) * p.batch;
    return few && p.head_dim * size % 16 == 0 && fits(p.q, p.q_stride) &&
           fits(p.k, p.k_stride) && fits(p.v, p.v_stride);
}

int launch_rows(const VarlenParams& p, cudaStream_t stream) {
    const long long blocks = rows_kernel_items(p) * p.splits;
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "attention launch exceeds the CUDA grid limit");
    }
    const unsigned count = static_cast<unsigned>(blocks);
    if (p.bf16) {
        return launch_few(p, queries_per_block(p), head_chunks(p), count, stream);
    }
    const int chunks = p.head_dim / kElems;
    if (chunks <= 4) {
        return launch_lanes<4>(p, count, stream);
    }
    if (chunks <= 8) {
        return launch_lanes<8>(p, count, stream);
    }
    return chunks <= 16 ? launch_lanes<16>(p, count, stream) : launch_lanes<32>(p, count, stream);
}

int launch_join(const VarlenParams& p, cudaStream_t stream) {
    const long long blocks = static_cast<long long>(p.q_tokens) * p.q_heads;
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "attention launch exceeds the CUDA grid limit");
    }
    // Always a dependent launch: the kernel before it is this call's own, which lets its
    // dependents start early, and the join waits for its end before reading the parts.
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config,
                       p.bf16 ? &attention_join_kernel<__nv_bfloat16>
                              : &attention_join_kernel<float>,
                       p);
    return host::after_launch("attention_join_kernel");
}

} // namespace cuvit::attn
