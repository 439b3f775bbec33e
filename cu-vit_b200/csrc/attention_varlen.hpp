// Attention over packed sequences: the checked problem its kernels share, and what a call that
// splits its keys leaves for the kernel that joins the parts.
#pragma once

#include "cuvit_b200.h"
#include "runtime.hpp"

#include <cuda_runtime.h>

namespace cuvit::attn {

constexpr int kMaxSplits = 64;

// Rows are heads * head_dim elements, strides in elements, defaults resolved.
struct VarlenParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int* q_offsets;
    const int* kv_offsets;
    int batch;
    int q_tokens;
    int kv_tokens;
    int q_heads;
    int kv_heads;
    int group; // query heads per key head
    int head_dim;
    int causal;
    int bf16;
    float scale_log2; // scale * log2(e): weights are powers of two of (scores - maximum)
    long long q_stride;
    long long k_stride;
    long long v_stride;
    long long out_stride;
    // Splits of every sequence's keys. With more than one, split i of query row t, head h
    // leaves its weighted sum of values, not yet divided by the sum of weights, at
    // part_out[((i * q_tokens + t) * q_heads + h) * head_dim] and its maximum (times scale_log2)
    // and sum of weights at part_stats[(i * q_tokens + t) * q_heads + h].
    int splits;
    float* part_out;
    float2* part_stats;
};

// Few query rows per sequence (attention_few.cu for bfloat16, attention_rows.cu for float): one pass
// over the keys for up to kMaxRows rows (queries times the heads that share a key head) at a time.
constexpr int kMaxRows = 8;
bool rows_kernel_takes(const VarlenParams& p);
int rows_kernel_rows(const VarlenParams& p);
long long rows_kernel_items(const VarlenParams& p); // blocks of a launch per split
int launch_rows(const VarlenParams& p, cudaStream_t stream);
int launch_few(const VarlenParams& p, int queries_per_block, int head_chunks, unsigned blocks,
               cudaStream_t stream);

// bfloat16 on the tensor cores (attention_tiles.cu).
bool tiles_kernel_takes(const VarlenParams& p);
long long tiles_kernel_items(const VarlenParams& p); // work items per split
int launch_tiles(const VarlenParams& p, cudaStream_t stream);

// Floats on the tensor cores, any alignment (attention_split.cu).
long long split_kernel_items(const VarlenParams& p); // blocks of a launch per split
int launch_split(const VarlenParams& p, unsigned* status, cudaStream_t stream);

// Joins the splits: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
int launch_join(const VarlenParams& p, cudaStream_t stream);

} // namespace cuvit::attn
