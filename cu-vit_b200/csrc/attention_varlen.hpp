// Attention over packed sequences: the checked problem its kernels share.
#pragma once

#include "cuvit_b200.h"
#include "runtime.hpp"

#include <cuda_runtime.h>

namespace cuvit::attn {

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
    float scale_log2; // scale * log2(e): weights are powers of two of (scores - maximum)
    long long q_stride;
    long long k_stride;
    long long v_stride;
    long long out_stride;
};

} // namespace cuvit::attn
