// Packed sequences: which rows a block of query rows stands for. Offsets come from the device
// and are clamped into the packed matrix here, so that wrong ones cannot lead outside it.
#pragma once

#include <cuda_runtime.h>

namespace cuvit::attn {

struct Sequence {
    int index; // -1: the block has no rows
    int q_begin, q_end; // the sequence's query rows
    int q_first;        // the block's first query row
    int kv_begin, kv_end;
};

__device__ __forceinline__ int clamped_offset(const int* offsets, int i, int limit) {
    return min(max(__ldg(offsets + i), 0), limit);
}

// Block b of the sequences' query rows cut into blocks of `rows`. Sequence s owns the blocks from
// q_offsets[s] / rows + s on: never fewer than it needs, since ceil(n / r) is at most
// floor((o + n) / r) - floor(o / r) + 1, and never past q_tokens / rows + batch, so the launch
// knows a bound for the blocks without knowing the lengths, and a block finds its sequence by
// binary search without a table of block counts.
__device__ __forceinline__ Sequence find_block(const int* q_offsets, const int* kv_offsets,
                                               int batch, int q_tokens, int kv_tokens,
                                               long long block, int rows) {
    int low = 0;
    int high = batch; // the largest s in [0, batch) whose blocks start at or before this one
    while (high - low > 1) {
        const int middle = low + (high - low) / 2;
        const long long start = clamped_offset(q_offsets, middle, q_tokens) / rows +
                                static_cast<long long>(middle);
        if (start <= block) {
            low = middle;
        } else {
            high = middle;
        }
    }
    Sequence s;
    s.index = -1;
    s.q_begin = clamped_offset(q_offsets, low, q_tokens);
    s.q_end = max(clamped_offset(q_offsets, low + 1, q_tokens), s.q_begin);
    s.kv_begin = clamped_offset(kv_offsets, low, kv_tokens);
    s.kv_end = max(clamped_offset(kv_offsets, low + 1, kv_tokens), s.kv_begin);
    const long long local = block - (s.q_begin / rows + static_cast<long long>(low));
    const long long first = s.q_begin + local * rows;
    s.q_first = 0;
    if (local >= 0 && first < s.q_end) {
        s.index = low;
        s.q_first = static_cast<int>(first);
    }
    return s;
}

// find_block by a whole warp: 32 pivots at a time instead of one, so two rounds of loads find one of
// 1024 sequences.
__device__ __forceinline__ Sequence find_block_warp(const int* q_offsets, const int* kv_offsets,
                                                    int batch, int q_tokens, int kv_tokens,
                                                    long long block, int rows) {
    const int lane = threadIdx.x % 32;
    int low = 0;
    int count = batch; // the sequence is one of [low, low + count)
    while (count > 1) {
        const int step = (count + 31) / 32;
        const int pivot = low + lane * step;
        bool before = lane == 0;
        if (lane > 0 && lane * step < count) {
            before = clamped_offset(q_offsets, pivot, q_tokens) / rows +
                         static_cast<long long>(pivot) <=
                     block;
        }
        const unsigned starts = __ballot_sync(0xFFFFFFFFu, before);
        const int last = 31 - __clz(starts); // starts hold for a run of lanes from 0 on
        low += last * step;
        count = min(step, count - last * step);
    }
    Sequence s;
    s.index = -1;
    s.q_begin = clamped_offset(q_offsets, low, q_tokens);
    s.q_end = max(clamped_offset(q_offsets, low + 1, q_tokens), s.q_begin);
    s.kv_begin = clamped_offset(kv_offsets, low, kv_tokens);
    s.kv_end = max(clamped_offset(kv_offsets, low + 1, kv_tokens), s.kv_begin);
    const long long local = block - (s.q_begin / rows + static_cast<long long>(low));
    const long long first = s.q_begin + local * rows;
    s.q_first = 0;
    if (local >= 0 && first < s.q_end) {
        s.index = low;
        s.q_first = static_cast<int>(first);
    }
    return s;
}

// The keys [first, end) of a sequence's `keys` that split i of n goes through.
__device__ __forceinline__ void split_keys(int keys, int i, int n, int& first, int& end) {
    const int each = (keys + n - 1) / n;
    first = static_cast<int>(min(static_cast<long long>(keys), static_cast<long long>(i) * each));
    end = min(keys, first + each);
}

} // namespace cuvit::attn
