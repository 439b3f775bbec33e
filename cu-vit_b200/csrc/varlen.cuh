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

// Sequence i's rows; no block yet.
__device__ __forceinline__ Sequence sequence_of(const int* q_offsets, const int* kv_offsets,
                                                int q_tokens, int kv_tokens, int i) {
    Sequence s;
    s.index = -1;
    s.q_begin = clamped_offset(q_offsets, i, q_tokens);
    s.q_end = max(clamped_offset(q_offsets, i + 1, q_tokens), s.q_begin);
    s.q_first = 0;
    s.kv_begin = clamped_offset(kv_offsets, i, kv_tokens);
    s.kv_end = max(clamped_offset(kv_offsets, i + 1, kv_tokens), s.kv_begin);
    return s;
}

// Block `block` if it is sequence i's, whose blocks start at q_offsets[i] / rows + i.
__device__ __forceinline__ Sequence block_of(const int* q_offsets, const int* kv_offsets,
                                             int q_tokens, int kv_tokens, int i, long long block,
                                             int rows) {
    Sequence s = sequence_of(q_offsets, kv_offsets, q_tokens, kv_tokens, i);
    const long long local = block - (s.q_begin / rows + static_cast<long long>(i));
    const long long first = s.q_begin + local * rows;
    if (local >= 0 && first < s.q_end) {
        s.index = i;
        s.q_first = static_cast<int>(first);
    }
    return s;
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
    return block_of(q_offsets, kv_offsets, q_tokens, kv_tokens, low, block, rows);
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
    return block_of(q_offsets, kv_offsets, q_tokens, kv_tokens, low, block, rows);
}

// Up to 32 sequences in the order of their work, most first: lane i holds the i-th and where its
// blocks start. Handing out long sequences first leaves only short ones for the end of a launch.
struct Order {
    int sequence;
    long long start;
};

__device__ __forceinline__ Order order_sequences(const int* q_offsets, const int* kv_offsets,
                                                 int batch, int q_tokens, int kv_tokens, int rows) {
    const int lane = threadIdx.x % 32;
    int queries = 0;
    int keys = -1; // past the last sequence
    if (lane < batch) {
        const int q = clamped_offset(q_offsets, lane, q_tokens);
        const int k = clamped_offset(kv_offsets, lane, kv_tokens);
        queries = max(clamped_offset(q_offsets, lane + 1, q_tokens) - q, 0);
        keys = max(clamped_offset(kv_offsets, lane + 1, kv_tokens) - k, 0);
    }
    // A sequence's place, then the sequence of this lane's place.
    int place = 0;
    for (int i = 0; i < 32; ++i) {
        const int other = __shfl_sync(0xFFFFFFFFu, keys, i);
        place += other > keys || (other == keys && i < lane) ? 1 : 0;
    }
    Order order{};
    for (int i = 0; i < 32; ++i) {
        order.sequence = __shfl_sync(0xFFFFFFFFu, place, i) == lane ? i : order.sequence;
    }
    const int own = __shfl_sync(0xFFFFFFFFu, queries, order.sequence);
    const long long blocks = (own + static_cast<long long>(rows) - 1) / rows;
    long long end = blocks;
    for (int distance = 1; distance < 32; distance *= 2) {
        const long long before = __shfl_up_sync(0xFFFFFFFFu, end, distance);
        end += lane >= distance ? before : 0;
    }
    order.start = end - blocks;
    return order;
}

// Block `block` of the sequences in that order, a sequence's last rows first where `last_first`.
__device__ __forceinline__ Sequence find_ordered_block(const Order& order, const int* q_offsets,
                                                       const int* kv_offsets, int batch,
                                                       int q_tokens, int kv_tokens,
                                                       long long block, int rows,
                                                       bool last_first) {
    const unsigned starts = __ballot_sync(0xFFFFFFFFu, order.start <= block);
    const int place = 31 - __clz(starts);
    // Sequences without queries share the next one's start: the last of them is meant.
    const int sequence = __shfl_sync(0xFFFFFFFFu, order.sequence, place);
    long long local = block - __shfl_sync(0xFFFFFFFFu, order.start, place);
    if (sequence >= batch) { // past the last block: a lane without a sequence
        Sequence none{};
        none.index = -1;
        return none;
    }
    Sequence s = sequence_of(q_offsets, kv_offsets, q_tokens, kv_tokens, sequence);
    const long long blocks = (s.q_end - s.q_begin + static_cast<long long>(rows) - 1) / rows;
    if (local < blocks) {
        local = last_first ? blocks - 1 - local : local;
        s.index = sequence;
        s.q_first = static_cast<int>(s.q_begin + local * rows);
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
