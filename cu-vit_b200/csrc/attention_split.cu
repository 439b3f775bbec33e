// Packed attention of floats on the tensor cores (tcgen05): both products as three of TF32 halves
// (split_tf32.cuh), softmax in FP32, one pass over the keys.
//
// A CTA has 128 query rows of one head and goes through tiles of 64 keys (32 for heads wider than
// 64, which leave tensor memory no room for more). Q's halves stay in tensor memory, scores come
// into one of two buffers there, weights go back as halves, and a tile's weighted values are added
// to registers, so no accumulator sums more than 64 products or a head's width.
//
// 4096 tokens, 8 heads of 64: 285 us, 121 TFLOP/s (products in the FP32 pipe: 954 us); heads of 128
// 665 us; 8 x 197 tokens, 12 heads 35 us (78). The tensor core would allow three times that (its
// products take 1540 cycles of the 4600 a tile of 64 keys and 64 elements takes): what bounds it is
// the softmax warps' chain of waits (scores, maximum, exponentials, previous sum, weights), and a
// quarter is the loading warps' share of the issue slots. A second set of softmax warps on alternate
// tiles would need more registers than an SM has.
//
//   first 8 (wide heads: 16) warps   softmax: two (four) threads per row, each with its part of a
//                tile's keys; they exchange the row's maximum through shared memory, and each keeps
//                its part of the output row
//   next 8       bring keys and values in (each thread its own pieces, several tiles ahead, without
//                any wait for one another), split them, and lay them out for the tensor core:
//                keys as they are, values transposed
//   last warp    issues the products: S(0), S(1), PV(0), S(2), PV(1), ...
#include "attention_varlen.hpp"
#include "ptx.cuh"
#include "split_tf32.cuh"
#include "varlen.cuh"

#include <cstdint>

namespace cuvit::attn {
namespace {

constexpr int kRows = 128;
constexpr int kMaxParts = 4;
// A tile is 1024 16-byte pieces (64 keys of 64 or 32 of 128), four to a place.
constexpr int kPieces = 4;
constexpr int kPlaces = 256;
constexpr int kGroup = 16; // columns of a tensor-memory access

constexpr int kHalfBytes = 16384; // a tile's hi or lo
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr int kTiles = 4; // split tiles: the tensor core works on one, up to three wait
constexpr int kRaw = 4;   // tiles being fetched
constexpr int kRawBytes = kPlaces * kPieces * 16;
constexpr int kRawOffset = kTiles * kTileBytes;
constexpr int kTopOffset = kRawOffset + kRaw * kRawBytes; // [2][parts][kRows] floats
constexpr int kBarrierOffset = kTopOffset + 2 * kMaxParts * kRows * 4;
constexpr int kBarriers = 2 * kTiles + 1 + 4 + 2 + 4 + 1;
constexpr int kSmemBytes = 1024 + kBarrierOffset + 8 * kBarriers + 8;
static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
constexpr int kTmemColumns = 512;

template <bool Wide> // heads of 65 to 128
struct Shape {
    static constexpr int kKeys = Wide ? 32 : 64;
    // Threads of a row. Narrow heads' fit 96 registers with two (four, with 72: 369 us against 320 for
    // 4096 tokens, 8 heads of 64), wide ones spill with two (760 us against 659 for heads of 128).
    static constexpr int kParts = Wide ? 4 : 2;
    static constexpr int kSoftmaxWarps = 4 * kParts;
    static constexpr int kOwn = kKeys / kParts; // keys of a softmax thread
    static constexpr int kGroups = 2;           // 16-column groups of its part of the output
    static constexpr int kQ = 0;                   // hi, then lo
    static constexpr int kWidth = Wide ? 128 : 64; // of Q's halves and of the output
    static constexpr int kS = 2 * kWidth;          // two buffers
    static constexpr int kP = kS + 2 * kKeys;      // hi, then lo
    static constexpr int kO = kP + 2 * kKeys;
    static_assert(kO + kWidth <= kTmemColumns, "tensor memory");
    static constexpr int kLoadWarps = 8;
    static constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
    static constexpr int kThreads = 32 * (kMmaWarp + 1);
    static constexpr int kLoaders = 32 * kLoadWarps;
    static constexpr int kSets = kPlaces / kLoaders; // places of a loading thread
};

struct Flags {
    int in_vector;  // rows of q, k and v are whole aligned 16-byte vectors
    int out_vector; // rows of the output (or of the parts)
};

// The key or value tile at position i of the order they are used in: K0, K1, V0, K2, V1, ...
struct Tile {
    bool value;
    int index;
};

__device__ __forceinline__ Tile tile_at(int i, int tiles) {
    if (i == 0) {
        return {false, 0};
    }
    if (i == 2 * tiles - 1) {
        return {true, tiles - 1};
    }
    return i % 2 == 1 ? Tile{false, (i + 1) / 2} : Tile{true, i / 2 - 1};
}

template <int Bytes>
__device__ __forceinline__ void copy_async(uint32_t to, const float* from, bool live) {
    if constexpr (Bytes == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from),
                     "r"(live ? 16 : 0)
                     : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from),
                     "r"(live ? 4 : 0)
                     : "memory");
    }
}

template <bool Wide>
__global__ void __launch_bounds__(Shape<Wide>::kThreads, 1)
    attention_split_kernel(const __grid_constant__ VarlenParams p, const Flags flags,
                           unsigned* status) {
    using S = Shape<Wide>;
    constexpr int kKeys = S::kKeys;
    constexpr int kLoaders = S::kLoaders;
    constexpr int kSets = S::kSets;
    constexpr int kMmaWarp = S::kMmaWarp;
    constexpr int kParts = S::kParts;
    constexpr int kSoftmaxWarps = S::kSoftmaxWarps;
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    // Causal: a sequence's last rows, which see most keys, first.
    const int index = static_cast<int>(p.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    const int item = index / p.splits;
    const int split = index - item * p.splits;
    const int block = item / p.q_heads;
    const int head = item - block * p.q_heads;
    const Sequence s = find_block_warp(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                       block, kRows);
    if (s.index < 0) {
        return; // the whole block
    }
    const int rows = min(kRows, s.q_end - s.q_first);
    const int keys = s.kv_end - s.kv_begin;
    // Query row r of this block sees keys j <= r + reach.
    const long long reach =
        static_cast<long long>(s.q_first - s.q_begin) + keys - (s.q_end - s.q_begin);
    int first_key, last_key;
    split_keys(keys, split, p.splits, first_key, last_key);
    if (p.causal) {
        last_key = static_cast<int>(min(static_cast<long long>(last_key), max(0LL, reach + rows)));
    }
    const int tiles = last_key > first_key ? (last_key - first_key + kKeys - 1) / kKeys : 0;
    const int d = p.head_dim;
    const int padded = (d + 15) / 16 * 16;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = dev::smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_base);
    const uint32_t bars = base + kBarrierOffset;
    const auto tile_full = [&](int i) -> uint32_t { return bars + 8u * i; };
    const auto tile_empty = [&](int i) -> uint32_t { return bars + 8u * (kTiles + i); };
    const uint32_t q_full = bars + 8u * (2 * kTiles);
    const auto s_full = [&](int i) -> uint32_t { return bars + 8u * (2 * kTiles + 1 + i); };
    const auto s_empty = [&](int i) -> uint32_t { return bars + 8u * (2 * kTiles + 3 + i); };
    const uint32_t p_full = bars + 8u * (2 * kTiles + 5);
    const uint32_t o_full = bars + 8u * (2 * kTiles + 6);
    const auto row_bar = [&](int i) -> uint32_t { return bars + 8u * (2 * kTiles + 7 + i); };
    const uint32_t drain_bar = bars + 8u * (2 * kTiles + 11);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarrierOffset + 8 * kBarriers);
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kTiles; ++i) {
            dev::mbar_init(tile_full(i), S::kLoadWarps);
            dev::mbar_init(tile_empty(i), 1);
        }
        dev::mbar_init(q_full, kSoftmaxWarps);
        for (int i = 0; i < 2; ++i) {
            dev::mbar_init(s_full(i), 1);
            dev::mbar_init(s_empty(i), kSoftmaxWarps);
        }
        dev::mbar_init(p_full, kSoftmaxWarps);
        dev::mbar_init(o_full, 1);
        for (int i = 0; i < 4; ++i) {
            dev::mbar_init(row_bar(i), kParts); // the warps of a quarter of the rows
        }
        dev::mbar_init(drain_bar, 1);
        dev::fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        dev::tmem_alloc(dev::smem_u32(tmem_slot), kTmemColumns);
        dev::tmem_relinquish();
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < kSoftmaxWarps) {
        // ---------------- softmax ----------------
        const int quarter = warp & 3;
        const int part = warp >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t mine = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        // This thread's 16-column groups of Q and of the output.
        const int group0 = part * S::kGroups;
        const int count = min(S::kGroups, max(0, padded / kGroup - group0));
        float* const tops = reinterpret_cast<float*>(smem + kTopOffset);

        const float* const q = static_cast<const float*>(p.q) + (s.q_first + row) * p.q_stride +
                               static_cast<long long>(head) * d;
#pragma unroll 1
        for (int g = group0; g < group0 + count && tiles > 0; ++g) {
            float x[4][4], hi[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int e = g * kGroup + 4 * c;
                if (flags.in_vector) {
                    const float4 four = row < rows && e < d
                                            ? __ldg(reinterpret_cast<const float4*>(q + e))
                                            : make_float4(0.0F, 0.0F, 0.0F, 0.0F);
                    x[c][0] = four.x;
                    x[c][1] = four.y;
                    x[c][2] = four.z;
                    x[c][3] = four.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[c][j] = row < rows && e + j < d ? __ldg(q + e + j) : 0.0F;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[c][j] *= p.scale_log2;
                }
            }
            // Once per block: always in the checked form.
            float lo[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                dev::split4_checked(x[c], hi[c], lo[c]);
            }
            __syncwarp(); // tensor-memory accesses are warp-wide
            dev::tmem_store_floats(mine + S::kQ + g * kGroup, hi);
            dev::tmem_store_floats(mine + S::kQ + S::kWidth + g * kGroup, lo);
        }
        dev::tmem_wait_store();
        dev::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            dev::mbar_arrive(q_full);
        }

        float o[S::kGroups][kGroup];
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
#pragma unroll
            for (int j = 0; j < kGroup; ++j) {
                o[g][j] = 0.0F;
            }
        }
        float maximum = -INFINITY; // of the row, times scale and log2 e
        float sum = 0.0F;          // of this thread's weights
        float pending = 1.0F;      // what o is to be multiplied by
        uint32_t row_phase = 0, o_phase = 0;
        // Hands this thread's value of the row to the others; `all` are in their order.
        const auto exchange = [&](int buffer, float value, float (&all)[kParts]) -> bool {
            float* const at = tops + buffer * kParts * kRows + row;
            at[part * kRows] = value;
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(row_bar(quarter));
            }
            const bool done = dev::mbar_wait_warp(row_bar(quarter), row_phase, status);
            row_phase ^= 1u;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                all[i] = at[i * kRows];
            }
            return done;
        };
        const auto drain = [&]() -> bool {
            if (!dev::mbar_wait_warp(o_full, o_phase, status)) {
                return false;
            }
            o_phase ^= 1u;
            dev::tc_fence_after();
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
                if (g < count) { // warp-uniform
                    uint32_t part[kGroup];
                    dev::tmem_load_16(mine + S::kO + (group0 + g) * kGroup, part);
                    dev::tmem_wait_load_of(part);
#pragma unroll
                    for (int j = 0; j < kGroup; ++j) {
                        o[g][j] = fmaf(o[g][j], pending, __uint_as_float(part[j]));
                    }
                }
            }
            dev::tc_fence_before();
            return true;
        };
        // The end of the keys that the row sees, less this thread's place in a tile.
        const int seen =
            (p.causal ? static_cast<int>(
                            min(static_cast<long long>(last_key), max(0LL, reach + row + 1)))
                      : last_key) -
            part * S::kOwn;
        bool ok = true;
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile) {
            const int buffer = tile & 1;
            if (!dev::mbar_wait_warp(s_full(buffer), (tile >> 1) & 1, status)) {
                ok = false;
                break;
            }
            dev::tc_fence_after();
            float w[S::kOwn / 4][4];
            const uint32_t scores = mine + S::kS + buffer * kKeys + part * S::kOwn;
            constexpr int kRead = S::kOwn < kGroup ? S::kOwn : kGroup;
#pragma unroll
            for (int g = 0; g < S::kOwn / kRead; ++g) {
                uint32_t raw[kRead];
                if constexpr (kRead == 16) {
                    dev::tmem_load_16(scores + g * kRead, raw);
                } else {
                    dev::tmem_load_8(scores, raw);
                }
                dev::tmem_wait_load_of(raw);
#pragma unroll
                for (int j = 0; j < kRead; ++j) {
                    w[(g * kRead + j) / 4][j % 4] = __uint_as_float(raw[j]);
                }
            }
            dev::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(s_empty(buffer));
            }
            const int first = first_key + tile * kKeys;
            const int limit = seen - first; // of these keys
            if (__any_sync(0xFFFFFFFFu, limit < S::kOwn)) {
#pragma unroll
                for (int i = 0; i < S::kOwn; ++i) {
                    w[i / 4][i % 4] = i < limit ? w[i / 4][i % 4] : -INFINITY;
                }
            }
            float top = w[0][0];
#pragma unroll
            for (int i = 1; i + 1 < S::kOwn; i += 2) {
                top = dev::max3(top, w[i / 4][i % 4], w[(i + 1) / 4][(i + 1) % 4]);
            }
            top = fmaxf(top, w[S::kOwn / 4 - 1][3]);
            float all[kParts];
            ok = exchange(buffer, top, all);
            if (!ok) {
                break;
            }
            float raised = maximum;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                raised = fmaxf(raised, all[i]);
            }
            // A row without a key so far: any finite stand-in keeps 2^(-inf - m) at zero.
            const float stand = raised == -INFINITY ? 0.0F : raised;
            const float factor = dev::ex2_approx(maximum - stand);
            maximum = raised;
            float partial[4] = {};
#pragma unroll
            for (int i = 0; i < S::kOwn; ++i) {
                w[i / 4][i % 4] = dev::ex2_approx(w[i / 4][i % 4] - stand);
                partial[i % 4] += w[i / 4][i % 4];
            }
            sum = fmaf(sum, factor, (partial[0] + partial[1]) + (partial[2] + partial[3]));
            // The previous weights' products are done: their sum is taken and their place free.
            if (tile > 0 && !drain()) {
                ok = false;
                break;
            }
            pending = factor;
            uint64_t check = 0u; // weights are at most 1, or NaN, which lo keeps
#pragma unroll
            for (int c = 0; c < S::kOwn / 4; c += 2) {
                float hi[2][4];
                dev::split4(w[c], hi[0], check);
                dev::split4(w[c + 1], hi[1], check);
                const uint32_t to = mine + S::kP + part * S::kOwn + 4 * c;
                dev::tmem_store_8(to, hi[0], hi[1]);
                dev::tmem_store_8(to + kKeys, w[c], w[c + 1]);
            }
            dev::tmem_wait_store();
            dev::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(p_full);
            }
        }
        if (ok && tiles > 0) {
            ok = drain();
        }
        if (ok) {
            float all[kParts];
            ok = exchange(tiles & 1, sum, all);
            sum = 0.0F;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                sum += all[i];
            }
        }
        if (ok && row < rows) {
            float* to;
            float inverse = 1.0F;
            if (p.splits > 1) {
                const long long at =
                    (static_cast<long long>(split) * p.q_tokens + s.q_first + row) * p.q_heads +
                    head;
                to = p.part_out + at * d;
                if (part == 0) {
                    p.part_stats[at] = make_float2(maximum, sum);
                }
            } else {
                to = static_cast<float*>(p.out) + (s.q_first + row) * p.out_stride +
                     static_cast<long long>(head) * d;
                inverse = sum == 0.0F ? 0.0F : 1.0F / sum;
            }
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int e = (group0 + g) * kGroup + 4 * c;
                    if (g >= count || e >= d) {
                        continue;
                    }
                    const float four[4] = {o[g][4 * c] * inverse, o[g][4 * c + 1] * inverse,
                                           o[g][4 * c + 2] * inverse, o[g][4 * c + 3] * inverse};
                    if (flags.out_vector) {
                        *reinterpret_cast<float4*>(to + e) =
                            make_float4(four[0], four[1], four[2], four[3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (e + j < d) {
                                to[e + j] = four[j];
                            }
                        }
                    }
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ---------------- keys and values ----------------
        const int t = threadIdx.x - 32 * kSoftmaxWarps;
        const int pieces = padded / 4; // of a row
        const float* const k = static_cast<const float*>(p.k) + s.kv_begin * p.k_stride +
                               static_cast<long long>(head / p.group) * d;
        const float* const v = static_cast<const float*>(p.v) + s.kv_begin * p.v_stride +
                               static_cast<long long>(head / p.group) * d;
        // Keys: piece t + 256 u of the tile, row-major. Values: a block of four keys by four
        // elements, eight lanes on consecutive key blocks, so that both the loads (a sector a
        // row) and the transposed stores (eight different bank groups) are whole.
        int k_row[kSets][kPieces], k_element[kSets][kPieces];
        int v_row[kSets], v_element[kSets];
#pragma unroll
        for (int n = 0; n < kSets; ++n) {
            const int place = t + kLoaders * n;
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
                const int piece = place + kPlaces * u;
                k_row[n][u] = piece / pieces;
                k_element[n][u] = 4 * (piece - k_row[n][u] * pieces);
            }
            v_row[n] = 4 * (Wide ? place % 8 : place % 8 + 8 * (place / 8 % 2));
            v_element[n] = 4 * (Wide ? place / 8 : place / 16);
        }
        const uint32_t raw0 = base + kRawOffset + 16u * t;
        const auto fetch = [&](int i) {
            if (i >= 2 * tiles) {
                return;
            }
            const Tile tile = tile_at(i, tiles);
            const int first = first_key + tile.index * kKeys;
            const uint32_t to = raw0 + (i % kRaw) * kRawBytes;
            const float* const from = tile.value ? v : k;
            const long long stride = tile.value ? p.v_stride : p.k_stride;
#pragma unroll
            for (int n = 0; n < kSets; ++n) {
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    const int r = tile.value ? v_row[n] + u : k_row[n][u];
                    const int e = tile.value ? v_element[n] : k_element[n][u];
                    const bool live = r < kKeys && first + r < last_key && e < d;
                    const float* const at = live ? from + (first + r) * stride + e : from;
                    const uint32_t here = to + 16 * (u * kPlaces + n * kLoaders);
                    if (flags.in_vector) {
                        copy_async<16>(here, at, live);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool one = live && e + j < d;
                            copy_async<4>(here + 4 * j, one ? at + j : from, one);
                        }
                    }
                }
            }
        };
#pragma unroll
        for (int i = 0; i < kRaw - 1; ++i) {
            fetch(i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
#pragma unroll 1
        for (int i = 0; i < 2 * tiles; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRaw - 2) : "memory");
            const Tile tile = tile_at(i, tiles);
            const uint32_t from = raw0 + (i % kRaw) * kRawBytes;
            const int slot = i % kTiles;
            const uint32_t to = base + slot * kTileBytes;
            bool free = false;
#pragma unroll
            for (int n = 0; n < kSets; ++n) {
                float x[kPieces][4], hi[kPieces][4];
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    dev::ld_shared_v4(from + 16 * (u * kPlaces + n * kLoaders), x[u]);
                }
                uint64_t check = 0u;
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    dev::split4(x[u], hi[u], check);
                }
                if (dev::any_special(check)) {
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) {
                        float again[4]; // lo has taken x's place
                        dev::ld_shared_v4(from + 16 * (u * kPlaces + n * kLoaders), again);
                        dev::split4_checked(again, hi[u], x[u]);
                    }
                }
                if (n == 0) {
                    free = dev::mbar_wait_warp(tile_empty(slot), ((i / kTiles) & 1) ^ 1u, status);
                    if (!free) {
                        break;
                    }
                }
                if (tile.value) {
                    // Row e of the transposed tile: 32 keys are 128 bytes, swizzled.
                    if (v_element[n] < padded) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int e = v_element[n] + j;
                            const uint32_t at = to + (v_row[n] / 32) * padded * 128 + e * 128 +
                                                ((v_row[n] % 32 / 4 ^ (e & 7)) << 4);
                            const float h[4] = {hi[0][j], hi[1][j], hi[2][j], hi[3][j]};
                            const float l[4] = {x[0][j], x[1][j], x[2][j], x[3][j]};
                            dev::st_shared_v4(at, h);
                            dev::st_shared_v4(at + kHalfBytes, l);
                        }
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) {
                        const int r = k_row[n][u];
                        if (r < kKeys) {
                            const int e = k_element[n][u];
                            const uint32_t at = to + (e / 32) * kKeys * 128 + r * 128 +
                                                ((e % 32 / 4 ^ (r & 7)) << 4);
                            dev::st_shared_v4(at, hi[u]);
                            dev::st_shared_v4(at + kHalfBytes, x[u]);
                        }
                    }
                }
            }
            if (!free) {
                break;
            }
            fetch(i + kRaw - 1); // into the place read in the previous round
            asm volatile("cp.async.commit_group;" ::: "memory");
            dev::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(tile_full(slot));
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---------------- products: the warp stays together, one lane issues ----------------
        const uint32_t base0 = __shfl_sync(0xFFFFFFFFu, base, 0);
        const uint32_t tmem0 = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint32_t idesc_s = dev::make_idesc(2u, kRows, kKeys, false, false);
        const uint32_t idesc_o = dev::make_idesc(2u, kRows, padded, false, false);
        const int steps = padded / 8;
        bool ok = tiles == 0 || dev::mbar_wait_warp(q_full, 0, status);
        for (int i = 0; i < 2 * tiles && ok; ++i) {
            const Tile tile = tile_at(i, tiles);
            const int slot = i % kTiles;
            if (!dev::mbar_wait_warp(tile_full(slot), (i / kTiles) & 1, status)) {
                ok = false;
                break;
            }
            const uint32_t data = base0 + slot * kTileBytes;
            if (tile.value) {
                if (!dev::mbar_wait_warp(p_full, tile.index & 1, status)) {
                    ok = false;
                    break;
                }
                dev::tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < kKeys / 8; ++kk) {
                    const uint64_t hi = dev::smem_desc_sw128(
                        data + (kk / 4) * padded * 128 + kk % 4 * 32, 16, 1024);
                    const uint64_t lo = hi + kHalfBytes / 16;
                    const uint32_t w = tmem0 + S::kP + 8 * kk;
                    dev::mma_ts_tf32_warp(tmem0 + S::kO, w + kKeys, hi, idesc_o, kk > 0 ? 1u : 0u);
                    dev::mma_ts_tf32_warp(tmem0 + S::kO, w, lo, idesc_o, 1u);
                    dev::mma_ts_tf32_warp(tmem0 + S::kO, w, hi, idesc_o, 1u);
                }
                dev::tc_commit_warp(tile_empty(slot));
                dev::tc_commit_warp(o_full);
            } else {
                const int buffer = tile.index & 1;
                if (!dev::mbar_wait_warp(s_empty(buffer), ((tile.index >> 1) & 1) ^ 1u, status)) {
                    ok = false;
                    break;
                }
                dev::tc_fence_after();
                const uint32_t to = tmem0 + S::kS + buffer * kKeys;
#pragma unroll 2
                for (int kk = 0; kk < steps; ++kk) {
                    const uint64_t hi = dev::smem_desc_sw128(
                        data + (kk / 4) * kKeys * 128 + kk % 4 * 32, 16, 1024);
                    const uint64_t lo = hi + kHalfBytes / 16;
                    const uint32_t a = tmem0 + S::kQ + 8 * kk;
                    dev::mma_ts_tf32_warp(to, a + S::kWidth, hi, idesc_s, kk > 0 ? 1u : 0u);
                    dev::mma_ts_tf32_warp(to, a, lo, idesc_s, 1u);
                    dev::mma_ts_tf32_warp(to, a, hi, idesc_s, 1u);
                }
                dev::tc_commit_warp(tile_empty(slot));
                dev::tc_commit_warp(s_full(buffer));
            }
        }
        if (!ok) {
            // No product still reads or writes when the CTA ends.
            dev::tc_commit_warp(drain_bar);
            dev::mbar_drain_wait(drain_bar, 0);
        }
    }

    __syncwarp();
    dev::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        dev::tc_fence_after();
        dev::tmem_dealloc(tmem, kTmemColumns);
    }
}

} // namespace

long long split_kernel_items(const VarlenParams& p) {
    return (static_cast<long long>(p.q_tokens) / kRows + p.batch) * p.q_heads;
}

int launch_split(const VarlenParams& p, unsigned* status, cudaStream_t stream) {
    const auto whole = [](const void* base, long long stride) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride % 4 == 0;
    };
    Flags flags{};
    flags.in_vector = p.head_dim % 4 == 0 && whole(p.q, p.q_stride) && whole(p.k, p.k_stride) &&
                              whole(p.v, p.v_stride)
                          ? 1
                          : 0;
    flags.out_vector =
        p.head_dim % 4 == 0 && (p.splits > 1 || whole(p.out, p.out_stride)) ? 1 : 0;
    const long long blocks = split_kernel_items(p) * p.splits;
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "attention launch exceeds the CUDA grid limit");
    }
    const bool wide = p.head_dim > 64;
    auto* kernel = wide ? &attention_split_kernel<true> : &attention_split_kernel<false>;
    CUVIT_TRY_CUDA(host::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmemBytes));
    const int threads = wide ? Shape<true>::kThreads : Shape<false>::kThreads;
    host::pdl_launch(kernel, dim3(static_cast<unsigned>(blocks)),
                     dim3(static_cast<unsigned>(threads)), kSmemBytes, stream, p, flags, status);
    return host::after_launch("attention_split_kernel");
}

} // namespace cuvit::attn
