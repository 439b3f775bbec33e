// Attention over packed sequences on the tensor cores, bfloat16 operands.
//
//   S = Q K^T for 128 query rows and 128 keys at a time into tensor memory; P = 2^(S scale - m);
//   O += P V, with m and the sum of P kept per row.
//
// A CTA works on (256 query rows, head, split of the keys) items: its own block index, then those of
// blocks that have not started, which it takes over one by one (cluster launch control), so that
// sequences of very different lengths balance over the SMs without a counter in memory. The load
// warp asks for the next item, finds its sequence and hands it to the other warps through a ring,
// all while they still work on the previous ones. Items with most keys come first (up to 32
// sequences are ordered by their lengths; causal: a sequence's last rows first). The 256 rows
// are two tiles of 128 whose chains alternate: while the tensor core works for one tile, the other
// tile's rows take their maxima and exponentials, so neither waits for the other longer than it
// must. Keys and values stream through a ring of TMA stages shared by both tiles.
//
//   warps 0..7    rows: one thread per row, warp w with tile w / 4 and tensor memory lanes
//                 32 (w % 4) .. + 31, so that every SM sub-partition runs one warp of each tile
//   warp 8        items and loads (one lane loading)
//   warp 9        MMA issue for both tiles in turn: P V and the next S of tile 0, then of tile 1,
//                 which is what keeps the tiles' chains half a step apart (with an issuer each they
//                 run in phase, and tensor core and exponentials wait for each other)
//   warp 10       tensor memory
//
// * m follows the true maximum only when that has risen by more than 2^8: P stays below 2^8, sums
//   below 2^8 per key, well inside FP32's and bfloat16's range, and results do not change, since m
//   cancels in the quotient. So a step takes its exponentials with the m it has, one read of the
//   scores giving both them and their maximum; only where a maximum turns out too high (in the first
//   step, where m is 0, also too low) are O and the sums rescaled and the scores read again.
// * NaN and minus infinity take that second reading too, in its exact form: the exponentials on the
//   FMA pipe would make something finite of both.
// * Scores are read 32 at a time, the next 32 in flight meanwhile. Two threads per row (64 scores
//   each, maxima or a "too high" flag exchanged every step) took 1.94 ms where this takes 1.81 ms
//   (16384 tokens, 16 heads of 128: 1214 TFLOP/s, of 1672 measured for one large product; heads of
//   64: 1.27 ms, 867 TFLOP/s, bound by exponentials: 3.4 of the special-function units' 4.5 10^12
//   a second, a quarter of them on the FMA pipe). Their exchanges cost more than the shorter rows
//   saved.
// * head_dim <= 64: P has tensor memory of its own, so the next S is issued as soon as the rows
//   have read the current one. Up to 128: P overlays S (S 2 x 128, O 2 x 128 columns fill the 512),
//   and the next S follows P V. (Steps of 96 keys, which leave P a place of its own for heads up to
//   112: 336 us against 292 for images of 64 to 4096 tokens, 16 heads of 72. A step's waits take
//   about 1.4 us whatever its keys.)
// * A sequence may end inside a tile. K rows past the end only make scores that are replaced by
//   -inf. V rows past the end would be multiplied by P = 0, which leaves NaN where they hold NaN
//   or infinity (they belong to other sequences, or to nobody): the at most 15 of them that the
//   last 16-key step still reads are overwritten with zeros in shared memory first.
// * Tensor memory is read and written by whole warps (.sync.aligned): no lane leaves or skips
//   ahead in the row warps' loops, and stores that only some lanes make are followed by a
//   __syncwarp.
#include "attention_varlen.hpp"
#include "ptx.cuh"
#include "varlen.cuh"

#include <cuda_bf16.h>

#include <cstdint>
#include <type_traits>

namespace cuvit::attn {
namespace {

constexpr int kTile = 128;              // query rows of a tile, keys of a step
constexpr int kAtomBytes = kTile * 128; // 128 rows of 64 bfloat16
constexpr int kRowWarps = 8;
constexpr int kLoadWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kTmemWarp = 10;
constexpr int kThreads = 352;
constexpr float kRescaleAbove = 8.0F; // log2
// Above this |m scale| (log2) the plain and the exact form of P would differ by more than 2^-14.
constexpr float kLargeMaximum = 1024.0F;
// A step's weights add up to 2^15 at most where none is NaN (the FMA pipe's form makes 2^128 of it).
constexpr float kLargeSum = 1.0e30F;
// Exponentials of these pairs of a 32-key chunk run on the FMA pipe (see attention.cu).
constexpr uint32_t kPolyPairs = 0x8888u;

constexpr int kItemSlots = 2;
// A warp may wait for its next item as long as another tile's rows take: seconds for 10^8 keys.
constexpr unsigned long long kItemWaitNs = 60000000000ull;
constexpr int kItemBytes = 48;

template <int Atoms>
struct Shape {
    static constexpr bool kOverlay = Atoms == 2; // P in the columns of S
    static constexpr int kQBytes = Atoms * kAtomBytes;
    static constexpr int kSlotBytes = Atoms * kAtomBytes;
    static constexpr int kSlots = Atoms == 2 ? 5 : 8;
    static constexpr int kSlotOffset = 2 * kQBytes;
    static constexpr int kBarrierOffset = kSlotOffset + kSlots * kSlotBytes;
    // full, empty per slot; q_full[2], q_empty, drain, s_full[2], s_free[2], p_full[2], o_done[2],
    // item_full, item_empty per item slot, the launch control's answer
    static constexpr int kBarriers = 2 * kSlots + 12 + 2 * kItemSlots + 1;
    static constexpr int kItemOffset = (kBarrierOffset + 8 * kBarriers + 15) / 16 * 16;
    static constexpr int kAnswerOffset = kItemOffset + kItemSlots * kItemBytes;
    static constexpr int kTmemSlotOffset = kAnswerOffset + 16;
    static constexpr int kSmemBytes = 1024 + kTmemSlotOffset + 16;
    static constexpr uint32_t kOColumn = 256;
    static constexpr uint32_t kOPitch = Atoms == 2 ? 128 : 64;
    static constexpr uint32_t kPColumn = Atoms == 2 ? 0 : 384;
    static constexpr uint32_t kPPitch = Atoms == 2 ? 128 : 64;
    static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
};

// What the warps know of an item, in shared memory.
struct Item {
    int rows; // query rows of the block (1..256); 0: no more items
    int head;
    int split;
    int q_first;   // the block's first query row
    int kv_first;  // the split's first key row
    int keys;      // of the split
    int reach;     // row r of the block sees the split's first (reach + r) keys, at least 0
    int steps[2];  // key tiles of each query tile
    int unused[3];
};
static_assert(sizeof(Item) == kItemBytes, "items are handed over as whole vectors");

__device__ __forceinline__ int tile_steps(int rows, int keys, int reach, int t) {
    const int live = min(kTile, rows - t * kTile);
    const int seen = min(static_cast<long long>(keys),
                         static_cast<long long>(reach) + t * kTile + live - 1);
    return live <= 0 || seen <= 0 ? 0 : (seen + kTile - 1) / kTile;
}

// Item `index` by a whole warp; rows 0 where the block has none. Up to 32 sequences come in the
// order of their work, more in their own order (causal: backwards, rows that see most first).
__device__ __forceinline__ Item find_item(const VarlenParams& p, const Order& order,
                                          long long index, long long items) {
    Item item{};
    const bool ordered = p.batch <= 32;
    index = p.causal && !ordered ? items - 1 - index : index;
    item.split = static_cast<int>(index % p.splits);
    index /= p.splits;
    item.head = static_cast<int>(index % p.q_heads);
    index /= p.q_heads;
    const Sequence s =
        ordered ? find_ordered_block(order, p.q_offsets, p.kv_offsets, p.batch, p.q_tokens,
                                     p.kv_tokens, index, 2 * kTile, p.causal != 0)
                : find_block_warp(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                  index, 2 * kTile);
    item.rows = s.index < 0 ? 0 : min(2 * kTile, s.q_end - s.q_first);
    item.q_first = s.q_first;
    const int keys = s.kv_end - s.kv_begin;
    // Whole tiles per split, so that only a sequence's end falls inside a tile.
    const int tiles = (keys + kTile - 1) / kTile;
    const int each = (tiles + p.splits - 1) / p.splits;
    const int first = min(keys, min(tiles, item.split * each) * kTile);
    const int end = min(keys, min(tiles, (item.split + 1) * each) * kTile);
    item.kv_first = s.kv_begin + first;
    item.keys = end - first;
    // The first row's share of the split's keys (rows see the split's keys at most).
    const long long reach = static_cast<long long>(s.q_first - s.q_begin) + 1 + keys -
                            (s.q_end - s.q_begin) - first;
    item.reach = p.causal ? static_cast<int>(
                                max(-4LL * kTile, min(static_cast<long long>(item.keys), reach)))
                          : item.keys;
    item.steps[0] = tile_steps(item.rows, item.keys, item.reach, 0);
    item.steps[1] = tile_steps(item.rows, item.keys, item.reach, 1);
    return item;
}

// Scores at or past `limit` become -inf.
__device__ __forceinline__ void mask(uint32_t (&s)[32], int limit) {
#pragma unroll
    for (int c = 0; c < 32; ++c) {
        s[c] = c < limit ? s[c] : 0xFF800000u;
    }
}

__device__ __forceinline__ float maximum(const uint32_t (&s)[32]) {
    float m[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        m[c] = __uint_as_float(s[16 * c]);
#pragma unroll
        for (int j = 1; j < 15; j += 2) {
            m[c] = dev::max3(m[c], __uint_as_float(s[16 * c + j]),
                             __uint_as_float(s[16 * c + j + 1]));
        }
        m[c] = fmaxf(m[c], __uint_as_float(s[16 * c + 15]));
    }
    return fmaxf(m[0], m[1]);
}

// P = 2^(scale (s - m)) of 32 scores, packed, and their sum. The plain form
// folds scale and m into one multiply-add, off by a row-wide factor 2^d, |d| <= 2^-24 |m scale|
// (it cancels in the quotient), and takes some exponentials on the FMA pipe. The exact form, for
// tiles with masked scores and rows with a very large m, subtracts first, so that no m overflows
// the exponent, and keeps to the special-function unit, whose 2^-inf is zero (the polynomial's is
// 2^-125).
template <bool Exact>
__device__ __forceinline__ float exponentials(const uint32_t (&s)[32], float scale, float m,
                                              uint32_t (&packed)[16]) {
    const uint64_t scale2 = dev::f32x2(scale, scale);
    const float minus = Exact ? -m : -m * scale;
    const uint64_t minus2 = dev::f32x2(minus, minus);
    uint64_t sums[2] = {dev::f32x2(0.0F, 0.0F), dev::f32x2(0.0F, 0.0F)};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const uint64_t s2 = dev::f32x2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1]));
        const uint64_t x2 = Exact ? dev::mul_f32x2(dev::add_f32x2(s2, minus2), scale2)
                                  : dev::fma_f32x2(s2, scale2, minus2);
        const float2 x = dev::f32x2_split(x2);
        float2 e;
        if (!Exact && ((kPolyPairs >> j) & 1u)) {
            e = dev::exp2_poly2<true>(x.x, x.y);
        } else {
            e = make_float2(dev::ex2_approx(x.x), dev::ex2_approx(x.y));
        }
        packed[j] = dev::pack_bf16x2(e.x, e.y);
        sums[j & 1] = dev::add_f32x2(sums[j & 1], dev::f32x2(e.x, e.y));
    }
    const float2 total = dev::f32x2_split(dev::add_f32x2(sums[0], sums[1]));
    return total.x + total.y;
}

// S = Q K^T: k_steps steps of 16 elements, 4 to an atom. By the whole warp.
template <int Atoms>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint64_t q_desc, uint64_t k_desc,
                                             uint32_t idesc, int k_steps) {
    constexpr uint64_t kAtomStep = kAtomBytes >> 4; // descriptors count 16-byte units
    if (k_steps == 4 * Atoms) {
#pragma unroll
        for (int kk = 0; kk < 4 * Atoms; ++kk) {
            const uint64_t at = static_cast<uint64_t>(kk >> 2) * kAtomStep + 2u * (kk & 3);
            dev::mma_ss_f16_warp(d_tmem, q_desc + at, k_desc + at, idesc, kk > 0 ? 1u : 0u);
        }
    } else {
#pragma unroll 1
        for (int kk = 0; kk < k_steps; ++kk) {
            const uint64_t at = static_cast<uint64_t>(kk >> 2) * kAtomStep + 2u * (kk & 3);
            dev::mma_ss_f16_warp(d_tmem, q_desc + at, k_desc + at, idesc, kk > 0 ? 1u : 0u);
        }
    }
}

// O (+)= P V: v_steps steps of 16 keys. By the whole warp.
__device__ __forceinline__ void issue_outputs(uint32_t d_tmem, uint32_t p_tmem, uint64_t v_desc,
                                              uint32_t idesc, int v_steps, uint32_t accumulate) {
    if (v_steps == kTile / 16) {
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk) {
            dev::mma_ts_f16_warp(d_tmem, p_tmem + 8 * kk,
                                 v_desc + static_cast<uint64_t>(kk) * (2048 >> 4), idesc,
                                 kk > 0 ? 1u : accumulate);
        }
    } else {
#pragma unroll 1
        for (int kk = 0; kk < v_steps; ++kk) {
            dev::mma_ts_f16_warp(d_tmem, p_tmem + 8 * kk,
                                 v_desc + static_cast<uint64_t>(kk) * (2048 >> 4), idesc,
                                 kk > 0 ? 1u : accumulate);
        }
    }
}

template <int Atoms, bool Short>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap map_q,
                           const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ VarlenParams p, unsigned* const status) {
    using S = Shape<Atoms>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = dev::smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_base);
    const uint32_t bars = base + S::kBarrierOffset;
    const auto full = [&](int i) -> uint32_t { return bars + 8u * i; };
    const auto empty = [&](int i) -> uint32_t { return bars + 8u * (S::kSlots + i); };
    const uint32_t more = bars + 16u * S::kSlots;
    const uint32_t q_full = more;        // + 8 t
    const uint32_t q_empty = more + 16;
    const uint32_t drain = more + 24;
    const uint32_t s_full = more + 32;   // + 8 t
    const uint32_t s_free = more + 48;   // + 8 t
    const uint32_t p_full = more + 64;   // + 8 t
    const uint32_t o_done = more + 80;   // + 8 t
    const uint32_t item_full = more + 96;  // + 8 slot
    const uint32_t item_empty = item_full + 8 * kItemSlots;
    const uint32_t answer_full = item_empty + 8 * kItemSlots;
    const auto item_slot = [&](int i) -> Item* {
        return reinterpret_cast<Item*>(smem + S::kItemOffset) + i;
    };

    // Through a shuffle, so that the compiler knows it is the same for the warp.
    const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) / 32, 0);
    const int lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kSlots; ++i) {
            dev::mbar_init(full(i), 1);
            dev::mbar_init(empty(i), 1);
        }
        for (uint32_t t = 0; t < 2; ++t) {
            dev::mbar_init(q_full + 8 * t, 1);
            dev::mbar_init(s_full + 8 * t, 1);
            dev::mbar_init(s_free + 8 * t, kRowWarps / 2);
            dev::mbar_init(p_full + 8 * t, kRowWarps / 2);
            dev::mbar_init(o_done + 8 * t, 1);
        }
        for (uint32_t i = 0; i < kItemSlots; ++i) {
            dev::mbar_init(item_full + 8 * i, 1);
            dev::mbar_init(item_empty + 8 * i, kRowWarps + 1); // the rows' warps and the issuer
        }
        dev::mbar_init(answer_full, 1);
        dev::mbar_init(q_empty, 1);
        dev::mbar_init(drain, 1);
        dev::fence_barrier_init();
    }
    if (warp == kTmemWarp) {
        dev::tmem_alloc(base + S::kTmemSlotOffset, 512);
        dev::tmem_relinquish();
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = __shfl_sync(
        0xFFFFFFFFu, *reinterpret_cast<const uint32_t*>(smem + S::kTmemSlotOffset), 0);
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();

    if (warp == kLoadWarp) {
        // ---------------- items and loads ----------------
        if (lane == 0) {
            dev::tma_prefetch_descriptor(&map_q);
            dev::tma_prefetch_descriptor(&map_k);
            dev::tma_prefetch_descriptor(&map_v);
        }
        int slot = 0;
        uint32_t phase = 0;
        uint32_t q_phase = 0;                // items with keys so far
        uint32_t q_loads0 = 0, q_loads1 = 0; // loads of each query tile so far
        int item_at = 0;
        uint32_t item_phase = 0;
        uint32_t answers = 0; // taken so far
        bool asked = false;
        bool ok = true;
        const auto load_kv = [&](const CUtensorMap* map, int kv_head, int row) {
            if (!dev::mbar_wait(empty(slot), phase ^ 1u, status)) {
                ok = false;
                return;
            }
            dev::mbar_arrive_expect_tx(full(slot), S::kSlotBytes);
            for (int a = 0; a < Atoms; ++a) {
                const int c[3] = {64 * a, kv_head, row};
                dev::tma_load(base + S::kSlotOffset + slot * S::kSlotBytes + a * kAtomBytes, map,
                              full(slot), 3, c);
            }
            if (++slot == S::kSlots) {
                slot = 0;
                phase ^= 1u;
            }
        };
        const auto load_q = [&](int t, int head, int row) {
            dev::mbar_arrive_expect_tx(q_full + 8 * t, S::kQBytes);
            for (int a = 0; a < Atoms; ++a) {
                const int c[3] = {64 * a, head, row};
                dev::tma_load(base + t * S::kQBytes + a * kAtomBytes, &map_q, q_full + 8 * t, 3, c);
            }
        };
        Order order{};
        if (p.batch <= 32) {
            order = order_sequences(p.q_offsets, p.kv_offsets, p.batch, p.q_tokens, p.kv_tokens,
                                    2 * kTile);
        }
        uint32_t index = blockIdx.x;
        bool more_items = true;
        while (true) {
            Item item{};
            if (more_items) {
                // Asked for while this item's loads wait for room.
                if (lane == 0) {
                    dev::mbar_arrive_expect_tx(answer_full, 16);
                    dev::launch_control_try_cancel(base + S::kAnswerOffset, answer_full);
                }
                __syncwarp();
                asked = true;
                item = find_item(p, order, index, gridDim.x);
            }
            if (!more_items || item.rows > 0) {
                ok = dev::mbar_wait_warp(item_empty + 8 * item_at, item_phase ^ 1u, status,
                                         kItemWaitNs);
                if (!ok) {
                    break;
                }
                if (lane == 0) {
                    *item_slot(item_at) = item;
                    dev::mbar_arrive(item_full + 8 * item_at);
                }
                __syncwarp();
                if (++item_at == kItemSlots) {
                    item_at = 0;
                    item_phase ^= 1u;
                }
                if (!more_items) {
                    break;
                }
            }
            const int steps = max(item.steps[0], item.steps[1]);
            if (item.rows > 0 && steps > 0) {
                if (lane == 0) {
                    ok = dev::mbar_wait(q_empty, (q_phase & 1u) ^ 1u, status);
                    if (ok && item.steps[0] > 0) {
                        load_q(0, item.head, item.q_first);
                    }
                    if (ok && item.steps[1] > 0) {
                        load_q(1, item.head, item.q_first + kTile);
                    }
                    q_loads0 += ok && item.steps[0] > 0 ? 1u : 0u;
                    q_loads1 += ok && item.steps[1] > 0 ? 1u : 0u;
                    const int kv_head = item.head / p.group;
                    const int row = item.kv_first;
                    // In the order the MMA warp takes them.
                    if (ok) {
                        load_kv(&map_k, kv_head, row);
                    }
                    for (int j = 0; j < steps && ok; ++j) {
                        if (S::kOverlay) {
                            load_kv(&map_v, kv_head, row + j * kTile);
                        }
                        if (ok && j + 1 < steps) {
                            load_kv(&map_k, kv_head, row + (j + 1) * kTile);
                        }
                        if (ok && !S::kOverlay) {
                            load_kv(&map_v, kv_head, row + j * kTile);
                        }
                    }
                }
                ++q_phase;
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) {
                    break;
                }
            }
            ok = dev::mbar_wait_warp(answer_full, answers & 1u, status);
            if (!ok) {
                break;
            }
            ++answers;
            asked = false;
            more_items = dev::launch_control_answer(base + S::kAnswerOffset, &index);
            // The answer has been read before the next one may be written.
            dev::fence_proxy_async_shared();
            __syncwarp();
        }
        if (!ok && lane == 0) {
            // Every copy asked for lands before the CTA's shared memory goes.
            for (int i = 0; i < S::kSlots; ++i) {
                dev::mbar_drain_wait(full(i), phase ^ (i < slot ? 0u : 1u));
            }
            if (q_loads0 > 0) {
                dev::mbar_drain_wait(q_full, (q_loads0 - 1) & 1u);
            }
            if (q_loads1 > 0) {
                dev::mbar_drain_wait(q_full + 8, (q_loads1 - 1) & 1u);
            }
            if (asked) {
                dev::mbar_drain_wait(answer_full, answers & 1u);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ---------------- MMA issue (the whole warp, one lane issuing) ----------------
        const int k_steps = (p.head_dim + 15) / 16;
        const uint32_t idesc_o = dev::make_idesc(1u, kTile, 16 * k_steps, false, true);
        // Descriptors are built once and stepped by adding to their start-address field.
        const uint64_t q_desc0 = dev::smem_desc_sw128(base, 16, 1024);
        const uint64_t k_desc0 = dev::smem_desc_sw128(base + S::kSlotOffset, 16, 1024);
        const uint64_t v_desc0 = dev::smem_desc(base + S::kSlotOffset, kAtomBytes, 1024,
                                                dev::kLayoutSwizzle128);
        constexpr uint64_t kSlotStep = S::kSlotBytes >> 4;
        constexpr uint64_t kQStep = S::kQBytes >> 4;
        int slot = 0;
        uint32_t phase = 0;
        uint32_t q_phase[2] = {0u, 0u};
        uint32_t free_phase[2] = {0u, 0u};
        uint32_t p_phase[2] = {0u, 0u};
        bool ok = true;
        int item_at = 0;
        uint32_t item_phase = 0;
        while (ok) {
            ok = dev::mbar_wait_warp(item_full + 8 * item_at, item_phase, status, kItemWaitNs);
            if (!ok) {
                break;
            }
            const auto uniform = [](int value) { return __shfl_sync(0xFFFFFFFFu, value, 0); };
            const Item* const item = item_slot(item_at);
            const int rows = uniform(item->rows);
            const int tile_steps[2] = {uniform(item->steps[0]), uniform(item->steps[1])};
            const int keys = uniform(item->keys);
            if (lane == 0) {
                dev::mbar_arrive(item_empty + 8 * item_at);
            }
            __syncwarp();
            if (++item_at == kItemSlots) {
                item_at = 0;
                item_phase ^= 1u;
            }
            if (rows == 0) {
                break;
            }
            const int steps = max(tile_steps[0], tile_steps[1]);
            if (steps == 0) {
                continue;
            }
            // The first scores.
            {
                const int keys16 = (min(kTile, keys) + 15) & ~15;
                const uint32_t idesc = dev::make_idesc(1u, kTile, keys16, false, false);
                ok = dev::mbar_wait_warp(full(slot), phase, status);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (ok && tile_steps[t] > 0) {
                        ok = dev::mbar_wait_warp(q_full + 8 * t, q_phase[t], status);
                        q_phase[t] ^= 1u;
                        if (ok) {
                            dev::tc_fence_after();
                            issue_scores<Atoms>(tmem + t * kTile, q_desc0 + t * kQStep,
                                                k_desc0 + slot * kSlotStep, idesc, k_steps);
                            dev::tc_commit_warp(s_full + 8 * t);
                        }
                    }
                }
                if (!ok) {
                    break;
                }
                dev::tc_commit_warp(empty(slot));
                if (steps == 1) {
                    dev::tc_commit_warp(q_empty);
                }
                if (++slot == S::kSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
            for (int j = 0; j < steps; ++j) {
                // Slots of this step: these values and the next keys, in the loads' order.
                const bool next = j + 1 < steps;
                int slot2 = slot + 1;
                uint32_t phase2 = phase;
                if (slot2 == S::kSlots) {
                    slot2 = 0;
                    phase2 ^= 1u;
                }
                const bool keys_first = !S::kOverlay && next;
                const int v_slot = keys_first ? slot2 : slot;
                const uint32_t v_phase = keys_first ? phase2 : phase;
                const int k_slot = keys_first ? slot : slot2;
                const uint32_t k_phase = keys_first ? phase : phase2;
                const int next16 = (min(kTile, keys - (j + 1) * kTile) + 15) & ~15;
                const uint32_t idesc_next =
                    dev::make_idesc(1u, kTile, next ? next16 : 16, false, false);
                ok = dev::mbar_wait_warp(full(v_slot), v_phase, status);
                if (ok && next) {
                    ok = dev::mbar_wait_warp(full(k_slot), k_phase, status);
                }
                if (!ok) {
                    break;
                }
                const int live = min(kTile, keys - j * kTile);
                const int live16 = (live + 15) & ~15;
                if (live < live16) {
                    // Values behind the sequence's end that the last 16-key step reads.
                    const float zero[4] = {0.0F, 0.0F, 0.0F, 0.0F};
                    for (int a = 0; a < Atoms; ++a) {
                        const uint32_t rows = base + S::kSlotOffset + v_slot * S::kSlotBytes +
                                              a * kAtomBytes + live * 128;
                        for (int i = lane; i < (live16 - live) * 8; i += 32) {
                            dev::st_shared_v4(rows + 16 * i, zero);
                        }
                    }
                    dev::fence_proxy_async_shared();
                    __syncwarp();
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (!ok || j >= tile_steps[t]) {
                        continue;
                    }
                    const bool more_scores = j + 1 < tile_steps[t];
                    const auto next_scores = [&]() {
                        dev::tc_fence_after();
                        issue_scores<Atoms>(tmem + t * kTile, q_desc0 + t * kQStep,
                                            k_desc0 + k_slot * kSlotStep, idesc_next, k_steps);
                        dev::tc_commit_warp(s_full + 8 * t);
                    };
                    if (!S::kOverlay) {
                        // The next scores as soon as the rows have read these. (s_free completes
                        // once per step, whether or not more scores follow.)
                        if (more_scores) {
                            ok = dev::mbar_wait_warp(s_free + 8 * t, free_phase[t], status);
                            if (ok) {
                                next_scores();
                            }
                        }
                        free_phase[t] ^= 1u;
                    }
                    ok = ok && dev::mbar_wait_warp(p_full + 8 * t, p_phase[t], status);
                    p_phase[t] ^= 1u;
                    if (ok) {
                        dev::tc_fence_after();
                        issue_outputs(tmem + S::kOColumn + t * S::kOPitch,
                                             tmem + S::kPColumn + t * S::kPPitch,
                                             v_desc0 + v_slot * kSlotStep, idesc_o, live16 / 16,
                                             j > 0 ? 1u : 0u);
                        dev::tc_commit_warp(o_done + 8 * t);
                        if (S::kOverlay && more_scores) {
                            next_scores();
                        }
                    }
                }
                if (!ok) {
                    break;
                }
                dev::tc_commit_warp(empty(v_slot));
                if (next) {
                    dev::tc_commit_warp(empty(k_slot));
                }
                if (j + 2 == steps) {
                    dev::tc_commit_warp(q_empty); // the last scores have been issued
                }
                // This step took the values' slot and, if keys followed, theirs.
                slot = next ? slot2 : slot;
                phase = next ? phase2 : phase;
                if (++slot == S::kSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
        // Every MMA issued has finished before the CTA's shared and tensor memory go.
        dev::tc_commit_warp(drain);
        dev::mbar_drain_wait(drain, 0);
        __syncwarp();
    } else if (warp < kRowWarps) {
        // ---------------- rows ----------------
        const int t = warp >> 2;
        const int quarter = warp & 3; // the tensor memory lanes this warp may access
        const int row = quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_tmem = tmem + lanes + t * kTile;
        const uint32_t p_tmem = tmem + lanes + S::kPColumn + t * S::kPPitch;
        const uint32_t o_tmem = tmem + lanes + S::kOColumn + t * S::kOPitch;
        const int o_columns = 16 * ((p.head_dim + 15) / 16);
        uint32_t s_phase = 0;
        uint32_t o_phase = 0; // of the tile's next P V to complete
        bool ok = true;
        // One arrival for the warp's tensor memory accesses so far.
        const auto arrive = [&](uint32_t bar) {
            dev::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(bar);
            }
            __syncwarp();
        };
        int item_at = 0;
        uint32_t item_phase = 0;
        while (ok) {
            ok = dev::mbar_wait_warp(item_full + 8 * item_at, item_phase, status, kItemWaitNs);
            if (!ok) {
                break;
            }
            const Item* const item = item_slot(item_at);
            const int block_rows = item->rows;
            const int head = item->head;
            const int split = item->split;
            const int steps = item->steps[t];
            // Keys of the split that this row sees.
            const int row_keys = max(0, min(item->keys, item->reach + t * kTile + row));
            const long long token = static_cast<long long>(item->q_first) + t * kTile + row;
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(item_empty + 8 * item_at);
            }
            __syncwarp();
            if (++item_at == kItemSlots) {
                item_at = 0;
                item_phase ^= 1u;
            }
            if (block_rows == 0) {
                break;
            }
            const int rows = block_rows - t * kTile; // may be 0 or less
            if (rows <= 0) {
                continue;
            }
            const bool live_warp = quarter * 32 < rows;
            // Of the warp's rows the first ones exist. What stands behind them is another
            // sequence's, or nobody's, and takes no part in the warp's choices.
            const unsigned live_rows = 0xFFFFFFFFu >> (32 - min(32, max(1, rows - quarter * 32)));
            float m = 0.0F; // unscaled
            float sum = 0.0F;
            for (int j = 0; j < steps && ok; ++j) {
                ok = dev::mbar_wait_warp(s_full + 8 * t, s_phase, status);
                s_phase ^= 1u;
                if (!ok) {
                    break;
                }
                dev::tc_fence_after();
                if (live_warp) {
                    const int limit = row_keys - j * kTile;
                    const bool masked = __any_sync(0xFFFFFFFFu, limit < kTile);
                    uint32_t packed[4][16];
                    float added = 0.0F;
                    float top = -INFINITY;
                    // Without branches inside, so that one chunk's maxima run under another's
                    // exponentials: a warp has its scheduler almost to itself here.
                    const auto weigh = [&](auto exact) {
                        uint32_t s[2][32];
                        dev::tmem_load_32(s_tmem, s[0]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            dev::tmem_wait_load_of(s[c & 1]);
                            if (c < 3) {
                                dev::tmem_load_32(s_tmem + 32 * (c + 1), s[(c + 1) & 1]);
                            }
                            if constexpr (exact.value) {
                                mask(s[c & 1], limit - 32 * c);
                            }
                            top = fmaxf(top, maximum(s[c & 1]));
                            added += exponentials<exact.value>(s[c & 1], p.scale_log2, m,
                                                               packed[c]);
                        }
                    };
                    const unsigned large_rows =
                        __ballot_sync(0xFFFFFFFFu, fabsf(m * p.scale_log2) > kLargeMaximum);
                    const bool exact = masked || (large_rows & live_rows) != 0u;
                    if (Short && exact) {
                        // Chunks that no row of the warp sees are zeros.
                        const int seen = __reduce_max_sync(0xFFFFFFFFu, limit);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (32 * c < seen) { // the whole warp
                                uint32_t s[32];
                                dev::tmem_load_32(s_tmem + 32 * c, s);
                                dev::tmem_wait_load_of(s);
                                mask(s, limit - 32 * c);
                                top = fmaxf(top, maximum(s));
                                added += exponentials<true>(s, p.scale_log2, m, packed[c]);
                            } else {
#pragma unroll
                                for (int x = 0; x < 16; ++x) {
                                    packed[c][x] = 0u;
                                }
                            }
                        }
                    } else if (exact) {
                        weigh(std::true_type{});
                    } else {
                        weigh(std::false_type{});
                    }
                    // A row without a weight so far has m = 0, which stays where the maximum is
                    // within 2^+-8 of it. NaN shows in the weights' sum.
                    const bool fresh = sum == 0.0F;
                    const bool some = top != -INFINITY;
                    const float above = (top - m) * p.scale_log2;
                    const unsigned raised_rows = __ballot_sync(
                        0xFFFFFFFFu, above > kRescaleAbove || !(added < kLargeSum) ||
                                         (some ? fresh && above < -kRescaleAbove : !exact));
                    const bool raise = (raised_rows & live_rows) != 0u;
                    if (!S::kOverlay && !raise) {
                        arrive(s_free + 8 * t);
                    }
                    if (!S::kOverlay && j > 0) {
                        // P V of the previous step has read P and written O.
                        ok = dev::mbar_wait_warp(o_done + 8 * t, o_phase, status);
                        o_phase ^= 1u;
                        if (!ok) {
                            break;
                        }
                        dev::tc_fence_after();
                    }
                    if (raise) {
                        if (j == 0) {
                            m = some ? top : 0.0F;
                        } else {
                            const float raised =
                                some && (fresh || above > kRescaleAbove) ? top : m;
                            const float factor =
                                fresh ? 0.0F : dev::ex2_approx((m - raised) * p.scale_log2);
                            m = raised;
                            sum *= factor;
#pragma unroll 1
                            for (int c = 0; c < o_columns; c += 16) {
                                uint32_t o[16];
                                dev::tmem_load_16(o_tmem + c, o);
                                dev::tmem_wait_load_of(o);
#pragma unroll
                                for (int x = 0; x < 16; ++x) {
                                    o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
                                }
                                dev::tmem_store_16(o_tmem + c, o);
                            }
                        }
                        added = 0.0F;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t s[32];
                            dev::tmem_load_32(s_tmem + 32 * c, s);
                            dev::tmem_wait_load_of(s);
                            if (masked) {
                                mask(s, limit - 32 * c);
                            }
                            added += exponentials<true>(s, p.scale_log2, m, packed[c]);
                        }
                        if (!S::kOverlay) {
                            arrive(s_free + 8 * t);
                        }
                    }
                    sum += added;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        dev::tmem_store_16(p_tmem + 16 * c, packed[c]);
                    }
                    dev::tmem_wait_store();
                } else if (!S::kOverlay) {
                    // A warp without rows keeps the others' pace: the next scores may come before
                    // they have handed over this step's P, and an arrival for that step would be
                    // counted into this one.
                    arrive(s_free + 8 * t);
                    if (j > 0) {
                        ok = dev::mbar_wait_warp(o_done + 8 * t, o_phase, status);
                        o_phase ^= 1u;
                        if (!ok) {
                            break;
                        }
                    }
                }
                arrive(p_full + 8 * t);
            }
            if (!ok) {
                break;
            }
            if (steps > 0) {
                // The last P V of this tile. With the overlay the phases of the earlier ones were
                // not waited for: each later S came after them.
                if (S::kOverlay) {
                    o_phase ^= static_cast<uint32_t>(steps - 1) & 1u;
                }
                ok = dev::mbar_wait_warp(o_done + 8 * t, o_phase, status);
                o_phase ^= 1u;
                if (!ok) {
                    break;
                }
                dev::tc_fence_after();
            }
            if (!live_warp) {
                continue; // the whole warp
            }
            const bool live = row < rows;
            const float inverse = sum == 0.0F ? 0.0F : 1.0F / sum;
            const long long part =
                (static_cast<long long>(split) * p.q_tokens + token) * p.q_heads + head;
            if (live && p.splits > 1) {
                p.part_stats[part] = make_float2(sum == 0.0F ? -INFINITY : m * p.scale_log2, sum);
            }
#pragma unroll 1
            for (int c = 0; c < p.head_dim; c += 32) {
                uint32_t o[32];
                // The read is warp-wide: lanes that store below, and those that do not, meet first.
                // (Columns past the last 16-column step hold anything and are not stored.)
                __syncwarp();
                if (steps > 0) {
                    dev::tmem_load_32(o_tmem + c, o);
                    dev::tmem_wait_load_of(o);
                }
                if (sum == 0.0F) { // no keys: what tensor memory holds is nobody's
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        o[x] = 0u;
                    }
                }
                if (live && p.splits > 1) {
                    float4* const out =
                        reinterpret_cast<float4*>(p.part_out + part * p.head_dim + c);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if (c + 4 * x < p.head_dim) {
                            out[x] = make_float4(
                                __uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                                __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
                        }
                    }
                } else if (live) {
                    uint4* const out = reinterpret_cast<uint4*>(
                        static_cast<__nv_bfloat16*>(p.out) + token * p.out_stride +
                        static_cast<long long>(head) * p.head_dim + c);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if (c + 8 * x < p.head_dim) {
                            uint32_t words[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                words[y] = dev::pack_bf16x2(
                                    __uint_as_float(o[8 * x + 2 * y]) * inverse,
                                    __uint_as_float(o[8 * x + 2 * y + 1]) * inverse);
                            }
                            out[x] = make_uint4(words[0], words[1], words[2], words[3]);
                        }
                    }
                }
            }
            __syncwarp();
            // O has been read before the next item's first P V, which follows this tile's p_full.
            dev::tc_fence_before();
        }
    }

    __syncthreads();
    if (warp == kTmemWarp) {
        dev::tc_fence_after();
        dev::tmem_dealloc(tmem, 512);
    }
}

template <int Atoms, bool Short>
int launch_atoms(const VarlenParams& p, const host::DeviceContext& context,
                 const CUtensorMap (&maps)[3], cudaStream_t stream) {
    auto* kernel = &attention_tiles_kernel<Atoms, Short>;
    constexpr int kBytes = Shape<Atoms>::kSmemBytes;
    CUVIT_TRY_CUDA(host::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kBytes));
    const long long items = tiles_kernel_items(p) * p.splits;
    if (items > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "attention launch exceeds the CUDA grid limit");
    }
    host::pdl_launch(kernel, dim3(static_cast<unsigned>(items)), dim3(kThreads), kBytes, stream,
                     maps[0], maps[1], maps[2], p, context.status);
    return host::after_launch("attention_tiles_kernel");
}

// [rows][heads][head_dim] with boxes of 64 elements of one head of 128 rows.
bool describe(const void* base, int head_dim, int heads, long long rows, long long stride,
              CUtensorMap* map) {
    host::TmaTensor t;
    t.base = base;
    t.type = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    t.element_bytes = 2;
    t.rank = 3;
    t.dims[0] = static_cast<uint64_t>(head_dim);
    t.dims[1] = static_cast<uint64_t>(heads);
    t.dims[2] = static_cast<uint64_t>(rows);
    t.strides_bytes[0] = static_cast<uint64_t>(head_dim) * 2;
    t.strides_bytes[1] = static_cast<uint64_t>(stride) * 2;
    t.box[0] = 64;
    t.box[1] = 1;
    t.box[2] = kTile;
    if (!host::tma_describable(t) || (map != nullptr && host::encode_tma(t, map) != CUVIT_OK)) {
        host::clear_error(); // another kernel serves what TMA cannot
        return false;
    }
    return true;
}

} // namespace

long long tiles_kernel_items(const VarlenParams& p) {
    return (p.q_tokens / (2 * kTile) + static_cast<long long>(p.batch)) * p.q_heads;
}

bool tiles_kernel_takes(const VarlenParams& p) {
    return p.bf16 && p.kv_tokens > 0 && p.head_dim % 8 == 0 &&
           reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % 8 == 0 &&
           describe(p.q, p.head_dim, p.q_heads, p.q_tokens, p.q_stride, nullptr) &&
           describe(p.k, p.head_dim, p.kv_heads, p.kv_tokens, p.k_stride, nullptr) &&
           describe(p.v, p.head_dim, p.kv_heads, p.kv_tokens, p.v_stride, nullptr);
}

int launch_tiles(const VarlenParams& p, cudaStream_t stream) {
    const host::DeviceContext* context = nullptr;
    CUVIT_TRY(host::current_context(&context));
    CUtensorMap maps[3];
    if (!describe(p.q, p.head_dim, p.q_heads, p.q_tokens, p.q_stride, &maps[0]) ||
        !describe(p.k, p.head_dim, p.kv_heads, p.kv_tokens, p.k_stride, &maps[1]) ||
        !describe(p.v, p.head_dim, p.kv_heads, p.kv_tokens, p.v_stride, &maps[2])) {
        return host::fail(CUVIT_CUDA_ERROR, "the attention operands' TMA descriptors failed");
    }
    // Sequences of less than two tiles on average: most tiles end inside, and the warps skip the
    // chunks behind (64 tokens, 16 heads of 64: 256 images 83 us against 95; 100 of 160 68 against 75;
    // 256 of 197, 12 heads, 151 against 156; where little is skipped the branches cost up to 6 %: 160 of
    // 100 68 against 65, 128 of 197 with heads of 80 120 against 114). Of longer ones a smaller part is
    // skipped, and whole tiles pay (300 tokens 86 against 87, 384 68 against 65, 16 images of 64 to 4096
    // with heads of 72 275 against 262, one of 16384 1327 against 1252), so they go without.
    const bool short_keys = p.kv_tokens <= 224LL * p.batch;
    if (p.head_dim <= 64) {
        return short_keys ? launch_atoms<1, true>(p, *context, maps, stream)
                          : launch_atoms<1, false>(p, *context, maps, stream);
    }
    return short_keys ? launch_atoms<2, true>(p, *context, maps, stream)
                      : launch_atoms<2, false>(p, *context, maps, stream);
}

} // namespace cuvit::attn
