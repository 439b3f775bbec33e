// FP32 linear layers on the tensor cores (tcgen05): out = residual + scale * act(x W^T + b)
// [* (up + b)], each operand split into two TF32 values.
//
// Three products of TF32 halves make one of floats (split_tf32.cuh). The accumulator collects 64 of k
// at a time (24 instructions) and hands them to registers, where the sum is rounded to nearest: the
// error then hardly grows with k (relative, root mean square against FP64: 4.7e-7 for k = 384,
// 5.4e-7 for 15360; summed in the accumulator throughout 9.4e-7 and, at k = 3840, 9e-6).
//
// Tile: 128 rows by up to 144 columns, in steps of 16 (of a gated layer, half gate and half up),
// one CTA per SM, persistent. What bounds it is shared memory: per 32 of k and 144 columns the
// copies write 34 KB, the splitters read those and write 36 KB, and the tensor core reads 54 KB,
// 158 KB or 1240 cycles where its products take 864. x's halves go to tensor memory, from where
// the tensor core reads them beside that traffic (from shared memory they would add 16 + 108 KB).
// Measured: 1576 x 1536 outputs, k = 384, GELU 30 us with cold caches (48 with both operands split in
// shared memory by the GEMM kernel's FP32 mode), of it about 10 us start and end; 8192 x 4096 x 4096
// 1.59 ms, 173 TFLOP/s of such products where that mode reached 130. What separates it from the
// bound is the splitting warps' latency (without the weight's splitting a quarter less); more of
// them (8 for the weight) leave the draining warps too few registers and take 15 % longer.
//
// Where the tiles do not fill the GPU, a cluster's CTAs share one, each with a slice of k; their sums
// meet in the memory of the CTA that owns the row, in the order of k.
//
//   warp 0        copies (TMA) into rings of kX and kW stages
//   warp 1        issues the products
//   warp 2        tensor memory
//   warps 4-15    take the partial sums (a third of the columns each, lane quarter = warp % 4) and
//                 write the outputs
//   warps 16-19   split x: stage -> tensor memory, a row per thread
//   warps 20-23   split the weight: hi in place, lo beside the stages
#include "activation.cuh"
#include "linear.hpp"
#include "ptx.cuh"
#include "split_tf32.cuh"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::linear {
namespace {

constexpr int kBlockM = 128;
constexpr int kBlockK = 32; // 128 bytes of a row
constexpr int kRowBytes = 128;
constexpr int kMaxN = 144;
constexpr int kMaxGatedN = 96; // 48 gate and 48 up columns
constexpr int kGroup = 16;     // columns a drain step takes
constexpr int kParts = 3;      // of a tile's columns
constexpr int kGroups = kMaxN / kGroup / kParts;
constexpr int kChunk = 2;      // k blocks summed in the tensor core
// Stages: about 1.5 us pass between a copy's issue and its arrival, three stages' products. x's
// are free once read; the weight's become hi in place and are held until their products are done.
constexpr int kX = 4;
constexpr int kW = 6;
constexpr int kSplit = 2; // x's halves, the weight's lo
constexpr int kThreads = 768;
constexpr int kDrainWarp = 4;
constexpr int kDrainWarps = 4 * kParts;
constexpr int kSplitXWarp = kDrainWarp + kDrainWarps;
constexpr int kSplitWWarp = kSplitXWarp + 4;
static_assert(32 * (kSplitWWarp + 4) == kThreads, "roles cover the block");

constexpr int kXBytes = kBlockM * kRowBytes;
constexpr int kWBytes = kMaxN * kRowBytes;
constexpr int kWOffset = kX * kXBytes;
constexpr int kLowOffset = kWOffset + kW * kWBytes;
constexpr int kSlabOffset = kLowOffset + kSplit * kWBytes;
constexpr int kSlabRows = 16;          // of a warp's 32 at a time
constexpr int kSlabPitch = kGroup + 4; // floats; rows' 16-byte accesses fall in different banks
constexpr int kSlabBytes = kSlabRows * kSlabPitch * 4;
// Slices' sums, in the stages' place: rows of the tile's columns and a vector, so that neighbouring
// rows fall in different banks.
constexpr int kPartPad = 4;
static_assert(4 * kBlockM * (kMaxN + kPartPad) <= kSlabOffset, "the slices' sums fit the stages");
constexpr int kMinSteps = 4; // of k in a slice
constexpr int kBarrierOffset = kSlabOffset + kDrainWarps * kSlabBytes;
constexpr int kBarriers = 2 * kX + 2 * kW + 2 * kSplit + 4 + 1;
constexpr int kSmemBytes = 1024 + kBarrierOffset + 8 * kBarriers + 8;
static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");

// Tensor memory: two partial sums, then the split stages of x (hi, then lo).
constexpr int kSumPitch = 160;
constexpr int kTmemX = 2 * kSumPitch;
constexpr int kTmemColumns = 512;
static_assert(kMaxN <= kSumPitch && kTmemX + kSplit * 2 * kBlockK <= kTmemColumns, "tensor memory");

struct SplitParams : OutRows {
    int slices;      // CTAs of a cluster that share a tile, each with its part of k
    int block_n;     // columns of the accumulator
    int out_columns; // block_n, or half of it for a gated layer
    int n_tiles, k_blocks, total_tiles;
    int columns_ok;      // bias and scale are 16-byte aligned
    unsigned* status;
};

template <bool Multiply>
__device__ __forceinline__ void with_columns(float (&v)[kGroup], const float* vector, int col0,
                                             int n, bool vector_ok) {
    if (vector_ok && col0 + kGroup <= n) {
#pragma unroll
        for (int q = 0; q < kGroup / 4; ++q) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(vector + col0) + q);
            const float four[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[4 * q + j] = Multiply ? v[4 * q + j] * four[j] : v[4 * q + j] + four[j];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            if (col0 + j < n) {
                const float b = __ldg(vector + col0 + j);
                v[j] = Multiply ? v[j] * b : v[j] + b;
            }
        }
    }
}

__device__ __forceinline__ void activate_group(int activation, float (&v)[kGroup]) {
    switch (activation) { // outside the loops: one branch for all values
    case CUVIT_ACTIVATION_GELU:
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            v[j] = dev::gelu_exact(v[j]);
        }
        break;
    case CUVIT_ACTIVATION_GELU_TANH:
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            v[j] = dev::gelu_tanh_exact(v[j]);
        }
        break;
    case CUVIT_ACTIVATION_SILU:
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            v[j] = dev::silu_exact(v[j]);
        }
        break;
    default:
        break;
    }
}

// Sliced: a cluster of s.slices CTAs to each tile. (One kernel for both spills more in the ordinary
// case.)
template <bool Sliced>
__global__ void __launch_bounds__(kThreads, 1)
    linear_split_kernel(const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ SplitParams s) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = dev::smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_base);
    const uint32_t bars = base + kBarrierOffset;
    const auto x_full = [&](int i) -> uint32_t { return bars + 8u * i; };
    const auto x_empty = [&](int i) -> uint32_t { return bars + 8u * (kX + i); };
    constexpr int kWBars = 2 * kX;
    const auto w_full = [&](int i) -> uint32_t { return bars + 8u * (kWBars + i); };
    const auto w_empty = [&](int i) -> uint32_t { return bars + 8u * (kWBars + kW + i); };
    constexpr int kSplitBars = kWBars + 2 * kW;
    const auto split_full = [&](int i) -> uint32_t { return bars + 8u * (kSplitBars + i); };
    const auto split_empty = [&](int i) -> uint32_t {
        return bars + 8u * (kSplitBars + kSplit + i);
    };
    constexpr int kAccBars = kSplitBars + 2 * kSplit;
    const auto acc_full = [&](int i) -> uint32_t { return bars + 8u * (kAccBars + i); };
    const auto acc_empty = [&](int i) -> uint32_t { return bars + 8u * (kAccBars + 2 + i); };
    const uint32_t drain_bar = bars + 8u * (kAccBars + 4);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarrierOffset + 8 * kBarriers);
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kX; ++i) {
            dev::mbar_init(x_full(i), 1);
            dev::mbar_init(x_empty(i), 4); // warps
        }
        for (int i = 0; i < kW; ++i) {
            dev::mbar_init(w_full(i), 1);
            dev::mbar_init(w_empty(i), 1);
        }
        for (int i = 0; i < kSplit; ++i) {
            dev::mbar_init(split_full(i), 8); // warps
            dev::mbar_init(split_empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            dev::mbar_init(acc_full(i), 1);
            dev::mbar_init(acc_empty(i), kDrainWarps);
        }
        dev::mbar_init(drain_bar, 1);
        dev::fence_barrier_init();
    }
    if (warp == 2) {
        dev::tmem_alloc(dev::smem_u32(tmem_slot), kTmemColumns);
        dev::tmem_relinquish();
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();

    const Params& p = s.p;
    const int slices = Sliced ? s.slices : 1;
    const int slice = Sliced ? static_cast<int>(dev::cluster_ctarank()) : 0;
    const int tile0 = static_cast<int>(blockIdx.x) / slices;
    const int tile_step = static_cast<int>(gridDim.x) / slices;
    const int k_first =
        Sliced ? static_cast<int>(static_cast<long long>(s.k_blocks) * slice / slices) : 0;
    const int k_end =
        Sliced ? static_cast<int>(static_cast<long long>(s.k_blocks) * (slice + 1) / slices)
               : s.k_blocks;
    const int k_blocks = k_end - k_first; // of this CTA
    const int my_tiles = (s.total_tiles - tile0 + tile_step - 1) / tile_step;
    const int steps = my_tiles * k_blocks; // k blocks of all this CTA's tiles (host: in 31 bits)

    if (warp == 0 && lane == 0) {
        // ---------------- copies ----------------
        dev::tma_prefetch_descriptor(&map_x);
        dev::tma_prefetch_descriptor(&map_w);
        int xs = 0, ws = 0;
        uint32_t x_phase = 0, w_phase = 0;
        bool ok = true;
        for (int tile = tile0; tile < s.total_tiles && ok; tile += tile_step) {
            const int m_block = tile / s.n_tiles;
            const int n_block = tile - m_block * s.n_tiles;
            const int col = n_block * s.out_columns;
            for (int kb = k_first; kb < k_end; ++kb) {
                if (!dev::mbar_wait(w_empty(ws), w_phase ^ 1u, s.status)) {
                    ok = false;
                    break;
                }
                dev::mbar_arrive_expect_tx(w_full(ws), s.block_n * kRowBytes);
                const uint32_t w_at = base + kWOffset + ws * kWBytes;
                const int cw[2] = {kb * kBlockK, col};
                dev::tma_load(w_at, &map_w, w_full(ws), 2, cw);
                if (p.gated) {
                    const int cu[2] = {kb * kBlockK, p.n + col};
                    dev::tma_load(w_at + s.out_columns * kRowBytes, &map_w, w_full(ws), 2, cu);
                }
                if (++ws == kW) {
                    ws = 0;
                    w_phase ^= 1u;
                }
                if (!dev::mbar_wait(x_empty(xs), x_phase ^ 1u, s.status)) {
                    ok = false;
                    break;
                }
                dev::mbar_arrive_expect_tx(x_full(xs), kXBytes);
                const int cx[2] = {kb * kBlockK, m_block * kBlockM};
                dev::tma_load(base + xs * kXBytes, &map_x, x_full(xs), 2, cx);
                if (++xs == kX) {
                    xs = 0;
                    x_phase ^= 1u;
                }
            }
        }
        if (!ok) {
            // Every load issued lands before the CTA exits.
            for (int i = 0; i < kW; ++i) {
                dev::mbar_drain_wait(w_full(i), w_phase ^ (i < ws ? 0u : 1u));
            }
            for (int i = 0; i < kX; ++i) {
                dev::mbar_drain_wait(x_full(i), x_phase ^ (i < xs ? 0u : 1u));
            }
        }
    } else if (warp == 1) {
        // ---------------- products: the warp stays together, one lane issues ----------------
        const uint32_t idesc = dev::make_idesc(2u, kBlockM, s.block_n, false, false);
        const uint32_t w0 = __shfl_sync(0xFFFFFFFFu, base, 0);
        const uint32_t tmem0 = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        int ws = 0, split = 0, acc = 0;
        uint32_t split_phase = 0, acc_phase = 0;
        bool ok = true;
        for (int tile = 0; tile < my_tiles && ok; ++tile) {
            for (int kb = 0; kb < k_blocks; ++kb) {
                const uint32_t sums = tmem0 + acc * kSumPitch;
                const bool first = kb % kChunk == 0;
                if ((first && !dev::mbar_wait_warp(acc_empty(acc), acc_phase ^ 1u, s.status)) ||
                    !dev::mbar_wait_warp(split_full(split), split_phase, s.status)) {
                    ok = false;
                    break;
                }
                dev::tc_fence_after();
                const uint64_t hi =
                    dev::smem_desc_sw128(w0 + kWOffset + ws * kWBytes, 16, 1024);
                const uint64_t lo =
                    dev::smem_desc_sw128(w0 + kLowOffset + split * kWBytes, 16, 1024);
                const uint32_t x_hi = tmem0 + kTmemX + split * 2 * kBlockK;
#pragma unroll
                for (int kk = 0; kk < kBlockK / 8; ++kk) { // 32 bytes on: 2 in a descriptor
                    dev::mma_ts_tf32_warp(sums, x_hi + kBlockK + kk * 8, hi + 2 * kk, idesc,
                                          !first || kk > 0 ? 1u : 0u);
                    dev::mma_ts_tf32_warp(sums, x_hi + kk * 8, lo + 2 * kk, idesc, 1u);
                    dev::mma_ts_tf32_warp(sums, x_hi + kk * 8, hi + 2 * kk, idesc, 1u);
                }
                dev::tc_commit_warp(w_empty(ws));
                dev::tc_commit_warp(split_empty(split));
                if (kb % kChunk == kChunk - 1 || kb == k_blocks - 1) {
                    dev::tc_commit_warp(acc_full(acc));
                    acc ^= 1;
                    acc_phase ^= acc == 0 ? 1u : 0u;
                }
                ws = ws + 1 == kW ? 0 : ws + 1;
                if (++split == kSplit) {
                    split = 0;
                    split_phase ^= 1u;
                }
            }
        }
        if (!ok) {
            // No product still reads or writes when the CTA ends.
            dev::tc_commit_warp(drain_bar);
            dev::mbar_drain_wait(drain_bar, 0);
        }
    } else if (warp >= kDrainWarp && warp < kSplitXWarp) {
        // ---------------- sums and outputs ----------------
        const int quarter = warp & 3;
        const int part = (warp - kDrainWarp) / 4;
        float* const slab =
            reinterpret_cast<float*>(smem + kSlabOffset + (warp - kDrainWarp) * kSlabBytes);
        // This warp's groups of 16 accumulator columns: consecutive ones, or for a gated layer
        // one of the gate and the same of up.
        const int groups = s.block_n / kGroup;
        const int each = (groups + kParts - 1) / kParts;
        const int from0 = (p.gated ? part : part * each) * kGroup;
        const int from_step = (p.gated ? groups / 2 : 1) * kGroup;
        const int count = p.gated ? (part < groups / 2 ? 2 : 0) : min(each, groups - part * each);
        const uint32_t sums = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int tile = tile0; tile < s.total_tiles && ok; tile += tile_step) {
            float v[kGroups][kGroup];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                for (int j = 0; j < kGroup; ++j) {
                    v[g][j] = 0.0F;
                }
            }
            for (int kb = 0; kb < k_blocks; kb += kChunk) {
                if (!dev::mbar_wait_warp(acc_full(acc), acc_phase, s.status)) {
                    ok = false;
                    break;
                }
                dev::tc_fence_after();
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    if (g < count) { // warp-uniform
                        uint32_t part_sums[kGroup];
                        dev::tmem_load_16(sums + acc * kSumPitch + from0 + g * from_step,
                                          part_sums);
                        dev::tmem_wait_load_of(part_sums);
#pragma unroll
                        for (int j = 0; j < kGroup; ++j) {
                            v[g][j] += __uint_as_float(part_sums[j]);
                        }
                    }
                }
                dev::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    dev::mbar_arrive(acc_empty(acc));
                }
                acc ^= 1;
                acc_phase ^= acc == 0 ? 1u : 0u;
            }
            if constexpr (Sliced) {
                // The only tile: its sums go to the CTA that owns the row, into the stages' place.
                dev::cluster_sync(); // no CTA's stages are in use any more
                const int row = quarter * 32 + lane;
                const int owned = kBlockM / slices;
                const int owner = row / owned;
                const uint32_t part =
                    dev::map_to_rank(base, owner) +
                    4u * ((slice * owned + row - owner * owned) * (s.block_n + kPartPad));
                const bool live = ok && tile / s.n_tiles * kBlockM + row < p.m;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                    for (int q = 0; q < kGroup / 4; ++q) {
                        if (g < count && live) {
                            const float four[4] = {v[g][4 * q], v[g][4 * q + 1], v[g][4 * q + 2],
                                                   v[g][4 * q + 3]};
                            store_remote(part + 4u * (from0 + g * from_step + 4 * q), four);
                        }
                    }
                }
                break;
            }
            if (!ok) {
                break;
            }
            const int m_block = tile / s.n_tiles;
            const int n_block = tile - m_block * s.n_tiles;
            const int row0 = m_block * kBlockM + quarter * 32;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int col0 = n_block * s.out_columns + from0 + g * from_step;
                if (g >= count || (p.gated && g > 0) || col0 >= p.n || row0 >= p.m) {
                    continue; // warp-uniform
                }
                if (p.bias != nullptr) {
                    with_columns<false>(v[g], p.bias, col0, p.n, s.columns_ok);
                }
                activate_group(p.activation, v[g]);
                if (g == 0 && p.gated) {
                    if (p.bias != nullptr) {
                        with_columns<false>(v[1], p.bias + p.n, col0, p.n,
                                            s.columns_ok && p.n % 4 == 0);
                    }
#pragma unroll
                    for (int j = 0; j < kGroup; ++j) {
                        v[g][j] *= v[1][j];
                    }
                }
                if (p.scale != nullptr) {
                    with_columns<true>(v[g], p.scale, col0, p.n, s.columns_ok);
                }
                // A row per lane becomes eight rows of four lanes, half of the rows at a time.
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    __syncwarp(); // the previous half's reads
                    if (lane / kSlabRows == half) {
#pragma unroll
                        for (int q = 0; q < kGroup / 4; ++q) {
                            *reinterpret_cast<float4*>(slab + lane % kSlabRows * kSlabPitch +
                                                       4 * q) =
                                make_float4(v[g][4 * q], v[g][4 * q + 1], v[g][4 * q + 2],
                                            v[g][4 * q + 3]);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < kSlabRows / 8; ++i) {
                        const int r = 8 * i + lane / 4;
                        const int c = 4 * (lane % 4);
                        const float4 sums =
                            *reinterpret_cast<const float4*>(slab + r * kSlabPitch + c);
                        const float four[4] = {sums.x, sums.y, sums.z, sums.w};
                        const int row = row0 + half * kSlabRows + r;
                        const int valid = min(4, p.n - col0 - c);
                        if (row < p.m && valid > 0) {
                            write_four(s, row, col0 + c, four, valid);
                        }
                    }
                }
            }
        }
    } else if (warp >= kSplitXWarp && warp < kSplitWWarp) {
        // ---------------- x's halves ----------------
        const int row = threadIdx.x - 32 * kSplitXWarp; // of the tile, and tensor memory's lane
        const uint32_t halves =
            tmem + kTmemX + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        int xs = 0, split = 0;
        uint32_t x_phase = 0, split_phase = 0;
        for (int step = 0; step < steps; ++step) {
            if (!dev::mbar_wait_warp(x_full(xs), x_phase, s.status) ||
                !dev::mbar_wait_warp(split_empty(split), split_phase ^ 1u, s.status)) {
                break;
            }
            dev::tc_fence_after(); // the products that read this stage
            const uint32_t from = base + xs * kXBytes + row * kRowBytes;
            const auto at = [&](int q) { return from + ((q ^ (row & 7)) << 4); };
            float x[2][4][4];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                dev::ld_shared_v4(at(q), x[q / 4][q % 4]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float hi[4][4];
                uint64_t check = 0u;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    dev::split4(x[h][q], hi[q], check);
                }
                if (dev::any_special(check)) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float again[4]; // lo has taken x's place
                        dev::ld_shared_v4(at(4 * h + q), again);
                        dev::split4_checked(again, hi[q], x[h][q]);
                    }
                }
                const uint32_t to = halves + split * 2 * kBlockK + 16 * h;
                dev::tmem_store_floats(to, hi);
                dev::tmem_store_floats(to + kBlockK, x[h]);
            }
            dev::tmem_wait_store();
            dev::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(x_empty(xs));
                dev::mbar_arrive(split_full(split));
            }
            if (++xs == kX) {
                xs = 0;
                x_phase ^= 1u;
            }
            if (++split == kSplit) {
                split = 0;
                split_phase ^= 1u;
            }
        }
    } else if (warp >= kSplitWWarp) {
        // ---------------- the weight's halves ----------------
        const int t = threadIdx.x - 32 * kSplitWWarp;
        const int rounds = s.block_n / 16; // 16-byte vectors per thread
        constexpr int kBatch = 3;
        int ws = 0, split = 0;
        uint32_t w_phase = 0, split_phase = 0;
        for (int step = 0; step < steps; ++step) {
            if (!dev::mbar_wait_warp(w_full(ws), w_phase, s.status) ||
                !dev::mbar_wait_warp(split_empty(split), split_phase ^ 1u, s.status)) {
                break;
            }
            const uint32_t hi_at = base + kWOffset + ws * kWBytes + 16u * t;
            const uint32_t lo_at = base + kLowOffset + split * kWBytes + 16u * t;
            float next[kBatch][4];
            const auto load = [&](int first) {
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    if (first + q < rounds) {
                        dev::ld_shared_v4(hi_at + 2048u * (first + q), next[q]);
                    }
                }
            };
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
                next[q][0] = next[q][1] = next[q][2] = next[q][3] = 0.0F;
            }
            load(0);
#pragma unroll 1
            for (int first = 0; first < rounds; first += kBatch) {
                float w[kBatch][4], hi[kBatch][4];
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[q][j] = next[q][j];
                    }
                }
                load(first + kBatch);
                uint64_t check = 0u;
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    dev::split4(w[q], hi[q], check);
                }
                if (dev::any_special(check)) {
#pragma unroll
                    for (int q = 0; q < kBatch; ++q) {
                        if (first + q < rounds) {
                            float again[4];
                            dev::ld_shared_v4(hi_at + 2048u * (first + q), again);
                            dev::split4_checked(again, hi[q], w[q]);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    if (first + q < rounds) {
                        dev::st_shared_v4(hi_at + 2048u * (first + q), hi[q]);
                        dev::st_shared_v4(lo_at + 2048u * (first + q), w[q]);
                    }
                }
            }
            dev::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(split_full(split));
            }
            if (++ws == kW) {
                ws = 0;
                w_phase ^= 1u;
            }
            if (++split == kSplit) {
                split = 0;
                split_phase ^= 1u;
            }
        }
    }

    __syncwarp(); // lanes of the copying and issuing warps come together
    if constexpr (Sliced) {
        if (warp < kDrainWarp || warp >= kSplitXWarp) {
            dev::cluster_sync(); // the draining warps' first
        }
        __syncwarp();
        dev::cluster_sync(); // all slices are here
        const float* const parts = reinterpret_cast<const float*>(smem);
        const int owned = kBlockM / slices;
        const int pitch = s.block_n + kPartPad;
        const int vectors = s.out_columns / 4;
        const int m_block = tile0 / s.n_tiles;
        const int col0 = (tile0 - m_block * s.n_tiles) * s.out_columns;
        const int row0 = m_block * kBlockM + slice * owned;
        const int rows = min(owned, p.m - row0);
        for (int i = threadIdx.x; i < rows * vectors; i += kThreads) {
            const int row = i / vectors;
            const int at = 4 * (i - row * vectors);
            finish_four(s, row0 + static_cast<long long>(row), col0 + at, at, s.out_columns + at,
                        [&](int from, float(&v)[4]) {
                            sum_slices(parts + row * pitch + from, slices, owned * pitch, v);
                        });
        }
    }
    dev::tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        dev::tc_fence_after();
        dev::tmem_dealloc(tmem, kTmemColumns);
    }
}

// Columns of a tile and slices of k: what takes least time, a tile's 32 of k taking the shared-memory
// cycles counted above (256 for x, 7 per column), but 1200 at least, the length of the chain from
// copies to products. 1576 x 1536 outputs: 143 tiles of 144 columns, one wave, where 128 columns
// leave 156 tiles and a second wave of eight. 16 x 4096 with k = 4096: 32 tiles of 128 columns, 4
// CTAs to each, 41 us (one to each of 128 tiles of 32 columns: 93).
void choose_shape(long long row_blocks, int n, bool gated, int k_blocks, int sm_count,
                  const ClusterLimits& limits, int* block_n, int* slices) {
    long long best_cost = 0;
    *block_n = 0;
    for (int bn = gated ? kMaxGatedN : kMaxN; bn > 0; bn -= gated ? 32 : 16) {
        const int columns = gated ? bn / 2 : bn;
        const long long tiles = row_blocks * ((n + columns - 1LL) / columns);
        int parts = 1;
        for (int i = 1; i < 4 && tiles <= limits.of[i] && k_blocks >= kMinSteps << i; ++i) {
            parts = 1 << i;
        }
        const long long step = 256 + 7 * bn > 1200 ? 256 + 7 * bn : 1200;
        const long long waves = (tiles * parts + sm_count - 1) / sm_count;
        // The exchange costs about as much as two steps.
        const long long cost =
            waves * ((k_blocks + parts - 1) / parts + (parts > 1 ? 2 : 0)) * step;
        if (*block_n == 0 || cost < best_cost) {
            *block_n = bn;
            *slices = parts;
            best_cost = cost;
        }
    }
}

} // namespace

bool launch_split(const Params& p, const host::DeviceContext& context, cudaStream_t stream,
                  int* result) {
    if (!host::is_blackwell(context) || p.k == 0) {
        return false;
    }
    const long long row_blocks = (p.m + kBlockM - 1LL) / kBlockM;
    SplitParams s{};
    s.p = p;
    s.k_blocks = (p.k + kBlockK - 1) / kBlockK;
    choose_shape(row_blocks, p.n, p.gated != 0, s.k_blocks, context.sm_count,
                 cluster_limits<&linear_split_kernel<true>>(kThreads, kSmemBytes), &s.block_n,
                 &s.slices);
    s.out_columns = p.gated ? s.block_n / 2 : s.block_n;
    const long long n_tiles = (p.n + s.out_columns - 1LL) / s.out_columns;
    const long long total = row_blocks * n_tiles;
    s.n_tiles = static_cast<int>(n_tiles);
    s.total_tiles = static_cast<int>(total);
    const long long tiles_each = (total + context.sm_count - 1) / context.sm_count;
    CUtensorMap map_x, map_w;
    if (total + context.sm_count > 0x7FFFFFFFLL || tiles_each > 0x7FFFFFFFLL / s.k_blocks ||
        !describe(p.x, false, p.k, p.m, p.ldx, kBlockM, &map_x) ||
        !describe(p.w, false, p.k, p.n * (p.gated ? 2LL : 1LL), p.ldw, s.out_columns, &map_w)) {
        return false;
    }
    const int out_bytes = p.out_kind == CUVIT_DTYPE_BF16 ? 2 : 4;
    s.out_vector = access_bytes(p.out, p.ldo * out_bytes);
    s.residual_vector = p.residual != nullptr ? access_bytes(p.residual, p.ldr * out_bytes) : 16;
    s.columns_ok = reinterpret_cast<uintptr_t>(p.bias) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.scale) % 16 == 0;
    s.status = context.status;
    const auto start = [&]() -> int {
        const long long blocks =
            s.slices > 1 ? total * s.slices : (total < context.sm_count ? total : context.sm_count);
        if (s.slices == 1) {
            CUVIT_TRY_CUDA(host::allow_dynamic_smem(
                reinterpret_cast<const void*>(&linear_split_kernel<false>), kSmemBytes));
        }
        launch_cluster(s.slices > 1 ? &linear_split_kernel<true> : &linear_split_kernel<false>,
                       s.slices, static_cast<unsigned>(blocks), kThreads, kSmemBytes, stream, map_x,
                       map_w, s);
        return host::after_launch("linear_split_kernel");
    };
    *result = start();
    return true;
}

} // namespace cuvit::linear
