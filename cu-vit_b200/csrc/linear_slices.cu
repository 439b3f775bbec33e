// bfloat16 linear layers with too few output tiles to fill the GPU (a few hundred rows and fewer):
// a cluster of 2, 4 or 8 CTAs shares a tile, each going through its slice of k, and adds up the
// slices over distributed shared memory.
//
// Bound by latency: with one CTA per tile, 64 columns of a weight of 4096 x 4096 come through one
// SM's copies, 64 steps of about 0.25 us. Divided, every SM streams its part of the weight. Each
// CTA's sums leave tensor memory for the CTA that owns their columns, which adds the slices in the
// order of k, in FP32, and finishes its columns (bias, activation, gate, scale, residual, rounding).
//
// 16 x 4096 x 4096: 18.5 us (28.7 with one CTA per tile, 20.5 with six stages of fixed size: what is in
// flight bounds it, so a stage holds only the rows of x that there are); 64 x 1280 x 1280 12.2 us
// (16.4), of which about 8 are launch, exchange and end: calls one behind another, with their host's
// share; replayed from a graph 14.1 and 7.5 us.
//
//   warp 0      copies (TMA) into a ring of stages
//   warp 1      issues the products
//   warp 2      tensor memory
//   warps 4-7   hand the sums out (a row per thread); then all warps finish the owned columns
#include "activation.cuh"
#include "linear.hpp"
#include "ptx.cuh"

#include <cuda_bf16.h>

#include <cstdint>

namespace cuvit::linear {
namespace {

constexpr int kBlockM = 128;
constexpr int kBlockK = 64; // 128 bytes of a row
constexpr int kRowBytes = 128;
constexpr int kThreads = 256;
constexpr int kHandOut = 4; // the first of four warps that read tensor memory
constexpr int kMaxStages = 16;
constexpr int kMaxSlices = 8;
constexpr int kMinSteps = 4; // of k in a slice

// N: accumulator columns; of a gated layer half gate and half up. A stage holds the rows of x that
// there are, then N of the weight. The products read 128 rows of x all the same: what follows in
// shared memory makes rows of the sums that nobody reads.
template <int N>
struct Shape {
    static constexpr int kWBytes = N * kRowBytes;
    static constexpr int kRingBytes = (N == 64 ? 6 : 4) * (kBlockM * kRowBytes + kWBytes);
    static constexpr int kPartOffset = kRingBytes;
    // The owned columns' sums of every slice: rows of N / slices floats and one vector between rows,
    // so that neighbouring rows fall in different banks.
    static constexpr int kPartBytes = 4 * kBlockM * (N + 4 * kMaxSlices);
    static constexpr int kBarrierOffset = kPartOffset + kPartBytes;
    static constexpr int kBarriers = 2 * kMaxStages + 2;
    static constexpr int kSmemBytes = 1024 + kBarrierOffset + 8 * kBarriers + 8;
    static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
    static_assert(kPartBytes >= kBlockM * kRowBytes, "the last stage's reads of x stay inside");
};

struct SliceParams : OutRows {
    int out_columns; // of a tile: N, or half of it for a gated layer
    int n_tiles, k_blocks;
    int slices;
    int x_rows; // rows of x a stage holds
    int stages;
    unsigned* status;
};

template <int N>
__global__ void __launch_bounds__(kThreads, 1)
    linear_slices_kernel(const __grid_constant__ CUtensorMap map_x,
                         const __grid_constant__ CUtensorMap map_w,
                         const __grid_constant__ SliceParams s) {
    using S = Shape<N>;
    constexpr int kWBytes = S::kWBytes;
    constexpr int kPartOffset = S::kPartOffset;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = dev::smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_base);
    const uint32_t bars = base + S::kBarrierOffset;
    const auto full = [&](int i) -> uint32_t { return bars + 8u * i; };
    const auto empty = [&](int i) -> uint32_t { return bars + 8u * (kMaxStages + i); };
    const uint32_t sums_full = bars + 8u * 2 * kMaxStages;
    const uint32_t drain_bar = sums_full + 8u;
    uint32_t* const tmem_slot =
        reinterpret_cast<uint32_t*>(smem + S::kBarrierOffset + 8 * S::kBarriers);
    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < s.stages; ++i) {
            dev::mbar_init(full(i), 1);
            dev::mbar_init(empty(i), 1);
        }
        dev::mbar_init(sums_full, 1);
        dev::mbar_init(drain_bar, 1);
        dev::fence_barrier_init();
    }
    if (warp == 2) {
        dev::tmem_alloc(dev::smem_u32(tmem_slot), N);
        dev::tmem_relinquish();
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    dev::cluster_sync(); // every CTA of the cluster runs before any writes to another's memory
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();

    const Params& p = s.p;
    const int rank = static_cast<int>(dev::cluster_ctarank());
    const int tile = static_cast<int>(blockIdx.x) / s.slices;
    const int m_block = tile / s.n_tiles;
    const int col0 = (tile - m_block * s.n_tiles) * s.out_columns;
    const int first = static_cast<int>(static_cast<long long>(s.k_blocks) * rank / s.slices);
    const int end = static_cast<int>(static_cast<long long>(s.k_blocks) * (rank + 1) / s.slices);
    const int owned = s.out_columns / s.slices; // columns of the output that a CTA finishes
    const int pitch = N / s.slices + 4;   // floats
    const int rows = min(kBlockM, p.m - m_block * kBlockM);
    const int x_bytes = s.x_rows * kRowBytes;
    const int stage_bytes = x_bytes + kWBytes;

    if (warp == 0 && lane == 0) {
        // ---------------- copies ----------------
        dev::tma_prefetch_descriptor(&map_x);
        dev::tma_prefetch_descriptor(&map_w);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = first; kb < end; ++kb) {
            ok = dev::mbar_wait(empty(stage), phase ^ 1u, s.status);
            if (!ok) {
                break;
            }
            dev::mbar_arrive_expect_tx(full(stage), stage_bytes);
            const uint32_t at = base + stage * stage_bytes;
            const int cw[2] = {kb * kBlockK, col0};
            dev::tma_load(at + x_bytes, &map_w, full(stage), 2, cw);
            if (p.gated) {
                const int cu[2] = {kb * kBlockK, p.n + col0};
                dev::tma_load(at + x_bytes + kWBytes / 2, &map_w, full(stage), 2, cu);
            }
            const int cx[2] = {kb * kBlockK, m_block * kBlockM};
            dev::tma_load(at, &map_x, full(stage), 2, cx);
            if (++stage == s.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (!ok) {
            // Every load issued lands before the CTA exits.
            for (int i = 0; i < s.stages; ++i) {
                dev::mbar_drain_wait(full(i), phase ^ (i < stage ? 0u : 1u));
            }
        }
    } else if (warp == 1) {
        // ---------------- products: the warp stays together, one lane issues ----------------
        const uint32_t idesc = dev::make_idesc(1u, kBlockM, N, false, false);
        const uint32_t base0 = __shfl_sync(0xFFFFFFFFu, base, 0);
        const uint32_t tmem0 = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = first; kb < end; ++kb) {
            ok = dev::mbar_wait_warp(full(stage), phase, s.status);
            if (!ok) {
                break;
            }
            dev::tc_fence_after();
            const uint64_t x = dev::smem_desc_sw128(base0 + stage * stage_bytes, 16, 1024);
            const uint64_t w =
                dev::smem_desc_sw128(base0 + stage * stage_bytes + x_bytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < kBlockK / 16; ++kk) { // 32 bytes on: 2 in a descriptor
                dev::mma_ss_f16_warp(tmem0, x + 2 * kk, w + 2 * kk, idesc,
                                     kb > first || kk > 0 ? 1u : 0u);
            }
            dev::tc_commit_warp(empty(stage));
            if (++stage == s.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (ok) {
            dev::tc_commit_warp(sums_full);
        } else {
            // No product still reads or writes when the CTA ends.
            dev::tc_commit_warp(drain_bar);
            dev::mbar_drain_wait(drain_bar, 0);
        }
    } else if (warp >= kHandOut) {
        // ---------------- sums to their columns' owners ----------------
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        if (dev::mbar_wait_warp(sums_full, 0, s.status)) {
            dev::tc_fence_after();
            const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
            // This slice's rows in an owner's memory.
            const uint32_t part = base + kPartOffset + 4u * ((rank * kBlockM + row) * pitch);
#pragma unroll 1
            for (int c = 0; c < N; c += 16) {
                uint32_t raw[16];
                __syncwarp(); // the read is warp-wide: lanes with and without a row meet first
                dev::tmem_load_16(from + c, raw);
                dev::tmem_wait_load_of(raw);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int column = c + 4 * q; // gate and up columns of one output go together
                    const bool up = p.gated && column >= N / 2;
                    const int output = up ? column - N / 2 : column;
                    const int owner = output / owned;
                    const int at = output - owner * owned + (up ? owned : 0);
                    const float four[4] = {
                        __uint_as_float(raw[4 * q]), __uint_as_float(raw[4 * q + 1]),
                        __uint_as_float(raw[4 * q + 2]), __uint_as_float(raw[4 * q + 3])};
                    if (row < rows) {
                        store_remote(dev::map_to_rank(part + 4u * at, owner), four);
                    }
                }
            }
            dev::tc_fence_before();
        }
    }
    __syncwarp();
    dev::cluster_sync(); // all slices are here

    // ---------------- the owned columns ----------------
    const float* const parts = reinterpret_cast<const float*>(smem + kPartOffset);
    const int vectors = owned / 4;
    for (int i = threadIdx.x; i < rows * vectors; i += kThreads) {
        const int row = i / vectors;
        const int at = 4 * (i - row * vectors);
        finish_four(s, static_cast<long long>(m_block) * kBlockM + row, col0 + rank * owned + at, at,
                    owned + at, [&](int from, float(&v)[4]) {
                        sum_slices(parts + row * pitch + from, s.slices, kBlockM * pitch, v);
                    });
    }

    dev::tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        dev::tc_fence_after();
        dev::tmem_dealloc(tmem, N);
    }
}

} // namespace

// A step of 64 of k takes 0.32, 0.34 or 0.45 us with 64, 128 or 256 columns (a tile per SM, 128 rows:
// 1024 x 4096 x 4096 takes 89, 51 and 37 us in 4, 2 and 1 waves), and an exchange of slices as
// much as three steps and one for every 1000 sums of a tile. 700 x 1280 x 5120: 60 tiles of 128
// columns and two slices, 27 us (33 with one CTA to each of 120 tiles of 64).
TileChoice choose_tiles(const Params& p, const host::DeviceContext& context) {
    const long long row_blocks = (p.m + kBlockM - 1LL) / kBlockM;
    const int k_blocks = (p.k + kBlockK - 1) / kBlockK;
    const auto tiles_of = [&](int bn) {
        const int columns = p.gated ? bn / 2 : bn;
        return row_blocks * ((p.n + columns - 1LL) / columns);
    };
    const auto step = [](int bn) { return bn == 64 ? 0.32 : (bn == 128 ? 0.34 : 0.45); };
    TileChoice choice{256, 1, 0};
    double best = 0.0;
    for (const int bn : {256, 128, 64}) {
        if (p.gated && bn == 64) {
            continue; // half a tile's columns of one operand stay a whole 32-column step
        }
        const long long waves = (tiles_of(bn) + context.sm_count - 1) / context.sm_count;
        const double cost = static_cast<double>(waves) * k_blocks * step(bn);
        if (best == 0.0 || cost < best) {
            best = cost;
            choice.block_n = bn;
        }
    }
    for (const int bn : {128, 64}) {
        const long long tiles = tiles_of(bn);
        if (tiles * 2 > context.sm_count) {
            continue;
        }
        const ClusterLimits limits =
            bn == 64 ? cluster_limits<&linear_slices_kernel<64>>(kThreads, Shape<64>::kSmemBytes)
                     : cluster_limits<&linear_slices_kernel<128>>(kThreads, Shape<128>::kSmemBytes);
        for (int i = 1; i < 4 && tiles <= limits.of[i] && k_blocks >= kMinSteps << i; ++i) {
            const double exchange = 3.0 + 1.0e-3 * bn * (p.m < kBlockM ? p.m : kBlockM);
            const double cost = (((k_blocks - 1) >> i) + 1 + exchange) * step(bn);
            if (cost < best) {
                best = cost;
                choice.slices = 1 << i;
                choice.slice_n = bn;
            }
        }
    }
    return choice;
}

bool launch_slices(const Params& p, const TileChoice& choice, const host::DeviceContext& context,
                   cudaStream_t stream, int* result) {
    SliceParams s{};
    s.p = p;
    s.slices = choice.slices;
    s.out_columns = p.gated ? choice.slice_n / 2 : choice.slice_n;
    const long long row_blocks = (p.m + kBlockM - 1LL) / kBlockM;
    const long long n_tiles = (p.n + s.out_columns - 1LL) / s.out_columns;
    const long long tiles = row_blocks * n_tiles; // no more than clusters fit the GPU
    s.k_blocks = (p.k + kBlockK - 1) / kBlockK;
    s.n_tiles = static_cast<int>(n_tiles);
    s.x_rows = p.m < kBlockM ? (p.m + 7) / 8 * 8 : kBlockM;
    CUtensorMap map_x, map_w;
    if (!describe(p.x, true, p.k, p.m, p.ldx, s.x_rows, &map_x) ||
        !describe(p.w, true, p.k, p.n * (p.gated ? 2LL : 1LL), p.ldw, s.out_columns, &map_w)) {
        return false;
    }
    const int out_bytes = p.out_kind == CUVIT_DTYPE_BF16 ? 2 : 4;
    s.out_vector = access_bytes(p.out, p.ldo * out_bytes);
    s.residual_vector = p.residual != nullptr ? access_bytes(p.residual, p.ldr * out_bytes) : 16;
    s.status = context.status;
    const auto start = [&](auto* kernel, int ring_bytes, int w_bytes, int smem_bytes) {
        const int stages = ring_bytes / (s.x_rows * kRowBytes + w_bytes);
        s.stages = stages < kMaxStages ? stages : kMaxStages;
        launch_cluster(kernel, s.slices, static_cast<unsigned>(tiles * s.slices), kThreads,
                       smem_bytes, stream, map_x, map_w, s);
        return host::after_launch("linear_slices_kernel");
    };
    *result = choice.slice_n == 64
                  ? start(&linear_slices_kernel<64>, Shape<64>::kRingBytes, Shape<64>::kWBytes,
                          Shape<64>::kSmemBytes)
                  : start(&linear_slices_kernel<128>, Shape<128>::kRingBytes, Shape<128>::kWBytes,
                          Shape<128>::kSmemBytes);
    return true;
}

} // namespace cuvit::linear
