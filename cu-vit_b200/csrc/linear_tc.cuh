// Linear layers on the tcgen05 GEMM kernels: their parameters and the epilogue that turns an
// accumulator tile into out = residual + scale * act(y + bias) [* (up + bias)].
//
// Each epilogue warp takes 32 rows of the tile, a slab row (128 bytes) of columns at a time. The
// residual's chunk is brought into the slab while the accumulator is read and activated, each lane
// adds its own row there in FP32 and writes the rounded row back, and the chunk leaves by TMA.
// Rows that TMA cannot describe (a row distance that is no multiple of 16 bytes: 3420 bfloat16
// columns) move between global memory and the slab with the widest vectors their alignment allows,
// consecutive lanes on consecutive bytes of a row.
//
// 50432 x 768 x 768 bfloat16: 51.1 us without any of it (a library product: 50.1), bias 52.5, bias and
// scale 55.0, with the residual 62.7; 16411 x 3420 x 1280 gated SiLU 205 us, 1400 TFLOP/s. (A second
// slab per warp, with the next chunk of the residual on its way while one is added, in place of one
// of six operand stages: 64.2 us.)
#pragma once

#include "activation.cuh"
#include "gemm_tc.cuh"

namespace cuvit::gemm {

struct LinearParams : TcParams {
    static constexpr bool kLinear = true;
    int activation; // cuvit_activation
    int gated;
    const float* scale;
    int scale_vector_ok;
    int up_vector_ok; // bias + n is 16-byte aligned
    const void* residual;
    long long ldr;
    int residual_tma;
    int out_vector;      // bytes per access of out / residual rows on the copied path
    int residual_vector;
    CUtensorMap map_residual;
};

// Copies 32 rows of row_bytes (64 or 128) between a slab (16-byte chunk j of row r at chunk
// j ^ (r % 8)) and global rows of which `rows` and valid_bytes exist, Vec bytes at a time.
template <int Vec, bool ToGlobal>
__device__ __forceinline__ void copy_rows(uint8_t* slab, uint8_t* global, long long pitch, int rows,
                                          int row_bytes, int valid_bytes, int element, int lane) {
    const int units = row_bytes / Vec;
    const int shift = 31 - __clz(units);
#pragma unroll 4
    for (int i = lane; i < 32 * units; i += 32) {
        const int r = i >> shift;
        const int byte = (i & (units - 1)) * Vec;
        uint8_t* const at = slab + r * kSwizzleBytes + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
        uint8_t* const far = global + r * pitch + byte;
        if (r >= rows || byte >= valid_bytes) {
            continue;
        }
        if (byte + Vec <= valid_bytes) {
            const auto move = [&](auto* to, const auto* from) { *to = *from; };
            if constexpr (Vec == 16) {
                ToGlobal ? move(reinterpret_cast<uint4*>(far), reinterpret_cast<uint4*>(at))
                         : move(reinterpret_cast<uint4*>(at), reinterpret_cast<uint4*>(far));
            } else if constexpr (Vec == 8) {
                ToGlobal ? move(reinterpret_cast<uint2*>(far), reinterpret_cast<uint2*>(at))
                         : move(reinterpret_cast<uint2*>(at), reinterpret_cast<uint2*>(far));
            } else if constexpr (Vec == 4) {
                ToGlobal ? move(reinterpret_cast<uint32_t*>(far), reinterpret_cast<uint32_t*>(at))
                         : move(reinterpret_cast<uint32_t*>(at), reinterpret_cast<uint32_t*>(far));
            } else {
                ToGlobal ? move(reinterpret_cast<uint16_t*>(far), reinterpret_cast<uint16_t*>(at))
                         : move(reinterpret_cast<uint16_t*>(at), reinterpret_cast<uint16_t*>(far));
            }
        } else { // the row ends inside this access
            for (int b = 0; byte + b < valid_bytes; b += element) {
                if (element == 4) {
                    auto* const near4 = reinterpret_cast<uint32_t*>(at + b);
                    auto* const far4 = reinterpret_cast<uint32_t*>(far + b);
                    ToGlobal ? *far4 = *near4 : *near4 = *far4;
                } else {
                    auto* const near2 = reinterpret_cast<uint16_t*>(at + b);
                    auto* const far2 = reinterpret_cast<uint16_t*>(far + b);
                    ToGlobal ? *far2 = *near2 : *near2 = *far2;
                }
            }
        }
    }
}

template <bool ToGlobal>
__device__ __forceinline__ void copy_rows(int vector, uint8_t* slab, uint8_t* global,
                                          long long pitch, int rows, int row_bytes, int valid_bytes,
                                          int element, int lane) {
    switch (vector) {
    case 16:
        copy_rows<16, ToGlobal>(slab, global, pitch, rows, row_bytes, valid_bytes, element, lane);
        break;
    case 8:
        copy_rows<8, ToGlobal>(slab, global, pitch, rows, row_bytes, valid_bytes, element, lane);
        break;
    case 4:
        copy_rows<4, ToGlobal>(slab, global, pitch, rows, row_bytes, valid_bytes, element, lane);
        break;
    default:
        copy_rows<2, ToGlobal>(slab, global, pitch, rows, row_bytes, valid_bytes, element, lane);
        break;
    }
}

// v[j] op= vector[col0 + j] for the columns below n.
template <bool Multiply>
__device__ __forceinline__ void apply_columns(float (&v)[32], const float* vector, int col0, int n,
                                              bool vector_ok) {
    if (vector_ok && col0 + 32 <= n) {
        const float4* const four = reinterpret_cast<const float4*>(vector + col0);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float4 b = __ldg(four + q);
            const uint64_t lo = dev::f32x2(v[4 * q], v[4 * q + 1]);
            const uint64_t hi = dev::f32x2(v[4 * q + 2], v[4 * q + 3]);
            const uint64_t b_lo = dev::f32x2(b.x, b.y);
            const uint64_t b_hi = dev::f32x2(b.z, b.w);
            const float2 l =
                dev::f32x2_split(Multiply ? dev::mul_f32x2(lo, b_lo) : dev::add_f32x2(lo, b_lo));
            const float2 h =
                dev::f32x2_split(Multiply ? dev::mul_f32x2(hi, b_hi) : dev::add_f32x2(hi, b_hi));
            v[4 * q] = l.x;
            v[4 * q + 1] = l.y;
            v[4 * q + 2] = h.x;
            v[4 * q + 3] = h.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (col0 + j < n) {
                const float b = __ldg(vector + col0 + j);
                v[j] = Multiply ? v[j] * b : v[j] + b;
            }
        }
    }
}

// The epilogue of one warp's part of a tile: rows row_base .. + 31, one half of the tile's output
// columns. False when a bounded wait gave up (no load is then in flight).
template <int BN>
__device__ bool linear_tile(const LinearParams& p, const CUtensorMap* tma_c, uint32_t tmem_cols,
                            int n_block, int row_base, int half, uint8_t* slab, uint32_t slab_addr,
                            uint32_t residual_bar, uint32_t& residual_phase, int lane) {
    const int tile_columns = p.gated ? BN / 2 : BN;
    const int warp_columns = tile_columns / 2;
    const bool bf16 = p.c_kind == 1;
    const int element = bf16 ? 2 : 4;
    const int chunk = bf16 && warp_columns >= 64 ? 64 : 32;
    const int row_bytes = chunk * element;
    const int rows = p.m - row_base; // may exceed 32, or be 0 or less
    if (rows <= 0) {
        return true; // uniform across the warp
    }
    uint4* const own = reinterpret_cast<uint4*>(slab + lane * kSwizzleBytes);
#pragma unroll 1
    for (int c = half * warp_columns; c < (half + 1) * warp_columns; c += chunk) {
        const int col0 = n_block * tile_columns + c;
        if (col0 >= p.n) {
            break; // uniform across the warp
        }
        const int valid_bytes = min(chunk, p.n - col0) * element;
        // The previous chunk must have left the slab, and ordinary accesses to it come before
        // the copy engine's.
        dev::fence_proxy_async_shared();
        if (p.c_tma && lane == 0) {
            dev::bulk_wait_group_read0();
        }
        __syncwarp();
        if (p.residual != nullptr) {
            if (p.residual_tma) {
                if (lane == 0) {
                    dev::mbar_arrive_expect_tx(residual_bar, kSlabBytes);
                    const int coords[2] = {col0, row_base};
                    dev::tma_load(slab_addr, &p.map_residual, residual_bar, 2, coords);
                }
            } else {
                copy_rows<false>(p.residual_vector, slab,
                                 static_cast<uint8_t*>(const_cast<void*>(p.residual)) +
                                     (row_base * p.ldr + col0) * element,
                                 p.ldr * element, rows, row_bytes, valid_bytes, element, lane);
                __syncwarp();
            }
        }
#pragma unroll 1
        for (int s = 0; s < chunk; s += 32) {
            float v[32];
            __syncwarp(); // the accumulator's reads are warp-wide
            load_accumulator<32, BN, false>(tmem_cols + c + s, v);
            if (p.bias != nullptr) {
                apply_columns<false>(v, p.bias, col0 + s, p.n, p.bias_vector_ok);
            }
            if (bf16) {
                dev::activate<true>(p.activation, v);
            } else {
                dev::activate<false>(p.activation, v);
            }
            if (p.gated) {
                float up[32];
                load_accumulator<32, BN, false>(tmem_cols + BN / 2 + c + s, up);
                if (p.bias != nullptr) {
                    apply_columns<false>(up, p.bias + p.n, col0 + s, p.n, p.up_vector_ok);
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    v[j] *= up[j];
                }
            }
            if (p.scale != nullptr) {
                apply_columns<true>(v, p.scale, col0 + s, p.n, p.scale_vector_ok);
            }
            if (p.residual != nullptr && p.residual_tma && s == 0) {
                const bool landed = dev::mbar_wait(residual_bar, residual_phase, p.status);
                if (!__all_sync(0xFFFFFFFFu, landed)) {
                    if (lane == 0) {
                        dev::mbar_drain_wait(residual_bar, residual_phase);
                    }
                    return false;
                }
                residual_phase ^= 1u;
            }
            if (bf16) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint4& slot = own[(s / 8 + q) ^ (lane & 7)];
                    if (p.residual != nullptr) {
                        const uint4 old = slot;
                        const uint32_t words[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[8 * q + 2 * j] += __uint_as_float(words[j] << 16);
                            v[8 * q + 2 * j + 1] += __uint_as_float(words[j] & 0xFFFF0000u);
                        }
                    }
                    slot = make_uint4(dev::pack_bf16x2(v[8 * q], v[8 * q + 1]),
                                      dev::pack_bf16x2(v[8 * q + 2], v[8 * q + 3]),
                                      dev::pack_bf16x2(v[8 * q + 4], v[8 * q + 5]),
                                      dev::pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
                }
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    uint4& slot = own[q ^ (lane & 7)];
                    if (p.residual != nullptr) {
                        const uint4 old = slot;
                        v[4 * q] += __uint_as_float(old.x);
                        v[4 * q + 1] += __uint_as_float(old.y);
                        v[4 * q + 2] += __uint_as_float(old.z);
                        v[4 * q + 3] += __uint_as_float(old.w);
                    }
                    if (p.c_kind == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[4 * q + j] = dev::round_to_tf32(v[4 * q + j]);
                        }
                    }
                    slot = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                      __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
                }
            }
        }
        if (p.c_tma) {
            dev::fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) {
                const int coords[2] = {col0, row_base};
                dev::tma_store<false>(tma_c, slab_addr, 2, coords);
                dev::bulk_commit_group();
            }
        } else {
            __syncwarp();
            copy_rows<true>(p.out_vector, slab,
                            static_cast<uint8_t*>(p.c) + (row_base * p.ldc + col0) * element,
                            p.ldc * element, rows, row_bytes, valid_bytes, element, lane);
            __syncwarp();
        }
    }
    return true;
}

} // namespace cuvit::gemm
