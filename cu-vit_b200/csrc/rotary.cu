// Rotary positions with several axes, and per-head norms of queries and keys with the rotation
// in the same pass.
//
// For a head x of token t:  y = x / sqrt(mean(x^2) + eps) * gamma + beta        (RMS)
//                           y = (x - mean) / sqrt(var + eps) * gamma + beta     (layer)
//                           y = x                                               (rotation alone)
// then each pair (y_a, y_b) of axis c turns by the angle positions[c][t] * rate, in FP32 with
// one rounding at the store. The angle is formed in fixed point: rates are kept in units of
// 2^-64 turn, so position * rate modulo 2^64 is the fraction of a turn without any range
// reduction, and no position loses accuracy (FP32 angles are off by 6e-3 rad at position 1e5).
#include "cuvit_b200.h"
#include "ptx.cuh"
#include "runtime.hpp"

#include <cuda_bf16.h>

#include <cmath>
#include <cstdint>
#include <cstring>

namespace cuvit::rotary {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 256;
constexpr int kNormNone = -1;

struct Side {
    const void* in;
    void* out;
    const float* gamma;
    const float* beta;
    long long in_stride;
    long long out_stride;
    int heads;
};

struct Params {
    Side side[2]; // queries, keys
    int tokens;
    int head_dim;
    int pairs; // rotated pairs per head
    int adjacent;
    float epsilon;
    const int* positions;
    long long position_stride;
    cuvit_rotary rotary;
};

template <typename T>
__device__ __forceinline__ float load_value(const T* p) {
    if constexpr (sizeof(T) == 2) {
        return __bfloat162float(*p);
    } else {
        return *p;
    }
}

template <typename T>
__device__ __forceinline__ void store_value(T* p, float v) {
    if constexpr (sizeof(T) == 2) {
        *p = __float2bfloat16_rn(v);
    } else {
        *p = v;
    }
}

// Elements of pair i of a head: the rotated pairs first, then what is left of the head, paired
// the same way (those turn by nothing).
__device__ __forceinline__ void pair_elements(int i, int pairs, int half_dim, int adjacent, int& a,
                                              int& b) {
    if (adjacent) {
        a = 2 * i;
        b = 2 * i + 1;
    } else if (i < pairs) {
        a = i;
        b = i + pairs;
    } else {
        a = 2 * pairs + (i - pairs);
        b = a + (half_dim - pairs);
    }
}

// cos and sin of pair i's angle at token t (1 and 0 past the rotated pairs).
__device__ __forceinline__ float2 turn_of(const Params& p, int t, int i) {
    if (i >= p.pairs) {
        return make_float2(1.0F, 0.0F);
    }
    int axis = 0;
    while (axis + 1 < p.rotary.axes && i >= p.rotary.first[axis + 1]) {
        ++axis;
    }
    const long long position = p.positions[axis * p.position_stride + t];
    const uint64_t fraction = static_cast<uint64_t>(position) * p.rotary.turns[i];
    // The top 32 bits as a signed number of half turns in [-1, 1): within 2^-25 of a half turn.
    const float half_turns =
        static_cast<float>(static_cast<int>(fraction >> 32)) * 4.656612873077393e-10F;
    float s, c;
    sincospif(half_turns, &s, &c);
    return make_float2(c, s);
}

__device__ __forceinline__ float warp_sum(float value) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        value += __shfl_xor_sync(0xFFFFFFFFu, value, offset);
    }
    return value;
}

// Any even head_dim and any alignment: one warp per head, scalar loads.
template <typename T, int Norm>
__global__ void __launch_bounds__(kThreads) qk_scalar_kernel(const __grid_constant__ Params p) {
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    const int lane = threadIdx.x % 32;
    const int heads = p.side[0].heads + p.side[1].heads;
    const long long item = static_cast<long long>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    const int t = static_cast<int>(item / heads);
    if (t >= p.tokens) {
        return; // the whole warp
    }
    int head = static_cast<int>(item - static_cast<long long>(t) * heads);
    const Side& side = head < p.side[0].heads ? p.side[0] : p.side[1];
    head -= head < p.side[0].heads ? 0 : p.side[0].heads;
    const T* const in = static_cast<const T*>(side.in) + t * side.in_stride +
                        static_cast<long long>(head) * p.head_dim;
    T* const out = static_cast<T*>(side.out) + t * side.out_stride +
                   static_cast<long long>(head) * p.head_dim;
    const int half = p.head_dim / 2;
    constexpr int kPer = kMaxHeadDim / 2 / 32;
    float x[kPer], y[kPer];
    float sum = 0.0F;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = lane + 32 * j;
        x[j] = y[j] = 0.0F;
        if (i < half) {
            int a, b;
            pair_elements(i, p.pairs, half, p.adjacent, a, b);
            x[j] = load_value(in + a);
            y[j] = load_value(in + b);
        }
        sum += x[j] + y[j];
    }
    if constexpr (Norm != kNormNone) {
        float mean = 0.0F;
        if constexpr (Norm == CUVIT_NORM_LAYER) {
            mean = warp_sum(sum) / static_cast<float>(p.head_dim);
        }
        float squares = 0.0F;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (lane + 32 * j < half) {
                x[j] -= mean;
                y[j] -= mean;
                squares = fmaf(x[j], x[j], fmaf(y[j], y[j], squares));
            }
        }
        squares = warp_sum(squares);
        const float scale = 1.0F / sqrtf(squares / static_cast<float>(p.head_dim) + p.epsilon);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = lane + 32 * j;
            if (i < half) {
                int a, b;
                pair_elements(i, p.pairs, half, p.adjacent, a, b);
                x[j] = x[j] * scale * (side.gamma != nullptr ? side.gamma[a] : 1.0F) +
                       (side.beta != nullptr ? side.beta[a] : 0.0F);
                y[j] = y[j] * scale * (side.gamma != nullptr ? side.gamma[b] : 1.0F) +
                       (side.beta != nullptr ? side.beta[b] : 0.0F);
            }
        }
    }
    __syncwarp(); // every lane has read its elements before any is written over (in place)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = lane + 32 * j;
        if (i < half) {
            int a, b;
            pair_elements(i, p.pairs, half, p.adjacent, a, b);
            if (i < p.pairs) {
                const float2 turn = turn_of(p, t, i);
                store_value(out + a, x[j] * turn.x - y[j] * turn.y);
                store_value(out + b, fmaf(x[j], turn.y, y[j] * turn.x));
            } else {
                store_value(out + a, x[j]);
                store_value(out + b, y[j]);
            }
        }
    }
}

// ---- vector kernel ------------------------------------------------------------------------
//
// Bound by HBM (each element read once and written once). A lane holds V pairs of one head: two
// vectors of V elements that turn together (V elements apart by the pairing, or next to each
// other), so the rotation needs no exchange between lanes and a norm one sum over the `chunks`
// lanes of a head, as many heads side by side in a warp as fit (6 of 5 lanes for head_dim 80; with
// heads padded to 8 lanes 3 in 8 would idle). A block takes a few tokens and first fills a table of
// their turns in shared memory: one sine and cosine per (token, pair), however many heads share it.
// Its lane groups are the heads of `slots` tokens, each going from token to token with its own head,
// so that a step is its loads, arithmetic and stores; finding a head and its gains for each of the
// heads in turn took more instructions than they. The next token's vectors are loaded before the
// current one's are used.
//
// 12544 tokens, 16 + 16 heads of 80: 26 us, 5.0 TB/s; with RMS norms, 50432 tokens, 12 + 12 heads of
// 64: 67 us, 4.6 TB/s, of 6.5 for a copy. What keeps norms from the copy's rate is the chain of sum,
// root, gains and turns in every step, which 36 warps an SM do not quite hide.
template <int Norm>
constexpr int kMaxWarps = Norm == kNormNone ? 12 : 9;
// Norms spill a little at 56 registers, but four blocks of nine warps beat three (69 and 74 us for
// 50432 tokens, 12 + 12 heads of 64); two tokens ahead instead of one, for fewer warps: 96 us.
template <int Norm>
constexpr int kMinBlocks = Norm == kNormNone ? 3 : 4;
constexpr int kTableVectors = 512; // float4 of two turns each: 8 KB
constexpr int kMaxHeads = 1 << 18; // of both sides: the second grid dimension stays in 16 bits

struct VectorShape {
    int chunks;       // lanes per head
    int warp_groups;  // heads side by side in a warp: 32 / chunks
    int heads;        // of a block (a second grid dimension goes through the others)
    int slots;        // tokens side by side in a block
    int block_tokens; // tokens of a block
    int warps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T value[V];
};

// Sum over the `count` lanes from lane `first` on, of which this is number `position`, the same in
// all of them: halves added onto halves, then handed out.
__device__ __forceinline__ float group_sum(float value, int first, int position, int count) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) {
        if (offset < count) { // the same for the launch
            const float other = __shfl_down_sync(0xFFFFFFFFu, value, offset);
            value += position + offset < count && position < offset ? other : 0.0F;
        }
    }
    return __shfl_sync(0xFFFFFFFFu, value, first);
}

// A lane's V elements as V / 2 packed pairs.
template <typename T, int V>
__device__ __forceinline__ void unpack2(const Vec<T, V>& raw, uint64_t (&out)[V / 2]) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
        if constexpr (sizeof(T) == 2) {
            uint32_t word;
            memcpy(&word, &raw.value[2 * j], 4);
            out[j] = dev::f32x2(__uint_as_float(word << 16), __uint_as_float(word & 0xFFFF0000u));
        } else {
            out[j] = dev::f32x2(raw.value[2 * j], raw.value[2 * j + 1]);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store2(T* p, const uint64_t (&in)[V / 2]) {
    Vec<T, V> raw;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
        const float2 pair = dev::f32x2_split(in[j]);
        if constexpr (sizeof(T) == 2) {
            const uint32_t word = dev::pack_bf16x2(pair.x, pair.y);
            memcpy(&raw.value[2 * j], &word, 4);
        } else {
            raw.value[2 * j] = pair.x;
            raw.value[2 * j + 1] = pair.y;
        }
    }
    *reinterpret_cast<Vec<T, V>*>(p) = raw;
}

// V consecutive floats of shared memory as pairs.
template <int V>
__device__ __forceinline__ void shared_pairs(const float* p, uint64_t (&out)[V / 2]) {
    if constexpr (V >= 4) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const ulonglong2 two = reinterpret_cast<const ulonglong2*>(p)[j];
            out[2 * j] = two.x;
            out[2 * j + 1] = two.y;
        }
    } else {
        out[0] = *reinterpret_cast<const uint64_t*>(p);
    }
}

template <typename T, int V, int Norm, bool Adjacent>
__global__ void __launch_bounds__(32 * kMaxWarps<Norm>, kMinBlocks<Norm>)
    qk_vector_kernel(const __grid_constant__ Params p, const VectorShape s) {
    __shared__ float4 table[kTableVectors];
    __shared__ __align__(16) float gains[Norm == kNormNone ? 1 : 4][kMaxHeadDim];
    dev::grid_dependency_wait();
    dev::grid_launch_dependents();
    constexpr int kPairs = V / 2;
    const int token0 = static_cast<int>(blockIdx.x) * s.block_tokens;
    const int tokens = min(s.block_tokens, p.tokens - token0);
    const int half = p.head_dim / 2;

    const int lane = threadIdx.x % 32;
    const int group_of_warp = lane / s.chunks;
    const int chunk = lane - group_of_warp * s.chunks;
    const int first_lane = group_of_warp * s.chunks;
    const int group = static_cast<int>(threadIdx.x) / 32 * s.warp_groups + group_of_warp;
    const int slot = group / s.heads;
    int head = static_cast<int>(blockIdx.y) * s.heads + group - slot * s.heads; // queries first
    const bool key = head >= p.side[0].heads;
    const Side& side = p.side[key ? 1 : 0];
    head -= key ? p.side[0].heads : 0;
    const bool in_group = group_of_warp < s.warp_groups && slot < s.slots && head < side.heads;
    int first, second; // this lane's elements
    if constexpr (Adjacent) {
        first = 2 * V * chunk;
        second = first + V;
    } else {
        pair_elements(V * chunk, p.pairs, half, 0, first, second);
    }
    const long long in_step = s.slots * side.in_stride;
    const long long out_step = s.slots * side.out_stride;
    const long long token = token0 + static_cast<long long>(slot);
    const T* in = static_cast<const T*>(side.in) + token * side.in_stride +
                  static_cast<long long>(head) * p.head_dim;
    T* out = static_cast<T*>(side.out) + token * side.out_stride +
             static_cast<long long>(head) * p.head_dim;
    Vec<T, V> x_next{}, y_next{};
    const auto load_token = [&](int t) {
        if (t < tokens && in_group) {
            x_next = *reinterpret_cast<const Vec<T, V>*>(in + first);
            y_next = *reinterpret_cast<const Vec<T, V>*>(in + second);
        }
        in += in_step;
    };
    load_token(slot);

    // Two neighbouring pairs of a token per float4, placed so that the lanes of a head read
    // consecutive vectors: chunk c's pairs 2q, 2q + 1 at q * chunks + c, as cos, cos, sin, sin for
    // pairs in two halves (whose elements are packed with their neighbours) and cos, sin, cos, sin
    // for adjacent ones.
    const int threads = 32 * s.warps;
    for (int i = threadIdx.x; i < tokens * half; i += threads) {
        const int t = i / half;
        const int pair = i - t * half;
        const int c = pair / V;
        const int within = pair - c * V;
        float* const at = reinterpret_cast<float*>(
            table + t * (half / 2) + (within / 2) * s.chunks + c);
        const float2 turn = turn_of(p, token0 + t, pair);
        at[Adjacent ? 2 * (within & 1) : within & 1] = turn.x;
        at[Adjacent ? 2 * (within & 1) + 1 : 2 + (within & 1)] = turn.y;
    }
    if constexpr (Norm != kNormNone) {
        for (int i = threadIdx.x; i < 2 * p.head_dim; i += threads) {
            const int k = i >= p.head_dim ? 1 : 0;
            const int e = i - k * p.head_dim;
            gains[2 * k][e] = p.side[k].gamma != nullptr ? p.side[k].gamma[e] : 1.0F;
            gains[2 * k + 1][e] = p.side[k].beta != nullptr ? p.side[k].beta[e] : 0.0F;
        }
    }
    __syncthreads();

    const bool offsets = p.side[0].beta != nullptr || p.side[1].beta != nullptr;
    const float inverse_dim = 1.0F / static_cast<float>(p.head_dim);
    const float4* turns = table + slot * (half / 2) + chunk;
    // Of this lane's pairs the first ones turn. The others stay what they are: turned by (1, 0), a
    // NaN or an infinity would reach its partner.
    const int turned_pairs = p.pairs - V * chunk;
    // All groups go round together: the sums need every lane of a warp.
    for (int t = slot; t - slot < tokens; t += s.slots) {
        uint64_t x[kPairs], y[kPairs];
        unpack2(x_next, x);
        unpack2(y_next, y);
        load_token(t + s.slots);
        if constexpr (Norm != kNormNone) {
            if constexpr (Norm == CUVIT_NORM_LAYER) {
                uint64_t sums = dev::add_f32x2(x[0], y[0]);
#pragma unroll
                for (int j = 1; j < kPairs; ++j) {
                    sums = dev::add_f32x2(sums, dev::add_f32x2(x[j], y[j]));
                }
                const float2 both = dev::f32x2_split(sums);
                const float mean =
                    group_sum(both.x + both.y, first_lane, chunk, s.chunks) * inverse_dim;
                const uint64_t mean2 = dev::f32x2(mean, mean);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    x[j] = dev::sub_f32x2(x[j], mean2);
                    y[j] = dev::sub_f32x2(y[j], mean2);
                }
            }
            uint64_t squares2 = dev::mul_f32x2(x[0], x[0]);
            squares2 = dev::fma_f32x2(y[0], y[0], squares2);
#pragma unroll
            for (int j = 1; j < kPairs; ++j) {
                squares2 = dev::fma_f32x2(x[j], x[j], squares2);
                squares2 = dev::fma_f32x2(y[j], y[j], squares2);
            }
            const float2 both = dev::f32x2_split(squares2);
            const float squares = group_sum(both.x + both.y, first_lane, chunk, s.chunks);
            const float scale = rsqrtf(fmaf(squares, inverse_dim, p.epsilon));
            const uint64_t scale2 = dev::f32x2(scale, scale);
            const float* const gamma = gains[key ? 2 : 0];
            uint64_t gain[kPairs];
            shared_pairs<V>(gamma + first, gain);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                x[j] = dev::mul_f32x2(dev::mul_f32x2(x[j], scale2), gain[j]);
            }
            shared_pairs<V>(gamma + second, gain);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                y[j] = dev::mul_f32x2(dev::mul_f32x2(y[j], scale2), gain[j]);
            }
            if (offsets) {
                const float* const beta = gains[key ? 3 : 1];
                shared_pairs<V>(beta + first, gain);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    x[j] = dev::add_f32x2(x[j], gain[j]);
                }
                shared_pairs<V>(beta + second, gain);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    y[j] = dev::add_f32x2(y[j], gain[j]);
                }
            }
        }
        if (t < tokens && in_group) {
            if constexpr (Adjacent) {
                // Pair j of the chunk is element pair j of x followed by y: with the turn (c, s),
                // (a, b) becomes (a c - b s, b c + a s).
                const auto turn = [](uint64_t pair, float c, float d) {
                    const float2 v = dev::f32x2_split(pair);
                    return dev::fma_f32x2(dev::f32x2(-v.y, v.x), dev::f32x2(d, d),
                                          dev::mul_f32x2(pair, dev::f32x2(c, c)));
                };
                constexpr int kQuarter = kPairs / 2;
#pragma unroll
                for (int q = 0; q < kPairs; ++q) {
                    const float4 two = turns[q * s.chunks];
                    uint64_t& even = kQuarter == 0 ? x[0] : (q < kQuarter ? x[2 * q]
                                                                          : y[2 * (q - kQuarter)]);
                    uint64_t& odd = kQuarter == 0 ? y[0] : (q < kQuarter ? x[2 * q + 1]
                                                                         : y[2 * (q - kQuarter) + 1]);
                    even = 2 * q < turned_pairs ? turn(even, two.x, two.y) : even;
                    odd = 2 * q + 1 < turned_pairs ? turn(odd, two.z, two.w) : odd;
                }
            } else if (turned_pairs > 0) { // all of them or none (vector_width)
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const ulonglong2 two =
                        *reinterpret_cast<const ulonglong2*>(turns + j * s.chunks);
                    const uint64_t turned = dev::sub_f32x2(dev::mul_f32x2(x[j], two.x),
                                                           dev::mul_f32x2(y[j], two.y));
                    y[j] = dev::fma_f32x2(x[j], two.y, dev::mul_f32x2(y[j], two.x));
                    x[j] = turned;
                }
            }
            store2<T, V>(out + first, x);
            store2<T, V>(out + second, y);
        }
        out += out_step;
        turns += s.slots * (half / 2);
    }
}

// Widest vectors the sizes and alignments allow: a lane's two vectors must lie within the
// rotated or the unrotated part of a head, start on a multiple of their size, and fit a warp.
template <typename T>
int vector_width(const Params& p) {
    const int half = p.head_dim / 2;
    for (int v = 16 / static_cast<int>(sizeof(T)); v >= 2; v /= 2) {
        const int bytes = v * static_cast<int>(sizeof(T));
        bool ok = half % v == 0 && half / v <= 32 && p.side[0].heads <= kMaxHeads / 2 &&
                  p.side[1].heads <= kMaxHeads / 2;
        ok = ok && (p.adjacent || (p.pairs % v == 0 && (half - p.pairs) % v == 0));
        for (const Side& side : p.side) {
            if (side.heads == 0) {
                continue;
            }
            const auto fits = [bytes](const void* base, long long stride) {
                return reinterpret_cast<uintptr_t>(base) % bytes == 0 &&
                       stride * static_cast<long long>(sizeof(T)) % bytes == 0;
            };
            ok = ok && fits(side.in, side.in_stride) && fits(side.out, side.out_stride);
        }
        if (ok) {
            return v;
        }
    }
    return 1;
}

template <typename T, int V, int Norm>
int launch_vector(const Params& p, int sm_count, cudaStream_t stream) {
    VectorShape s{};
    const int half = p.head_dim / 2;
    s.chunks = half / V;
    s.warp_groups = 32 / s.chunks;
    const int heads = p.side[0].heads + p.side[1].heads;
    // Warps of a block: the number from 4 on that leaves fewest lane groups without a head, next to
    // 8 of equals.
    double best = 0.0;
    for (const int warps : {8, 9, 7, 10, 6, 11, 5, 12, 4}) {
        if (warps > kMaxWarps<Norm>) {
            continue;
        }
        const int groups = warps * s.warp_groups;
        const int parts = (heads + groups - 1) / groups;
        const int taken = parts > 1 ? heads : groups / heads * heads;
        const double used = static_cast<double>(taken) / (static_cast<double>(parts) * groups);
        if (used > best + 0.02) {
            best = used;
            s.warps = warps;
        }
    }
    const int table_tokens = kTableVectors * 2 / half;
    const int groups = s.warps * s.warp_groups;
    s.heads = heads < groups ? heads : groups;
    s.slots = groups / s.heads < table_tokens ? groups / s.heads : table_tokens;
    // Tokens of a block: as many steps as the table holds, but no more than give every SM 12 blocks.
    const int steps = p.tokens / (12 * sm_count * s.slots);
    const int most = table_tokens / s.slots;
    s.block_tokens = s.slots * (steps < 1 ? 1 : (steps < most ? steps : most));
    const int blocks = (p.tokens - 1) / s.block_tokens + 1;
    const int parts = (heads + s.heads - 1) / s.heads;
    host::pdl_launch(p.adjacent ? qk_vector_kernel<T, V, Norm, true>
                                : qk_vector_kernel<T, V, Norm, false>,
                     dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(parts)),
                     dim3(static_cast<unsigned>(32 * s.warps)), 0, stream, p, s);
    return host::after_launch("qk_vector_kernel");
}

template <typename T, int Norm>
int launch_scalar(const Params& p, cudaStream_t stream) {
    const long long heads = p.side[0].heads + p.side[1].heads;
    const long long blocks = (heads * p.tokens + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7FFFFFFFLL) {
        return host::fail(CUVIT_LENGTH_ERROR, "rotary launch exceeds the CUDA grid limit");
    }
    host::pdl_launch(qk_scalar_kernel<T, Norm>, dim3(static_cast<unsigned>(blocks)),
                     dim3(kThreads), 0, stream, p);
    return host::after_launch("qk_scalar_kernel");
}

template <typename T, int Norm>
int launch_norm(const Params& p, int sm_count, cudaStream_t stream) {
    switch (vector_width<T>(p)) {
    case 8:
        if constexpr (sizeof(T) == 2) {
            return launch_vector<T, 8, Norm>(p, sm_count, stream);
        }
        [[fallthrough]];
    case 4:
        return launch_vector<T, 4, Norm>(p, sm_count, stream);
    case 2:
        return launch_vector<T, 2, Norm>(p, sm_count, stream);
    default:
        return launch_scalar<T, Norm>(p, stream);
    }
}

template <typename T>
int launch_typed(const Params& p, int norm, int sm_count, cudaStream_t stream) {
    switch (norm) {
    case CUVIT_NORM_RMS:
        return launch_norm<T, CUVIT_NORM_RMS>(p, sm_count, stream);
    case CUVIT_NORM_LAYER:
        return launch_norm<T, CUVIT_NORM_LAYER>(p, sm_count, stream);
    default:
        return launch_norm<T, kNormNone>(p, sm_count, stream);
    }
}

int check_rotary(const cuvit_rotary& r, int head_dim) {
    bool ok = r.axes >= 1 && r.axes <= CUVIT_ROTARY_MAX_AXES && r.first[0] == 0 &&
              (r.pairing == CUVIT_ROTARY_HALVES || r.pairing == CUVIT_ROTARY_ADJACENT);
    for (int a = 0; ok && a < r.axes; ++a) {
        ok = r.first[a + 1] >= r.first[a] && r.first[a + 1] <= CUVIT_ROTARY_MAX_PAIRS;
    }
    if (!ok || r.first[r.axes] < 1) {
        return host::fail(CUVIT_INVALID_ARGUMENT,
                          "the rotary axes were not set up by cuvit_rotary_init()");
    }
    if (2 * r.first[r.axes] > head_dim) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "the rotary axes turn more pairs than a head has");
    }
    return CUVIT_OK;
}

int run(const void* q, const void* k, void* q_out, void* k_out, const cuvit_qk_norm* norm,
        const int32_t* positions, const cuvit_rotary* rotary, const cuvit_qk_problem* problem,
        cudaStream_t stream) {
    if (problem == nullptr) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "query / key problem cannot be null");
    }
    const cuvit_qk_problem& c = *problem;
    if (c.tokens < 0 || c.q_heads < 0 || c.k_heads < 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "query / key dimensions cannot be negative");
    }
    if (c.head_dim < 2 || c.head_dim > kMaxHeadDim || c.head_dim % 2 != 0) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "head_dim must be even, from 2 to 256");
    }
    if (c.dtype != CUVIT_DTYPE_F32 && c.dtype != CUVIT_DTYPE_BF16) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "queries and keys must be F32 or BF16");
    }
    if (rotary != nullptr) {
        CUVIT_TRY(check_rotary(*rotary, c.head_dim));
    }
    if (norm != nullptr && ((norm->kind != CUVIT_NORM_RMS && norm->kind != CUVIT_NORM_LAYER) ||
                            !(norm->epsilon >= 0.0F) || std::isinf(norm->epsilon))) {
        return host::fail(CUVIT_INVALID_ARGUMENT,
                          "unknown norm, or an epsilon that is negative or not finite");
    }
    if (c.tokens == 0 || (c.q_heads == 0 && c.k_heads == 0)) {
        return CUVIT_OK;
    }
    if (rotary != nullptr && positions == nullptr) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "positions cannot be null");
    }

    Params p{};
    p.tokens = c.tokens;
    p.head_dim = c.head_dim;
    const int element = c.dtype == CUVIT_DTYPE_BF16 ? 2 : 4;
    const void* const ins[2] = {q, k};
    void* const outs[2] = {q_out, k_out};
    const int heads[2] = {c.q_heads, c.k_heads};
    const int64_t in_strides[2] = {c.q_stride, c.k_stride};
    const int64_t out_strides[2] = {c.q_out_stride, c.k_out_stride};
    host::RowSpan in_spans[2]{}, out_spans[2]{};
    for (int s = 0; s < 2; ++s) {
        Side& side = p.side[s];
        side.heads = heads[s];
        if (heads[s] == 0) {
            continue;
        }
        if (ins[s] == nullptr || outs[s] == nullptr) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "queries and keys cannot be null");
        }
        if (reinterpret_cast<uintptr_t>(ins[s]) % element != 0 ||
            reinterpret_cast<uintptr_t>(outs[s]) % element != 0) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "queries and keys must be aligned to their type");
        }
        const int64_t width = static_cast<int64_t>(heads[s]) * c.head_dim;
        side.in = ins[s];
        side.out = outs[s];
        side.in_stride = in_strides[s] != 0 ? in_strides[s] : width;
        side.out_stride = out_strides[s] != 0 ? out_strides[s] : width;
        if (side.in_stride < width || side.out_stride < width) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "a token stride is smaller than its heads");
        }
        const int64_t limit = (int64_t{1} << 58) / c.tokens;
        if (side.in_stride > limit || side.out_stride > limit) {
            return host::fail(CUVIT_LENGTH_ERROR, "a token stride is too large");
        }
        in_spans[s] = {ins[s], c.tokens, width * element, side.in_stride * element};
        out_spans[s] = {outs[s], c.tokens, width * element, side.out_stride * element};
        if (norm != nullptr) {
            side.gamma = s == 0 ? norm->q_gamma : norm->k_gamma;
            side.beta = s == 0 ? norm->q_beta : norm->k_beta;
            if (reinterpret_cast<uintptr_t>(side.gamma) % 4 != 0 ||
                reinterpret_cast<uintptr_t>(side.beta) % 4 != 0) {
                return host::fail(CUVIT_INVALID_ARGUMENT,
                                  "norm gains and offsets must be aligned to their type");
            }
        }
    }
    for (int o = 0; o < 2; ++o) {
        for (int i = 0; i < 2; ++i) {
            const bool in_place = o == i && ins[i] == outs[o] &&
                                  p.side[i].in_stride == p.side[i].out_stride;
            if (!in_place && host::rows_overlap(out_spans[o], in_spans[i])) {
                return host::fail(CUVIT_INVALID_ARGUMENT,
                                  "an output overlaps an input that is not its own");
            }
        }
    }
    if (host::rows_overlap(out_spans[0], out_spans[1])) {
        return host::fail(CUVIT_INVALID_ARGUMENT, "the outputs overlap");
    }
    p.epsilon = norm != nullptr ? norm->epsilon : 0.0F;
    if (rotary != nullptr) {
        p.rotary = *rotary;
        p.pairs = rotary->first[rotary->axes];
        p.adjacent = rotary->pairing == CUVIT_ROTARY_ADJACENT ? 1 : 0;
        p.positions = positions;
        p.position_stride = c.position_stride != 0 ? c.position_stride : c.tokens;
        if (p.position_stride < 0 || p.position_stride > (int64_t{1} << 58)) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "the position stride is out of range");
        }
        if (reinterpret_cast<uintptr_t>(positions) % 4 != 0) {
            return host::fail(CUVIT_INVALID_ARGUMENT, "positions must be aligned to their type");
        }
    }
    // What every block reads must not change under it.
    const int64_t gain_bytes = static_cast<int64_t>(c.head_dim) * 4;
    for (const host::RowSpan& out : out_spans) {
        bool shared = p.positions != nullptr &&
                      host::rows_overlap(out, {p.positions, rotary->axes, c.tokens * int64_t{4},
                                               p.position_stride * 4});
        for (const Side& side : p.side) {
            for (const float* gains : {side.gamma, side.beta}) {
                shared = shared || (gains != nullptr &&
                                    host::rows_overlap(out, {gains, 1, gain_bytes, gain_bytes}));
            }
        }
        if (shared) {
            return host::fail(CUVIT_INVALID_ARGUMENT,
                              "an output overlaps the positions or the norm's gains or offsets");
        }
    }
    const host::DeviceContext* context = nullptr;
    CUVIT_TRY(host::current_context(&context));
    CUVIT_TRY(host::check_operands({p.side[0].in, p.side[0].out, p.side[1].in, p.side[1].out,
                                    p.positions, p.side[0].gamma, p.side[0].beta, p.side[1].gamma,
                                    p.side[1].beta}));
    const int kind = norm != nullptr ? norm->kind : kNormNone;
    return c.dtype == CUVIT_DTYPE_BF16
               ? launch_typed<__nv_bfloat16>(p, kind, context->sm_count, stream)
               : launch_typed<float>(p, kind, context->sm_count, stream);
}

} // namespace
} // namespace cuvit::rotary

extern "C" {

int cuvit_rotary_init(cuvit_rotary* rotary, int axes, const int* sections, double base,
                      int pairing, int ladder) {
    return cuvit::host::guarded([&]() {
        using cuvit::host::fail;
        if (rotary == nullptr || sections == nullptr) {
            return fail(CUVIT_INVALID_ARGUMENT, "rotary axes and sections cannot be null");
        }
        if (axes < 1 || axes > CUVIT_ROTARY_MAX_AXES) {
            return fail(CUVIT_INVALID_ARGUMENT, "rotary positions have 1 to 4 axes");
        }
        int total = 0;
        for (int a = 0; a < axes; ++a) {
            if (sections[a] < 0 || sections[a] > CUVIT_ROTARY_MAX_PAIRS - total) {
                return fail(CUVIT_INVALID_ARGUMENT,
                            "rotary sections must be at least 0 and hold at most 128 pairs in all");
            }
            total += sections[a];
        }
        if (total == 0) {
            return fail(CUVIT_INVALID_ARGUMENT, "the rotary axes turn no pair");
        }
        if (!std::isfinite(base) || base < 1.0) {
            return fail(CUVIT_INVALID_ARGUMENT, "the rotary base must be finite and at least 1");
        }
        if ((pairing != CUVIT_ROTARY_HALVES && pairing != CUVIT_ROTARY_ADJACENT) ||
            (ladder != CUVIT_ROTARY_LADDER_AXIS && ladder != CUVIT_ROTARY_LADDER_SHARED)) {
            return fail(CUVIT_INVALID_ARGUMENT, "unknown rotary pairing or ladder");
        }
        cuvit_rotary r{};
        r.axes = axes;
        r.pairing = pairing;
        constexpr long double kTwoPi = 6.283185307179586476925286766559L;
        for (int a = 0; a < axes; ++a) {
            r.first[a + 1] = r.first[a] + sections[a];
            for (int j = 0; j < sections[a]; ++j) {
                const int i = r.first[a] + j;
                const long double exponent =
                    ladder == CUVIT_ROTARY_LADDER_AXIS
                        ? static_cast<long double>(j) / sections[a]
                        : static_cast<long double>(i) / total;
                // A rate is at most 1 radian a step, so the fraction of a turn is below 1/6.
                const long double rate = powl(static_cast<long double>(base), -exponent);
                r.turns[i] = static_cast<uint64_t>(ldexpl(rate / kTwoPi, 64));
            }
        }
        for (int a = axes; a < CUVIT_ROTARY_MAX_AXES; ++a) {
            r.first[a + 1] = r.first[axes];
        }
        *rotary = r;
        return static_cast<int>(CUVIT_OK);
    });
}

int cuvit_rotary_qk(const void* q, const void* k, void* q_out, void* k_out,
                    const int32_t* positions, const cuvit_rotary* rotary,
                    const cuvit_qk_problem* problem, cuvit_stream_t stream) {
    return cuvit::host::guarded([&]() {
        if (rotary == nullptr) {
            return cuvit::host::fail(CUVIT_INVALID_ARGUMENT, "rotary axes cannot be null");
        }
        return cuvit::rotary::run(q, k, q_out, k_out, nullptr, positions, rotary, problem,
                                  reinterpret_cast<cudaStream_t>(stream));
    });
}

int cuvit_qk_norm_rotary(const void* q, const void* k, void* q_out, void* k_out,
                         const cuvit_qk_norm* norm, const int32_t* positions,
                         const cuvit_rotary* rotary, const cuvit_qk_problem* problem,
                         cuvit_stream_t stream) {
    return cuvit::host::guarded([&]() {
        if (norm == nullptr) {
            return cuvit::host::fail(CUVIT_INVALID_ARGUMENT, "the norm cannot be null");
        }
        return cuvit::rotary::run(q, k, q_out, k_out, norm, positions, rotary, problem,
                                  reinterpret_cast<cudaStream_t>(stream));
    });
}

} // extern "C"
