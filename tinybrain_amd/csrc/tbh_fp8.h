// tbh_fp8.h -- block-scaled FP8 matrices: their layout and the pieces that
// their kernels share (tbh_fp8.hip, tbh_moe.hip).
//
// A matrix of N outputs by K inputs is stored as tiles of 16 outputs x 128
// inputs, 2 KiB each, padded with zeros to whole blocks of 128 outputs, the eight
// tiles of a block (what shares a scale) together: [ceil(N / 128)][ceil(K / 128)][8].
// In a tile, byte i of 16-byte piece (h, g, r) is output r, input
// 64 h + 16 g + i, pieces in the order h, g, r: lane (g, r) = 16 g + r of a
// wave finds both halves of its matrix operand with two loads that each cover
// 1 KiB, and both operands of a product use the same order, so that which
// input a lane holds cancels.
#pragma once

#include <string>

#include "tbh_internal.h"

namespace tbh {
namespace fp8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 128;        // outputs and inputs that share a scale
constexpr int kTileBytes = 2048;

inline int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// A matrix in that layout on the device.
struct Matrix {
    const uint8_t *tiles;      // [row_blocks][k_blocks][8][2048]
    const float *scales;       // [row_blocks][k_blocks]
};

// Writes `count` matrices of N x K e4m3 bytes (row-major, one after the other) as tiles,
// one matrix after the other: tile t of block b goes to place (t / group * k_blocks + b) *
// group * step + t % group * step of its matrix's (places of `step` tiles; tbh_fp8.hip).
hipError_t launch_repack(const uint8_t *data, int64_t N, int64_t K, int64_t count, int64_t group, int64_t step,
                         uint8_t *tiles, hipStream_t s);

// Where tile t of block b of a matrix in groups of eight tiles starts.
__device__ __forceinline__ int64_t tile_at(int64_t t, int64_t b, int64_t k_blocks) {
    return ((t >> 3) * k_blocks + b) * (8 * kTileBytes) + (t & 7) * kTileBytes;
}

// Copies `bytes` from host or device memory into a new device allocation.
hipError_t copy_in(void **out, const void *from, size_t bytes, hipStream_t s);

inline size_t type_size(int32_t t) { return t == TBH_BF16 ? 2 : 4; }

// a . b of a whole 128-deep block on the FP8 instruction: A's row r16 and B's
// column r16 per lane; the result's lane holds rows 4 (lane / 16) + 0 .. 3 of
// column r16.  The instruction cuts its sums: 1.4e-5 .. 5e-5 of the result's
// size are lost (measured, values of one size .. of spread e^2), less than a
// hundredth of what rounding to bf16 does, but far more than fp32 sums.  A product keeps some 17
// bits below the block's largest: with one input of 128 ten to ten thousand times the others the error of a
// bf16 result is 1.0001 to 1.0015 times that of its rounding.
__device__ __forceinline__ f32x4 mfma_block(i32x8 a, i32x8 b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// A lane's 16 bytes of a tile as bf16, exactly: its operands of two instructions
// of 32 inputs, whose sums are as good as fp32 ones (1e-8 of the result's size).
__device__ __forceinline__ void widen(i32x4 v, bf16x8 (&o)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * s + i], 1.0f, false);
            const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * s + i], 1.0f, true);
            o[s][4 * i] = lo[0], o[s][4 * i + 1] = lo[1], o[s][4 * i + 2] = hi[0], o[s][4 * i + 3] = hi[1];
        }
}

__device__ __forceinline__ f32x4 mfma_wide(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The largest of the four lanes that hold one row's block (lane, and those 16, 32 and 48 away).
__device__ __forceinline__ uint32_t row_most(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// A lane's 32 elements of a row's block as they are stored: inputs 16 g .. 16 g + 15 of both halves.
template <class T>
struct Block {
    static constexpr int kWords = sizeof(T) == 4 ? 16 : 8;      // of a half
    uint32_t v[2][kWords];
};

// p: the row at input 16 g of the block; elements at and behind `left` are 0.
template <class T>
__device__ __forceinline__ void load_block(Block<T> &x, const T *p, int left, bool vec) {
    constexpr int N = Block<T>::kWords;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int rest = left - 64 * h;
        if (vec && rest >= 16) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const u32x4 q = *(const u32x4 *)((const uint32_t *)(p + 64 * h) + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) x.v[h][4 * i + j] = q[j];
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x.v[h][i] = i < rest ? __builtin_bit_cast(uint32_t, p[64 * h + i]) : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint16_t *u = (const uint16_t *)p + 64 * h + 2 * i;
                x.v[h][i] = (2 * i < rest ? u[0] : 0u) | (2 * i + 1 < rest ? (uint32_t)u[1] << 16 : 0u);
            }
        }
    }
}

// Quantizes a row's block of 128, of which this lane holds 32 and the three
// lanes 16, 32 and 48 away the others: scale s, the least power of two (at
// least 2^-126) with max |x| <= 448 s over the finite elements, and e4m3(x / s),
// ties to even: the conversion scales exactly and rounds once, and makes NaN of
// what is not finite.
template <class T>
__device__ __forceinline__ float quantize_block(const Block<T> &x, i32x8 &q) {
    uint32_t most = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = max(most, x.v[h][i] & 0x7FFFFFFFu);
    } else {
        u16x2 m{0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.v[h][i] & 0x7FFF7FFFu));
        most = (uint32_t)max(m[0], m[1]) << 16;
    }
    if (most >= 0x7F800000u) {        // rare: the largest of what is finite
        most = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < Block<T>::kWords; ++i) {
                const uint32_t w = x.v[h][i];
                const uint32_t a = (sizeof(T) == 4 ? w : w << 16) & 0x7FFFFFFFu, b = sizeof(T) == 4 ? 0u : w & 0x7FFF0000u;
                most = max(most, max(a < 0x7F800000u ? a : 0u, b < 0x7F800000u ? b : 0u));
            }
    }
    most = row_most(most);
    // 448 = 1.75 * 2^8: a mantissa above 1.75 needs the next power
    int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = max(e, -126);
    const float s = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);      // e in -126 .. 120
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s16x2 w{0, 0};
            if constexpr (sizeof(T) == 4) {
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = __builtin_bit_cast(float, x.v[h][4 * i + j]);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, f[0], f[1], s, false);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, f[2], f[3], s, true);
            } else {
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, x.v[h][2 * i]), s, false);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, x.v[h][2 * i + 1]), s, true);
            }
            q[4 * h + i] = __builtin_bit_cast(int, w);
        }
    return s;
}

// Four results of one row from column n on: those at and behind N are left out.
template <class T>
__device__ __forceinline__ void store4(T *p, f32x4 v, int64_t left, bool vec) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            *(f32x4 *)p = v;
        } else {
            *(bf16x4 *)p = bf16x4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

}  // namespace fp8
}  // namespace tbh

struct tbh_fp8_weight {
    tbh_device *dev = nullptr;
    int64_t K = 0, N = 0;
    int64_t kb = 0, nb = 0;          // blocks of 128 along K and N
    uint8_t *tiles = nullptr;        // [nb][kb][8][2048]
    float *scales = nullptr;         // [nb][kb]
};
