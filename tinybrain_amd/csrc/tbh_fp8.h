// tbh_fp8.h -- block-scaled FP8 matrices: their layout and the pieces that
// their kernels share (tbh_fp8.hip, tbh_moe.hip).
//
// A matrix of N outputs by K inputs is stored as tiles of 16 outputs x 128
// inputs, 2 KiB each, [ceil(N / 16)][ceil(K / 128)], padded with zeros to 128
// outputs.  In a tile, byte i of 16-byte piece (h, g, r) is output r, input
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
    const uint8_t *tiles;      // [row_blocks * 8][k_blocks][2048]
    const float *scales;       // [row_blocks][k_blocks]
};

// Writes `count` matrices of N x K e4m3 bytes (row-major, one after the other) as tiles;
// tile row t of matrix i goes to tiles + (i * row_tiles + t * step) * k_blocks * 2048, with
// row_tiles tile rows per matrix in the result (tbh_fp8.hip).
hipError_t launch_repack(const uint8_t *data, int64_t N, int64_t K, int64_t count, int64_t row_tiles, int64_t step,
                         uint8_t *tiles, hipStream_t s);

// Copies `bytes` from host or device memory into a new device allocation.
hipError_t copy_in(void **out, const void *from, size_t bytes, hipStream_t s);

inline size_t type_size(int32_t t) { return t == TBH_BF16 ? 2 : 4; }

// a . b of a whole 128-deep block on the FP8 instruction: A's row r16 and B's
// column r16 per lane; the result's lane holds rows 4 (lane / 16) + 0 .. 3 of
// column r16.  The instruction cuts its sums: 1.4e-5 .. 5e-5 of the result's
// size are lost (measured, values of one size .. of spread e^2), less than a
// hundredth of what rounding to bf16 does, but far more than fp32 sums.
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

// 16 elements of a row as float: those at and behind `left` are 0.
template <class T>
__device__ __forceinline__ void load16(const T *p, int left, bool vec, float (&x)[16]) {
    if (vec && left >= 16) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 v = *(const f32x4 *)(p + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const u32x4 v = *(const u32x4 *)(p + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[8 * i + 2 * j] = __builtin_bit_cast(float, v[j] << 16);
                    x[8 * i + 2 * j + 1] = __builtin_bit_cast(float, v[j] & 0xFFFF0000u);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i < left ? (float)p[i] : 0.0f;
    }
}

// The largest of the four lanes that hold one row's block (lane, and those 16, 32 and 48 away).
__device__ __forceinline__ uint32_t row_most(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// Quantizes a row's block of 128, of which this lane holds 32 and the three
// lanes 16, 32 and 48 away the others: scale s, the least power of two (at
// least 2^-126) with max |x| <= 448 s over the finite elements, and e4m3(x / s),
// ties to even.  x / s is exact, so that the one rounding is the last.  Not
// finite: NaN.
__device__ __forceinline__ float quantize_block(const float (&x)[2][16], i32x8 &q) {
    uint32_t most = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t u = __builtin_bit_cast(uint32_t, x[h][i]) & 0x7FFFFFFFu;
            most = max(most, u >= 0x7F800000u ? 0u : u);
        }
    most = row_most(most);
    // 448 = 1.75 * 2^8: a mantissa above 1.75 needs the next power
    int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = max(e, -126);
    const float inv = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);   // 2^-e, e in -126 .. 120
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = x[h][4 * i + j] * inv;
                // (the conversion takes an infinity to 448 or NaN by a mode of the wave)
                if (__builtin_isinf(v[j])) v[j] = __builtin_nanf("");
            }
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
            q[4 * h + i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
        }
    return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
}

template <class T>
__device__ __forceinline__ T rounded(float v) {
    return (T)v;
}

// Four results of one row from column n on: those at and behind N are left out.
template <class T>
__device__ __forceinline__ void store4(T *p, f32x4 v, int64_t left, bool vec) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            *(f32x4 *)p = v;
        } else {
            typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
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
    uint8_t *tiles = nullptr;        // [nb * 8][kb][2048]
    float *scales = nullptr;         // [nb][kb]
};
