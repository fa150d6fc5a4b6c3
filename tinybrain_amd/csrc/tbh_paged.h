// tbh_paged.h -- element types and host checks that the paged-cache calls
// share (tbh_paged.hip, tbh_paged_attn.hip).
#pragma once

#include <string>

#include "tbh_internal.h"

namespace tbh {
namespace paged {

constexpr int kMaxHeadDim = 256;
constexpr int kMaxBlockSize = 1024;

template <class T>
struct Vec8;   // eight consecutive elements as stored
template <>
struct Vec8<float> {
    float4 a, b;
};
template <>
struct Vec8<__bf16> {
    uint4 a;
};

__device__ __forceinline__ void unpack(const Vec8<float> &v, float (&x)[8]) {
    x[0] = v.a.x, x[1] = v.a.y, x[2] = v.a.z, x[3] = v.a.w;
    x[4] = v.b.x, x[5] = v.b.y, x[6] = v.b.z, x[7] = v.b.w;
}

__device__ __forceinline__ void unpack(const Vec8<__bf16> &v, float (&x)[8]) {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
        x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void pack(Vec8<float> &v, const float (&x)[8]) {
    v.a = float4{x[0], x[1], x[2], x[3]};
    v.b = float4{x[4], x[5], x[6], x[7]};
}

__device__ __forceinline__ void pack(Vec8<__bf16> &v, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]) << 16;
    v.a = uint4{w[0], w[1], w[2], w[3]};
}

inline size_t type_size(int32_t t) { return t == TBH_BF16 ? 2 : 4; }
inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// The layout fields every paged call reads; what: the call's name.
inline tbh_status check_layout(const char *what, const tbh_device *dev, const tbh_paged_layout *l, bool cache) {
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!dev || !l) return bad("NULL device or layout");
    if (l->num_blocks < 0 || l->max_requests < 0 || l->max_blocks < 0) return bad("negative size");
    if (l->block_size < 1 || l->block_size > kMaxBlockSize || (l->block_size & (l->block_size - 1)))
        return bad("block_size must be a power of two, 1 .. 1024");
    if ((int64_t)l->num_blocks * l->block_size > INT32_MAX) return bad("num_blocks * block_size exceeds 2^31 - 1");
    if ((int64_t)l->max_requests * l->max_blocks > INT32_MAX)
        return bad("max_requests * max_blocks exceeds 2^31 - 1");
    // positions and the tile behind the last one, and a tile of requests, in 32 bits
    if ((int64_t)l->max_blocks * l->block_size > 1 << 30) return bad("max_blocks * block_size exceeds 2^30");
    if (l->max_requests > 1 << 30) return bad("max_requests exceeds 2^30");
    if (!cache) return TBH_OK;
    if (l->num_kv_heads <= 0 || l->head_dim <= 0) return bad("invalid heads or head_dim");
    if (l->type != TBH_F32 && l->type != TBH_BF16) return bad("unknown cache type");
    if (l->head_dim > kMaxHeadDim)
        return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": head_dim > 256");
    return TBH_OK;
}

}  // namespace paged
}  // namespace tbh
