// tbh_paged_attn.hip -- attention of a step's new tokens over a paged cache
// (tbh_paged_attention_device).
#include <algorithm>
#include <cmath>

#include "tbh_paged.h"
#include "tbh_wave.h"

namespace tbh {
namespace {

using namespace paged;

struct PagedArgs {
    const void *q, *kc, *vc;
    void *out;
    const int32_t *start, *ctx, *table;
    int64_t q_stride, out_stride, tokens;
    int32_t requests, most, num_blocks, shift;   // shift: log2 of the block size
    int32_t nh, nkv, hd, rep;
    float scale;
};

template <class T>
__device__ __forceinline__ float elem(const void *p, int64_t i) {
    return (float)((const T *)p)[i];
}

// Last request whose first row is at most t (those before it may have none).
__device__ __forceinline__ int32_t request_of(const PagedArgs &a, int32_t t) {
    int32_t lo = 0, hi = a.requests;
    while (lo < hi) {
        const int32_t mid = (lo + hi + 1) >> 1;
        if (a.start[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Element index of a request's position in the cache arrays at head kvh, or -1
// where the table has no block.
__device__ __forceinline__ int64_t place(const PagedArgs &a, int32_t b, int32_t pos, int kvh) {
    const int32_t id = a.table[(int64_t)b * a.most + (pos >> a.shift)];
    if ((uint32_t)id >= (uint32_t)a.num_blocks) return -1;
    return ((((int64_t)id * a.nkv + kvh) << a.shift) + (pos & ((1 << a.shift) - 1))) * a.hd;
}

// Any head dimension, type and alignment: one wave per (token, query head),
// 64 positions a pass, a position per lane for the scores and an output
// dimension per lane for the values.
template <class XT, class CT>
__global__ __launch_bounds__(256) void paged_rows(const PagedArgs a) {
    __shared__ float qs[4][kMaxHeadDim];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + w;
    if (row >= a.tokens * a.nh) return;
    const int64_t t = row / a.nh;
    const int h = (int)(row % a.nh), kvh = h / a.rep;
    const int32_t b = request_of(a, (int32_t)t);
    if (b >= a.requests) return;                 // behind the last request's rows
    const int64_t held = min((int64_t)max(a.ctx[b], 0), (int64_t)a.most << a.shift);
    const int64_t behind = (int64_t)a.start[b + 1] - 1 - t;   // rows of the request after this one
    const int32_t last = (int32_t)min(held - 1, held - 1 - behind);   // this row's position
    for (int d = lane; d < a.hd; d += 64) qs[w][d] = elem<XT>(a.q, t * a.q_stride + (int64_t)h * a.hd + d);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");

    float m = -INFINITY, l = 0.0f, o[kMaxHeadDim / 64] = {};
    bool seen = false;
    for (int32_t p0 = 0; p0 <= last; p0 += 64) {
        const int32_t pos = p0 + lane;
        const int64_t at = pos <= last ? place(a, b, pos, kvh) : -1;
        const uint64_t valid = __ballot(at >= 0);
        if (!valid) continue;
        seen = true;
        float s = -INFINITY;
        if (at >= 0) {
            float dot = 0.0f;
            for (int d = 0; d < a.hd; ++d) dot += qs[w][d] * elem<CT>(a.kc, at + d);
            s = dot * a.scale;
        }
        const float nm = fmaxf(m, wave::max(s));
        const float ref = nm == -INFINITY ? 0.0f : nm;
        const float corr = expf(m - ref), p = at >= 0 ? expf(s - ref) : 0.0f;
        l = l * corr + wave::sum(p);
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 64; ++i) o[i] *= corr;
        for (uint64_t v = valid; v; v &= v - 1) {
            const int j = __builtin_ctzll(v);
            const float pj = wave::lane_value(p, j);
            const int64_t vj = __shfl(at, j);
#pragma unroll
            for (int i = 0; i < kMaxHeadDim / 64; ++i)
                if (lane + 64 * i < a.hd) o[i] += pj * elem<CT>(a.vc, vj + lane + 64 * i);
        }
        m = nm;
    }
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 64; ++i)
        if (lane + 64 * i < a.hd)
            ((XT *)a.out)[t * a.out_stride + (int64_t)h * a.hd + lane + 64 * i] = (XT)(seen ? o[i] / l : 0.0f);
}

template <class XT, class CT>
hipError_t launch_paged(const PagedArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((paged_rows<XT, CT>), dim3((unsigned)((a.tokens * a.nh + 3) / 4)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace tbh

using namespace tbh;

extern "C" {

tbh_status tbh_paged_attention_device(tbh_device *dev, const tbh_paged_layout *layout,
                                      const tbh_paged_queries *queries, const void *k_cache, const void *v_cache,
                                      const int32_t *block_table, void *stream) {
    const char *what = "tbh_paged_attention";
    tbh_status st = check_layout(what, dev, layout, true);
    if (st != TBH_OK) return st;
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!queries) return bad("queries is NULL");
    const tbh_paged_queries &q = *queries;
    if (q.tokens < 0 || q.tokens > INT32_MAX) return bad("tokens out of range");
    if (q.type != TBH_F32 && q.type != TBH_BF16) return bad("unknown type");
    if (q.num_heads <= 0 || q.num_heads % layout->num_kv_heads != 0)
        return bad("num_heads must be a multiple of num_kv_heads");
    if (std::isnan(q.scale) || std::isinf(q.scale)) return bad("scale must be finite");
    if (q.max_query_len < 0 || q.max_context_len < 0) return bad("negative length bound");
    const int64_t nq = (int64_t)layout->head_dim * q.num_heads;
    if (q.tokens * q.num_heads > INT32_MAX)
        return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": more than 2^31 rows of heads");
    if (q.tokens == 0 || layout->max_requests == 0) return TBH_OK;
    if (!q.q || !q.out || !q.query_start || !q.context_lens) return bad("NULL pointer");
    if (q.tokens > 1 && (q.q_stride < nq || q.out_stride < nq)) return bad("a stride is shorter than its row");
    if (layout->max_blocks > 0 && !block_table) return bad("NULL block_table");
    if (layout->num_blocks > 0 && (!k_cache || !v_cache)) return bad("NULL cache");
    if (!aligned(k_cache, 16) || !aligned(v_cache, 16)) return bad("the cache must be 16-byte aligned");
    if (q.q == q.out) return bad("out must not be q");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    PagedArgs a{};
    a.q = q.q;
    a.kc = k_cache;
    a.vc = v_cache;
    a.out = q.out;
    a.start = q.query_start;
    a.ctx = q.context_lens;
    a.table = block_table;
    a.q_stride = q.q_stride;
    a.out_stride = q.out_stride;
    a.tokens = q.tokens;
    a.requests = layout->max_requests;
    a.most = layout->max_blocks;
    a.num_blocks = layout->num_blocks;
    a.shift = __builtin_ctz((unsigned)layout->block_size);
    a.nh = q.num_heads;
    a.nkv = layout->num_kv_heads;
    a.hd = layout->head_dim;
    a.rep = q.num_heads / layout->num_kv_heads;
    a.scale = q.scale != 0.0f ? q.scale : 1.0f / std::sqrt((float)layout->head_dim);
    const hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    switch ((q.type == TBH_BF16) * 2 + (layout->type == TBH_BF16)) {
    case 0: e = launch_paged<float, float>(a, s); break;
    case 1: e = launch_paged<float, __bf16>(a, s); break;
    case 2: e = launch_paged<__bf16, float>(a, s); break;
    default: e = launch_paged<__bf16, __bf16>(a, s); break;
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "paged attention launch");
}

}  // extern "C"
