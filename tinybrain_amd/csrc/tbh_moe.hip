// tbh_moe.hip -- a mixture-of-experts layer on block-scaled FP8 weights, for a
// few tokens:
//   z = x . router^T;  the top_k largest z of a token are its experts, with
//   weights p = softmax(z) (over all experts, or over the chosen ones)
//   y = sum over its experts e of p_e (silu(x . G_e) * (x . U_e)) . D_e
// Few tokens are bound by reading the chosen experts' weights once: rows of x
// and h stay as exact as they came, as bf16 or as three bf16 pieces of an fp32,
// and the weights are widened to bf16 (exactly) on their way to the matrix
// instruction.
#include <algorithm>
#include <cmath>
#include <memory>

#include "tbh_fp8.h"

struct tbh_moe {
    tbh_device *dev = nullptr;
    int64_t H = 0, I = 0, hb = 0, ib = 0;     // blocks of 128
    int32_t E = 0;
    float *router = nullptr;                  // [E][H]
    uint8_t *gate_up = nullptr;               // [E][ib * 8][gate, up][hb][2048]
    uint8_t *down = nullptr;                  // [E][hb * 8][ib][2048]
    float *gate_scales = nullptr, *up_scales = nullptr;   // [E][ib][hb]
    float *down_scales = nullptr;             // [E][hb][ib]
};

namespace tbh {
namespace moe {
namespace {

using fp8::blocks_of;
using fp8::f32x4;
using fp8::i32x4;
using fp8::kBlock;
using fp8::kTileBytes;
using fp8::u32x4;
using fp8::bf16x4;
using fp8::bf16x8;

constexpr int kMaxExperts = 512, kMaxTopK = 32;
constexpr int kMaxTokens = 64;      // of one part of a call
constexpr int kListHead = 2;        // expert, number of its tokens

struct Args {
    const void *x;
    void *y;
    int64_t ldx, ldy;
    const float *router;
    const uint8_t *gate_up, *down;
    const float *gate_scales, *up_scales, *down_scales;
    int32_t *ids;            // [T][top_k]
    float *weights;          // [T][top_k]
    __bf16 *xp;              // [P][T][hb * 128]
    __bf16 *hp;              // [P][T * top_k][ib * 128]
    int32_t *lists;          // [used][kListHead + kMaxTokens]: an expert, its tokens' places in ids
    int T, E, H, I, hb, ib, top_k, used;
    bool normalize;
};

// v as P pieces that sum to it: bf16 as it is, fp32 cut after 8 bits, twice.
template <int P>
__device__ __forceinline__ void pieces_of(float v, __bf16 (&p)[P]) {
    if constexpr (P == 1) {
        p[0] = (__bf16)v;
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u;
            p[i] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
            v -= __builtin_bit_cast(float, u);
        }
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// A block takes a token: its pieces, its experts and their weights.  Logits are
// summed in 64 bits: which of two near ones is the larger decides an expert.
template <class T, int P>
__global__ __launch_bounds__(256) void moe_route(Args a) {
    __shared__ double z[kMaxExperts];
    __shared__ int32_t chosen[kMaxTopK];
    __shared__ float part[kMaxTopK];
    __shared__ float sums[4];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = (const T *)a.x + (int64_t)t * a.ldx;
    const int hp = a.hb * kBlock;
    for (int k = tid; k < hp; k += 256) {
        __bf16 p[P];
        pieces_of<P>(k < a.H ? (float)x[k] : 0.0f, p);
#pragma unroll
        for (int i = 0; i < P; ++i) a.xp[((int64_t)i * a.T + t) * hp + k] = p[i];
    }
    for (int e = wave; e < a.E; e += 4) {
        const float *r = a.router + (int64_t)e * a.H;
        double s = 0.0;
        for (int k = lane; k < a.H; k += 64) s = __builtin_fma((double)(float)x[k], (double)r[k], s);
        s = wave_sum(s);
        // NaN is in no order: an expert like any other, behind the rest
        if (lane == 0) z[e] = s != s ? -HUGE_VAL : s;
    }
    __syncthreads();
    double most = -HUGE_VAL;
    for (int e = 0; e < a.E; ++e) most = fmax(most, z[e]);
    float sum = 0.0f;
    for (int e = tid; e < a.E; e += 256) {
        const double v = z[e];
        int rank = 0;
        for (int o = 0; o < a.E; ++o) rank += z[o] > v || (z[o] == v && o < e);
        const float w = expf((float)(v - most));
        if (rank < a.top_k) chosen[rank] = e, part[rank] = w;
        sum += w;
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (tid < a.top_k) {
        float all = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (a.normalize) {
            all = 0.0f;
            for (int i = 0; i < a.top_k; ++i) all += part[i];
        }
        a.ids[t * a.top_k + tid] = chosen[tid];
        a.weights[t * a.top_k + tid] = part[tid] / all;
    }
}

// The number of the y-th expert that some token has chosen and the places of
// its tokens, in order; -1 if there are not so many.
__device__ __forceinline__ int find_expert(const Args &a, int y, uint32_t (&used)[kMaxExperts / 32], int32_t *slots,
                                           int *count) {
    const int tid = threadIdx.x, lane = tid & 63, n = a.T * a.top_k;
    if (tid < kMaxExperts / 32) used[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        const int id = a.ids[i];
        atomicOr(&used[id >> 5], 1u << (id & 31));
    }
    __syncthreads();
    int e = -1, left = y;
    for (int w = 0; w < kMaxExperts / 32 && e < 0; ++w) {
        uint32_t u = used[w];
        const int c = __builtin_popcount(u);
        if (left >= c) {
            left -= c;
            continue;
        }
        for (; left > 0; --left) u &= u - 1;
        e = w * 32 + __builtin_ctz(u);
    }
    if (e < 0) return -1;
    if (tid < 64) {
        int found = 0;
        for (int base = 0; base < n; base += 64) {
            const bool mine = base + lane < n && a.ids[base + lane] == e;
            const uint64_t m = __ballot(mine);
            if (mine) slots[found + __builtin_popcountll(m & ((1ull << lane) - 1))] = base + lane;
            found += __builtin_popcountll(m);
        }
        if (lane == 0) *count = found;
    }
    __syncthreads();
    return e;
}

// One 128-deep block: acc[c] += scale * (tile . rows), for CT columns tiles of rows.
// row[c]: the lane's row of column tile c at input 16 g of the block; stride: from one
// piece to the next.
template <int P, int CT>
__device__ __forceinline__ void block_product(const uint8_t *tile, float scale, const __bf16 *const (&row)[CT],
                                              int64_t stride, f32x4 (&acc)[CT]) {
    const i32x4 w[2] = {*(const i32x4 *)tile, *(const i32x4 *)(tile + 1024)};
    f32x4 part[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) part[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bf16x8 o[2];
        fp8::widen(w[h], o);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 x = *(const bf16x8 *)(row[c] + p * stride + 64 * h + 8 * s);
                    part[c] = fp8::mfma_wide(o[s], x, part[c]);
                }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_fmaf(part[c][i], scale, acc[c][i]);
}

// h of 16 inner columns for an expert's tokens c0 .. c0 + 16 CT.
template <int P, int CT>
__device__ __forceinline__ void up_tokens(const Args &a, int e, int tile, const int32_t *slots, int c0, int count,
                                          f32x4 (*red)[64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int hp = a.hb * kBlock;
    const __bf16 *row[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        // a column past the last token repeats it; its result is not stored
        const int slot = slots[min(c0 + c * 16 + r16, count - 1)];
        row[c] = a.xp + (int64_t)(slot / a.top_k) * hp + 16 * g;
    }
    f32x4 gate[CT], up[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) gate[c] = up[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t *wt = a.gate_up + ((int64_t)e * a.ib * 8 + tile) * 2 * a.hb * kTileBytes + lane * 16;
    const int64_t sb = ((int64_t)e * a.ib + tile / 8) * a.hb, stride = (int64_t)a.T * hp;
    const int b0 = a.hb * wave / 4, b1 = a.hb * (wave + 1) / 4;
    for (int b = b0; b < b1; ++b) {
        const __bf16 *at[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) at[c] = row[c] + b * kBlock;
        block_product<P, CT>(wt + (int64_t)b * kTileBytes, a.gate_scales[sb + b], at, stride, gate);
        block_product<P, CT>(wt + (int64_t)(a.hb + b) * kTileBytes, a.up_scales[sb + b], at, stride, up);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        red[wave * 2 * CT + 2 * c][lane] = gate[c];
        red[wave * 2 * CT + 2 * c + 1][lane] = up[c];
    }
    __syncthreads();
    if (wave < CT) {
        const int c = wave;
        f32x4 gv = red[2 * c][lane], uv = red[2 * c + 1][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            gv += red[w * 2 * CT + 2 * c][lane];
            uv += red[w * 2 * CT + 2 * c + 1][lane];
        }
        const int at = c0 + c * 16 + r16;
        if (at < count) {
            const int ip = a.ib * kBlock;
            bf16x4 o[P];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __bf16 p[P];
                pieces_of<P>(gv[i] / (1.0f + expf(-gv[i])) * uv[i], p);
#pragma unroll
                for (int j = 0; j < P; ++j) o[j][i] = p[j];
            }
#pragma unroll
            for (int j = 0; j < P; ++j)
                *(bf16x4 *)(a.hp + ((int64_t)j * a.T * a.top_k + slots[at]) * ip + tile * 16 + 4 * g) = o[j];
        }
    }
    __syncthreads();
}

// Gate and up products of 16 inner columns of one expert and h = silu(gate) * up;
// the waves part the inputs.
template <int P>
__global__ __launch_bounds__(256) void moe_up(Args a) {
    __shared__ uint32_t used[kMaxExperts / 32];
    __shared__ int32_t slots[kMaxTokens];
    __shared__ int count;
    __shared__ f32x4 red[4 * 4][64];
    const int e = find_expert(a, blockIdx.y, used, slots, &count);
    if (blockIdx.x == 0) {
        int32_t *l = a.lists + blockIdx.y * (kListHead + kMaxTokens);
        if (threadIdx.x == 0) l[0] = e, l[1] = e < 0 ? 0 : count;
        if (e >= 0 && (int)threadIdx.x < count) l[kListHead + threadIdx.x] = slots[threadIdx.x];
    }
    if (e < 0) return;
    int c0 = 0;
    for (; count - c0 > 16; c0 += 32) up_tokens<P, 2>(a, e, blockIdx.x, slots, c0, count, red);
    if (c0 < count) up_tokens<P, 1>(a, e, blockIdx.x, slots, c0, count, red);
}

// 16 outputs of all tokens: the waves part the (expert, block of inputs) pairs and
// each adds its share of a token's sum to its own row in LDS; joined in order.
template <class T, int P>
__global__ __launch_bounds__(512) void moe_down(Args a) {
    extern __shared__ f32x4 sums[];       // [8][T][4]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4, tile = blockIdx.x;
    f32x4 *own = sums + wave * a.T * 4;
    for (int i = lane; i < a.T * 4; i += 64) own[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int active = 0;
    for (int y = 0; y < a.used; y += 64)
        active += __builtin_popcountll(__ballot(y + lane < a.used && a.lists[(y + lane) * (kListHead + kMaxTokens) + 1] > 0));
    const int total = active * a.ib;
    int i = (int)((int64_t)total * wave / 8);
    const int end = (int)((int64_t)total * (wave + 1) / 8);
    const int ip = a.ib * kBlock;
    const int64_t stride = (int64_t)a.T * a.top_k * ip;
    __builtin_amdgcn_wave_barrier();
    while (i < end) {
        const int y = i / a.ib, b0 = i - y * a.ib, b1 = min(a.ib, b0 + end - i);
        const int32_t *l = a.lists + y * (kListHead + kMaxTokens);
        const int e = l[0], count = l[1];
        const uint8_t *wt = a.down + ((int64_t)e * a.hb * 8 + tile) * a.ib * kTileBytes + lane * 16;
        const float *sw = a.down_scales + ((int64_t)e * a.hb + tile / 8) * a.ib;
        for (int c0 = 0; c0 < count; c0 += 16) {
            const int at = c0 + r16, slot = l[kListHead + min(at, count - 1)];
            const __bf16 *row = a.hp + (int64_t)slot * ip + 16 * g;
            f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
            for (int b = b0; b < b1; ++b) {
                const __bf16 *const rows[1] = {row + b * kBlock};
                block_product<P, 1>(wt + (int64_t)b * kTileBytes, sw[b], rows, stride, acc);
            }
            if (at < count) {
                const float p = a.weights[slot];
                f32x4 *to = own + (slot / a.top_k) * 4 + g;
                f32x4 v = *to;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(acc[0][j], p, v[j]);
                *to = v;
            }
        }
        i += b1 - b0;
    }
    __syncthreads();
    for (int j = tid; j < a.T * 16; j += 512) {
        const int t = j >> 4, n = tile * 16 + (j & 15);
        float v = 0.0f;
        for (int w = 0; w < 8; ++w) v += ((const float *)sums)[w * a.T * 16 + j];
        if (n < a.H) ((T *)a.y)[(int64_t)t * a.ldy + n] = (T)v;
    }
}

template <class T, int P>
hipError_t launch(const Args &a, hipStream_t s) {
    hipLaunchKernelGGL((moe_route<T, P>), dim3((unsigned)a.T), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_up<P>), dim3((unsigned)(a.ib * 8), (unsigned)a.used), dim3(256), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((moe_down<T, P>), dim3((unsigned)((a.H + 15) / 16)), dim3(512), (size_t)a.T * 8 * 64, s, a);
    return hipGetLastError();
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace of a part of T tokens; sets the pointers when `base` is given.
size_t carve(Args &a, int P, char *base) {
    size_t at = 0;
    auto take = [&](size_t n) {
        char *p = base ? base + at : nullptr;
        at += round256(n);
        return p;
    };
    const size_t rows = (size_t)a.T * a.top_k;
    a.ids = (int32_t *)take(rows * 4);
    a.weights = (float *)take(rows * 4);
    a.lists = (int32_t *)take((size_t)a.used * (kListHead + kMaxTokens) * 4);
    a.xp = (__bf16 *)take((size_t)P * a.T * a.hb * kBlock * 2);
    a.hp = (__bf16 *)take((size_t)P * rows * a.ib * kBlock * 2);
    return at;
}

size_t workspace_of(const tbh_moe &m, int32_t x_type, int64_t tokens, int32_t top_k) {
    Args a{};
    a.T = (int)std::min<int64_t>(tokens, kMaxTokens);
    a.top_k = top_k;
    a.hb = (int)m.hb;
    a.ib = (int)m.ib;
    a.used = std::min(m.E, a.T * top_k);
    return carve(a, x_type == TBH_BF16 ? 1 : 3, nullptr);
}

constexpr int64_t kMaxWidth = 1 << 17;

}  // namespace
}  // namespace moe
}  // namespace tbh

using namespace tbh;
using namespace tbh::moe;

extern "C" {

tbh_status tbh_moe_destroy(tbh_moe *m) {
    if (!m) return TBH_OK;
    if (m->dev) (void)use_device(m->dev->ordinal);
    hipError_t e = hipSuccess;
    for (void *p : {(void *)m->router, (void *)m->gate_up, (void *)m->down, (void *)m->gate_scales, (void *)m->up_scales,
                    (void *)m->down_scales})
        if (p) {
            const hipError_t f = hipFree(p);
            if (e == hipSuccess) e = f;
        }
    delete m;
    return e == hipSuccess ? TBH_OK : hip_error(e, "tbh_moe_destroy");
}

tbh_status tbh_moe_create(tbh_device *dev, const tbh_moe_desc *desc, tbh_moe **out) {
    const char *what = "tbh_moe_create";
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!out) return bad("out is NULL");
    *out = nullptr;
    if (!dev || !desc) return bad("NULL device or descriptor");
    const tbh_moe_desc &d = *desc;
    if (d.hidden <= 0 || d.intermediate <= 0 || d.experts <= 0) return bad("sizes must be positive");
    if (!d.router || !d.gate || !d.up || !d.down || !d.gate_scales || !d.up_scales || !d.down_scales)
        return bad("NULL pointer");
    if (d.hidden > kMaxWidth || d.intermediate > kMaxWidth || d.experts > kMaxExperts)
        return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": a width above 2^17 or more than 512 experts");
    tbh_status st = use_device(dev->ordinal);
    if (st != TBH_OK) return st;
    std::unique_ptr<tbh_moe, tbh_status (*)(tbh_moe *)> m(new (std::nothrow) tbh_moe, tbh_moe_destroy);
    if (!m) return set_error(TBH_E_OOM, std::string(what) + ": out of host memory");
    m->dev = dev;
    m->H = d.hidden;
    m->I = d.intermediate;
    m->E = d.experts;
    m->hb = blocks_of(m->H);
    m->ib = blocks_of(m->I);
    const size_t E = (size_t)m->E, scales = E * m->hb * m->ib * 4, bytes = E * m->H * m->I;
    const size_t tiles = E * m->hb * m->ib * 8 * kTileBytes;
    std::lock_guard<std::mutex> lock(dev->mu);
    const hipStream_t s = dev->stream;
    hipError_t e = fp8::copy_in((void **)&m->router, d.router, E * m->H * 4, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->gate_scales, d.gate_scales, scales, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->up_scales, d.up_scales, scales, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->down_scales, d.down_scales, scales, s);
    if (e == hipSuccess) e = hipMalloc((void **)&m->gate_up, 2 * tiles);
    if (e == hipSuccess) e = hipMalloc((void **)&m->down, tiles);
    auto repack = [&](const uint8_t *from, int64_t N, int64_t K, int64_t row_tiles, int64_t step, uint8_t *to) {
        void *raw = nullptr;
        if (e == hipSuccess) e = fp8::copy_in(&raw, from, bytes, s);
        if (e == hipSuccess) e = fp8::launch_repack((const uint8_t *)raw, N, K, m->E, row_tiles, step, to, s);
        const hipError_t waited = hipStreamSynchronize(s);
        if (e == hipSuccess) e = waited;
        if (raw) (void)hipFree(raw);
    };
    repack(d.gate, m->I, m->H, m->ib * 16, 2, m->gate_up);
    repack(d.up, m->I, m->H, m->ib * 16, 2, m->gate_up ? m->gate_up + m->hb * kTileBytes : nullptr);
    repack(d.down, m->H, m->I, m->hb * 8, 1, m->down);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return hip_error(e, what);
    }
    *out = m.release();
    return TBH_OK;
}

static tbh_status check_moe(const char *what, const tbh_moe *m, int32_t x_type, int64_t tokens, int32_t top_k) {
    auto bad = [&](const char *t) { return set_error(TBH_E_INVALID, std::string(what) + ": " + t); };
    if (!m) return bad("NULL layer");
    if (x_type != TBH_F32 && x_type != TBH_BF16) return bad("unknown x_type");
    if (tokens < 0) return bad("negative tokens");
    if (top_k < 1 || top_k > m->E) return bad("top_k must be 1 .. experts");
    if (top_k > kMaxTopK) return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": top_k > 32");
    return TBH_OK;
}

tbh_status tbh_moe_workspace(const tbh_moe *m, int32_t x_type, int64_t tokens, int32_t top_k, int64_t *bytes) {
    const tbh_status st = check_moe("tbh_moe_workspace", m, x_type, tokens, top_k);
    if (st != TBH_OK) return st;
    if (!bytes) return set_error(TBH_E_INVALID, "tbh_moe_workspace: NULL pointer");
    *bytes = (int64_t)workspace_of(*m, x_type, tokens, top_k);
    return TBH_OK;
}

tbh_status tbh_moe_device(const tbh_moe *m, const void *x, int32_t x_type, int64_t tokens, int64_t x_stride, int32_t top_k,
                          int32_t normalize, void *y, int64_t y_stride, int32_t *experts, float *weights, void *workspace,
                          int64_t workspace_bytes, void *stream) {
    const char *what = "tbh_moe";
    auto bad = [&](const char *t) { return set_error(TBH_E_INVALID, std::string(what) + ": " + t); };
    tbh_status st = check_moe(what, m, x_type, tokens, top_k);
    if (st != TBH_OK) return st;
    if (tokens == 0) return TBH_OK;
    if (!x || !y) return bad("NULL x or y");
    if (tokens > 1 && (x_stride < m->H || y_stride < m->H)) return bad("a stride is shorter than its row");
    const size_t size = fp8::type_size(x_type);
    if ((uintptr_t)x % size || (uintptr_t)y % size || (uintptr_t)experts % 4 || (uintptr_t)weights % 4)
        return bad("a pointer is not aligned to its type");
    if (workspace && ((uintptr_t)workspace & 255)) return bad("the workspace must be 256-byte aligned");
    const size_t need = workspace_of(*m, x_type, tokens, top_k);
    if (workspace && (workspace_bytes < 0 || (size_t)workspace_bytes < need)) return bad("the workspace is too small");
    if ((st = use_device(m->dev->ordinal)) != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    const auto held = hold_launches(m->dev, s);
    char *room = (char *)(workspace ? workspace : stream_workspace(m->dev, s, need));
    if (!room)
        return set_error(TBH_E_OOM, std::string(what) + ": no workspace (a captured stream needs an earlier eager call, or a "
                                                        "workspace of the caller's)");
    hipError_t e = hipSuccess;
    for (int64_t at = 0; at < tokens && e == hipSuccess; at += kMaxTokens) {
        Args a{};
        a.T = (int)std::min<int64_t>(kMaxTokens, tokens - at);
        a.top_k = top_k;
        a.E = m->E;
        a.H = (int)m->H;
        a.I = (int)m->I;
        a.hb = (int)m->hb;
        a.ib = (int)m->ib;
        a.used = std::min(m->E, a.T * top_k);
        a.normalize = normalize != 0;
        carve(a, x_type == TBH_BF16 ? 1 : 3, room);
        if (experts) a.ids = experts + at * top_k;
        if (weights) a.weights = weights + at * top_k;
        a.x = (const char *)x + at * x_stride * size;
        a.y = (char *)y + at * y_stride * size;
        a.ldx = x_stride;
        a.ldy = y_stride;
        a.router = m->router;
        a.gate_up = m->gate_up;
        a.down = m->down;
        a.gate_scales = m->gate_scales;
        a.up_scales = m->up_scales;
        a.down_scales = m->down_scales;
        e = x_type == TBH_BF16 ? launch<__bf16, 1>(a, s) : launch<float, 3>(a, s);
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "moe launch");
}

}  // extern "C"
