// tbh_paged_attn.hip -- attention of a step's new tokens over a paged cache
// (tbh_paged_attention_device).  Figures: us a call among others, both of its
// launches; where a trace is named, one launch from its first wave to its last.
#include <algorithm>
#include <cmath>

#include "tbh_dma.h"
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
        const int32_t mid = lo + ((hi - lo + 1) >> 1);
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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// One row's part of the softmax over positions [c0, end), by one wave: 64
// positions a pass, every `step`, a position per lane for the scores and an output
// dimension per lane (lane, lane + 64, ...) for the values.  m: largest score in
// powers of two, l and o: sums relative to it.  qs: the wave's LDS, head_dim floats.
// AHEAD: positions whose values are in flight at once, 8, or 1 where the rare row is
// taken inside a kernel that needs the registers.
struct RowPart {
    float m, l, o[kMaxHeadDim / 64];
    bool seen;             // a position of the range is in a block
};

template <class CT, bool VEC>
__device__ __forceinline__ float dot_key(const PagedArgs &a, int64_t at, const float *qs) {
    float dot = 0.0f;
    if (VEC && a.hd % 8 == 0) {
        const CT *k = (const CT *)a.kc + at;
#pragma unroll 4
        for (int d = 0; d < a.hd; d += 8) {
            float x[8];
            unpack(*(const Vec8<CT> *)(k + d), x);
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += qs[d + i] * x[i];
        }
    } else {
        for (int d = 0; d < a.hd; ++d) dot += qs[d] * elem<CT>(a.kc, at + d);
    }
    return dot;
}

template <class XT, class CT, int AHEAD>
__device__ __forceinline__ RowPart row_part(const PagedArgs &a, int32_t b, int64_t t, int head, int32_t c0, int32_t end,
                                            float *qs, int32_t step = 64) {
    const int lane = threadIdx.x & 63, kvh = head / a.rep;
    const float c2 = a.scale * 1.44269504f;
    wave::lds_fence();
    for (int d = lane; d < a.hd; d += 64) qs[d] = elem<XT>(a.q, t * a.q_stride + (int64_t)head * a.hd + d);
    wave::lds_fence();
    RowPart r{-INFINITY, 0.0f, {}, false};
    for (int32_t p0 = c0; p0 < end; p0 += step) {
        const int64_t at = p0 + lane < end ? place(a, b, p0 + lane, kvh) : -1;
        const uint64_t valid = __ballot(at >= 0);
        if (!valid) continue;
        r.seen = true;
        const float s = at >= 0 ? dot_key<CT, (AHEAD > 1)>(a, at, qs) * c2 : -INFINITY;
        const float nm = fmaxf(r.m, wave::max(s));
        const float ref = nm == -INFINITY ? 0.0f : nm;
        const float corr = exp2_fast(r.m - ref), p = at >= 0 ? exp2_fast(s - ref) : 0.0f;
        r.l = r.l * corr + wave::sum(p);
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 64; ++i) r.o[i] *= corr;
        for (uint64_t left = valid; AHEAD == 1 && left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const float pj = wave::lane_value(p, j);
            const int64_t from = __shfl(at, j);
#pragma unroll
            for (int i = 0; i < kMaxHeadDim / 64; ++i)
                if (lane + 64 * i < a.hd) r.o[i] += pj * elem<CT>(a.vc, from + lane + 64 * i);
        }
        for (int j0 = 0; AHEAD > 1 && j0 < 64; j0 += AHEAD) {
            if (!(valid >> j0 & ((1ull << AHEAD) - 1))) continue;
            int64_t from[AHEAD];
            float pj[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                pj[j] = wave::lane_value(p, j0 + j);
                from[j] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j0 + j) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((int)at, j0 + j));
            }
#pragma unroll
            for (int i = 0; i < kMaxHeadDim / 64; ++i) {
                if (64 * i >= a.hd) break;
                const int d = min(lane + 64 * i, a.hd - 1);
                float x[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) x[j] = elem<CT>(a.vc, max(from[j], (int64_t)0) + d);   // block 0's: not used
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) r.o[i] += from[j] >= 0 ? pj[j] * x[j] : 0.0f;
            }
        }
        r.m = nm;
    }
    return r;
}

// The row's result from all of its positions.
template <class XT>
__device__ __forceinline__ void store_row(const PagedArgs &a, int64_t t, int head, const RowPart &r) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 64; ++i)
        if (lane + 64 * i < a.hd)
            ((XT *)a.out)[t * a.out_stride + (int64_t)head * a.hd + lane + 64 * i] = (XT)(r.seen ? r.o[i] / r.l : 0.0f);
}

// Any head dimension, block size and alignment: a block per (token, query head),
// whose four waves take passes of 64 positions in turn and meet in LDS.  Bound by
// the latency of its loads.  us, bf16 cache, 32 heads on 8 of 80: 130 for a row over
// 4000 positions (381 with one wave a row), 119 for 64 rows over 1000 (143), 265 for
// 256 rows over 1024 (292); heads of 256: 210 (708), 313 (301), 630 (647).
template <class XT, class CT>
__global__ __launch_bounds__(256) void paged_rows(const PagedArgs a) {
    __shared__ float qs[4][kMaxHeadDim], so[4][kMaxHeadDim];
    __shared__ float sm[4], sl[4];
    __shared__ bool sseen[4];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.tokens * a.nh) return;
    const int64_t t = row / a.nh;
    const int h = (int)(row % a.nh);
    const int32_t b = request_of(a, (int32_t)t);
    if (b >= a.requests || a.start[b] > t || a.start[b] < 0) return;   // not a request's row
    const int64_t held = min((int64_t)max(a.ctx[b], 0), (int64_t)a.most << a.shift);
    const int64_t behind = (int64_t)a.start[b + 1] - 1 - t;   // rows of the request after this one
    const int32_t last = (int32_t)min(held - 1, held - 1 - behind);   // this row's position
    const RowPart p = row_part<XT, CT, 8>(a, b, t, h, 64 * w, last + 1, qs[w], 256);
    if (lane == 0) {
        sm[w] = p.m;
        sl[w] = p.l;
        sseen[w] = p.seen;
    }
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 64; ++i)
        if (lane + 64 * i < a.hd) so[w][lane + 64 * i] = p.o[i];
    __syncthreads();
    if (w != 0) return;
    RowPart r{-INFINITY, 0.0f, {}, false};
#pragma unroll
    for (int k = 0; k < 4; ++k) r.m = fmaxf(r.m, sm[k]);
    for (int k = 0; k < 4; ++k) {
        if (!sseen[k]) continue;
        r.seen = true;
        const float f = exp2_fast(sm[k] - (r.m == -INFINITY ? 0.0f : r.m));   // 0 for scores of -inf alone
        r.l += f * sl[k];
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 64; ++i)
            if (lane + 64 * i < a.hd) r.o[i] += f * so[k][lane + 64 * i];
    }
    store_row<XT>(a, t, h, r);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A request's rows as the kernels below take them: row r of a key/value head
// is token r / rep, query head r % rep of its group.
struct Request {
    int32_t first, n;      // its rows of q that exist
    int32_t rows;          // n * rep
    int32_t held;          // positions in the cache
    int32_t base;          // position of its first row, negative where rows exceed positions
};

__device__ __forceinline__ Request request(const PagedArgs &a, int32_t b) {
    Request r;
    const int64_t first = a.start[b], end = a.start[b + 1];
    r.held = (int32_t)min((int64_t)max(a.ctx[b], 0), (int64_t)a.most << a.shift);
    r.first = (int32_t)first;
    const bool ok = first >= 0 && first < a.tokens && end > first;
    r.n = ok ? (int32_t)(min(end, a.tokens) - first) : 0;
    r.base = ok ? (int32_t)(r.held - (end - first)) : 0;
    r.rows = r.n * a.rep;
    return r;
}

// How a range of `len` positions is cut for at most `splits` blocks: parts of
// `chunk` positions, a multiple of 128 and at least the caller's.
struct Cut {
    int32_t parts, chunk;
};
__device__ __forceinline__ Cut cut(int32_t len, int32_t splits, int32_t least) {
    const int32_t even = (len + splits - 1) / splits;
    const int32_t chunk = max(least, (even + 127) / 128 * 128);
    return {max(1, (len + chunk - 1) / chunk), chunk};
}

struct SplitArgs {
    PagedArgs a;
    int32_t units;         // (16 rows, key/value head) pairs
    int32_t splits, least; // see cut
    int32_t slots;         // rows of a unit in the partials, at most 16
    int32_t long_rows;     // requests of more rows are tile_block's
    bool scan;             // units are groups of 16 rows of any request, else requests
    bool qvec;             // q rows are 16-byte aligned
    uint32_t base;         // the launch's first block, of both kinds
    float2 *ml;            // partials [unit][split][slots]: (max, sum)
    float *po;             // and sums of p v, [unit][split][slots][head_dim]
};

// 16 rows of one key/value head.
struct Group {
    Request q;
    int32_t b, kvh, row0, rows;    // rows: of this group
    int32_t len;                   // positions its last row sees
};

// Finds group `index` of the requests' groups of ROWS rows, heads fastest, a
// request's last rows first: they see the most positions.  pair_up: the second
// half of a request's groups follows from its first rows on, so that blocks that
// run side by side, half the launch apart, see as many positions as the others.
template <int ROWS>
__device__ __forceinline__ bool find_group(const PagedArgs &a, uint32_t index, int32_t more_than, bool pair_up,
                                           Group &g) {
    const int lane = threadIdx.x & 63;
    g.kvh = (int)(index % (uint32_t)a.nkv);
    int32_t left = (int32_t)(index / (uint32_t)a.nkv);
    for (int32_t b0 = 0; b0 < a.requests; b0 += 64) {
        Request r{};
        if (b0 + lane < a.requests) r = request(a, b0 + lane);
        const int32_t mine = r.rows > more_than ? (r.rows + ROWS - 1) / ROWS : 0;
        int32_t in = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int32_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        const int32_t total = __builtin_amdgcn_readlane(in, 63);
        if (left < total) {
            const int l = __builtin_ctzll(__ballot(in > left));
            g.b = b0 + l;
            const int32_t n = __builtin_amdgcn_readlane(mine, l), k = left - (__builtin_amdgcn_readlane(in, l) - n);
            const int32_t half = (n + 1) / 2;
            g.row0 = (pair_up && k >= half ? k - half : n - 1 - k) * ROWS;
            g.q.first = __builtin_amdgcn_readlane(r.first, l);
            g.q.n = __builtin_amdgcn_readlane(r.n, l);
            g.q.rows = __builtin_amdgcn_readlane(r.rows, l);
            g.q.held = __builtin_amdgcn_readlane(r.held, l);
            g.q.base = __builtin_amdgcn_readlane(r.base, l);
            return true;
        }
        left -= total;
    }
    return false;
}

template <int ROWS>
__device__ __forceinline__ void set_rows(const PagedArgs &a, Group &g, int32_t row0) {
    g.row0 = row0;
    g.rows = min(ROWS, g.q.rows - row0);
    g.len = min(g.q.held, max(0, g.q.base + (row0 + g.rows - 1) / a.rep + 1));
}

// Largest value, sum over the four lanes that hold one row (lane % 16).  A
// half swap of v with itself leaves one partner's value in its first result and
// the other's in its second, in both partners.
struct Both {
    float x, y;
};
__device__ __forceinline__ Both half_swap16(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t x = r[0], y = r[1];
    return {__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ Both half_swap32(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t x = r[0], y = r[1];
    return {__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float row4_max(float v) {
    const Both a = half_swap16(v), b = half_swap32(fmaxf(a.x, a.y));
    return fmaxf(b.x, b.y);
}
__device__ __forceinline__ float row4_sum(float v) {
    const Both a = half_swap16(v), b = half_swap32(a.x + a.y);
    return b.x + b.y;
}

// x as a sum of NP bf16 values: exact for NP = 3 (8 + 8 + 8 bits), rounded for 1.
// One for bf16 rows, whose q is exact so and whose probabilities are rounded, each
// off by at most 2^-8 of itself.  The sum that divides is that of the rounded ones
// (split_block: of the exact ones), so a result is off by at most 2^-8 of sum p |v -
// out| (of sum p |v|), as much as its own rounding to bf16 where values are about as
// large as their mean, more where they cancel: against 64 bits 2.2e-3 over 2048 rows
// over 4096 positions, 1.7e-3 with exact probabilities, whose three products take
// 253 us for 116.  fp32 rows keep fp32's precision.
template <int NP>
__device__ __forceinline__ void pieces(float x, __bf16 (&p)[NP]) {
    p[0] = (__bf16)x;
    if constexpr (NP == 3) {
        const float r = x - (float)p[0];
        const bool finite = fabsf((float)p[0]) < INFINITY;   // inf and NaN are held by the first piece
        p[1] = (__bf16)(finite ? r : 0.0f);
        p[2] = (__bf16)(finite ? r - (float)p[1] : 0.0f);
    }
}

// Eight elements of row n of q from dimension d on (0 behind the head).
template <class XT>
__device__ __forceinline__ void load_q8(const PagedArgs &a, int64_t t, int head, int d, bool vec, float (&x)[8]) {
    const XT *p = (const XT *)a.q + t * a.q_stride + (int64_t)head * a.hd + d;
    if (vec) {
        unpack(*(const Vec8<XT> *)p, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
    }
}

// The same of a probability: finite, or NaN, which every piece then is.
template <int NP>
__device__ __forceinline__ void pieces_of_p(float x, __bf16 (&p)[NP]) {
    p[0] = (__bf16)x;
    if constexpr (NP == 3) {
        const float r = x - (float)p[0];
        p[1] = (__bf16)r;
        p[2] = (__bf16)(r - (float)p[1]);
    }
}

template <int N>
struct __attribute__((aligned(4))) Words {
    uint32_t w[N];
};

// The two products of 32 positions (two tiles of 16, each inside a block) with
// 16 rows, operands straight from the cache.  Scores are formed transposed,
// keys x queries, so that lane (g = lane / 16, n = lane % 16) holds positions 4g
// + i of each tile for row n: the layout in which the second product, values
// transposed x probabilities, takes its right operand, if its reduction index
// 8g + c (bf16) or g (fp32) is read as position 4g + c % 4 of tile c / 4, or 4g +
// i in the i-th instruction.  VD = HD / 16 consecutive dimensions of a value
// row per lane: lane (g, n) ends with outputs 4 VD g .. 4 VD (g + 1) of row n.
template <class XT, class CT, int HD>
struct Step;

template <class XT, int HD>
struct Step<XT, __bf16, HD> {
    static constexpr int NP = sizeof(XT) == 4 ? 3 : 1;   // bf16 pieces of q and p
    static constexpr int NJ = HD / 32, VD = HD / 16, VW = VD / 2;
    bf16x8 q[NP][NJ];
    bf16x8 k[2][NJ];
    Words<VW> v[2][4];

    __device__ __forceinline__ void load_q(const PagedArgs &a, int64_t t, int head, int g, bool vec) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float x[8];
            load_q8<XT>(a, t, head, 32 * j + 8 * g, vec, x);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                __bf16 p[NP];
                pieces<NP>(x[c], p);
#pragma unroll
                for (int i = 0; i < NP; ++i) q[i][j][c] = p[i];
            }
        }
    }
    __device__ __forceinline__ void load_keys(int t, const __bf16 *p, int g, int n) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) k[t][j] = *(const bf16x8 *)(p + n * HD + 32 * j + 8 * g);
    }
    __device__ __forceinline__ void load_values(int t, const __bf16 *p, int g, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[t][i] = *(const Words<VW> *)(p + (4 * g + i) * HD + VD * n);
    }
    __device__ __forceinline__ void drop_value(int t, int i) {
#pragma unroll
        for (int w = 0; w < VW; ++w) v[t][i].w[w] = 0;
    }
    __device__ __forceinline__ f32x4 scores(int t) const {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = NP - 1; i >= 0; --i)              // the smallest pieces first
#pragma unroll
            for (int j = 0; j < NJ; ++j) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t][j], q[i][j], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void values(const f32x4 (&p)[2], f32x4 (&o)[VD]) const {
        bf16x8 pp[NP];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            __bf16 x[NP];
            pieces_of_p<NP>(p[c / 4][c % 4], x);
#pragma unroll
            for (int i = 0; i < NP; ++i) pp[i][c] = x[i];
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {              // dimension 2w + h of eight positions
                uint32_t e[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    e[c] = __builtin_amdgcn_perm(v[c / 2][2 * (c % 2) + 1].w[w], v[c / 2][2 * (c % 2)].w[w],
                                                 h ? 0x07060302u : 0x05040100u);
                const bf16x8 vv = __builtin_bit_cast(bf16x8, uint4{e[0], e[1], e[2], e[3]});
#pragma unroll
                for (int i = NP - 1; i >= 0; --i)
                    o[2 * w + h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pp[i], o[2 * w + h], 0, 0, 0);
            }
    }
};

template <class XT, int HD>
struct Step<XT, float, HD> {
    static constexpr int NJ = HD / 16, VD = HD / 16;
    float q[NJ][4];
    f32x4 k[2][NJ];
    Words<VD> v[2][4];

    __device__ __forceinline__ void load_q(const PagedArgs &a, int64_t t, int head, int g, bool) {
        const XT *p = (const XT *)a.q + t * a.q_stride + (int64_t)head * a.hd + 4 * g;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) q[j][c] = (float)p[16 * j + c];
    }
    __device__ __forceinline__ void load_keys(int t, const float *p, int g, int n) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) k[t][j] = *(const f32x4 *)(p + n * HD + 16 * j + 4 * g);
    }
    __device__ __forceinline__ void load_values(int t, const float *p, int g, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[t][i] = *(const Words<VD> *)(p + (4 * g + i) * HD + VD * n);
    }
    __device__ __forceinline__ void drop_value(int t, int i) {
#pragma unroll
        for (int w = 0; w < VD; ++w) v[t][i].w[w] = 0;
    }
    __device__ __forceinline__ f32x4 scores(int t) const {
        f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};   // two chains: half the rounding of one
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                s[c & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][j][c], q[j][c], s[c & 1], 0, 0, 0);
        return s[0] + s[1];
    }
    __device__ __forceinline__ void values(const f32x4 (&p)[2], f32x4 (&o)[VD]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < VD; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, v[t][i].w[d]), p[t][i], o[d],
                                                                0, 0, 0);
    }
};

// Few rows per request (single tokens of grouped heads, short chunks): 16 rows
// and one part of the positions a block, its four waves taking steps of 32
// positions in turn and meeting in LDS at the end.  Operands go from memory to
// registers: each byte of the cache is used by one wave alone, so LDS would only
// add a trip.  Bound by reading the cache: 64 requests of 100 .. 8192 positions, 32
// heads on 8 of 128, fp32 rows over a bf16 cache 107 to 114 us, 470 MB at 4.1 to 4.4
// TB/s (a large copy: 4.7); by latency where there is little: a row over 4096 fp32
// positions of 4 heads of 64 7.4 us.
template <int HD>
struct SplitLds {
    float so[4][16][HD + 4];
    float2 sml[4][16];
    int odd;
};

template <class XT, class CT, int HD>
__device__ __forceinline__ void split_block(const SplitArgs &sa, uint32_t block, SplitLds<HD> &lds) {
    constexpr int VD = HD / 16;
    auto &so = lds.so;
    auto &sml = lds.sml;
    int &odd = lds.odd;
    const PagedArgs &a = sa.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, n = lane & 15;
    // The units run fastest: consecutive blocks go to different XCDs, and with the
    // parts fastest one XCD would get every request's first part and another only
    // those of the longest (64 requests of 100 .. 8192 positions: 216 us for 107).
    const uint32_t unit = block % (uint32_t)sa.units, split = block / (uint32_t)sa.units;
    Group gr;
    bool alone = false;            // more rows than a unit has places for: no parts
    if (sa.scan) {
        if (!find_group<16>(a, unit, 0, false, gr)) return;
    } else {
        gr.kvh = (int)(unit % (uint32_t)a.nkv);
        gr.b = (int32_t)(unit / (uint32_t)a.nkv);
        gr.q = request(a, gr.b);
        gr.row0 = 0;
        if (gr.q.rows == 0 || gr.q.rows > sa.long_rows) return;
        alone = gr.q.rows > sa.slots;
    }
    const int32_t end_row = sa.scan ? gr.row0 + 1 : gr.q.rows;
    const int32_t *table = a.table + (int64_t)gr.b * a.most;
    const float c2 = a.scale * 1.44269504f;   // scores in powers of two
    const int32_t head_rows = HD << a.shift, in_block = (1 << a.shift) - 1;
    const int64_t block_rows = (int64_t)head_rows * a.nkv;
    const CT *kb = (const CT *)a.kc + (int64_t)gr.kvh * head_rows, *vb = (const CT *)a.vc + (int64_t)gr.kvh * head_rows;

    for (int32_t row0 = gr.row0; row0 < end_row; row0 += 16) {
        set_rows<16>(a, gr, row0);
        const Cut ct = alone ? Cut{1, max(gr.len, 1)} : cut(gr.len, sa.splits, sa.least);
        if ((int32_t)split >= ct.parts) return;
        const int32_t c0 = split * ct.chunk, c1 = min(gr.len, c0 + ct.chunk);
        const int32_t r = row0 + min(n, gr.rows - 1);
        const int32_t token = r / a.rep;
        const int32_t last = min(gr.q.base + token, gr.q.held - 1);   // this row's position
        const int32_t first_last = min(gr.q.base + row0 / a.rep, gr.q.held - 1);   // the first row's
        Step<XT, CT, HD> st;

        // A step's keys are loaded once the step before has used its own, values
        // likewise.  The blocks of 32 steps (two tiles each) are looked up at once,
        // one per lane.
        auto window = [&](int32_t p) {
            const int32_t x = p + 128 * (lane >> 1) + 16 * (lane & 1);
            return x < c1 ? table[x >> a.shift] : -1;
        };
        struct Pair {
            int32_t id[2];
        };
        int32_t p0 = c0 + 32 * w;
        int32_t ids = window(p0);
        auto pair = [&](int32_t p) {           // of the step at p, in the window
            const int i = (p - c0) >> 7 & 31;
            return Pair{{__builtin_amdgcn_readlane(ids, 2 * i), __builtin_amdgcn_readlane(ids, 2 * i + 1)}};
        };
        auto there = [&](const Pair &x, int t) { return (uint32_t)x.id[t] < (uint32_t)a.num_blocks; };
        auto at = [&](const Pair &x, int t, int32_t p0) {   // a tile without a block: any block's rows, not used
            return (int64_t)(there(x, t) ? x.id[t] : 0) * block_rows + ((p0 + 16 * t) & in_block) * HD;
        };
        Pair cur = pair(p0);
        st.load_q(a, gr.q.first + token, gr.kvh * a.rep + r % a.rep, g, sa.qvec);
        if (p0 < c1) {
#pragma unroll
            for (int t = 0; t < 2; ++t) st.load_keys(t, kb + at(cur, t, p0), g, n);
#pragma unroll
            for (int t = 0; t < 2; ++t) st.load_values(t, vb + at(cur, t, p0), g, n);
        }

        float m = -INFINITY, l = 0.0f;   // l: this lane's positions only
        int32_t first = INT32_MAX;       // this wave's first position in a block
        f32x4 o[VD];
#pragma unroll
        for (int d = 0; d < VD; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (; p0 < c1; p0 += 128) {
            if (((p0 - c0) >> 7 & 31) == 31) ids = window(p0 + 128);
            const Pair nxt = pair(p0 + 128);
            const bool th[2] = {there(cur, 0), there(cur, 1)};
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = st.scores(t);
#pragma unroll
            for (int t = 0; t < 2; ++t) st.load_keys(t, kb + at(nxt, t, p0 + 128), g, n);   // behind the part: block 0
            float nm = m;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (th[t]) first = min(first, p0 + 16 * t);
                const int32_t lim = th[t] ? last - (p0 + 16 * t + 4 * g) : -1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[t][i] = i <= lim ? s[t][i] * c2 : -INFINITY;
                    nm = fmaxf(nm, s[t][i]);
                }
            }
            if (!th[0] || !th[1] || p0 + 32 > c1) {   // what lies there may be NaN: 0 * NaN
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!th[t] || p0 + 16 * t + 4 * g + i >= c1) st.drop_value(t, i);
            }
            nm = row4_max(nm);
            const float ref = nm == -INFINITY ? 0.0f : nm;
            const float corr = exp2_fast(m - ref);
            m = nm;
            l *= corr;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[t][i] = exp2_fast(s[t][i] - ref);
                    l += s[t][i];
                }
            if (__any(corr != 1.0f)) {
#pragma unroll
                for (int d = 0; d < VD; ++d) o[d] *= corr;
            }
            st.values(s, o);
#pragma unroll
            for (int t = 0; t < 2; ++t) st.load_values(t, vb + at(nxt, t, p0 + 128), g, n);
            cur = nxt;
        }
        l = row4_sum(l);
        if (m == -INFINITY) l = first <= last ? 1.0f : 0.0f;   // positions seen, each of score -inf; none at all

        // the four waves' parts
        __syncthreads();
        if (tid == 0) odd = 0;
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) so[w][n][4 * VD * g + VD * i + d] = o[d][i];
        if (g == 0) sml[w][n] = float2{m, l};
        __syncthreads();
        for (int e = tid; e < gr.rows * HD; e += 256) {
            const int rr = e / HD, d = e % HD;
            float mm = -INFINITY, ll = 0.0f, v = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) mm = fmaxf(mm, sml[i][rr].x);
            float none = 0.0f;           // a wave has seen positions
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 ml = sml[i][rr];
                const float f = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - mm);
                none = fmaxf(none, ml.y);
                ll += f * ml.y;
                v += f * so[i][rr][d];
            }
            if (mm == -INFINITY) ll = none;
            if (!(fabsf(v) < INFINITY)) odd = 1;
            if (ct.parts == 1) {
                const int32_t tt = (row0 + rr) / a.rep;
                const int head = gr.kvh * a.rep + (row0 + rr) % a.rep;
                // nothing seen: 0; only scores of -inf: 0 / 0
                const float res = mm == -INFINITY ? (ll > 0.0f ? NAN : 0.0f) : v / ll;
                ((XT *)a.out)[(int64_t)(gr.q.first + tt) * a.out_stride + (int64_t)head * HD + d] = (XT)res;
            } else {
                const int64_t at = ((int64_t)unit * sa.splits + split) * sa.slots + rr;
                if (d == 0) sa.ml[at] = float2{mm, ll};
                sa.po[at * HD + d] = v;
            }
        }
        if (first_last + 1 >= c1) continue;      // every row sees all of the part (uniform)
        // An inf or NaN among the values that some rows do not see became NaN in
        // theirs, 0 times it: those parts once more, a row at a time.
        __syncthreads();
        if (!odd) continue;
        for (int rr = w; rr < gr.rows; rr += 4) {
            const int32_t tt = (row0 + rr) / a.rep;
            const int head = gr.kvh * a.rep + (row0 + rr) % a.rep;
            const int32_t end = min(c1, gr.q.base + tt + 1);
            const RowPart x = row_part<XT, CT, 1>(a, gr.b, gr.q.first + tt, head, c0, end, &so[w][0][0]);
            if (ct.parts == 1) {
                store_row<XT>(a, gr.q.first + tt, head, x);
            } else {
                const int64_t at = ((int64_t)unit * sa.splits + split) * sa.slots + rr;
                if (lane == 0) sa.ml[at] = x.m == -INFINITY ? float2{x.m, x.seen ? 1.0f : 0.0f} : float2{x.m, x.l};
                for (int i = 0; 64 * i + lane < HD; ++i) sa.po[at * HD + 64 * i + lane] = x.o[i];
            }
        }
    }
}

template <class XT, class CT, int HD>
__global__ __launch_bounds__(256) void paged_split(const SplitArgs sa) {
    __shared__ __attribute__((aligned(16))) SplitLds<HD> lds;
    split_block<XT, CT, HD>(sa, sa.base + blockIdx.x, lds);
}

// Joins split_block's parts: a wave per unit and row, HD / 4 lanes across the head,
// the parts dealt over its groups of lanes, four loads each in flight.  Lane i holds
// part i's factor.  Bound by latency: 4.1 us after a row over 4096 positions, 4.8
// after 64 requests of up to 8192 (5.9 with a block per row).
template <class XT, int HD>
__device__ __forceinline__ void split_merge(const SplitArgs &sa, uint32_t block) {
    constexpr int T = HD / 4, G = 64 / T;
    const PagedArgs &a = sa.a;
    const int lane = threadIdx.x & 63, d4 = lane % T, sg = lane / T;
    const uint32_t index = block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rr = index % (uint32_t)sa.slots, unit = index / (uint32_t)sa.slots;
    if (unit >= (uint32_t)sa.units) return;
    const int64_t at0 = (int64_t)unit * sa.splits * sa.slots + rr;
    const float2 mine = sa.ml[at0 + (int64_t)min(lane, sa.splits - 1) * sa.slots];   // before the request is known
    Group gr;
    if (sa.scan) {
        if (!find_group<16>(a, unit, 0, false, gr)) return;
    } else {
        gr.kvh = (int)(unit % (uint32_t)a.nkv);
        gr.b = (int32_t)(unit / (uint32_t)a.nkv);
        gr.q = request(a, gr.b);
        gr.row0 = 0;
        if (gr.q.rows == 0 || gr.q.rows > sa.long_rows || gr.q.rows > sa.slots) return;
    }
    set_rows<16>(a, gr, gr.row0);
    const Cut ct = cut(gr.len, sa.splits, sa.least);
    if (ct.parts == 1 || (int32_t)rr >= gr.rows) return;
    const float *po = sa.po + at0 * HD + 4 * d4;
    const bool part = lane < ct.parts;
    const float mm = wave::max(part ? mine.x : -INFINITY);
    const float f = part && mine.x != -INFINITY ? exp2_fast(mine.x - mm) : 0.0f;
    const float l = wave::sum(part && f != 0.0f ? f * mine.y : 0.0f);
    const bool any = __any(part && mine.y > 0.0f);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < ct.parts; s0 += 4 * G) {
        f32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = *(const f32x4 *)(po + (int64_t)min(s0 + G * i + sg, ct.parts - 1) * sa.slots * HD);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + G * i + sg;
            const float fs = __shfl(f, min(s, 63));
            if (s < ct.parts && sg < G) o += fs * v[i];
        }
    }
#pragma unroll
    for (int w = G / 2; w; w /= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_down(o[i], w * T);
    if (sg != 0) return;
    const int32_t row = gr.row0 + rr;
    XT *out = (XT *)a.out + (int64_t)(gr.q.first + row / a.rep) * a.out_stride +
              (int64_t)(gr.kvh * a.rep + row % a.rep) * HD + 4 * d4;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (XT)(mm == -INFINITY ? (any ? NAN : 0.0f) : o[i] / l);
}

template <class XT, int HD>
__global__ __launch_bounds__(256) void paged_split_merge(const SplitArgs sa) {
    split_merge<XT, HD>(sa, sa.base + blockIdx.x);
}

constexpr int64_t kMaxSplits = 64;   // a lane each in split_merge

// Positions a part of split_block has at least, for `units` units: enough blocks
// to fill the chip, parts no longer than 1024 (a batch's longest request would
// else end long after the others: 64 requests of 109 .. 7927 positions 111 us, 126
// without, 159 with 256) and no shorter than 128 (a step per wave).
int32_t split_least(int64_t units, int64_t context, int64_t cus) {
    const int64_t parts = std::max<int64_t>(1, 4 * cus / std::max<int64_t>(units, 1));
    const int64_t even = (context + parts - 1) / parts;
    return (int32_t)std::min<int64_t>(1024, std::max<int64_t>(128, (even + 127) / 128 * 128));
}

// Partials of `rows` rows: (max, sum) pairs, then rows of head_dim floats.
size_t partial_head(int64_t rows) { return ((size_t)rows * sizeof(float2) + 255) / 256 * 256; }
size_t partial_bytes(int64_t rows, int hd) { return partial_head(rows) + ((size_t)rows * hd * sizeof(float) + 255) / 256 * 256; }

// Most bytes of a launch's partials, of tiles and of few rows each: units and parts
// are the most that the call's bounds allow, whatever its lengths are (1024 requests
// of a table of 131072 positions, 8 heads of 128, no bounds: 4.3 GB).  Fewer parts
// leave a request that is much longer than the others to fewer blocks, but also fewer
// blocks without work: 256 requests of 100 .. 2000 positions and one of 131072, one
// row each, 641 us without a limit, 624 with 256 MiB, 505 with 128, 484 with 64, 612
// with 32; without bounds 689, 521, 654, 882, 1495; 1024 such requests 1939, 1067,
// 1073, 1358, 1721 and 2052, 1408, 1751, 1737, 1735.
constexpr size_t kMaxPartials = (size_t)128 << 20;
int32_t splits_within(int64_t splits, int64_t rows, int hd) {   // rows: of one split
    const size_t each = (size_t)rows * ((size_t)hd * sizeof(float) + sizeof(float2));
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>(splits, (int64_t)(kMaxPartials / std::max<size_t>(each, 1))));
}

SplitArgs plan_split(const PagedArgs &a, int64_t query, int64_t context, bool tiles, size_t elem, int64_t cus) {
    SplitArgs sa{};
    sa.a = a;
    sa.qvec = aligned(a.q, 16) && (a.q_stride * (int64_t)elem) % 16 == 0;
    sa.scan = !tiles && query * a.rep > 16;
    const int64_t units = (sa.scan ? a.tokens * a.rep / 16 + std::min<int64_t>(a.requests, a.tokens) : a.requests) *
                          (int64_t)a.nkv;
    sa.units = (int32_t)std::min<int64_t>(units, INT32_MAX);
    sa.long_rows = tiles ? 16 : INT32_MAX;
    sa.slots = (int32_t)std::min<int64_t>(16, query * a.rep);
    sa.least = split_least(units, context, cus);
    // at most 2^22 blocks, most of which will have no part
    sa.splits = (int32_t)std::max<int64_t>(
        1, std::min<int64_t>({(context + sa.least - 1) / sa.least, kMaxSplits, (1 << 22) / std::max<int64_t>(units, 1)}));
    sa.splits = splits_within(sa.splits, units * sa.slots, a.hd);
    return sa;
}

struct TileArgs {
    PagedArgs a;
    int32_t units;         // (ROWS rows, key/value head) pairs
    int32_t splits, least; // see cut
    bool pair_up;          // see find_group
    bool qvec;             // q rows are 16-byte aligned
    uint32_t blocks, merge_blocks;   // of the launch that takes split_block's work too
    float2 *ml;            // partials [unit][split][ROWS]: (max, sum)
    float *po;             // and sums of p v, [unit][split][ROWS][head_dim]
};

// Rows of a tile (ROWS): 64, 16 a wave; 128, two column groups a wave, for bf16 rows
// over a bf16 cache whose tiles fill the chip even so, heads of 64 twice over: half
// the LDS reads per product (us with 128 and with 64, 32 heads on 8 of 128: 2048 rows
// over 4096 119 and 143, 1000 over 1000 47 and 28; on 4 of 64: 2048 over 2048 47 and 39,
// 8192 over 8192 351 and 393).  With more matrix work per LDS read (three pieces of fp32
// rows: 301 and 313; the fp32 instruction) 64 always.
constexpr int kWideRows = 128;

// As in split_block: the wave's rows one at a time, where one may have met an inf
// or NaN that it does not see.
template <class XT, class CT, int HD, int ROWS>
__device__ __forceinline__ void rows_apart(const TileArgs &ta, const Group &gr, uint32_t unit, uint32_t split,
                                           int32_t parts, int32_t c0, int32_t c1, int32_t wrow, int32_t wrows,
                                           float *qs) {
    const PagedArgs &a = ta.a;
    const int lane = threadIdx.x & 63;
    for (int rr = 0; rr < wrows; ++rr) {
        const int32_t tt = (wrow + rr) / a.rep;
        const int head = gr.kvh * a.rep + (wrow + rr) % a.rep;
        const RowPart x = row_part<XT, CT, 1>(a, gr.b, gr.q.first + tt, head, c0, min(c1, gr.q.base + tt + 1), qs);
        if (parts == 1) {
            store_row<XT>(a, gr.q.first + tt, head, x);
        } else {
            const int64_t r = ((int64_t)unit * ta.splits + split) * ROWS + wrow + rr - gr.row0;
            if (lane == 0) ta.ml[r] = x.m == -INFINITY ? float2{x.m, x.seen ? 1.0f : 0.0f} : float2{x.m, x.l};
            for (int i = 0; 64 * i + lane < HD; ++i) ta.po[r * HD + 64 * i + lane] = x.o[i];
        }
    }
}

// Many rows per request over a bf16 cache.  A block takes ROWS rows of one
// key/value head and one part of the positions: four waves of 16 or 32 rows,
// tiles of 64 positions in two LDS buffers, each wave copying 16 positions of the
// next tile straight to LDS while this one is multiplied, one barrier a tile.
// The copies go through a buffer resource per 16 positions that ends with them,
// so positions behind the part or without a block read as zeros.  The products
// are those of Step: scores transposed, so that the probabilities need no
// shuffle; keys are read from LDS as stored, values through the transposing LDS
// read (four positions of one dimension per lane).  LDS rows are swizzled, 16-byte
// pieces of keys by the row, 32-byte pieces of values likewise, so that both
// reads touch every bank once; the copies permute their global addresses for it.
// Bound by the matrix instructions and the exponentials that they wait for: 2048
// rows over 4096 positions, 32 heads on 8 of 128, bf16 throughout 116 to 120 us, 103
// GFLOP at 860 to 890 TFLOP/s (a large product: 1143); in a trace 133, of whose cycles
// matrix instructions take 38 in a hundred and vector instructions 40, with no LDS
// conflicts.  Prompts of 150 .. 301 fp32 rows of 12 heads of 64: 17 us in a trace, in
// which launch, look-ups and the first tile count for more than the three pieces'
// products.
template <int HD>
struct TileLds {
    __attribute__((aligned(256))) unsigned char k[2][64 * HD * 2], v[2][64 * HD * 2];   // 32 positions of fp32
    float qs[4][HD];
};

template <class XT, int HD, int ROWS>
__device__ __forceinline__ void tile_block(const TileArgs &ta, uint32_t block, TileLds<HD> &lds, __bf16) {
    constexpr int NP = sizeof(XT) == 4 ? 3 : 1, CG = ROWS / 64;
    constexpr int NJ = HD / 32, ND = HD / 16;
    constexpr int CR = HD / 8, NL = CR / 4;                // 16-byte pieces per row, copies per wave and tile
    constexpr int KD = 16 / CR, VD2 = 8 / ND;              // rows per 256 bytes of LDS, as 16- and 32-byte pieces count
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    uint16_t (*kl)[64 * HD] = (uint16_t (*)[64 * HD])lds.k, (*vl)[64 * HD] = (uint16_t (*)[64 * HD])lds.v;
    auto &qs = lds.qs;
    const PagedArgs &a = ta.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, n = lane & 15;
    const uint32_t unit = block % (uint32_t)ta.units, split = block / (uint32_t)ta.units;
    Group gr;
    if (!find_group<ROWS>(a, unit, 16, ta.pair_up, gr)) return;
    set_rows<ROWS>(a, gr, gr.row0);
    const Cut ct = cut(gr.len, ta.splits, ta.least);
    if ((int32_t)split >= ct.parts) return;
    const int32_t c0 = split * ct.chunk, c1 = min(gr.len, c0 + ct.chunk);
    const int32_t *table = a.table + (int64_t)gr.b * a.most;
    const float c2 = fabsf(a.scale) * 1.44269504f;   // a negative scale turns q's sign
    const int32_t head_rows = HD << a.shift, in_block = (1 << a.shift) - 1;
    const int64_t block_rows = (int64_t)head_rows * a.nkv;
    const __bf16 *kb = (const __bf16 *)a.kc + (int64_t)gr.kvh * head_rows;
    const __bf16 *vb = (const __bf16 *)a.vc + (int64_t)gr.kvh * head_rows;

    // Wave w copies positions 16 w .. of a tile, NL pieces of 1 KiB of keys and of values.
    uint32_t koff[NL], voff[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int r = (64 * j + lane) / CR, c = (64 * j + lane) % CR;
        koff[j] = 16 * (r * CR + (c ^ (r / KD & (CR - 1))));
        voff[j] = 16 * (r * CR + ((((c >> 1) ^ (r / VD2 & (ND - 1))) << 1) | (c & 1)));
    }
    const uint32_t kdst = dma::lds_addr(&kl[0][16 * w * HD]), vdst = dma::lds_addr(&vl[0][16 * w * HD]);
    // The blocks of 64 sub-tiles of 16 positions, one per lane: those of this
    // tile's window and of the next.  (A look-up per tile would stall the wave
    // for its latency, behind the copies in flight.)
    auto window = [&](int32_t p) {
        return p + 16 * lane < c1 ? table[(p + 16 * lane) >> a.shift] : -1;
    };
    int32_t ids = window(c0), ids_next = window(c0 + 1024);
    auto copy = [&](int buf, int32_t p0, int32_t from) {   // from: the window's ids
        const int32_t p = p0 + 16 * w;
        const int32_t id = __builtin_amdgcn_readlane(from, (p - c0) >> 4 & 63);
        const bool ok = p < c1 && (uint32_t)id < (uint32_t)a.num_blocks;
        const int64_t at = (int64_t)(ok ? id : 0) * block_rows + (p & in_block) * HD;
        const int bytes = ok ? min(16, c1 - p) * HD * 2 : 0;
        const dma::i32x4 kr = dma::make_rsrc(kb + at, bytes), vr = dma::make_rsrc(vb + at, bytes);
        const uint32_t kd = __builtin_amdgcn_readfirstlane(kdst + buf * 128 * HD);
        const uint32_t vd = __builtin_amdgcn_readfirstlane(vdst + buf * 128 * HD);
#pragma unroll
        for (int j = 0; j < NL; ++j) dma::dma16(kd + 1024 * j, kr, koff[j], 0);
#pragma unroll
        for (int j = 0; j < NL; ++j) dma::dma16(vd + 1024 * j, vr, voff[j], 0);
    };
    if (c0 < c1) copy(0, c0, ids);   // else nothing waits for it
    uint64_t blocks = __ballot((uint32_t)ids < (uint32_t)a.num_blocks);   // sub-tiles of the window that have one

    // this wave's rows and their positions
    const int32_t wrow = gr.row0 + 16 * CG * w, wrows = min(16 * CG, gr.row0 + gr.rows - wrow);   // may be none
    int32_t row[CG], last[CG];
    bf16x8 q[CG][NP][NJ];
#pragma unroll
    for (int c = 0; c < CG; ++c) {
        row[c] = min(wrow + 16 * c + n, gr.row0 + gr.rows - 1);
        const int32_t token = row[c] / a.rep;
        last[c] = min(gr.q.base + token, gr.q.held - 1);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float x[8];
            load_q8<XT>(a, gr.q.first + token, gr.kvh * a.rep + row[c] % a.rep, 32 * j + 8 * g, ta.qvec, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                __bf16 p[NP];
                pieces<NP>(a.scale < 0.0f ? -x[e] : x[e], p);
#pragma unroll
                for (int i = 0; i < NP; ++i) q[c][i][j][e] = p[i];
            }
        }
    }
    // positions of the wave's first and last row
    const int32_t low = min(gr.q.base + wrow / a.rep, gr.q.held - 1);
    const int32_t high = wrows > 0 ? min(gr.q.base + (wrow + wrows - 1) / a.rep, gr.q.held - 1) : -1;

    // mr: what the exponents of l and o are relative to, in powers of two: a
    // score at most kLag below the row's largest (moving it with every new
    // maximum cost a tenth of the kernel's vector instructions); -inf: no score
    // above -inf yet.  l: sums of p as the second product has them, by a row of ones
    constexpr float kLag = 8.0f;
    float mr[CG];
    int32_t first = INT32_MAX;                // first position in a block
    f32x4 l[CG], o[CG][ND];
#pragma unroll
    for (int c = 0; c < CG; ++c) {
        mr[c] = -INFINITY;
        l[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < ND; ++d) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.0f;
    // eight positions of dimension 16 d + n (see Step), from a buffer of values
    auto value = [&](int buf, int d, int u) {
        s16x4 h[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = 32 * u + 16 * t + 4 * g + n / 4;
            const int vs = ((d ^ (r / VD2 & (ND - 1))) << 1) | (n >> 1 & 1);
            h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)&vl[buf][r * HD + 8 * vs + 4 * (n & 1)]);
        }
        return s16x8{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
    };
    int buf = 0;
    for (int32_t p0 = c0; p0 < c1; p0 += 64, buf ^= 1) {
        // this tile has landed, and every wave is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int32_t at = (p0 - c0) >> 4 & 63;       // of the window
        if (at == 0 && p0 != c0) {
            ids = ids_next;
            ids_next = window(p0 + 1024);
            blocks = __ballot((uint32_t)ids < (uint32_t)a.num_blocks);
        }
        if (p0 + 64 < c1) copy(buf ^ 1, p0 + 64, at == 60 ? ids_next : ids);
        if (p0 > high) continue;
        f32x4 s[CG][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            bf16x8 k[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                k[j] = *(const bf16x8 *)&kl[buf][(16 * t + n) * HD + 8 * ((4 * j + g) ^ (n / KD & (CR - 1)))];
#pragma unroll
            for (int c = 0; c < CG; ++c) {
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = NP - 1; i >= 0; --i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[j], q[c][i][j], x, 0, 0, 0);
                s[c][t] = x;
            }
        }
        // sub-tiles of the part, those without a block
        const int part = p0 + 64 <= c1 ? 15 : (1 << ((c1 - p0 + 15) >> 4)) - 1, hole = (int)(~blocks >> at) & part;
        if (first == INT32_MAX && hole != part) first = p0 + 16 * __builtin_ctz(part & ~hole);
        const bool border = p0 + 63 > low;   // some row does not see all of the tile
        if (hole || border) {
#pragma unroll
            for (int c = 0; c < CG; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int32_t lim = hole >> t & 1 ? -1 : last[c] - (p0 + 16 * t + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c][t][i] = i <= lim ? s[c][t][i] : -INFINITY;
                }
        }
        bf16x8 pp[CG][NP][2];
#pragma unroll
        for (int c = 0; c < CG; ++c) {
            float nm = s[c][0][0];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) nm = fmaxf(nm, s[c][t][i]);
            nm = row4_max(nm) * c2;
            const bool move = nm > mr[c] + kLag;
            if (__any(move)) {
                const float to = move ? nm : mr[c], corr = move ? exp2_fast(mr[c] - to) : 1.0f;
                mr[c] = to;
                l[c] *= corr;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[c][d] *= corr;
            }
            const float ref = mr[c] == -INFINITY ? 0.0f : mr[c];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[c][t][i] = exp2_fast(fmaf(s[c][t][i], c2, -ref));
                    __bf16 x[NP];
                    pieces_of_p<NP>(s[c][t][i], x);
#pragma unroll
                    for (int k = 0; k < NP; ++k) pp[c][k][t / 2][4 * (t & 1) + i] = x[k];
                }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = NP - 1; k >= 0; --k)
                    l[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pp[c][k][u], l[c], 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf16x8 v = __builtin_bit_cast(bf16x8, value(buf, d, u));
#pragma unroll
                for (int c = 0; c < CG; ++c)
#pragma unroll
                    for (int k = NP - 1; k >= 0; --k)
                        o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pp[c][k][u], o[c][d], 0, 0, 0);
            }
    }
    bool odd = false;                             // inf or NaN in a row
#pragma unroll
    for (int c = 0; c < CG; ++c) {
        if (wrow + 16 * c + n >= gr.row0 + gr.rows) continue;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= !(fabsf(o[c][d][i]) < INFINITY);
        const bool none = mr[c] == -INFINITY, seen = first <= last[c];
        if (ct.parts == 1) {
            // nothing seen: 0; only scores of -inf: 0 / 0
            XT *out = (XT *)a.out + (int64_t)(gr.q.first + row[c] / a.rep) * a.out_stride +
                      (int64_t)(gr.kvh * a.rep + row[c] % a.rep) * HD + 4 * g;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out[16 * d + i] = (XT)(none ? (seen ? NAN : 0.0f) : o[c][d][i] / l[c][0]);
        } else {
            const int64_t r = ((int64_t)unit * ta.splits + split) * ROWS + row[c] - gr.row0;
            if (g == 0) ta.ml[r] = none ? float2{-INFINITY, seen ? 1.0f : 0.0f} : float2{mr[c], l[c][0]};
#pragma unroll
            for (int d = 0; d < ND; ++d) *(f32x4 *)(ta.po + r * HD + 16 * d + 4 * g) = o[c][d];
        }
    }
    if (low + 1 >= c1 || !__any(odd)) return;
    rows_apart<XT, __bf16, HD, ROWS>(ta, gr, unit, split, ct.parts, c0, c1, wrow, wrows, qs[w]);
}

// Many rows per request over an fp32 cache, as above but on the fp32 matrix
// instruction (256 flop per clock and CU, which bounds it): four waves of 16
// rows, tiles of 32 positions, a wave copying eight of them.  The products are
// those of Step: values need no transposing read, as the instruction's reduction
// takes one position per lane.  Outputs are dealt four consecutive dimensions of
// every 64 to a lane, so that 16 lanes read 256 bytes of a value row at once;
// keys' 16-byte pieces are swizzled by the row.  A tile's values are summed before
// they join the running sums: an eighth of the roundings.  31 single tokens and a
// chunk of 333, 32 heads on 4 of 64, fp32: 26 us in a trace with split_block's share, 7
// tiles of 32 positions a block, each a wait and 64 matrix instructions of 32 cycles.
template <class XT, int HD, int ROWS>
__device__ __forceinline__ void tile_block(const TileArgs &ta, uint32_t block, TileLds<HD> &lds, float) {
    static_assert(ROWS == 64, "16 rows a wave");
    constexpr int POS = 32;
    constexpr int NJ = HD / 16, NH = HD / 64;
    constexpr int CR = HD / 4, NL = 8 * CR / 64;           // 16-byte pieces per row, copies per wave and tile
    float (*kl)[POS * HD] = (float (*)[POS * HD])lds.k, (*vl)[POS * HD] = (float (*)[POS * HD])lds.v;
    auto &qs = lds.qs;
    const PagedArgs &a = ta.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, n = lane & 15;
    const uint32_t unit = block % (uint32_t)ta.units, split = block / (uint32_t)ta.units;
    Group gr;
    if (!find_group<ROWS>(a, unit, 16, ta.pair_up, gr)) return;
    set_rows<ROWS>(a, gr, gr.row0);
    const Cut ct = cut(gr.len, ta.splits, ta.least);
    if ((int32_t)split >= ct.parts) return;
    const int32_t c0 = split * ct.chunk, c1 = min(gr.len, c0 + ct.chunk);
    const int32_t *table = a.table + (int64_t)gr.b * a.most;
    const float c2 = fabsf(a.scale) * 1.44269504f;         // a negative scale turns q's sign
    const int32_t head_rows = HD << a.shift, in_block = (1 << a.shift) - 1;
    const int64_t block_rows = (int64_t)head_rows * a.nkv;
    const float *kb = (const float *)a.kc + (int64_t)gr.kvh * head_rows;
    const float *vb = (const float *)a.vc + (int64_t)gr.kvh * head_rows;

    // wave w copies positions 8 w .. of a tile
    uint32_t koff[NL], voff[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int r = (64 * j + lane) / CR, c = (64 * j + lane) % CR;
        koff[j] = 16 * (r * CR + (c ^ (8 * (w & 1) + r)));   // the row's place among 16
        voff[j] = 16 * (64 * j + lane);
    }
    const uint32_t kdst = dma::lds_addr(&kl[0][8 * w * HD]), vdst = dma::lds_addr(&vl[0][8 * w * HD]);
    auto window = [&](int32_t p) {                         // as above
        return p + 16 * lane < c1 ? table[(p + 16 * lane) >> a.shift] : -1;
    };
    int32_t ids = window(c0), ids_next = window(c0 + 1024);
    auto copy = [&](int buf, int32_t p0, int32_t from) {
        const int32_t p = p0 + 8 * w;
        const int32_t id = __builtin_amdgcn_readlane(from, (p - c0) >> 4 & 63);
        const bool ok = p < c1 && (uint32_t)id < (uint32_t)a.num_blocks;
        const int64_t at = (int64_t)(ok ? id : 0) * block_rows + (p & in_block) * HD;
        const int bytes = ok ? min(8, c1 - p) * HD * 4 : 0;
        const dma::i32x4 kr = dma::make_rsrc(kb + at, bytes), vr = dma::make_rsrc(vb + at, bytes);
        const uint32_t kd = __builtin_amdgcn_readfirstlane(kdst + buf * POS * HD * 4);
        const uint32_t vd = __builtin_amdgcn_readfirstlane(vdst + buf * POS * HD * 4);
#pragma unroll
        for (int j = 0; j < NL; ++j) dma::dma16(kd + 1024 * j, kr, koff[j], 0);
#pragma unroll
        for (int j = 0; j < NL; ++j) dma::dma16(vd + 1024 * j, vr, voff[j], 0);
    };
    if (c0 < c1) copy(0, c0, ids);   // else nothing waits for it
    uint64_t blocks = __ballot((uint32_t)ids < (uint32_t)a.num_blocks);

    const int32_t wrow = gr.row0 + 16 * w, wrows = min(16, gr.row0 + gr.rows - wrow);   // may be none
    const int32_t row = min(wrow + n, gr.row0 + gr.rows - 1), token = row / a.rep;
    const int32_t last = min(gr.q.base + token, gr.q.held - 1);
    float q[NJ][4];
    {
        const XT *x = (const XT *)a.q + (gr.q.first + token) * a.q_stride +
                      (int64_t)(gr.kvh * a.rep + row % a.rep) * HD + 4 * g;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) q[j][c] = a.scale < 0.0f ? -(float)x[16 * j + c] : (float)x[16 * j + c];
    }
    const int32_t low = min(gr.q.base + wrow / a.rep, gr.q.held - 1);
    const int32_t high = wrows > 0 ? min(gr.q.base + (wrow + wrows - 1) / a.rep, gr.q.held - 1) : -1;

    constexpr float kLag = 8.0f;                           // as above
    float mr = -INFINITY, l = 0.0f;                        // l: this lane's positions only
    int32_t first = INT32_MAX;
    f32x4 o[4 * NH];
#pragma unroll
    for (int d = 0; d < 4 * NH; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    int buf = 0;
    for (int32_t p0 = c0; p0 < c1; p0 += POS, buf ^= 1) {
        // this tile has landed, and every wave is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int32_t at = (p0 - c0) >> 4 & 63;            // of the window
        if (at == 0 && p0 != c0) {
            ids = ids_next;
            ids_next = window(p0 + 1024);
            blocks = __ballot((uint32_t)ids < (uint32_t)a.num_blocks);
        }
        if (p0 + POS < c1) copy(buf ^ 1, p0 + POS, at == 62 ? ids_next : ids);
        if (p0 > high) continue;
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};   // two chains: half the rounding of one
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4 k = *(const f32x4 *)&kl[buf][(16 * t + n) * HD + 4 * ((4 * j + g) ^ n)];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    x[c & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c], q[j][c], x[c & 1], 0, 0, 0);
            }
            s[t] = x[0] + x[1];
        }
        // sub-tiles of the part, those without a block
        const int part = p0 + 16 < c1 ? 3 : 1, hole = (int)(~blocks >> at) & part;
        if (first == INT32_MAX && hole != part) first = p0 + 16 * __builtin_ctz(part & ~hole);
        if (hole || p0 + POS - 1 > low) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int32_t lim = hole >> t & 1 ? -1 : last - (p0 + 16 * t + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = i <= lim ? s[t][i] : -INFINITY;
            }
        }
        float nm = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) nm = fmaxf(nm, s[t][i]);
        nm = row4_max(nm) * c2;
        const bool move = nm > mr + kLag;
        if (__any(move)) {
            const float to = move ? nm : mr, corr = move ? exp2_fast(mr - to) : 1.0f;
            mr = to;
            l *= corr;
#pragma unroll
            for (int d = 0; d < 4 * NH; ++d) o[d] *= corr;
        }
        const float ref = mr == -INFINITY ? 0.0f : mr;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = exp2_fast(fmaf(s[t][i], c2, -ref));
        l += ((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])) + ((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
        f32x4 pv[4 * NH];
#pragma unroll
        for (int d = 0; d < 4 * NH; ++d) pv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const f32x4 v = *(const f32x4 *)&vl[buf][(16 * t + 4 * g + i) * HD + 64 * h + 4 * n];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        pv[4 * h + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c], s[t][i], pv[4 * h + c], 0, 0, 0);
                }
#pragma unroll
        for (int d = 0; d < 4 * NH; ++d) o[d] += pv[d];
    }
    l = row4_sum(l);

    // lane (g, n): outputs 64 h + 16 g + 4 i + c of row n
    bool odd = false;                                      // inf or NaN in a row
    if (wrow + n < gr.row0 + gr.rows) {
#pragma unroll
        for (int d = 0; d < 4 * NH; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= !(fabsf(o[d][i]) < INFINITY);
        const bool none = mr == -INFINITY, seen = first <= last;
        const int64_t r = ((int64_t)unit * ta.splits + split) * ROWS + row - gr.row0;
        XT *out = (XT *)a.out + (int64_t)(gr.q.first + token) * a.out_stride +
                  (int64_t)(gr.kvh * a.rep + row % a.rep) * HD + 16 * g;
        if (ct.parts > 1 && g == 0) ta.ml[r] = none ? float2{-INFINITY, seen ? 1.0f : 0.0f} : float2{mr, l};
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 v = {o[4 * h][i], o[4 * h + 1][i], o[4 * h + 2][i], o[4 * h + 3][i]};
                if (ct.parts == 1) {
                    // nothing seen: 0; only scores of -inf: 0 / 0
#pragma unroll
                    for (int c = 0; c < 4; ++c) out[64 * h + 4 * i + c] = (XT)(none ? (seen ? NAN : 0.0f) : v[c] / l);
                } else {
                    *(f32x4 *)(ta.po + r * HD + 64 * h + 16 * g + 4 * i) = v;
                }
            }
    }
    if (low + 1 >= c1 || !__any(odd)) return;
    rows_apart<XT, float, HD, ROWS>(ta, gr, unit, split, ct.parts, c0, c1, wrow, wrows, qs[w]);
}

// Joins tile_block's parts: HD / 4 threads a row.  Bound by latency: 5 us in a trace after the
// prompts above and after the mixed batch, with split_merge's share.  (Eight parts'
// loads in flight at once: no difference.)
template <class XT, int HD, int ROWS>
__device__ __forceinline__ void tile_merge(const TileArgs &ta, uint32_t block) {
    constexpr int T = HD / 4, R = 256 / T;
    const PagedArgs &a = ta.a;
    const uint32_t unit = block / (ROWS / R);
    const int rr = (int)(block % (ROWS / R)) * R + threadIdx.x / T, d4 = threadIdx.x % T;
    Group gr;
    if (!find_group<ROWS>(a, unit, 16, ta.pair_up, gr)) return;
    set_rows<ROWS>(a, gr, gr.row0);
    const Cut ct = cut(gr.len, ta.splits, ta.least);
    if (ct.parts == 1 || rr >= gr.rows) return;
    const int64_t at0 = (int64_t)unit * ta.splits * ROWS + rr;
    float mm = -INFINITY, any = 0.0f;
#pragma unroll 4
    for (int s = 0; s < ct.parts; ++s) {
        const float2 x = ta.ml[at0 + (int64_t)s * ROWS];
        mm = fmaxf(mm, x.x);
        any = fmaxf(any, x.y);
    }
    float l = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < ct.parts; ++s) {
        const int64_t r = at0 + (int64_t)s * ROWS;
        const float2 x = ta.ml[r];
        const float f = x.x == -INFINITY ? 0.0f : exp2_fast(x.x - mm);
        if (x.x != -INFINITY) l += f * x.y;
        o += f * *(const f32x4 *)(ta.po + r * HD + 4 * d4);
    }
    const int32_t row = gr.row0 + rr;
    XT *out = (XT *)a.out + (int64_t)(gr.q.first + row / a.rep) * a.out_stride +
              (int64_t)(gr.kvh * a.rep + row % a.rep) * HD + 4 * d4;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (XT)(mm == -INFINITY ? (any > 0.0f ? NAN : 0.0f) : o[i] / l);
}

// One launch for a batch of chunks and single tokens: the tiles' blocks, then those
// of the requests with few rows, which fill in beside them (31 tokens and a
// 333-token chunk over fp32: 48 us in two launches and two merges, 35 when joined, 29 now); likewise
// their merges.
template <class XT, class CT, int HD, int ROWS>
__global__ __launch_bounds__(256, 2) void paged_both(const TileArgs ta, const SplitArgs sa) {
    __shared__ __attribute__((aligned(256))) union {
        TileLds<HD> tile;
        SplitLds<HD> split;
    } lds;
    const uint32_t block = sa.base + blockIdx.x;
    if (block < ta.blocks) tile_block<XT, HD, ROWS>(ta, block, lds.tile, CT{});
    else split_block<XT, CT, HD>(sa, block - ta.blocks, lds.split);
}

template <class XT, int HD, int ROWS>
__global__ __launch_bounds__(256) void paged_both_merge(const TileArgs ta, const SplitArgs sa) {
    const uint32_t block = sa.base + blockIdx.x;
    if (block < ta.merge_blocks) tile_merge<XT, HD, ROWS>(ta, block);
    else split_merge<XT, HD>(sa, block - ta.merge_blocks);
}

// Whether so many tiles fill two blocks per CU, nine in ten of them.
bool fills(int64_t tiles, int64_t cus) { return 10 * tiles >= 9 * 2 * cus; }

// Parts of tile_block's tiles: none where they fill the chip (2048 rows over 4096
// positions, on an earlier tile: 1.2 times the time in two parts, 1.45 in four: partials of fp32 rows
// cost more than evener blocks gain), else enough to fill it twice over, of at least 256 positions (a
// chunk of 8 rows over 4096: 16 us, 71 without; 600 over 4000 81, 89 without).
TileArgs plan_tile(const PagedArgs &a, int64_t query, int64_t context, int64_t tile_rows, size_t elem, int64_t cus) {
    TileArgs ta{};
    ta.a = a;
    ta.qvec = aligned(a.q, 16) && (a.q_stride * (int64_t)elem) % 16 == 0;
    const int64_t rows = a.tokens * a.rep;
    const int64_t units = (rows / tile_rows + std::min<int64_t>(a.requests, rows / 17 + 1)) * (int64_t)a.nkv;
    ta.units = (int32_t)std::min<int64_t>(units, INT32_MAX);
    // How many there are: chunks alike, as the step's bounds tell, have a last, partial
    // tile each (64 chunks of 5 rows over 1000: 67 us with parts for as many tiles as the
    // rows would fill, 50 so); else those that the rows fill, as the rest may be single tokens.
    const bool alike = 2 * a.tokens >= a.requests * query;
    const int64_t each = (rows + a.requests - 1) / a.requests;   // rows of a request, on average
    const int64_t tiles = alike ? a.requests * ((each + tile_rows - 1) / tile_rows) : rows / tile_rows;
    const int64_t full = std::max<int64_t>(1, tiles * a.nkv);
    const int64_t parts = fills(full, cus) ? 1 : std::max<int64_t>(1, 4 * cus / full);
    ta.least = 256;
    ta.splits = (int32_t)std::max<int64_t>(1, std::min({parts, (context + ta.least - 1) / ta.least, kMaxSplits}));
    ta.splits = splits_within(ta.splits, units * tile_rows, a.hd);
    // two blocks share a CU: all run at once, or the longest have to come first (512 blocks
    // of 2048 rows over 4096: 119 us, 121 without; over 8192: 244, 250)
    ta.pair_up = full <= 2 * cus;
    return ta;
}

// launch(grid) for all of them, from sa.base on.
template <class F>
hipError_t launch_blocks(int64_t blocks, SplitArgs &sa, F launch) {
    hipError_t e = hipSuccess;
    for (int64_t b = 0; e == hipSuccess && b < blocks; b += kMostBlocks) {
        sa.base = (uint32_t)b;
        launch(dim3((unsigned)std::min(blocks - b, kMostBlocks)));
        e = hipGetLastError();
    }
    return e;
}

template <class XT, class CT, int HD, int ROWS>
hipError_t launch_both(const TileArgs &ta, SplitArgs &sa, int64_t split_blocks, int64_t split_merges, hipStream_t s) {
    const hipError_t e = launch_blocks(ta.blocks + split_blocks, sa, [&](dim3 grid) {
        hipLaunchKernelGGL((paged_both<XT, CT, HD, ROWS>), grid, dim3(256), 0, s, ta, sa);
    });
    if (e != hipSuccess) return e;
    return launch_blocks(ta.merge_blocks + split_merges, sa, [&](dim3 grid) {
        hipLaunchKernelGGL((paged_both_merge<XT, HD, ROWS>), grid, dim3(256), 0, s, ta, sa);
    });
}

template <class XT, class CT, int HD>
hipError_t launch_matrix(tbh_device *dev, const PagedArgs &a, int64_t query, int64_t context, hipStream_t s) {
    const int64_t cus = std::max(1, dev->cu_count);
    // More than one group of 16 rows: tiles, or else groups apart.  us, bf16 throughout, 32
    // heads on 8 of 128: 8 chunks of 5 rows over 2000 positions 24 in tiles and 29 in groups,
    // 64 of 5 over 1000 50 and 56, 8 of 16 over 2000 27 and 39, a chunk of 32 over 1024 14 and
    // 17.  fp32, 32 on 4 of 64, gains from more rows on and loses before: a chunk of 8 over 4096
    // 23.0 and 20.5, one of 32 over 1024 21.1 and 15.9, 64 chunks of 5 over 1000 60.8 and 58.9, 8
    // of 5 and of 8 over 2000 30.6 and 30.0, 31.5 and 31.8, 8 of 16 33.9 and 45.9.  Heads of 32 and
    // 96 have no tile kernel: every 16 rows read the context (2048 rows over 4096: 188 and 375 us,
    // 82 at heads of 64, 116 at 128).
    const bool tiles = (HD == 64 || HD == 128) && query * a.rep > 16;
    SplitArgs sa = plan_split(a, query, context, tiles, sizeof(XT), cus);
    TileArgs ta{};
    int64_t R = 64;
    if (sizeof(XT) + sizeof(CT) == 4 && fills(a.tokens * a.rep / kWideRows * a.nkv * HD / 128, cus)) R = kWideRows;
    if (tiles) ta = plan_tile(a, query, context, R, sizeof(XT), cus);
    const int64_t tile_rows = tiles && ta.splits > 1 ? (int64_t)ta.units * ta.splits * R : 0;
    const int64_t split_rows = sa.splits > 1 ? (int64_t)sa.units * sa.splits * sa.slots : 0;
    if (tile_rows + split_rows > 0) {
        const size_t tb = tile_rows ? partial_bytes(tile_rows, HD) : 0, sb = split_rows ? partial_bytes(split_rows, HD) : 0;
        char *ws = (char *)stream_workspace(dev, s, tb + sb);
        if (ws) {
            ta.ml = (float2 *)ws;
            ta.po = (float *)(ws + partial_head(tile_rows));
            sa.ml = (float2 *)(ws + tb);
            sa.po = (float *)(ws + tb + partial_head(split_rows));
        } else {
            ta.splits = sa.splits = 1;   // no workspace (graph capture before any eager call): whole contexts
        }
    }
    const int64_t tile_blocks = tiles ? (int64_t)ta.units * ta.splits : 0, split_blocks = (int64_t)sa.units * sa.splits;
    const int64_t tile_merges = tiles && ta.splits > 1 ? (int64_t)ta.units * (R * HD / 1024) : 0;
    const int64_t split_merges = sa.splits > 1 ? ((int64_t)sa.units * sa.slots + 3) / 4 : 0;
    if (std::max(tile_blocks + split_blocks, tile_merges + split_merges) > INT32_MAX || sa.units == INT32_MAX ||
        ta.units == INT32_MAX)
        return hipErrorInvalidValue;
    ta.blocks = (uint32_t)tile_blocks;
    ta.merge_blocks = (uint32_t)tile_merges;
    if constexpr (HD == 64 || HD == 128) {
        if (tiles) {
            if constexpr (sizeof(XT) + sizeof(CT) == 4)
                if (R == kWideRows) return launch_both<XT, CT, HD, kWideRows>(ta, sa, split_blocks, split_merges, s);
            return launch_both<XT, CT, HD, 64>(ta, sa, split_blocks, split_merges, s);
        }
    }
    const hipError_t e = launch_blocks(split_blocks, sa, [&](dim3 grid) {
        hipLaunchKernelGGL((paged_split<XT, CT, HD>), grid, dim3(256), 0, s, sa);
    });
    if (e != hipSuccess) return e;
    return launch_blocks(split_merges, sa, [&](dim3 grid) {
        hipLaunchKernelGGL((paged_split_merge<XT, HD>), grid, dim3(256), 0, s, sa);
    });
}

template <class XT, class CT>
hipError_t launch_paged(tbh_device *dev, const PagedArgs &a, int64_t query, int64_t context, hipStream_t s) {
    // the matrix kernels take a tile of 16 positions from one block
    if (a.shift >= 4 && a.num_blocks > 0 && a.most > 0) {
        switch (a.hd) {
        case 32: return launch_matrix<XT, CT, 32>(dev, a, query, context, s);
        case 64: return launch_matrix<XT, CT, 64>(dev, a, query, context, s);
        case 96: return launch_matrix<XT, CT, 96>(dev, a, query, context, s);
        case 128: return launch_matrix<XT, CT, 128>(dev, a, query, context, s);
        default: break;
        }
    }
    const int64_t rows = a.tokens * a.nh, across = std::min(rows, kMostBlocks);
    hipLaunchKernelGGL((paged_rows<XT, CT>), dim3((unsigned)across, (unsigned)((rows + across - 1) / across)), dim3(256), 0,
                       s, a);
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
    const int64_t query = q.max_query_len ? std::min<int64_t>(q.max_query_len, q.tokens) : q.tokens;
    const int64_t table = (int64_t)layout->max_blocks * layout->block_size;
    const int64_t context = q.max_context_len ? std::min<int64_t>(q.max_context_len, table) : table;
    const auto held = hold_launches(dev, s);
    hipError_t e;
    switch ((q.type == TBH_BF16) * 2 + (layout->type == TBH_BF16)) {
    case 0: e = launch_paged<float, float>(dev, a, query, context, s); break;
    case 1: e = launch_paged<float, __bf16>(dev, a, query, context, s); break;
    case 2: e = launch_paged<__bf16, float>(dev, a, query, context, s); break;
    default: e = launch_paged<__bf16, __bf16>(dev, a, query, context, s); break;
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "paged attention launch");
}

}  // extern "C"
