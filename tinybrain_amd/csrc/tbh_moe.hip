// tbh_moe.hip -- a mixture-of-experts layer on block-scaled FP8 weights, for a
// few tokens:
//   z = x . router^T;  the top_k largest z of a token are its experts, with
//   weights p = softmax(z) (over all experts, or over the chosen ones)
//   y = sum over its experts e of p_e (silu(x . G_e) * (x . U_e)) . D_e
// Few tokens are bound by reading the chosen experts' weights once: rows of x
// stay as exact as they came, as bf16 or as three bf16 pieces of an fp32, h is two
// pieces of 16 bits together (bf16 rows, whose y is rounded to 8) or three, and the
// weights are widened to bf16 (exactly) on their way to the matrix instruction.
//   Three launches, as every chosen expert's h has to be whole before D_e, and the
// choice before either.  Their times in us (route, up, down; floor: the chosen experts'
// bytes at the 4.8 TB/s of a large copy):
//   1 token, 2 of 8 experts of 2048 x 5632, fp32 rows      8.5  11.8  10.0   (14.5)
//   13 tokens, 6 of 64 experts of 2048 x 1000, bf16       11.4  41.2  29.5   (59)
//   64 tokens, 4 of 32 experts of 4096 x 2048, bf16       13.2   111  69.8   (168)
// What is above the floor is the latency of launches and of loads that depend on
// one another (ids, lists, weights, the join), not the work.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "tbh_fp8.h"
#include "tbh_join.h"
#include "tbh_wave.h"

struct tbh_moe {
    tbh_device *dev = nullptr;
    int64_t H = 0, I = 0, hb = 0, ib = 0;     // blocks of 128
    int32_t E = 0;
    float *router = nullptr;                  // [E][hb * 128], padded with zeros
    uint8_t *gate_up = nullptr;               // [E][ib * 8][hb][gate, up][2048]
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
constexpr int kSplits = 4;          // parts of the inputs of a router's product
constexpr int kListHead = 2;        // expert, number of its tokens

struct Args {
    const void *x;
    void *y;
    int64_t ldx, ldy;
    const float *router;     // [E][hb * 128]
    const uint8_t *gate_up, *down;
    const float *gate_scales, *up_scales, *down_scales;
    int32_t *ids;            // [T][top_k]
    float *weights;          // [T][top_k]
    uint32_t *counters;
    double *logits;          // [splits][T][E]
    float *sums;             // [tiles of 32 outputs][parts][T][32]
    __bf16 *xp;              // [P][T][hb * 128], see pieces_of
    __bf16 *hp;              // [PH][T * top_k][ib * 128]
    int32_t *lists;          // [used][kListHead + kMaxTokens]: an expert, its tokens' places in ids
    int T, E, H, hb, ib, top_k, used, splits, parts;
    int tiles;               // of 16 outputs that a wave of moe_down takes
    bool normalize, vec;     // vec: rows of x can be read four elements at a time
};

// v as P pieces that sum to it: a bf16 as it is; of an fp32 what is cut after 8 bits, and the rest
// in the same way, the last piece rounded.  Three hold all of an fp32, two are off by at most 2^-16
// of it.  (An infinity is its first piece and zeros, not infinity less infinity.)
template <int P>
__device__ __forceinline__ void pieces_of(float v, __bf16 (&p)[P]) {
#pragma unroll
    for (int i = 0; i + 1 < P; ++i) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u;
        const float cut = __builtin_bit_cast(float, u);
        p[i] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
        v = v == cut ? 0.0f : v - cut;
    }
    p[P - 1] = (__bf16)v;
}

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Four consecutive elements of a row, those at and behind `left` 0.
template <class T>
__device__ __forceinline__ void load4(const T *p, int left, bool vec, float (&x)[4]) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 v = *(const f32x4 *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = v[i];
        } else {
            const bf16x4 v = *(const bf16x4 *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < left ? (float)p[i] : 0.0f;
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_most(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    v = dpp_most<wave::kXor1>(v);
    v = dpp_most<wave::kXor2>(v);
    v = dpp_most<wave::kHalfMirror>(v);
    v = dpp_most<wave::kRowMirror>(v);
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
    return max(max(a, b), max(c, d));
}

// The double whose key (sign flipped, or all bits of a negative one) is u.
__device__ __forceinline__ double from_key(uint64_t u) {
    return __builtin_bit_cast(double, u ^ (u >> 63 ? 1ull << 63 : ~0ull));
}

// A wave picks a token's experts, one after the other, from the a.splits parts of its
// logits: of up to 64 N experts, lane l holds l + 64 i.  Logits are compared as whole
// numbers in the same order, 32 bits at a time (0.75 us an expert with 64-bit maxima, 0.1 so).
template <int N>
__device__ __forceinline__ void choose(const Args &a, int t) {
    const int lane = threadIdx.x & 63;
    // all of the loads, which take a trip past the caches, before the first is used
    double z[N][kSplits];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double *p = a.logits + (int64_t)t * a.E + min(lane + 64 * i, a.E - 1);
#pragma unroll
        for (int s = 0; s < kSplits; ++s) z[i][s] = s < a.splits ? handed_over(p + (int64_t)s * a.T * a.E) : 0.0;
    }
    uint32_t hi[N], lo[N];        // 0: none, or taken
    float all = 0.0f;
    uint32_t first_hi = 0, first_lo = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        double sum = z[i][0];
#pragma unroll
        for (int s = 1; s < kSplits; ++s) sum += z[i][s];
        // NaN is in no order: an expert like any other, behind the rest; zeros are equal
        if (sum != sum) sum = -HUGE_VAL;
        if (sum == 0.0) sum = 0.0;
        z[i][0] = sum;
        uint64_t u = __builtin_bit_cast(uint64_t, sum);
        u ^= (int64_t)u < 0 ? ~0ull : 1ull << 63;
        const bool in = lane + 64 * i < a.E;
        hi[i] = in ? (uint32_t)(u >> 32) : 0, lo[i] = in ? (uint32_t)u : 0;
    }
    int id = 0;
    double own = 0.0;             // lane j: the logit of the j-th
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t h = 0, l = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) h = max(h, hi[i]);
        h = wave_most(h);
#pragma unroll
        for (int i = 0; i < N; ++i) l = max(l, hi[i] == h ? lo[i] : 0u);
        l = wave_most(l);
        int e = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t m = __ballot(hi[i] == h && lo[i] == l);
            if (m && e < 0) {
                const int at = __builtin_ctzll(m);
                e = 64 * i + at;
                if (lane == at) hi[i] = lo[i] = 0;
            }
        }
        if (j == 0) first_hi = h, first_lo = l;
        if (lane == j) id = e, own = from_key((uint64_t)h << 32 | l);
    }
    const double most = from_key((uint64_t)first_hi << 32 | first_lo);
    const float weight = lane < a.top_k ? expf((float)(own - most)) : 0.0f;
    if (a.normalize) {
        all = weight;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + 64 * i < a.E) all += expf((float)(z[i][0] - most));
    }
    all = wave::sum(all);
    if (lane < a.top_k) {
        a.ids[t * a.top_k + lane] = id;
        a.weights[t * a.top_k + lane] = weight / all;
    }
}

// Logits of 16 tokens and 16 experts over a part of the inputs, on the 64-bit matrix
// instruction: products of two floats are exact there, and which of two near logits
// is the larger decides an expert.  Lane (g, r) has inputs 4 g .. 4 g + 3 of each 16 of
// token r and of expert r; of the result, experts 4 i + g of token r.  The instruction
// takes 64 cycles, so that a tile is parted over 16 waves and a.splits blocks; the block
// that finishes a tile of tokens picks their experts, a wave a token.  Blocks of the
// first experts also write the rows' pieces.  Bound by latency: of 8.4 us for one token
// and 8 experts, 2.6 are the loads and products, 1.9 the sums over waves, 0.9 the count of
// the blocks, 1.0 the choice.
template <class T, int P>
__global__ __launch_bounds__(1024) void moe_route(Args a) {
    __shared__ double part[16][256];
    __shared__ uint32_t seen;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, t0 = blockIdx.y * 16, e0 = blockIdx.x * 16, hp = a.hb * kBlock;
    const int steps = a.hb * (kBlock / 16), w = blockIdx.z * 16 + wave, ws = a.splits * 16;
    const int s0 = steps * w / ws, s1 = steps * (w + 1) / ws;
    const bool live = t0 + r < a.T;
    const T *x = (const T *)a.x + (int64_t)(t0 + r) * a.ldx + 4 * g;
    const float *router = a.router + (int64_t)min(e0 + r, a.E - 1) * hp + 4 * g;
    f64x4 z{0.0, 0.0, 0.0, 0.0};
    constexpr int D = 4;
    for (int s = s0; s < s1; s += D) {
        float xv[D][4];
        f32x4 rv[D];
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int k = (s + d) * 16;
            const bool in = s + d < s1;
            rv[d] = in ? *(const f32x4 *)(router + k) : f32x4{0.f, 0.f, 0.f, 0.f};
            load4(x + k, in && live ? a.H - k - 4 * g : 0, a.vec, xv[d]);
        }
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (e0 == 0 && live && s + d < s1) {
                bf16x4 o[P];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __bf16 p[P];
                    pieces_of<P>(xv[d][i], p);
#pragma unroll
                    for (int j = 0; j < P; ++j) o[j][i] = p[j];
                }
#pragma unroll
                for (int j = 0; j < P; ++j)
                    *(bf16x4 *)(a.xp + ((int64_t)j * a.T + t0 + r) * hp + (s + d) * 16 + 4 * g) = o[j];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                z = __builtin_amdgcn_mfma_f64_16x16x4f64((double)rv[d][i], (double)xv[d][i], z, 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][r * 16 + 4 * j + g] = z[j];
    __syncthreads();
    const int t = t0 + (threadIdx.x >> 4), e = e0 + (threadIdx.x & 15);
    if (threadIdx.x < 256 && t < a.T && e < a.E) {
        double v = 0.0;
        for (int i = 0; i < 16; ++i) v += part[i][threadIdx.x];
        hand_over(a.logits + ((int64_t)blockIdx.z * a.T + t) * a.E + e, v);
    }
    if (!last_to_arrive(a.counters + blockIdx.y, gridDim.x * gridDim.z, &seen) || t0 + wave >= a.T) return;
    if (a.E <= 64) choose<1>(a, t0 + wave);
    else choose<kMaxExperts / 64>(a, t0 + wave);
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

// The rows of a matrix instruction's other operand: P pieces of kTokens<P> tokens side by
// side, so that an fp32 row costs no more instructions and loads than its pieces fill.
template <int P>
constexpr int kTokens = 16 / P;
// Column r16's token among them (P == 3: the last column repeats, and is not used).
template <int P>
__device__ __forceinline__ int token_of(int r16) {
    return min(r16 / P, kTokens<P> - 1);
}
template <int P>
__device__ __forceinline__ int piece_of(int r16) {
    return r16 % P;
}
// A token's sum over its pieces, in the column of its first.
template <int P>
__device__ __forceinline__ f32x4 over_pieces(f32x4 v) {
    // columns + 1, + 2
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (P == 2) v[i] += wave::dpp<0x101>(v[i]);
        if constexpr (P == 3) v[i] += wave::dpp<0x101>(v[i]) + wave::dpp<0x102>(v[i]);
    }
    return v;
}
template <int P>
__device__ __forceinline__ bool first_piece(int r16) {
    return r16 % P == 0 && r16 / P < kTokens<P>;
}

// acc[t][c] += scale[t] * (tile t . rows c) of one 128-deep block, for RT tiles and CT column
// tiles of rows that are the sum of PK pieces; row[c]: the lane's row at input 16 g of the block,
// its pieces `step` elements apart.
template <int PK, int RT, int CT>
__device__ __forceinline__ void block_product(const i32x4 (&w)[RT][2], const float (&scale)[RT], const __bf16 *const (&row)[CT],
                                              int64_t step, f32x4 (&acc)[RT][CT]) {
    bf16x8 x[CT][PK][4];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int q = 0; q < PK; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[c][q][i] = *(const bf16x8 *)(row[c] + q * step + 64 * (i >> 1) + 8 * (i & 1));
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        f32x4 part[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) part[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 o[2];
            fp8::widen(w[t][h], o);
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int q = 0; q < PK; ++q)
#pragma unroll
                    for (int s = 0; s < 2; ++s) part[c] = fp8::mfma_wide(o[s], x[c][q][2 * h + s], part[c]);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][c][i] = __builtin_fmaf(part[c][i], scale[t], acc[t][c][i]);
    }
}

__device__ __forceinline__ void load_tile(i32x4 (&w)[2], const uint8_t *p) {
    w[0] = *(const i32x4 *)p, w[1] = *(const i32x4 *)(p + 1024);
}

// h of 16 inner columns for an expert's tokens c0 .. c0 + CT kTokens.
template <int P, int PH, int CT>
__device__ __forceinline__ void up_tokens(const Args &a, int e, int tile, const int32_t *slots, int c0, int count,
                                          f32x4 (*red)[64]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    const int hp = a.hb * kBlock;
    const __bf16 *row[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        // a column past the last token repeats it; its result is not stored
        const int slot = slots[min(c0 + c * kTokens<P> + token_of<P>(r16), count - 1)];
        row[c] = a.xp + ((int64_t)piece_of<P>(r16) * a.T + slot / a.top_k) * hp + 16 * g;
    }
    f32x4 acc[2][CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[0][c] = acc[1][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t *wt = a.gate_up + ((int64_t)e * a.ib * 8 + tile) * 2 * a.hb * kTileBytes + lane * 16;
    const int64_t sb = ((int64_t)e * a.ib + tile / 8) * a.hb;
    const int b0 = a.hb * wave / 4, b1 = a.hb * (wave + 1) / 4;
    for (int b = b0; b < b1; ++b) {
        i32x4 w[2][2];
        load_tile(w[0], wt + (int64_t)b * (2 * kTileBytes));
        load_tile(w[1], wt + (int64_t)b * (2 * kTileBytes) + kTileBytes);
        const float s[2] = {a.gate_scales[sb + b], a.up_scales[sb + b]};
        const __bf16 *at[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) at[c] = row[c] + b * kBlock;
        block_product<1>(w, s, at, 0, acc);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        red[wave * 2 * CT + 2 * c][lane] = acc[0][c];
        red[wave * 2 * CT + 2 * c + 1][lane] = acc[1][c];
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
        gv = over_pieces<P>(gv), uv = over_pieces<P>(uv);
        const int at = c0 + c * kTokens<P> + token_of<P>(r16);
        if (at < count && first_piece<P>(r16)) {
            const int ip = a.ib * kBlock;
            bf16x4 o[PH];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __bf16 p[PH];
                pieces_of<PH>(gv[i] / (1.0f + expf(-gv[i])) * uv[i], p);
#pragma unroll
                for (int j = 0; j < PH; ++j) o[j][i] = p[j];
            }
#pragma unroll
            for (int j = 0; j < PH; ++j)
                *(bf16x4 *)(a.hp + ((int64_t)j * a.T * a.top_k + slots[at]) * ip + tile * 16 + 4 * g) = o[j];
        }
    }
    __syncthreads();
}

// Gate and up products of 16 inner columns of one expert and h = silu(gate) * up;
// the waves part the inputs.  Gate's and up's tiles lie side by side, so that a wave
// reads 4 KiB in a row a step.  Bound by memory: 32 experts of 4096 x 2048 (537 MB) in 111 us,
// 4.8 TB/s, 2 of 2048 x 5632 (46 MB) in 11.8, of which 1.0 is the search for the expert.  (Two
// or four steps' loads ahead of the products: no faster, the blocks of a CU hide each other's.)
template <int P, int PH>
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
    // two column tiles to a load of the weights while there are more than one's tokens (a whole call of 64
    // tokens, 2 of 8 experts of 4096 x 4096: 127 us against 136 one at a time, of fp32 224 and 248).  More
    // tokens load them again, from the caches.
    int c0 = 0;
    for (; count - c0 > kTokens<P>; c0 += 2 * kTokens<P>) up_tokens<P, PH, 2>(a, e, blockIdx.x, slots, c0, count, red);
    if (c0 < count) up_tokens<P, PH, 1>(a, e, blockIdx.x, slots, c0, count, red);
}

// 16 RT outputs of all tokens: the waves of a.parts blocks part the units of kUnit blocks
// of inputs of the active experts, the next unit's tiles in flight while one is
// multiplied; each wave adds its share of a token's sum to its own row in LDS, once an
// expert.  Joined in order, and over the blocks by the one that is last.  (A tile for one
// token needs twice as many loads of h as of weights, so that a wave takes two or four tiles a
// load of h, see size_up.)  Bound by memory where there are many experts (268 MB in 70 us, 3.8 TB/s, which
// with h in one piece of bf16 took 67), by the
// latency of the join for one token: 4.6 of 10 us are products.  (kUnit 1, 2 or 4: a whole call on
// 1 token 29.1, 28.9, 31.4 us, on 64, h in one piece, 177, 169, 169.)
constexpr int kDownWaves = 8, kUnit = 2;

template <class T, int P, int PK, int RT>
__global__ __launch_bounds__(64 * kDownWaves) void moe_down(Args a) {
    extern __shared__ f32x4 sums[];       // [waves][4 RT quads of outputs][T], then the experts' heads
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4, tile = blockIdx.x * RT, w = blockIdx.y * kDownWaves + wave;
    f32x4 *own = sums + wave * a.T * (4 * RT);
    int2 *heads = (int2 *)(sums + kDownWaves * a.T * (4 * RT));      // expert, number of its tokens
    for (int y = tid; y < a.used; y += 64 * kDownWaves) heads[y] = *(const int2 *)(a.lists + y * (kListHead + kMaxTokens));
    for (int i = lane; i < a.T * (4 * RT); i += 64) own[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    int active = 0;
    for (int y = 0; y < a.used; y += 64) active += __builtin_popcountll(__ballot(y + lane < a.used && heads[y + lane].y > 0));
    const int per = (a.ib + kUnit - 1) / kUnit, total = active * per, ws = a.parts * kDownWaves;
    const int first = (int)((int64_t)total * w / ws), end = (int)((int64_t)total * (w + 1) / ws);
    const int ip = a.ib * kBlock;
    i32x4 next[kUnit][RT][2];
    float next_s[kUnit];
    int y = first / per, b0 = (first - y * per) * kUnit;      // of the unit that is loaded next
    auto load = [&]() {
        const int e = __builtin_amdgcn_readfirstlane(heads[y].x);
        const int64_t row = ((int64_t)e * a.hb * 8 + tile) * a.ib;
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            const int b = min(b0 + u, a.ib - 1);
#pragma unroll
            for (int t = 0; t < RT; ++t) load_tile(next[u][t], a.down + (row + (int64_t)t * a.ib + b) * kTileBytes + lane * 16);
            next_s[u] = a.down_scales[((int64_t)e * a.hb + tile / 8) * a.ib + b];
        }
    };
    auto slot_of = [&](int c0, int count) {
        return a.lists[y * (kListHead + kMaxTokens) + kListHead + min(c0 + token_of<P>(r16), count - 1)];
    };
    auto add = [&](int slot, bool some, f32x4 (&acc)[RT][1]) {
        const float p = a.weights[slot];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const f32x4 sum = over_pieces<P>(acc[t][0]);
            if (!some || !first_piece<P>(r16)) continue;
            f32x4 *to = own + (4 * t + g) * a.T + slot / a.top_k;
            f32x4 v = *to;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(sum[j], p, v[j]);
            *to = v;
        }
    };
    const int64_t step = (int64_t)a.T * a.top_k * ip;         // a piece of all rows
    const __bf16 *hrow = a.hp + piece_of<P>(r16) * step + 16 * g;
    f32x4 acc[RT][1];
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    int count = 0, slot = 0;
    bool fresh = true;
    if (first < end) load();
    for (int i = first; i < end; ++i) {
        i32x4 now[kUnit][RT][2];
        float s[kUnit];
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            s[u] = next_s[u];
#pragma unroll
            for (int t = 0; t < RT; ++t) now[u][t][0] = next[u][t][0], now[u][t][1] = next[u][t][1];
        }
        if (fresh) {
            count = __builtin_amdgcn_readfirstlane(heads[y].y);
            slot = slot_of(0, count);
            clear();
        }
        const int yi = y, bi = b0;
        b0 += kUnit;
        fresh = b0 >= a.ib;
        if (fresh) ++y, b0 = 0;
        if (i + 1 < end) load();
        for (int c0 = 0; c0 < count; c0 += kTokens<P>) {
            int sl = slot;
            if (c0 > 0) {
                sl = a.lists[yi * (kListHead + kMaxTokens) + kListHead + min(c0 + token_of<P>(r16), count - 1)];
                clear();
            }
#pragma unroll
            for (int u = 0; u < kUnit; ++u) {
                if (bi + u >= a.ib) break;
                const __bf16 *const rows[1] = {hrow + (int64_t)sl * ip + (bi + u) * kBlock};
                float sc[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) sc[t] = s[u];
                block_product<PK>(now[u], sc, rows, step, acc);
            }
            // one column tile: its sums stay in registers until the expert's last unit
            if (count > kTokens<P> || fresh || i + 1 == end) add(sl, c0 + token_of<P>(r16) < count, acc);
        }
        if (count > kTokens<P>) clear();
    }
    __syncthreads();
    constexpr int kWide = 16 * RT;
    auto store = [&](int j, float v) {
        const int t = j / kWide, n = tile * 16 + j % kWide;
        if (n < a.H) ((T *)a.y)[(int64_t)t * a.ldy + n] = (T)v;
    };
    float *part = a.sums + (int64_t)blockIdx.x * a.parts * a.T * kWide;
    for (int j = tid; j < a.T * kWide; j += 64 * kDownWaves) {
        const int at = (j % kWide / 4 * a.T + j / kWide) * 4 + (j & 3);
        float v = 0.0f;
        for (int i = 0; i < kDownWaves; ++i) v += ((const float *)sums)[i * a.T * kWide + at];
        if (a.parts == 1) store(j, v);
        else hand_over(part + (int64_t)blockIdx.y * a.T * kWide + j, v);
    }
    if (a.parts == 1 || !last_to_arrive(a.counters + blockIdx.x, a.parts, (uint32_t *)sums)) return;
    for (int j = tid; j < a.T * kWide; j += 64 * kDownWaves) {
        float v = 0.0f;
        // (four at a time: a load past the caches takes a third of a microsecond)
        for (int i = 0; i < a.parts; i += 4) {
            float u[4];
#pragma unroll
            for (int o = 0; o < 4; ++o) u[o] = i + o < a.parts ? handed_over(part + (int64_t)(i + o) * a.T * kWide + j) : 0.0f;
#pragma unroll
            for (int o = 0; o < 4; ++o) v += u[o];
        }
        store(j, v);
    }
}

// x in P pieces, h in PC * PK: PC side by side as columns, PK one after the other; RT output tiles a wave.
template <class T, int P, int PC, int PK, int RT>
hipError_t launch(const Args &a, hipStream_t s) {
    hipLaunchKernelGGL((moe_route<T, P>), dim3((unsigned)(a.E + 15) / 16, (unsigned)(a.T + 15) / 16, (unsigned)a.splits),
                       dim3(1024), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_up<P, PC * PK>), dim3((unsigned)(a.ib * 8), (unsigned)a.used), dim3(256), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((moe_down<T, PC, PK, RT>), dim3((unsigned)((a.H + 16 * RT - 1) / (16 * RT)), (unsigned)a.parts),
                       dim3(64 * kDownWaves), (size_t)a.T * kDownWaves * (64 * RT) + (size_t)a.used * 8, s, a);
    return hipGetLastError();
}

// Sizes of a part of T tokens and the launch shapes that follow from them.
void size_up(Args &a, const tbh_moe &m, int32_t x_type, int64_t tokens, int32_t top_k) {
    a.T = (int)std::min<int64_t>(kMaxTokens, tokens);
    a.top_k = top_k;
    a.E = m.E;
    a.H = (int)m.H;
    a.hb = (int)m.hb;
    a.ib = (int)m.ib;
    a.used = std::min(m.E, a.T * top_k);
    // two steps of 16 inputs a wave at the least (1, 2 or 4 parts: a whole call on 1 token 33.3,
    // 30.5, 28.9 us, on 64 of width 4096 184, 174, 169)
    a.splits = std::max(1, std::min(kSplits, a.hb * (kBlock / 16) / 32));
    // a block a CU, of waves that have a unit at the least (one part a tile: 13 tokens of width 2048
    // 106 us, 73 so, 64 of 4096 194 and 169)
    // An h of bf16 rows has two pieces.  Side by side they are free while an expert has few tokens; past
    // four on the average they would ask for a second column tile, and follow one another in one of 16
    // tokens, with four output tiles to a load of h.  Side by side / one after the other in us, a whole
    // call: 13 tokens, 6 of 64 experts of 2048 x 1000 74.4 / 76.8, 5 tokens, 2 of 8 of 4096 x 14336 226 / 230,
    // 64 tokens, 8 of 128 of 2048 x 768 153 / 153, 4 of 32 of 4096 x 2048 204 / 175, 2 of 8 of 4096 x 4096 136 / 126.
    a.tiles = x_type == TBH_BF16 && a.T * top_k > 4 * m.E ? 4 : 2;
    const int tiles = (a.H + 16 * a.tiles - 1) / (16 * a.tiles), units = a.used * ((a.ib + kUnit - 1) / kUnit);
    a.parts = std::max(1, std::min((m.dev->cu_count + tiles - 1) / tiles, units / kDownWaves));
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace of a part of T tokens; sets the pointers when `base` is given.
size_t carve(Args &a, int32_t x_type, char *base) {
    const size_t P = x_type == TBH_BF16 ? 1 : 3, PH = x_type == TBH_BF16 ? 2 : 3;
    size_t at = 0;
    auto take = [&](size_t n) {
        char *p = base ? base + at : nullptr;
        at += round256(n);
        return p;
    };
    const size_t rows = (size_t)a.T * a.top_k;
    a.ids = (int32_t *)take(rows * 4);
    a.weights = (float *)take(rows * 4);
    a.logits = (double *)take((size_t)a.splits * a.T * a.E * 8);
    a.sums = (float *)take(a.parts > 1 ? (size_t)((a.H + 16 * a.tiles - 1) / (16 * a.tiles)) * a.parts * a.T * (64 * a.tiles) : 0);
    a.lists = (int32_t *)take((size_t)a.used * (kListHead + kMaxTokens) * 4);
    a.xp = (__bf16 *)take(P * a.T * a.hb * kBlock * 2);
    a.hp = (__bf16 *)take(PH * rows * a.ib * kBlock * 2);
    return at;
}

size_t workspace_of(const tbh_moe &m, int32_t x_type, int64_t tokens, int32_t top_k) {
    Args a{};
    size_up(a, m, x_type, tokens, top_k);
    // (more tokens have fewer parts of a tile, and a last part of few tokens may have more)
    size_t most = 0;
    for (int64_t t : {(int64_t)a.T, tokens % kMaxTokens}) {
        if (t == 0) continue;
        size_up(a, m, x_type, t, top_k);
        most = std::max(most, carve(a, x_type, nullptr));
    }
    return most;
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
    const size_t row = (size_t)m->hb * kBlock * 4;
    hipError_t e = hipMalloc((void **)&m->router, E * row);
    if (e == hipSuccess) e = hipMemsetAsync(m->router, 0, E * row, s);
    if (e == hipSuccess)
        e = hipMemcpy2DAsync(m->router, row, d.router, (size_t)m->H * 4, (size_t)m->H * 4, E, hipMemcpyDefault, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->gate_scales, d.gate_scales, scales, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->up_scales, d.up_scales, scales, s);
    if (e == hipSuccess) e = fp8::copy_in((void **)&m->down_scales, d.down_scales, scales, s);
    if (e == hipSuccess) e = hipMalloc((void **)&m->gate_up, 2 * tiles);
    if (e == hipSuccess) e = hipMalloc((void **)&m->down, tiles);
    auto repack = [&](const uint8_t *from, int64_t N, int64_t K, int64_t step, uint8_t *to) {
        void *raw = nullptr;
        if (e == hipSuccess) e = fp8::copy_in(&raw, from, bytes, s);
        if (e == hipSuccess) e = fp8::launch_repack((const uint8_t *)raw, N, K, m->E, 1, step, to, s);
        const hipError_t waited = hipStreamSynchronize(s);
        if (e == hipSuccess) e = waited;
        if (raw) (void)hipFree(raw);
    };
    repack(d.gate, m->I, m->H, 2, m->gate_up);
    repack(d.up, m->I, m->H, 2, m->gate_up ? m->gate_up + kTileBytes : nullptr);
    repack(d.down, m->H, m->I, 1, m->down);
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
    *bytes = (int64_t)(kCounterBytes + workspace_of(*m, x_type, tokens, top_k));
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
    const Span of_x(x, m->H, x_stride, size, tokens), of_y(y, m->H, y_stride, size, tokens);
    if (overlap(of_x, of_y)) return bad("y overlaps x");
    const Span chosen[2] = {Span(experts, (size_t)tokens * top_k * 4), Span(weights, (size_t)tokens * top_k * 4)};
    for (const Span &c : chosen)
        if (c.at && (overlap(c, of_x) || overlap(c, of_y))) return bad("experts or weights overlap x or y");
    if (experts && weights && overlap(chosen[0], chosen[1])) return bad("experts and weights overlap");
    if ((uintptr_t)x % size || (uintptr_t)y % size || (uintptr_t)experts % 4 || (uintptr_t)weights % 4)
        return bad("a pointer is not aligned to its type");
    if (workspace && ((uintptr_t)workspace & 255)) return bad("the workspace must be 256-byte aligned");
    const size_t need = workspace_of(*m, x_type, tokens, top_k);
    if (workspace && (workspace_bytes < 0 || (size_t)workspace_bytes < need + kCounterBytes)) return bad("the workspace is too small");
    if ((st = use_device(m->dev->ordinal)) != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    const bool vec = (uintptr_t)x % (4 * size) == 0 && (tokens == 1 || x_stride % 4 == 0);
    const auto held = hold_launches(m->dev, s);
    const Room room = room_of(m->dev, s, workspace, need);
    if (!room.counters)
        return set_error(TBH_E_OOM, std::string(what) + ": no workspace (a captured stream needs an earlier eager call, or a "
                                                        "workspace of the caller's)");
    hipError_t e = hipSuccess;
    for (int64_t at = 0; at < tokens && e == hipSuccess; at += kMaxTokens) {
        Args a{};
        size_up(a, *m, x_type, tokens - at, top_k);
        a.normalize = normalize != 0;
        a.vec = vec;
        a.counters = room.counters;
        carve(a, x_type, room.data);
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
        if (x_type == TBH_F32) e = launch<float, 3, 3, 1, 2>(a, s);
        else e = a.tiles == 4 ? launch<__bf16, 1, 1, 2, 4>(a, s) : launch<__bf16, 1, 2, 1, 2>(a, s);
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "moe launch");
}

}  // extern "C"
