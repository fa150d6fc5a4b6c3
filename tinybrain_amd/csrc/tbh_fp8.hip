// tbh_fp8.hip -- products with block-scaled FP8 weights:
//   y[m][n] = sum_b s[m][b] sw[n / 128][b] sum_{k in block b} q[m][k] w[n][k]
// with w and q in e4m3, a scale sw per 128 x 128 block of the weight and a
// scale s per row and 128 inputs of x, which the call chooses itself
// (quantize_block).  A 128-deep matrix instruction takes one block of K: its
// result is multiplied by both scales and added in fp32.
#include <algorithm>
#include <memory>
#include <new>

#include "tbh_dma.h"
#include "tbh_fp8.h"

namespace tbh {
namespace fp8 {
namespace {

// ---- weights ---------------------------------------------------------------
struct RepackArgs {
    const uint8_t *data;
    uint8_t *tiles;
    int64_t N, K, kb, group, step, pieces;
    int64_t src_tiles;      // tile rows of one matrix
};

// A thread writes one 16-byte piece.
__global__ __launch_bounds__(256) void fp8_repack(RepackArgs a) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < a.pieces; p += stride) {
        const int lane = (int)(p & 63), h = (int)(p >> 6) & 1;
        const int64_t tile = p >> 7, b = tile % a.kb, row_tile = tile / a.kb;
        const int64_t i = row_tile / a.src_tiles, t = row_tile % a.src_tiles;
        const int64_t n = t * 16 + (lane & 15), k = b * kBlock + h * 64 + (lane >> 4) * 16;
        uint32_t w[4] = {0, 0, 0, 0};
        if (n < a.N) {
            const uint8_t *from = a.data + (i * a.N + n) * a.K + k;
            if (k + 16 <= a.K && ((uintptr_t)from & 15) == 0) {
                const u32x4 v = *(const u32x4 *)from;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (k + j < a.K) w[j / 4] |= (uint32_t)from[j] << (8 * (j % 4));
            }
        }
        const int64_t to = (i * a.src_tiles * a.kb + (t / a.group * a.kb + b) * a.group + t % a.group) * a.step;
        *(u32x4 *)(a.tiles + to * kTileBytes + h * 1024 + lane * 16) = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// ---- few rows of x -----------------------------------------------------------
struct RowsArgs {
    Matrix w;
    const void *x;
    void *y;
    int64_t ldx, ldy, M;
    int K, N, kb;
    bool vec_x, vec_y;
};

// acc += s * (w . q) of a block, q scaled by f = its row's scale: on the FP8 instruction
// for a result of bf16, on the bf16 one for one of fp32 (x: q widened).
template <class YT>
struct Operand {
    i32x8 q;
};
template <>
struct Operand<float> {
    bf16x8 x[2][2];
};
__device__ __forceinline__ void set(Operand<__bf16> &o, i32x8 q) { o.q = q; }
__device__ __forceinline__ void set(Operand<float> &o, i32x8 q) {
    widen(i32x4{q[0], q[1], q[2], q[3]}, o.x[0]);
    widen(i32x4{q[4], q[5], q[6], q[7]}, o.x[1]);
}
__device__ __forceinline__ f32x4 dot(i32x4 lo, i32x4 hi, const Operand<__bf16> &o) {
    return mfma_block(i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, o.q);
}
__device__ __forceinline__ f32x4 dot(i32x4 lo, i32x4 hi, const Operand<float> &o) {
    bf16x8 w[2];
    widen(lo, w);
    f32x4 part = mfma_wide(w[0], o.x[0][0], f32x4{0.f, 0.f, 0.f, 0.f});
    part = mfma_wide(w[1], o.x[0][1], part);
    widen(hi, w);
    part = mfma_wide(w[0], o.x[1][0], part);
    return mfma_wide(w[1], o.x[1][1], part);
}

// The waves' sums of a block's tiles, added in order and stored.
template <class YT, int W, int RT, int CT>
__device__ __forceinline__ void join_waves(void *y, int64_t ldy, int64_t M, int N, bool vec, int64_t tile, int64_t m0,
                                           const f32x4 (&acc)[RT][CT], f32x4 (&red)[W][RT * CT][64]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < CT; ++c) red[wave][t * CT + c][lane] = acc[t][c];
    __syncthreads();
    for (int i = wave; i < RT * CT; i += W) {
        const int t = i / CT, c = i % CT;
        const int64_t m = m0 + c * 16 + r16, n = (tile + t) * 16 + 4 * g;
        f32x4 v = red[0][i][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][i][lane];
        if (m < M) store4((YT *)y + m * ldy + n, v, N - n, vec);
    }
}

// Up to 16 rows of x as the columns of tiles; a block owns 16 RT outputs, its W waves
// part K, KW blocks at a time, whose weights are all under way before the first is used.
// Every lane quantizes the 32 elements of its own operand: one launch, and no x in
// between, for which each block of outputs does so again.  Bound by the latency of a
// launch and one round of loads where the weight is small, by memory past that: one
// row, weights from memory, 2048 x 1024 5.5 us (0.4 TB/s), 4096 x 32768 28.3 us
// (4.7 TB/s, what a large copy reaches).
template <class XT, class YT, int W, int RT, int KW>
__global__ __launch_bounds__(64 * W) void fp8_rows(RowsArgs a) {
    __shared__ f32x4 red[W][RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int64_t tile = (int64_t)blockIdx.x * RT, m0 = (int64_t)blockIdx.y * 16, m = m0 + r16;
    f32x4 acc[RT][1];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int b0 = a.kb * wave / W, b1 = a.kb * (wave + 1) / W;
    const uint8_t *wt = a.w.tiles + tile_at(tile, 0, a.kb) + lane * 16;      // (RT tiles lie in one group)
    const float *sw = a.w.scales + tile / 8 * a.kb;
    const XT *xr = (const XT *)a.x + m * a.ldx + 16 * g;
    for (int b = b0; b < b1; b += KW) {
        i32x4 w[KW][RT][2];
        float s[KW];
#pragma unroll
        for (int u = 0; u < KW; ++u) {
            const int at = min(b + u, b1 - 1);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const uint8_t *p = wt + ((int64_t)at * 8 + t) * kTileBytes;
                w[u][t][0] = *(const i32x4 *)p, w[u][t][1] = *(const i32x4 *)(p + 1024);
            }
            s[u] = sw[at];
        }
#pragma unroll
        for (int u = 0; u < KW; ++u) {
            if (b + u >= b1) break;
            const int k = (b + u) * kBlock;
            Block<XT> x;
            load_block(x, xr + k, m < a.M ? a.K - k - 16 * g : 0, a.vec_x);
            i32x8 q;
            const float f = quantize_block(x, q) * s[u];
            Operand<YT> o;
            set(o, q);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const f32x4 part = dot(w[u][t][0], w[u][t][1], o);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][0][i] = __builtin_fmaf(part[i], f, acc[t][0][i]);
            }
        }
    }
    join_waves<YT, W, RT, 1>(a.y, a.ldy, a.M, a.N, a.vec_y, tile, m0, acc, red);
}

// ---- many rows of x ------------------------------------------------------------
struct QuantizeArgs {
    const void *x;
    uint8_t *tiles;      // as a weight's, of M rows; WIDE: of bf16, operands of one instruction together
    float *scales;       // [kb][row_tiles * 16]
    int64_t ldx, M, row_tiles;
    int K, kb;
    bool vec;
};

// A wave quantizes 16 rows x 128 and writes them in the layout of a weight.  Bound by
// memory: 4096 x 4096 of bf16 10.5 us (33.5 MB read, 17 written: 4.8 TB/s).
template <class XT, bool WIDE>
__global__ __launch_bounds__(256) void fp8_quantize(QuantizeArgs a) {
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= a.kb) return;
    const int64_t m = (int64_t)blockIdx.y * 16 + r16;
    const int k = b * kBlock + 16 * g;
    Block<XT> x;
    load_block(x, (const XT *)a.x + m * a.ldx + k, m < a.M ? a.K - k : 0, a.vec);
    i32x8 q;
    const float s = quantize_block(x, q);
    uint8_t *to = a.tiles + tile_at(blockIdx.y, b, a.kb) * (WIDE ? 2 : 1) + lane * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const i32x4 v{q[4 * h], q[4 * h + 1], q[4 * h + 2], q[4 * h + 3]};
        if constexpr (WIDE) {
            bf16x8 o[2];
            widen(v, o);
            *(bf16x8 *)(to + h * 2048) = o[0];
            *(bf16x8 *)(to + h * 2048 + 1024) = o[1];
        } else {
            *(i32x4 *)(to + h * 1024) = v;
        }
    }
    if (g == 0) a.scales[(int64_t)b * a.row_tiles * 16 + m] = s;
}

struct TilesArgs {
    Matrix w;
    const uint8_t *x;       // tiles
    const float *xs;        // [kb][row_tiles * 16]
    void *y;
    int64_t ldy, M, row_tiles;
    int N, kb, w_tiles;
    bool vec_y;
};

// 16 CT rows of quantized x and 16 RT outputs a block, waves over K as in fp8_rows, operands
// from memory straight to registers: no barrier but that of the join.  For products that
// do not fill the device with blocks of 128 x 256, bound by the latency of the loads and then by
// the caches, which serve x to every block of outputs and the weight to every block of rows:
// 21 rows by 4096 x 11008 10.3 us (4.4 TB/s of weight) behind the quantizing's 3.4, 333 of fp32
// by 5632 x 2048 14.2 behind 5.4, in which waves ask the L2 caches for 207 MB (counted, 14.6 TB/s) of
// operands that are 18 MB: two tiles by three take five loads for six products.
template <class YT, int W, int RT, int KW, int CT>
__global__ __launch_bounds__(64 * W) void fp8_few(TilesArgs a) {
    __shared__ f32x4 red[W][RT * CT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15;
    const int64_t tile = (int64_t)blockIdx.x * RT, x0 = (int64_t)blockIdx.y * CT, mp = a.row_tiles * 16;
    f32x4 acc[RT][CT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int b0 = a.kb * wave / W, b1 = a.kb * (wave + 1) / W;
    const uint8_t *wt = a.w.tiles + tile_at(tile, 0, a.kb) + lane * 16, *xt[CT];
    const float *sw = a.w.scales + tile / 8 * a.kb, *sx[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        // a column tile past the last repeats it; its results are not stored
        const int64_t x = min(x0 + c, a.row_tiles - 1);
        xt[c] = a.x + tile_at(x, 0, a.kb) + lane * 16;
        sx[c] = a.xs + x * 16 + r16;
    }
    for (int b = b0; b < b1; b += KW) {
        i32x4 w[KW][RT][2], x[KW][CT][2];
        float s[KW], f[KW][CT];
#pragma unroll
        for (int u = 0; u < KW; ++u) {
            const int at = min(b + u, b1 - 1);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const uint8_t *p = wt + ((int64_t)at * 8 + t) * kTileBytes;
                w[u][t][0] = *(const i32x4 *)p, w[u][t][1] = *(const i32x4 *)(p + 1024);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const uint8_t *p = xt[c] + (int64_t)at * (8 * kTileBytes);
                x[u][c][0] = *(const i32x4 *)p, x[u][c][1] = *(const i32x4 *)(p + 1024);
                f[u][c] = sx[c][(int64_t)at * mp];
            }
            s[u] = sw[at];
        }
#pragma unroll
        for (int u = 0; u < KW; ++u) {
            if (b + u >= b1) break;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const i32x4 lo = x[u][c][0], hi = x[u][c][1];
                Operand<YT> o;
                set(o, i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
                const float scale = f[u][c] * s[u];
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const f32x4 part = dot(w[u][t][0], w[u][t][1], o);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][c][i] = __builtin_fmaf(part[i], scale, acc[t][c][i]);
                }
            }
        }
    }
    join_waves<YT, W, RT, CT>(a.y, a.ldy, a.M, a.N, a.vec_y, tile, x0 * 16, acc, red);
}

constexpr uint32_t kPast = 0x7FFFFFF0u;   // past every buffer: reads as zeros

// A block's 16 WN TN outputs x 16 WM TM rows; waves WN x WM, each TN x TM tiles.
// A result of bf16 comes from the FP8 instruction; one of fp32 from the bf16 one,
// half as fast, with x widened by the pass that quantized it (WIDE) and the weight here.
// Two steps of 128 inputs in LDS: a step's one barrier says that its tiles have landed and
// that every wave is done with the step before, whose place the loads issued then take, a few
// behind each row of products (all at the step's start: 196 us and 364 of the 190 and 345 below).
// 4096 rows by 4096 x 11008: 182 to 203 us of this kernel by the card (medians of traces, 2.03 to 1.82
// PFLOP/s; loads alone 115, products
// alone 170), fp32 results 345 us with the quantizing.  Bound by the step: of its some 4100
// cycles (395000 a launch, three rounds of 32 steps) the matrix instructions are busy for 2050, LDS reads take 1536, loads 2800, and a
// barrier joins them; 160 KiB of LDS hold no third step.  (Two halves of a block's
// waves, one at LDS while the other multiplies: 210 us of then 203; cache lines touched two to
// four steps ahead: 233; instructions of 32 x 32 results: 197 of 190.  Matrix instructions alone, out of registers and with these fp32 sums, run
// such data at 3.0 PFLOP/s, where power brings the clock down to 1.6 GHz.)
template <class YT, int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tiles(TilesArgs a) {
    constexpr bool WIDE = sizeof(YT) == 4;
    constexpr int W = WN * WM, NT = WN * TN, MT = WM * TM, XB = (WIDE ? 2 : 1) * kTileBytes, XL = XB / 1024;
    constexpr int LOADS = (NT * 2 + MT * XL) / W;
    static_assert((NT * 2 + MT * XL) % W == 0 && MT * 64 <= 1024, "");
    static_assert(NT % 8 == 0 && MT % 8 == 0 && 8 % TN == 0, "whole groups of tiles; a wave's outputs share a scale");
    constexpr int kScales = NT * kTileBytes + MT * XB, kStage = kScales + 1024;
    static_assert(2 * kStage <= 160 * 1024, "");
    __shared__ __align__(16) char sm[2 * kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4, wn = wave % WN, wm = wave / WN;
    // blocks go to the XCDs in turn: each XCD gets tiles that lie together, four of the
    // weight by the rows', so that its cache serves both
    const int nt = (a.w_tiles + NT - 1) / NT, mt = (int)((a.row_tiles + MT - 1) / MT), total = nt * mt;
    const int each = (total + 7) / 8, t = (int)(blockIdx.x & 7) * each + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= each || t >= total) return;
    const int group = t / (4 * mt), rest = t - group * 4 * mt, wide = min(4, nt - group * 4);
    const int64_t n0 = (int64_t)(group * 4 + rest % wide) * NT, m0 = (int64_t)(rest / wide) * MT;   // in tiles
    // a block's groups of eight tiles, as far as there are any: the rest reads as zeros.  (The
    // rows' last group is not filled: what it holds there are columns of no row.)
    const int64_t row = (int64_t)a.kb * (8 * kTileBytes), xrow = (int64_t)a.kb * (8 * XB);
    const int64_t w_groups = min((int64_t)NT / 8, a.w_tiles / 8 - n0 / 8);
    const int64_t x_groups = min((int64_t)MT / 8, (a.row_tiles + 7) / 8 - m0 / 8);
    const dma::i32x4 wr = dma::make_rsrc(a.w.tiles + tile_at(n0, 0, a.kb), (int)(w_groups * row));
    const dma::i32x4 xr = dma::make_rsrc(a.x + tile_at(m0, 0, a.kb) * (XB / kTileBytes), (int)(x_groups * xrow));
    const int64_t mp = a.row_tiles * 16, sm0 = m0 * 16 + wm * TM * 16;
    const dma::i32x4 sr = dma::make_rsrc(a.xs, (int)((int64_t)a.kb * mp * 4));
    const uint32_t lds0 = dma::lds_addr(sm);
    // Loads i0 .. i1 - 1 of a wave for a step.  (The step past the last is the last again.)
    auto issue = [&](int step, int buf, int i0, int i1) {
        const uint32_t lds = lds0 + buf * kStage;
        const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane(min(step, a.kb - 1));
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            const int j = i * W + wave;      // 1 KiB of a tile
            const bool of_w = j < 2 * NT;
            const int t = of_w ? j >> 1 : (j - 2 * NT) / XL, part = of_w ? j & 1 : (j - 2 * NT) % XL;
            dma::dma16(__builtin_amdgcn_readfirstlane(lds + j * 1024), of_w ? wr : xr,
                       (uint32_t)((t >> 3) * (of_w ? row : xrow)) + (t & 7) * (of_w ? kTileBytes : XB) + part * 1024 + lane * 16,
                       b * (8 * (of_w ? kTileBytes : XB)));
        }
        // the scales of the block's rows
        if (i0 == 0 && wave == 0)
            dma::dma16(__builtin_amdgcn_readfirstlane(lds + kScales), sr,
                       lane < MT * 4 && m0 * 16 + lane * 4 < mp ? (uint32_t)(m0 * 64 + lane * 16) : kPast, b * (uint32_t)(mp * 4));
    };
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (a wave's outputs lie in one block of 128)
    const auto *sw = (const __attribute__((address_space(4))) float *)(a.w.scales + min((n0 + wn * TN) / 8, (int64_t)a.w_tiles / 8 - 1) * a.kb);
    issue(0, 0, 0, LOADS);
    for (int b = 0; b < a.kb; ++b) {
        const int buf = b & 1;
        const float s = sw[b];
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        const char *st = sm + buf * kStage;
        const char *wt = st + wn * TN * kTileBytes + lane * 16, *xt = st + NT * kTileBytes + wm * TM * XB + lane * 16;
        float f[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) f[j] = s * *(const float *)(st + kScales + ((wm * TM + j) * 16 + r16) * 4);
        auto add = [&](int i, int j, f32x4 part) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], f[j], acc[i][j][e]);
        };
        if constexpr (WIDE) {
            bf16x8 x[TM][4];
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) x[j][c] = *(const bf16x8 *)(xt + j * XB + c * 1024);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                bf16x8 w[2][2];
                issue(b + 1, buf ^ 1, i * LOADS / TN, (i + 1) * LOADS / TN);
#pragma unroll
                for (int h = 0; h < 2; ++h) widen(*(const i32x4 *)(wt + i * kTileBytes + h * 1024), w[h]);
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    f32x4 part{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 4; ++c) part = mfma_wide(w[c >> 1][c & 1], x[j][c], part);
                    add(i, j, part);
                }
            }
        } else {
            auto operand = [](const char *p) {
                const i32x4 lo = *(const i32x4 *)p, hi = *(const i32x4 *)(p + 1024);
                return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            i32x8 x[TM], next = operand(wt);
#pragma unroll
            for (int j = 0; j < TM; ++j) x[j] = operand(xt + j * kTileBytes);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const i32x8 w = next;
                issue(b + 1, buf ^ 1, i * LOADS / TN, (i + 1) * LOADS / TN);
                if (i + 1 < TN) next = operand(wt + (i + 1) * kTileBytes);
#pragma unroll
                for (int j = 0; j < TM; ++j) add(i, j, mfma_block(w, x[j]));
            }
        }
    }
    // the loads past the last step have still to land in this block's LDS
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int64_t m = sm0 + j * 16 + r16;
        if (m >= a.M) continue;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int64_t n = (n0 + wn * TN + i) * 16 + 4 * g;
            store4((YT *)a.y + m * a.ldy + n, acc[i][j], a.N - n, a.vec_y);
        }
    }
}

constexpr int64_t kRows = 16;

template <class YT, int WN, int WM, int TN, int TM>
hipError_t launch_tiles(const TilesArgs &a, hipStream_t s) {
    const int64_t nt = (a.w_tiles + WN * TN - 1) / (WN * TN), mt = (a.row_tiles + WM * TM - 1) / (WM * TM);
    hipLaunchKernelGGL((fp8_tiles<YT, WN, WM, TN, TM>), dim3((unsigned)((nt * mt + 7) / 8 * 8)), dim3(64 * WN * WM), 0, s, a);
    return hipGetLastError();
}

template <class YT, int W, int RT, int KW, int CT>
hipError_t launch_few_as(const TilesArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)(a.w_tiles / RT), (unsigned)((a.row_tiles + CT - 1) / CT));
    hipLaunchKernelGGL((fp8_few<YT, W, RT, KW, CT>), grid, dim3(64 * W), 0, s, a);
    return hipGetLastError();
}

// Pieces of 16 outputs x 64 rows.
int64_t units_of(int64_t w_tiles, int64_t row_tiles) { return w_tiles * ((row_tiles + 3) / 4); }

// A block's outputs and its waves: few blocks take few outputs each, on many waves; past what
// the device holds at once, fewer waves with more outputs read x less often.  K = 4096, bf16:
// 32 rows, RT 1 / 2: N = 4096 9.6 / 11.1 us, 8192 13.8 / 12.8.  CT = 4, RT 1 / 2 / 4:
// 64 rows of N = 4096 (256 units) 11.4 / 12.2 / 19.9, 128 rows of 8192 (1024) 26.6 /
// 18.3 / 20.8, 256 rows of 8192 (2048) 41.9 / 26.9 / 24.2.  CT = 3 where it leaves fewer tiles
// of x empty: 5632 x 2048, 48 rows 12.1 us against 13.3, 333 rows of fp32 19.6 against 21.4.
template <class YT, int CT>
hipError_t launch_few_of(const TilesArgs &a, hipStream_t s) {
    const int64_t units = units_of(a.w_tiles, a.row_tiles);
    if (units <= 300) return launch_few_as<YT, 16, 1, 2, CT>(a, s);
    if (units <= 1200) return launch_few_as<YT, 8, 2, 2, CT>(a, s);
    return launch_few_as<YT, 4, 4, 2, CT>(a, s);
}
template <class YT>
hipError_t launch_few(const TilesArgs &a, hipStream_t s) {
    if (a.row_tiles <= 2)
        return a.w_tiles <= 256 ? launch_few_as<YT, 16, 1, 2, 2>(a, s) : launch_few_as<YT, 16, 2, 1, 2>(a, s);
    const bool three = (a.row_tiles + 2) / 3 * 3 < (a.row_tiles + 3) / 4 * 4;
    return three ? launch_few_of<YT, 3>(a, s) : launch_few_of<YT, 4>(a, s);
}

// Which kernel a product of quantized rows takes: a step of 128 inputs costs fp8_few 0.25 ns
// a unit (fp32 results: 0.27), and fp8_tiles, for each 256 blocks begun, 1 us with 128
// outputs x 256 rows (bf16) and 1.5 with 256 x 256, or 1.8 with 256 x 128 (fp32 results); the
// least is taken.  bf16, few / 128 x 256 / 256 x 256 in us: 4096 x 11008 on 256 rows 33.9 / 39.0 /
// 60.4, 512 55.5 / 42.6 / 61.9, 1024 104.9 / 77.8 / 65.3; 2048 x 32000 on 64 rows 17.7 / 22.2 / 31.1,
// 384 65.3 / 46.9 / 41.3; fp32, few / 256 x 128: 4096 x 11008 on 512 rows 63.2 / 65.0, 768
// 93.2 / 121.8; 2048 x 32000 on 192 rows 40.7 / 39.4, 256 50.3 / 39.4.
enum class Plan { Few, Tiles, Large };
Plan plan_of(int64_t w_tiles, int64_t row_tiles, bool f32) {
    const auto rounds = [&](int64_t nt, int64_t mt) {
        return ((w_tiles + nt - 1) / nt * ((row_tiles + mt - 1) / mt) + 255) / 256;
    };
    const int64_t few = units_of(w_tiles, row_tiles) * (f32 ? 27 : 25);
    const int64_t large = rounds(16, f32 ? 8 : 16) * (f32 ? 180000 : 150000), tiles = f32 ? large : rounds(8, 16) * 100000;
    if (few < std::min(large, tiles)) return Plan::Few;
    return tiles < large || (!f32 && tiles == large) ? Plan::Tiles : Plan::Large;
}

template <class XT, class YT, int W, int RT, int KW>
hipError_t launch_rows_as(const RowsArgs &a, int64_t w_tiles, hipStream_t s) {
    const dim3 grid((unsigned)(w_tiles / RT), (unsigned)((a.M + 15) / 16));
    hipLaunchKernelGGL((fp8_rows<XT, YT, W, RT, KW>), grid, dim3(64 * W), 0, s, a);
    return hipGetLastError();
}

// One tile and many waves while each CU gets one block (K = 4096, one row of bf16, RT 1 / 2 / 4:
// N = 4096 8.3 / 9.2 / 12.3 us), then fewer blocks, which quantize x less often (8192
// 12.1 / 11.5 / 14.0, 32768 33.2 / 36.7 / 28.3; 16 rows 41.4 / 36.9 / 29.7).
template <class XT, class YT>
hipError_t launch_rows(const RowsArgs &a, int64_t w_tiles, hipStream_t s) {
    if (w_tiles <= 256) return launch_rows_as<XT, YT, 16, 1, 2>(a, w_tiles, s);
    if (w_tiles <= 512) return launch_rows_as<XT, YT, 16, 2, 2>(a, w_tiles, s);
    return launch_rows_as<XT, YT, 8, 4, 2>(a, w_tiles, s);
}

// Rows that fp8_rows takes, up to kRows or, of bf16, while every 16 x 16 results have a CU of
// their own: the pass that quantizes first costs a launch.  fp8_rows / pass and fp8_few: 2048 x
// 2048, 32 rows 5.4 / 7.5 us, 4096 x 1024, 32 rows 6.7 / 7.8 (of fp32, twice the loads and work
// to quantize, 10.2 / 7.9), 4096 x 4096, 32 rows 12.7 / 9.6; 16 rows 8.3 / 9.1.
bool direct(int64_t M, int64_t w_tiles, int32_t x_type) {
    return M <= kRows || (x_type == TBH_BF16 && w_tiles * ((M + 15) / 16) <= 256);
}

constexpr int64_t kMaxK = 1 << 20;       // a block's 16 tiles along K within 32 bits
constexpr int64_t kMaxN = 1 << 24;       // blocks of 16 outputs in one launch
constexpr int64_t kPartRows = 1 << 14;   // rows of one part of a long x

}  // namespace

hipError_t launch_repack(const uint8_t *data, int64_t N, int64_t K, int64_t count, int64_t group, int64_t step,
                         uint8_t *tiles, hipStream_t s) {
    RepackArgs a{};
    a.data = data;
    a.tiles = tiles;
    a.N = N;
    a.K = K;
    a.kb = blocks_of(K);
    a.group = group;
    a.step = step;
    a.src_tiles = blocks_of(N) * 8;
    a.pieces = count * a.src_tiles * a.kb * 128;
    const int64_t blocks = std::min<int64_t>((a.pieces + 255) / 256, 1 << 16);
    if (blocks == 0) return hipSuccess;
    hipLaunchKernelGGL(fp8_repack, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t copy_in(void **out, const void *from, size_t bytes, hipStream_t s) {
    hipError_t e = hipMalloc(out, std::max<size_t>(bytes, 16));
    if (e == hipSuccess && bytes) e = hipMemcpyAsync(*out, from, bytes, hipMemcpyDefault, s);
    return e;
}

}  // namespace fp8
}  // namespace tbh

using namespace tbh;
using namespace tbh::fp8;

extern "C" {

tbh_status tbh_fp8_weight_destroy(tbh_fp8_weight *w) {
    if (!w) return TBH_OK;
    if (w->dev) (void)use_device(w->dev->ordinal);
    hipError_t e = hipSuccess;
    for (void *p : {(void *)w->tiles, (void *)w->scales})
        if (p) {
            const hipError_t f = hipFree(p);
            if (e == hipSuccess) e = f;
        }
    delete w;
    return e == hipSuccess ? TBH_OK : hip_error(e, "tbh_fp8_weight_destroy");
}

tbh_status tbh_fp8_weight_create(tbh_device *dev, const tbh_fp8_desc *desc, tbh_fp8_weight **out) {
    const char *what = "tbh_fp8_weight_create";
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!out) return bad("out is NULL");
    *out = nullptr;
    if (!dev || !desc) return bad("NULL device or descriptor");
    if (desc->K <= 0 || desc->N <= 0) return bad("K and N must be positive");
    if (!desc->data || !desc->scales) return bad("NULL data or scales");
    if (desc->K > kMaxK || desc->N > kMaxN)
        return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": K above 2^20 or N above 2^24");
    tbh_status st = use_device(dev->ordinal);
    if (st != TBH_OK) return st;
    std::unique_ptr<tbh_fp8_weight, tbh_status (*)(tbh_fp8_weight *)> w(new (std::nothrow) tbh_fp8_weight,
                                                                        tbh_fp8_weight_destroy);
    if (!w) return set_error(TBH_E_OOM, std::string(what) + ": out of host memory");
    w->dev = dev;
    w->K = desc->K;
    w->N = desc->N;
    w->kb = blocks_of(desc->K);
    w->nb = blocks_of(desc->N);
    std::lock_guard<std::mutex> lock(dev->mu);
    void *raw = nullptr;
    hipError_t e = copy_in(&raw, desc->data, (size_t)(desc->K * desc->N), dev->stream);
    if (e == hipSuccess) e = copy_in((void **)&w->scales, desc->scales, (size_t)(w->kb * w->nb) * 4, dev->stream);
    if (e == hipSuccess) e = hipMalloc((void **)&w->tiles, (size_t)(w->nb * 8 * w->kb) * kTileBytes);
    if (e == hipSuccess)
        e = launch_repack((const uint8_t *)raw, w->N, w->K, 1, 8, 1, w->tiles, dev->stream);
    const hipError_t waited = hipStreamSynchronize(dev->stream);
    if (e == hipSuccess) e = waited;
    if (raw) (void)hipFree(raw);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return hip_error(e, what);
    }
    *out = w.release();
    return TBH_OK;
}

tbh_status tbh_fp8_matmul_workspace(const tbh_fp8_weight *w, int64_t M, int64_t *bytes) {
    if (!w || !bytes || M < 0) return set_error(TBH_E_INVALID, "tbh_fp8_matmul_workspace: NULL pointer or negative M");
    const int64_t rows = (std::min(M, kPartRows) + 127) & ~(int64_t)127;
    *bytes = rows * w->kb * (2 * kBlock + 4);      // widened, for results of fp32
    return TBH_OK;
}

tbh_status tbh_fp8_matmul_device(const tbh_fp8_weight *w, const void *x, int32_t x_type, int64_t M, int64_t K,
                                 int64_t x_stride, void *y, int32_t y_type, int64_t y_stride, void *workspace,
                                 int64_t workspace_bytes, void *stream) {
    const char *what = "tbh_fp8_matmul";
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!w) return bad("NULL weight");
    if (x_type != TBH_F32 && x_type != TBH_BF16) return bad("unknown x_type");
    if (y_type != TBH_F32 && y_type != TBH_BF16) return bad("unknown y_type");
    if (M < 0) return bad("negative M");
    if (K != w->K) return bad("Dimensions must match");
    if (M == 0) return TBH_OK;
    if (!x || !y) return bad("NULL x or y");
    if (M > 1 && (x_stride < K || y_stride < w->N)) return bad("a stride is shorter than its row");
    if (workspace && ((uintptr_t)workspace & 255)) return bad("the workspace must be 256-byte aligned");
    if (workspace_bytes < 0) return bad("negative workspace_bytes");
    const size_t xs = type_size(x_type), ys = type_size(y_type);
    if (overlap(Span(x, K, x_stride, xs, M), Span(y, w->N, y_stride, ys, M))) return bad("y overlaps x");
    if ((uintptr_t)x % xs || (uintptr_t)y % ys) return bad("x or y is not aligned to its type");
    tbh_status st = use_device(w->dev->ordinal);
    if (st != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    const bool vec_x = ((uintptr_t)x & 15) == 0 && (M == 1 || x_stride * xs % 16 == 0);
    const bool vec_y = (uintptr_t)y % (4 * ys) == 0 && (M == 1 || y_stride % 4 == 0);
    hipError_t e = hipSuccess;
    const auto held = hold_launches(w->dev, s);
    int64_t need = 0;
    (void)tbh_fp8_matmul_workspace(w, M, &need);
    void *room = nullptr;
    if (!direct(M, w->nb * 8, x_type)) {
        if (workspace) room = workspace_bytes >= need ? workspace : nullptr;
        else room = stream_workspace(w->dev, s, (size_t)need);
        if (workspace && !room) return bad("the workspace is too small");
    }
    const int64_t most = room ? kPartRows : 16 * 65535;
    for (int64_t at = 0; at < M && e == hipSuccess; at += most) {
        const int64_t rows = std::min(most, M - at);
        const char *xp = (const char *)x + at * x_stride * xs;
        char *yp = (char *)y + at * y_stride * ys;
        if (!room) {
            RowsArgs a{};
            a.w = {w->tiles, w->scales};
            a.x = xp;
            a.y = yp;
            a.ldx = x_stride;
            a.ldy = y_stride;
            a.M = rows;
            a.K = (int)K;
            a.N = (int)w->N;
            a.kb = (int)w->kb;
            a.vec_x = vec_x;
            a.vec_y = vec_y;
            const int64_t t = w->nb * 8;
            if (x_type == TBH_BF16)
                e = y_type == TBH_BF16 ? launch_rows<__bf16, __bf16>(a, t, s) : launch_rows<__bf16, float>(a, t, s);
            else
                e = y_type == TBH_BF16 ? launch_rows<float, __bf16>(a, t, s) : launch_rows<float, float>(a, t, s);
            continue;
        }
        QuantizeArgs q{};
        q.x = xp;
        q.ldx = x_stride;
        q.M = rows;
        q.row_tiles = (rows + 15) / 16;
        q.tiles = (uint8_t *)room;
        q.scales = (float *)(q.tiles + (q.row_tiles + 7) / 8 * 8 * w->kb * kTileBytes * (y_type == TBH_BF16 ? 1 : 2));
        q.K = (int)K;
        q.kb = (int)w->kb;
        q.vec = vec_x;
        const Plan plan = plan_of(w->nb * 8, q.row_tiles, y_type == TBH_F32);
        const bool narrow = plan == Plan::Few || y_type == TBH_BF16;
        const dim3 grid((unsigned)((w->kb + 3) / 4), (unsigned)q.row_tiles);
        if (x_type == TBH_BF16) {
            if (narrow) hipLaunchKernelGGL((fp8_quantize<__bf16, false>), grid, dim3(256), 0, s, q);
            else hipLaunchKernelGGL((fp8_quantize<__bf16, true>), grid, dim3(256), 0, s, q);
        } else {
            if (narrow) hipLaunchKernelGGL((fp8_quantize<float, false>), grid, dim3(256), 0, s, q);
            else hipLaunchKernelGGL((fp8_quantize<float, true>), grid, dim3(256), 0, s, q);
        }
        e = hipGetLastError();
        if (e != hipSuccess) break;
        TilesArgs a{};
        a.w = {w->tiles, w->scales};
        a.x = q.tiles;
        a.xs = q.scales;
        a.y = yp;
        a.ldy = y_stride;
        a.M = rows;
        a.row_tiles = q.row_tiles;
        a.N = (int)w->N;
        a.kb = (int)w->kb;
        a.w_tiles = (int)(w->nb * 8);
        a.vec_y = vec_y;
        if (plan == Plan::Few) e = y_type == TBH_BF16 ? launch_few<__bf16>(a, s) : launch_few<float>(a, s);
        else if (y_type == TBH_F32) e = launch_tiles<float, 4, 2, 4, 4>(a, s);
        else if (plan == Plan::Tiles) e = launch_tiles<__bf16, 2, 4, 4, 4>(a, s);
        else e = launch_tiles<__bf16, 2, 4, 8, 4>(a, s);
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "fp8 matmul launch");
}

}  // extern "C"
