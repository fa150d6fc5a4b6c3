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
    int64_t N, K, kb, row_tiles, step, pieces;
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
        const int64_t to = (i * a.row_tiles + t * a.step) * a.kb + b;
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

// Up to 16 rows of x as the columns of a tile; a block owns 16 RT outputs, its
// waves part K.  Every lane quantizes the 32 elements of its own operand.
template <class XT, class YT, int RT>
__global__ __launch_bounds__(256) void fp8_rows(RowsArgs a) {
    __shared__ f32x4 red[4][RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int64_t tile = (int64_t)blockIdx.x * RT, m = (int64_t)blockIdx.y * 16 + r16;
    const bool live = m < a.M;
    const XT *xr = (const XT *)a.x + m * a.ldx;
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int b0 = a.kb * wave / 4, b1 = a.kb * (wave + 1) / 4;
    for (int b = b0; b < b1; ++b) {
        i32x4 w[RT][2];
        float sw[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const uint8_t *p = a.w.tiles + ((tile + t) * a.kb + b) * kTileBytes + lane * 16;
            w[t][0] = *(const i32x4 *)p, w[t][1] = *(const i32x4 *)(p + 1024);
            sw[t] = a.w.scales[(tile + t) / 8 * a.kb + b];
        }
        float x[2][16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = b * kBlock + 64 * h + 16 * g;
            load16(xr + k, live ? a.K - k : 0, a.vec_x, x[h]);
        }
        i32x8 q;
        const float s = quantize_block(x, q);
        bf16x8 xw[2][2];
        widen(i32x4{q[0], q[1], q[2], q[3]}, xw[0]);
        widen(i32x4{q[4], q[5], q[6], q[7]}, xw[1]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            f32x4 part{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8 o[2];
                widen(w[t][h], o);
                part = mfma_wide(o[0], xw[h][0], part);
                part = mfma_wide(o[1], xw[h][1], part);
            }
            const float f = s * sw[t];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(part[i], f, acc[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= RT || !live) return;
    f32x4 v = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += red[w][wave][lane];
    const int64_t n = (tile + wave) * 16 + 4 * g;
    store4((YT *)a.y + m * a.ldy + n, v, a.N - n, a.vec_y);
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

// A wave quantizes 16 rows x 128.
template <class XT, bool WIDE>
__global__ __launch_bounds__(256) void fp8_quantize(QuantizeArgs a) {
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= a.kb) return;
    const int64_t m = (int64_t)blockIdx.y * 16 + r16;
    const XT *xr = (const XT *)a.x + m * a.ldx;
    float x[2][16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = b * kBlock + 64 * h + 16 * g;
        load16(xr + k, m < a.M ? a.K - k : 0, a.vec, x[h]);
    }
    i32x8 q;
    const float s = quantize_block(x, q);
    uint8_t *to = a.tiles + ((int64_t)blockIdx.y * a.kb + b) * (WIDE ? 2 : 1) * kTileBytes + lane * 16;
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

constexpr uint32_t kDead = 0x7FFFFFF0u;   // past every buffer: reads as zeros

// A block's 16 WN TN outputs x 16 WM TM rows; waves WN x WM, each TN x TM tiles.
// A result of bf16 comes from the FP8 instruction; one of fp32 from the bf16 one,
// half as fast, with x widened by the pass that quantized it (WIDE) and the weight here.
template <class YT, int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(64 * WN * WM) void fp8_tiles(TilesArgs a) {
    constexpr bool WIDE = sizeof(YT) == 4;
    constexpr int W = WN * WM, NT = WN * TN, MT = WM * TM, XB = (WIDE ? 2 : 1) * kTileBytes, XL = XB / 1024;
    constexpr int LOADS = (NT * 2 + MT * XL) / W;
    static_assert((NT * 2 + MT * XL) % W == 0 && TM * 64 <= 1024, "");
    constexpr int kScales = NT * kTileBytes + MT * XB, kStage = kScales + W * 1024;
    __shared__ __align__(16) char sm[2 * kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4, wn = wave % WN, wm = wave / WN;
    const int64_t n0 = (int64_t)blockIdx.x * NT, m0 = (int64_t)blockIdx.y * MT;   // in tiles
    const int64_t row = (int64_t)a.kb * kTileBytes, xrow = (int64_t)a.kb * XB;
    const dma::i32x4 wr = dma::make_rsrc(a.w.tiles + n0 * row, (int)(min((int64_t)NT, a.w_tiles - n0) * row));
    const dma::i32x4 xr = dma::make_rsrc(a.x + m0 * xrow, (int)(min((int64_t)MT, a.row_tiles - m0) * xrow));
    const int64_t mp = a.row_tiles * 16, sm0 = m0 * 16 + wm * TM * 16;
    const dma::i32x4 sr = dma::make_rsrc(a.xs, (int)min((int64_t)a.kb * mp * 4, (int64_t)kDead - 1));
    const uint32_t lds0 = dma::lds_addr(sm);
    auto issue = [&](int b, int buf) {
        const uint32_t lds = lds0 + buf * kStage;
        const bool in = b < a.kb;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int j = i * W + wave;      // 1 KiB of a tile
            const bool of_w = j < 2 * NT;
            const int t = of_w ? j >> 1 : (j - 2 * NT) / XL, part = of_w ? j & 1 : (j - 2 * NT) % XL;
            dma::dma16(__builtin_amdgcn_readfirstlane(lds + j * 1024), of_w ? wr : xr,
                       (uint32_t)((int64_t)t * (of_w ? row : xrow)) + part * 1024 + lane * 16,
                       in ? (uint32_t)b * (of_w ? kTileBytes : XB) : kDead);
        }
        // the scales of the wave's rows
        dma::dma16(__builtin_amdgcn_readfirstlane(lds + kScales + wave * 1024), sr,
                   lane < TM * 4 && sm0 + lane * 4 < mp ? (uint32_t)(sm0 * 4 + lane * 16) : kDead,
                   in ? (uint32_t)((int64_t)b * mp * 4) : kDead);
    };
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float *sw = a.w.scales + min((n0 + wn * TN) / 8, (int64_t)a.w_tiles / 8 - 1) * a.kb;
    float held = 0.0f;
    issue(0, 0);
    for (int b = 0; b < a.kb; ++b) {
        const int buf = b & 1;
        if ((b & 63) == 0) held = b + lane < a.kb ? sw[b + lane] : 0.0f;
        issue(b + 1, buf ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(LOADS + 1) : "memory");
        const char *st = sm + buf * kStage;
        const char *wt = st + wn * TN * kTileBytes + lane * 16, *xt = st + NT * kTileBytes + wm * TM * XB + lane * 16;
        const float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), b & 63));
        float f[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) f[j] = s * *(const float *)(st + kScales + wave * 1024 + (j * 16 + r16) * 4);
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
            i32x8 x[TM];
#pragma unroll
            for (int j = 0; j < TM; ++j) x[j] = operand(xt + j * kTileBytes);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const i32x8 w = operand(wt + i * kTileBytes);
#pragma unroll
                for (int j = 0; j < TM; ++j) add(i, j, mfma_block(w, x[j]));
            }
        }
        // the next step's loads fill this buffer
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
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

template <class YT>
hipError_t launch_tiles(const TilesArgs &a, hipStream_t s) {
    constexpr int NT = 8, MT = 8;
    const dim3 grid((unsigned)((a.w_tiles + NT - 1) / NT), (unsigned)((a.row_tiles + MT - 1) / MT));
    hipLaunchKernelGGL((fp8_tiles<YT, 2, 2, 4, 4>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <class XT, class YT>
hipError_t launch_rows(const RowsArgs &a, int64_t row_tiles, hipStream_t s) {
    constexpr int RT = 1;
    hipLaunchKernelGGL((fp8_rows<XT, YT, RT>), dim3((unsigned)(row_tiles / RT), (unsigned)((a.M + 15) / 16)), dim3(256), 0,
                       s, a);
    return hipGetLastError();
}

constexpr int64_t kMaxK = 1 << 20;       // a block's 16 tiles along K within 32 bits
constexpr int64_t kMaxN = 1 << 24;       // blocks of 16 outputs in one launch
constexpr int64_t kPartRows = 1 << 14;   // rows of one part of a long x

}  // namespace

hipError_t launch_repack(const uint8_t *data, int64_t N, int64_t K, int64_t count, int64_t row_tiles, int64_t step,
                         uint8_t *tiles, hipStream_t s) {
    RepackArgs a{};
    a.data = data;
    a.tiles = tiles;
    a.N = N;
    a.K = K;
    a.kb = blocks_of(K);
    a.row_tiles = row_tiles;
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
        e = launch_repack((const uint8_t *)raw, w->N, w->K, 1, w->nb * 8, 1, w->tiles, dev->stream);
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
    const int64_t rows = (std::min(M, kPartRows) + 15) & ~(int64_t)15;
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
    if (M > 32) {
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
        q.scales = (float *)(q.tiles + q.row_tiles * w->kb * kTileBytes * (y_type == TBH_BF16 ? 1 : 2));
        q.K = (int)K;
        q.kb = (int)w->kb;
        q.vec = vec_x;
        const dim3 grid((unsigned)((w->kb + 3) / 4), (unsigned)q.row_tiles);
        if (x_type == TBH_BF16) {
            if (y_type == TBH_BF16) hipLaunchKernelGGL((fp8_quantize<__bf16, false>), grid, dim3(256), 0, s, q);
            else hipLaunchKernelGGL((fp8_quantize<__bf16, true>), grid, dim3(256), 0, s, q);
        } else {
            if (y_type == TBH_BF16) hipLaunchKernelGGL((fp8_quantize<float, false>), grid, dim3(256), 0, s, q);
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
        e = y_type == TBH_BF16 ? launch_tiles<__bf16>(a, s) : launch_tiles<float>(a, s);
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "fp8 matmul launch");
}

}  // extern "C"
