// tbh_sample.hip -- tokens from logits (Sampler.swift): temperature, top-k,
// top-p and min-p, with one given random number per row.
//
// Every filter keeps a prefix of the row in the order (logit descending, index
// ascending), so the kept set is one pair (key, index): the last kept element.
// A row's prefix is found without a sort.  A histogram of the distance to the
// largest logit, of element counts (top-k) or weights (top-p), names the bin the
// border lies in.  If at most kCand elements lie in it and above it, they finish
// the row among themselves in LDS, where the bins' sums leave each only its own
// bin's to count.  Else those of the bin alone place the border, and the whole row
// is summed once more.  Bins of more elements (equal logits, high temperatures) are
// narrowed by key first.
//
// Weights exp((l - max) / T) are summed as 64-bit integers of 2^-43: sums are
// exact and do not depend on their order, and a token on the border of the
// cumulative sum is off by at most the weights' own rounding.  A weight is formed
// in double precision from a table of 2^(j / 64) and a polynomial of degree 5 on
// +-1/128 (its error, (ln 2 / 128)^6 / 720, is below 2^-54).
//
// One block of 1024 threads takes a row, in two to four passes over it.  Bound by
// the row's one CU: of 64 rows of 32000 a pass takes 5.7 us for the maximum, 13.6
// with the weights (about 35 operations in double precision each), 10 with counts;
// of 256 rows of 100000 16.7 (6.1 TB/s, memory), 37, 20.  us with all filters: 18 for
// one row of 32000, of which 5 are launch and latency; 36 for 64 rows, each its own
// settings; 121 for 256 rows of 100000 with top_p in a trace, vector instructions in 54
// of a hundred cycles (one in eight of them a multiply-add in double precision), LDS
// conflicts in 9.  Time grows with the vocabulary from there on: 64 rows of 262144 with
// top_p 211, without filters 115.
#include <algorithm>
#include <cstring>
#include <new>

#include "tbh_hostcall.h"
#include "tbh_internal.h"
#include "tbh_wave.h"

namespace tbh {
namespace {

constexpr int64_t kMaxVocab = (int64_t)1 << 20;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kCand = kThreads;                 // elements that finish a row among themselves, one per thread
constexpr int kEdge = 512;                      // of one bin, each of which counts the others before it
constexpr int kSeg = 256;                       // elements of one wave's piece of the row
constexpr int kSegs = kMaxVocab / kSeg;
constexpr double kOne = 8796093022208.0;        // 2^43

struct SampleArgs {
    const float *logits, *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
    int64_t ld;
    int32_t vocab;
};

// Order-preserving key of a logit; equal logits (-0 and 0) share one, NaN is 0.
__device__ __forceinline__ uint32_t key_of(float l) {
    if (l != l) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kNone = 0x007FFFFFu;         // key of -inf
__device__ __forceinline__ float logit_of(uint32_t key) {
    return key & 0x80000000u ? __builtin_bit_cast(float, key & 0x7FFFFFFFu) : __builtin_bit_cast(float, ~key);
}

struct Shared {
    uint32_t cnt[kBins];
    union {
        uint64_t wsum[kBins];
        uint64_t seg[kSegs];
    };
    uint64_t sums[kThreads];                    // partial sums; or weights of one piece
    uint32_t first[kBins];                  // elements in the bins before
    double pow2[64];                            // 2^(j / 64)
    uint32_t ckey[kCand];
    int32_t cidx[kCand];
    uint64_t cw[kCand];
    uint64_t red[kWaves];
    uint32_t redc[kWaves];
    uint64_t above_w;
    uint32_t above_c, bin, pop, n, key;
    int32_t idx;
};

// Sums, scans and extremes of a wave through DPP (a chain of __shfl steps goes
// through LDS: 0.4 us each here).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }

__device__ __forceinline__ uint32_t wave_sum32(uint32_t v) {
    v += dpp<wave::kXor1>(v);
    v += dpp<wave::kXor2>(v);
    v += dpp<wave::kHalfMirror>(v);
    v += dpp<wave::kRowMirror>(v);
    return lane_of(v, 0) + lane_of(v, 16) + lane_of(v, 32) + lane_of(v, 48);
}
__device__ __forceinline__ uint32_t wave_max32(uint32_t v) {
    v = max(v, dpp<wave::kXor1>(v));
    v = max(v, dpp<wave::kXor2>(v));
    v = max(v, dpp<wave::kHalfMirror>(v));
    v = max(v, dpp<wave::kRowMirror>(v));
    return max(max(lane_of(v, 0), lane_of(v, 16)), max(lane_of(v, 32), lane_of(v, 48)));
}
// of values below 2^50: two sums of 25 bits (64 of them fit 32); of any: of 22
__device__ __forceinline__ uint64_t wave_sum50(uint64_t v) {
    return ((uint64_t)wave_sum32((uint32_t)(v >> 25)) << 25) + wave_sum32((uint32_t)v & 0x1FFFFFFu);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
    return ((uint64_t)wave_sum32((uint32_t)(v >> 44)) << 44) + ((uint64_t)wave_sum32((uint32_t)(v >> 22) & 0x3FFFFFu) << 22) +
           wave_sum32((uint32_t)v & 0x3FFFFFu);
}
// Inclusive sums, lane by lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan32(uint32_t v) {
    v += shifted<0x111, 0xF>(v);    // row_shr 1, 2, 4, 8 within the 16-lane rows
    v += shifted<0x112, 0xF>(v);
    v += shifted<0x114, 0xF>(v);
    v += shifted<0x118, 0xF>(v);
    v += shifted<0x142, 0xA>(v);    // the last lane of rows 0 and 2 to rows 1 and 3,
    return v + shifted<0x143, 0xC>(v);   // of row 1 to rows 2 and 3
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
    return ((uint64_t)wave_scan32((uint32_t)(v >> 44)) << 44) + ((uint64_t)wave_scan32((uint32_t)(v >> 22) & 0x3FFFFFu) << 22) +
           wave_scan32((uint32_t)v & 0x3FFFFFu);
}

struct Row {
    const float *x;
    int32_t vocab;
    float cap;              // largest logit; of a row with inf: the largest finite float, standing for inf
    float half;             // 1/2 at temperatures above 1, where a distance past the largest float can count; else 1
    float cap_half;         // cap * half
    float bins;             // 64 / (temperature * half)
    double c;               // log2(e) / temperature
    const double *pow2;
    uint32_t top;           // the largest logit's key
    // kept so far: logits above `least`, or equal and of index at most idx
    float least;
    int32_t idx;

    __device__ __forceinline__ bool kept(float l, int32_t i) const { return l > least || (l == least && i <= idx); }
    // log2 of the weight of a kept logit, at least -64
    __device__ __forceinline__ double log_weight(float l) const {
        return fmax(((double)fminf(l, cap) - (double)cap) * c, -64.0);
    }
    // Distance to the largest logit in 1/64 of a power of e: from 2^-46 down the last bin.
    __device__ __forceinline__ uint32_t bin(float l) const {
        return (uint32_t)min(kBins - 1, (int)(fmaf(-half, fminf(l, cap), cap_half) * bins));
    }
    __device__ __forceinline__ uint64_t weight_of(double t) const {   // round(2^(43 + t)), -64 <= t <= 0
        constexpr double kShift = 6755399441055744.0;                 // 1.5 2^52: rounds to whole numbers
        const double kd = fma(t, 64.0, kShift);
        const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, kd);
        const double r = fma(kd - kShift, -1.0 / 64.0, t);
        double p = 1.3333558146428443e-3;                             // ln(2)^n / n!
        p = fma(p, r, 9.618129107628477e-3);
        p = fma(p, r, 5.550410866482158e-2);
        p = fma(p, r, 2.402265069591007e-1);
        p = fma(p, r, 6.931471805599453e-1);
        p = fma(p, r, 1.0);
        const double w = __builtin_amdgcn_ldexp(p * pow2[k & 63], (k >> 6) + 43);
        return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // 2^52: to whole numbers
    }
    __device__ __forceinline__ uint64_t weight(float l) const { return weight_of(log_weight(l)); }
    // Four at once.  The compiler would move each into the branch that uses it, where
    // its chain of dependent operations waits alone; the empty statement keeps them
    // side by side (a row of 32000 logits without filters: 29 us, 22 with it).
    __device__ __forceinline__ void weights4(const float (&e)[4], double (&lw)[4], uint64_t (&w)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) lw[j] = log_weight(e[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = weight_of(lw[j]);
        asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
    }
};

// Block sum of v in every thread.
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, Shared &sh) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) t += sh.red[i];
    return t;
}

// Cuts row.least / row.idx down to the shortest prefix whose count (BYW false) or
// weight reaches `target` (at least 1, and the kept elements reach it).
template <bool BYW>
__device__ void narrow(Row &row, uint64_t target, Shared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t hi = row.top, lo = key_of(row.least);
    uint64_t above = 0;                          // count or weight of the keys above hi
    for (;;) {
        const uint32_t span = hi - lo;
        const int shift = span < kBins ? 0 : 32 - __builtin_clz(span) - 11;
        for (int b = tid; b < kBins; b += kThreads) {
            sh.cnt[b] = 0;
            if (BYW) sh.wsum[b] = 0;
        }
        __syncthreads();
        for (int32_t i = tid; i < row.vocab; i += kThreads) {
            const float l = row.x[i];
            const uint32_t k = key_of(l);
            if (k <= hi && k >= lo && row.kept(l, i)) {
                const uint32_t b = (hi - k) >> shift;
                atomicAdd(&sh.cnt[b], 1u);
                if (BYW) atomicAdd((unsigned long long *)&sh.wsum[b], (unsigned long long)row.weight(l));
            }
        }
        __syncthreads();
        // bins 2 tid and 2 tid + 1: the first whose running sum reaches the target
        uint64_t v0 = BYW ? sh.wsum[2 * tid] : sh.cnt[2 * tid], v1 = BYW ? sh.wsum[2 * tid + 1] : sh.cnt[2 * tid + 1];
        const uint64_t in = wave_scan64(v0 + v1);
        if (lane == 63) sh.red[wave] = in;
        __syncthreads();
        uint64_t before = above;
        for (int i = 0; i < wave; ++i) before += sh.red[i];
        const uint64_t b0 = before + in - v0 - v1, b1 = b0 + v0, b2 = b1 + v1;
        if (b0 < target && b1 >= target) {
            sh.bin = 2 * tid;
            sh.above_w = b0;
            sh.pop = sh.cnt[2 * tid];
        } else if (b1 < target && b2 >= target) {
            sh.bin = 2 * tid + 1;
            sh.above_w = b1;
            sh.pop = sh.cnt[2 * tid + 1];
        }
        if (tid == 0) sh.n = 0;
        __syncthreads();
        above = sh.above_w;
        const uint32_t pop = sh.pop;
        const uint32_t h = hi - (sh.bin << shift);
        lo = h - lo < (1u << shift) ? lo : h - (1u << shift) + 1;
        hi = h;
        __syncthreads();
        if (pop <= kEdge || lo == hi) {
            if (pop > kEdge) break;
            // the candidates, each counting those before it
            for (int32_t i = tid; i < row.vocab; i += kThreads) {
                const float l = row.x[i];
                const uint32_t k = key_of(l);
                if (k <= hi && k >= lo && row.kept(l, i)) {
                    const uint32_t at = atomicAdd(&sh.n, 1u);
                    sh.ckey[at] = k;
                    sh.cidx[at] = i;
                    sh.cw[at] = BYW ? row.weight(l) : 1;
                }
            }
            __syncthreads();
            for (uint32_t c = tid; c < pop; c += kThreads) {
                const uint32_t k = sh.ckey[c];
                const int32_t ix = sh.cidx[c];
                uint64_t s = above;
                for (uint32_t j = 0; j < pop; ++j)
                    if (sh.ckey[j] > k || (sh.ckey[j] == k && sh.cidx[j] < ix)) s += sh.cw[j];
                if (s < target && s + sh.cw[c] >= target) {
                    sh.key = k;
                    sh.idx = ix;
                }
            }
            __syncthreads();
            row.least = logit_of(sh.key);
            row.idx = sh.idx;
            __syncthreads();
            return;
        }
    }
    // many equal logits: the border is the R-th of them in index order
    const float l = logit_of(hi);
    const uint64_t w = BYW ? row.weight(l) : 1;
    uint64_t left = (target - above + w - 1) / w;
    for (int32_t i0 = 0; i0 < row.vocab; i0 += kThreads) {
        const int32_t i = i0 + tid;
        const bool on = i < row.vocab && row.x[i] == l && row.kept(l, i);
        const uint64_t m = __ballot(on);
        if (lane == 0) sh.redc[wave] = __popcll(m);
        __syncthreads();
        uint32_t before = 0, total = 0;
        for (int k = 0; k < kWaves; ++k) {
            before += k < wave ? sh.redc[k] : 0;
            total += sh.redc[k];
        }
        if (on && before + __popcll(m & ((1ull << lane) - 1)) + 1 == left) sh.idx = i;
        __syncthreads();
        if (total >= left) break;
        left -= total;
    }
    row.least = l;
    row.idx = sh.idx;
    __syncthreads();
}

// The row's elements, four neighbours per thread and pass: pass p covers 4096 of
// them, wave w's part of it piece 16 p + w of 256.  Every use reads them again, a
// row stays in its XCD's cache: held in registers, eight passes unrolled, a row
// of 32000 took 20.5 us for 18.7 (no filters) and one of 1000 9.5 for 6.7, as the
// code grew eightfold.
template <bool VEC>
struct Elems {
    const float *x;
    int32_t vocab;

    __device__ __forceinline__ float4 at(int32_t i) const {
        if (VEC && i + 4 <= vocab) return *(const float4 *)(x + i);
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = i + k < vocab ? x[i + k] : -INFINITY;
        return float4{e[0], e[1], e[2], e[3]};
    }
    // f(piece, index of the first, four elements); elements behind the row are -inf
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int tid = threadIdx.x, wave = tid >> 6;
        const int32_t n = (vocab + 4095) / 4096;
        float4 a = at(4 * tid);
        for (int32_t p = 0; p < n; ++p) {
            const float4 b = p + 1 < n ? at(4096 * (p + 1) + 4 * tid) : a;   // the next, meanwhile
            f(16 * p + wave, 4096 * p + 4 * tid, a);
            a = b;
        }
    }
};

// One block per row.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void sample_rows(const SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    Row row;
    row.x = a.logits + r * a.ld;
    row.vocab = a.vocab;
    row.pow2 = sh.pow2;
    const Elems<VEC> el{row.x, a.vocab};
    if (tid < 64) sh.pow2[tid] = exp2(tid * (1.0 / 64.0));
    for (int b = tid; b < kBins; b += kThreads) {
        sh.cnt[b] = 0;
        sh.wsum[b] = 0;
    }
    if (tid == 0) sh.n = 0;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    const int32_t k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
    float u = a.u[r];

    // largest logit, first of equal ones
    uint32_t bk = 0, bi = 0;
    el.each([&](int, int32_t i, const float4 &v) {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t key = key_of(e[j]);
            if (key > bk) {                      // indices rise: the first of equal ones stays
                bk = key;
                bi = i + j;
            }
        }
    });
    const uint32_t wk = wave_max32(bk), wi = wave_max32(bk == wk ? ~bi : 0);
    uint64_t best = (uint64_t)wk << 32 | wi;
    if (lane == 0) sh.red[wave] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) best = best > sh.red[i] ? best : sh.red[i];
    __syncthreads();
    row.top = (uint32_t)(best >> 32);
    const uint32_t arg = ~(uint32_t)best;
    if (row.top <= kNone || !(t > 0.0f)) {
        if (tid == 0) {
            const bool none = row.top <= kNone;
            a.tokens[r] = none ? -1 : (int32_t)arg;
            if (a.probs) a.probs[r] = none ? 0.0f : 1.0f;
        }
        return;
    }
    const float largest = logit_of(row.top);
    const bool inf = largest == INFINITY;
    row.cap = inf ? 3.40282347e38f : largest;
    row.half = t > 1.0f ? 0.5f : 1.0f;
    row.cap_half = row.cap * row.half;
    row.bins = 64.0f / row.half / t;
    row.c = 1.4426950408889634 / (double)t;
    row.least = inf ? row.cap : -INFINITY;    // everything above -inf, or the infinities alone ...
    row.idx = -1;
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    // the least logarithm of a weight that min_p keeps (the largest, 0, always)
    const double cut = mp > 0.0f ? fmin(log2((double)mp), 0.0) : -INFINITY;

    // The border's bin, of the first `target` elements or of that much weight; the
    // histogram's sums become those of the bins before each.
    struct Border {
        uint64_t above;       // what lies in the bins before it
        uint32_t bin, pop, upto;   // its elements; those up to and with it
    };
    auto find = [&](bool by_weight, uint64_t target) {
        __syncthreads();
        const uint32_t c0 = sh.cnt[2 * tid], c1 = sh.cnt[2 * tid + 1];
        const uint64_t v0 = by_weight ? sh.wsum[2 * tid] : c0, v1 = by_weight ? sh.wsum[2 * tid + 1] : c1;
        const uint64_t in = wave_scan64(v0 + v1);
        const uint32_t cin = wave_scan32(c0 + c1);
        if (lane == 63) {
            sh.red[wave] = in;
            sh.redc[wave] = cin;
        }
        if (tid == 0) sh.bin = kBins;
        __syncthreads();
        uint64_t b0 = in - v0 - v1;
        uint32_t n0 = cin - c0 - c1;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            b0 += i < wave ? sh.red[i] : 0;
            n0 += i < wave ? sh.redc[i] : 0;
        }
        const uint64_t b1 = b0 + v0, b2 = b1 + v1;
        sh.first[2 * tid] = n0;
        sh.first[2 * tid + 1] = n0 + c0;
        if (by_weight) {
            sh.wsum[2 * tid] = b0;
            sh.wsum[2 * tid + 1] = b1;
        }
        if (b0 < target && b1 >= target) {
            sh.bin = 2 * tid;
            sh.above_w = b0;
            sh.pop = c0;
            sh.above_c = n0 + c0;
        } else if (b1 < target && b2 >= target) {
            sh.bin = 2 * tid + 1;
            sh.above_w = b1;
            sh.pop = c1;
            sh.above_c = n0 + c0 + c1;
        }
        __syncthreads();
        return Border{sh.above_w, sh.bin, sh.pop, sh.above_c};
    };
    // The weight of those of the first n candidates that come before candidate c =
    // this thread's column; the threads of a column share the others, and column
    // c's first thread (tid c) returns the sum.
    auto before_of = [&](uint32_t n) {
        const uint32_t cols = n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512, rows = kThreads / cols;
        const uint32_t c = tid & (cols - 1), s0 = tid / cols;
        const uint32_t key = c < n ? sh.ckey[c] : 0;
        const int32_t ix = c < n ? sh.cidx[c] : 0;
        uint64_t w = 0;
#pragma unroll 4
        for (uint32_t j = s0; j < n; j += rows)
            if (sh.ckey[j] > key || (sh.ckey[j] == key && sh.cidx[j] < ix)) w += sh.cw[j];
        sh.sums[tid] = w;
        __syncthreads();
        if (tid < (int)cols) {
#pragma unroll 4
            for (uint32_t q = 1; q < rows; ++q) w += sh.sums[q * cols + tid];
        }
        return w;
    };
    // The token: the first element in index order whose running sum of kept weights
    // passes u of the total.  sh.seg: sums of pieces of 256 elements; weight(i): of
    // element i of a piece.  By one wave.
    const int32_t segs = (a.vocab + kSeg - 1) / kSeg;
    auto draw = [&](uint64_t total, auto prepare, auto weight) {
        const uint64_t at = (uint64_t)((double)u * (double)total);      // below the total
        int32_t piece = -1, token = -1;
        uint64_t run = 0;
        for (int32_t g0 = 0; piece < 0 && g0 < segs; g0 += 64) {
            const uint64_t in = wave_scan64(g0 + lane < segs ? sh.seg[g0 + lane] : 0);
            const uint64_t over = __ballot(run + in > at);
            const int f = over ? __builtin_ctzll(over) : 64;
            if (over) piece = g0 + f;
            run += f ? __shfl(in, f - 1) : 0;
        }
        if (piece >= 0) {
            prepare(piece);
            uint64_t w[kSeg / 64];
#pragma unroll
            for (int j = 0; j < kSeg / 64; ++j) w[j] = weight(piece * kSeg + j * 64 + lane);
#pragma unroll
            for (int j = 0; j < kSeg / 64; ++j) {
                const uint64_t in = wave_scan64(w[j]);
                const uint64_t over = __ballot(run + in > at);
                if (over && token < 0) token = piece * kSeg + j * 64 + __builtin_ctzll(over);
                run += __shfl(in, 63);
            }
        }
        if (lane == 0) {
            a.tokens[r] = token;
            if (a.probs)
                a.probs[r] = token < 0 ? 0.0f : (float)(exp2(row.log_weight(row.x[token])) * (kOne / (double)total));
        }
    };
    // The row's token from all elements it may be: the n kept ones of bins 0 .. last,
    // put in the order of the bins, each counting those of its own bin before it (64
    // rows of 32000 with top_p near 512 elements: 69 us if each counts all of them).
    // all: the weight that top_p is of (0: the first k's).
    auto finish = [&](uint32_t last, uint32_t n, uint64_t all) {
        el.each([&](int, int32_t i, const float4 &v) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t b = row.bin(e[j]);
                if (b > last || !row.kept(e[j], i + j)) continue;
                const uint32_t at = sh.first[b] + atomicSub(&sh.cnt[b], 1u) - 1;
                sh.ckey[at] = key_of(e[j]);
                sh.cidx[at] = i + j;
            }
        });
        __syncthreads();
        const bool mine = tid < (int)n;
        const uint32_t key = mine ? sh.ckey[tid] : 0;
        const int32_t ix = mine ? sh.cidx[tid] : 0;
        const double lw = row.log_weight(logit_of(key));
        const uint64_t w = mine ? row.weight_of(lw) : 0;
        const uint32_t b = mine ? row.bin(logit_of(key)) : 0;
        sh.cw[tid] = w;
        if (p < 1.0f && !all) {                   // sh.wsum holds zeros
            if (mine) atomicAdd((unsigned long long *)&sh.wsum[b], (unsigned long long)w);
            __syncthreads();
            const uint64_t v0 = sh.wsum[2 * tid], v1 = sh.wsum[2 * tid + 1], in = wave_scan64(v0 + v1);
            if (lane == 63) sh.red[wave] = in;
            __syncthreads();
            uint64_t b0 = in - v0 - v1;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) b0 += i < wave ? sh.red[i] : 0;
            sh.wsum[2 * tid] = b0;
            sh.wsum[2 * tid + 1] = b0 + v0;
        }
        __syncthreads();
        uint32_t rank = mine ? sh.first[b] : 0;
        uint64_t before = mine ? sh.wsum[b] : 0;
        for (uint32_t j = rank, end = mine ? sh.first[b + 1] : 0; j < end; ++j)
            if (sh.ckey[j] > key || (sh.ckey[j] == key && sh.cidx[j] < ix)) {
                ++rank;
                before += sh.cw[j];
            }
        bool keep = mine && (k <= 0 || rank < (uint32_t)k);
        if (p < 1.0f) {
            const double want = ceil((double)p * (double)(all ? all : block_sum64(keep ? w : 0, sh)));
            keep &= before < (want >= 1.0 ? (uint64_t)want : 1);
        }
        if (mp > 0.0f) keep &= lw >= cut;
        const uint64_t total = block_sum64(keep ? w : 0, sh);
        sh.cw[tid] = keep ? w : 0;
        for (int32_t g = tid; g < segs; g += kThreads) sh.seg[g] = 0;
        if (tid < kSeg) sh.sums[tid] = 0;
        __syncthreads();
        if (keep) atomicAdd((unsigned long long *)&sh.seg[ix / kSeg], (unsigned long long)w);
        __syncthreads();
        if (wave != 0) return;
        draw(
            total,
            [&](int32_t piece) {
                for (uint32_t c = lane; c < n; c += 64)
                    if (sh.cidx[c] / kSeg == piece) sh.sums[sh.cidx[c] % kSeg] = sh.cw[c];
                wave::lds_fence();
            },
            [&](int32_t i) { return sh.sums[i % kSeg]; });
    };

    uint32_t edge = kBins, edge_pop = 0;          // the bin in which top_p's border lies, still to be placed
    uint64_t edge_above = 0, edge_target = 0;
    bool counted = false, whole = true;           // the histogram holds counts; nothing is cut off yet
    if (k > 0 && k < a.vocab) {
        el.each([&](int, int32_t i, const float4 &v) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t b = row.bin(e[j]);
                if (b < kBins - 1 && row.kept(e[j], i + j)) atomicAdd(&sh.cnt[b], 1u);   // the last weighs nothing
            }
        });
        counted = true;
        const Border bd = find(false, (uint64_t)k);
        if (bd.bin < (uint32_t)kBins) {           // else fewer than k elements weigh something: all are kept
            if (bd.upto <= kCand) {
                finish(bd.bin, bd.upto, 0);
                return;
            }
            narrow<false>(row, (uint64_t)k, sh);
            whole = false;
        }
    }
    if (p < 1.0f) {
        uint64_t s = 0;
        if (counted) {
            __syncthreads();
            for (int b = tid; b < kBins; b += kThreads) {
                sh.cnt[b] = 0;
                sh.wsum[b] = 0;
            }
            if (tid == 0) sh.n = 0;
            __syncthreads();
        }
        el.each([&](int, int32_t i, const float4 &v) {
            const float e[4] = {v.x, v.y, v.z, v.w};
            double lw[4];
            uint64_t w[4];
            row.weights4(e, lw, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t b = row.bin(e[j]);
                if (b < kBins - 1 && row.kept(e[j], i + j)) {
                    s += w[j];
                    atomicAdd(&sh.cnt[b], 1u);
                    atomicAdd((unsigned long long *)&sh.wsum[b], (unsigned long long)w[j]);
                }
            }
        });
        const uint64_t all = block_sum64(s, sh);
        const double want = ceil((double)p * (double)all);
        const uint64_t target = want >= 1.0 ? (uint64_t)want : 1;
        const Border bd = find(true, target);
        if (whole && bd.upto <= kCand) {
            finish(bd.bin, bd.upto, all);
            return;
        }
        if (bd.pop <= kEdge) {
            edge = bd.bin;
            edge_pop = bd.pop;
            edge_above = bd.above;
            edge_target = target;
        } else {
            narrow<true>(row, target, sh);
        }
    }

    auto weight = [&](float l, int32_t i) -> uint64_t {
        const double lw = row.log_weight(l);
        return row.kept(l, i) && lw >= cut ? row.weight_of(lw) : 0;
    };
    // sums of pieces of 256 elements, in index order; those of the border's bin
    // are set aside and added once it is placed among them
    __syncthreads();                              // the histogram's memory holds them
    uint64_t sum = 0;
    el.each([&](int piece, int32_t i, const float4 &v) {
        const float e[4] = {v.x, v.y, v.z, v.w};
        bool on[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            on[j] = row.kept(e[j], i + j);
            if (edge < (uint32_t)kBins) {
                const uint32_t b = row.bin(e[j]);
                if (on[j] && b == edge) {
                    const uint32_t at = atomicAdd(&sh.n, 1u);
                    sh.ckey[at] = key_of(e[j]);
                    sh.cidx[at] = i + j;
                }
                on[j] &= b < edge;
            }
        }
        uint64_t total = 0;
        if (__any(on[0] || on[1] || on[2] || on[3])) {
            double lw[4];
            uint64_t w[4], s = 0;
            row.weights4(e, lw, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) s += on[j] && lw[j] >= cut ? w[j] : 0;
            total = wave_sum50(s);
        }
        if (lane == 0 && piece < segs) sh.seg[piece] = total;
        sum += total;
    });
    if (edge < (uint32_t)kBins) {
        __syncthreads();
        if (tid < (int)edge_pop) sh.cw[tid] = row.weight(logit_of(sh.ckey[tid]));
        __syncthreads();
        const uint64_t before = edge_above + before_of(edge_pop);
        const bool mine = tid < (int)edge_pop && before < edge_target;
        const uint64_t w = mine ? sh.cw[tid] : 0;
        if (mine) {
            if (row.log_weight(logit_of(sh.ckey[tid])) >= cut)
                atomicAdd((unsigned long long *)&sh.seg[sh.cidx[tid] / kSeg], (unsigned long long)w);
            if (before + w >= edge_target) {      // the last one kept
                sh.key = sh.ckey[tid];
                sh.idx = sh.cidx[tid];
            }
        }
        sum += wave_sum64(mine && row.log_weight(logit_of(sh.ckey[tid])) >= cut ? w : 0);
        __syncthreads();
        row.least = logit_of(sh.key);
        row.idx = sh.idx;
    }
    if (lane == 0) sh.red[wave] = sum;
    __syncthreads();
    uint64_t total = 0;
    for (int i = 0; i < kWaves; ++i) total += sh.red[i];
    if (wave != 0) return;
    draw(total, [](int32_t) {}, [&](int32_t i) -> uint64_t { return i < a.vocab ? weight(row.x[i], i) : 0; });
}

tbh_status check_sample(const char *what, tbh_device *dev, const float *logits, int64_t ld, int64_t rows,
                        int64_t vocab, const float *u, const int32_t *tokens) {
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!dev) return bad("dev is NULL");
    if (rows < 0 || vocab < 0) return bad("negative size");
    if (rows > INT32_MAX) return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": more than 2^31 rows");
    if (vocab > kMaxVocab) return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": vocab above 2^20");
    if (rows > 1 && ld < vocab) return bad("ld is shorter than a row");
    if (rows > 0 && (!u || !tokens || (vocab > 0 && !logits))) return bad("NULL pointer");
    return TBH_OK;
}

hipError_t launch_sample(SampleArgs a, int64_t rows, hipStream_t s) {
    const bool vec = ((uintptr_t)a.logits & 15) == 0 && (a.ld % 4 == 0 || rows == 1);
    while (rows > 0) {
        const int64_t n = std::min(rows, kMostBlocks);
        if (vec) hipLaunchKernelGGL((sample_rows<true>), dim3((unsigned)n), dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((sample_rows<false>), dim3((unsigned)n), dim3(kThreads), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        rows -= n;
        if (rows == 0) break;
        a.logits += n * a.ld;
        for (const float **p : {&a.temperature, &a.top_p, &a.min_p, &a.u})
            if (*p) *p += n;
        if (a.top_k) a.top_k += n;
        if (a.probs) a.probs += n;
        a.tokens += n;
    }
    return hipSuccess;
}

}  // namespace
}  // namespace tbh

using namespace tbh;

extern "C" {

tbh_status tbh_sample_device(tbh_device *dev, const float *logits, int64_t ld, int64_t rows, int64_t vocab,
                             const float *temperature, const int32_t *top_k, const float *top_p,
                             const float *min_p, const float *u, int32_t *tokens, float *probs, void *stream) {
    tbh_status st = check_sample("tbh_sample", dev, logits, ld, rows, vocab, u, tokens);
    if (st != TBH_OK || rows == 0) return st;
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    SampleArgs a{logits, temperature, top_p, min_p, u, top_k, tokens, probs, ld, (int32_t)vocab};
    const hipError_t e = launch_sample(a, rows, (hipStream_t)stream);
    return e == hipSuccess ? TBH_OK : hip_error(e, "sample launch");
}

tbh_status tbh_sample(tbh_device *dev, const float *logits, int64_t rows, int64_t vocab, const float *temperature,
                      const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                      int32_t *tokens, float *probs) {
    tbh_status st = check_sample("tbh_sample", dev, logits, vocab, rows, vocab, u, tokens);
    if (st != TBH_OK || rows == 0) return st;
    const size_t n = (size_t)rows * 4, lb = n * (size_t)vocab;
    try {
        std::vector<int32_t> out((size_t)rows * 2);   // tokens, then probs
        st = host_call(dev, "tbh_sample",
                       {{logits, lb},
                        {temperature, temperature ? n : 0},
                        {top_k, top_k ? n : 0},
                        {top_p, top_p ? n : 0},
                        {min_p, min_p ? n : 0},
                        {u, n}},
                       out.data(), 2 * n, [&](const std::vector<const void *> &d, void *o, hipStream_t s) {
                           SampleArgs a{(const float *)d[0], (const float *)d[1], (const float *)d[3],
                                        (const float *)d[4], (const float *)d[5], (const int32_t *)d[2],
                                        (int32_t *)o, (float *)o + rows, vocab, (int32_t)vocab};
                           return launch_sample(a, rows, s);
                       });
        if (st != TBH_OK) return st;
        std::copy(out.begin(), out.begin() + rows, tokens);
        if (probs) std::memcpy(probs, out.data() + rows, n);
    } catch (const std::bad_alloc &) {
        return set_error(TBH_E_OOM, "tbh_sample: host memory");
    }
    return TBH_OK;
}

}  // extern "C"
