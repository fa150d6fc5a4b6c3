// tbh_sample.hip -- tokens from logits (Sampler.swift): temperature, top-k,
// top-p and min-p, with one given random number per row.
//
// Every filter keeps a prefix of the row in the order (logit descending, index
// ascending), so the kept set is one pair (key, index): the last kept element.
// A row's prefix is found without a sort: histograms of element counts (top-k)
// or weights (top-p) over ever narrower ranges of keys, then, once the border
// lies among at most kCand elements, each of them counts the others before it.
//
// Weights exp((l - max) / T) are formed in double precision and summed as
// 64-bit integers of 2^-43: sums are exact and do not depend on their order,
// and a token on the border of the cumulative sum is off by at most the weights'
// own rounding.
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
constexpr int kCand = 512;
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

struct Shared {
    uint32_t cnt[kBins];
    union {
        uint64_t wsum[kBins];
        uint64_t seg[kSegs];
    };
    uint32_t ckey[kCand], cidx[kCand];
    uint64_t cw[kCand];
    uint64_t red[kWaves];
    uint32_t redc[kWaves];
    uint64_t above_w;
    uint32_t above_c, bin, pop, n, key, idx;
    int32_t token;
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

struct Row {
    const float *x;
    int32_t vocab;
    double m, inv_t;        // largest logit, 1 / temperature (1 where m is inf: all others weigh nothing)
    uint32_t top;           // its key
    // kept so far: key above `key`, or equal and index at most idx
    uint32_t key;
    uint32_t idx;

    __device__ __forceinline__ bool kept(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
    __device__ __forceinline__ double share(float l) const {   // exp((l - max) / T)
        return (double)l == m ? 1.0 : exp(((double)l - m) * inv_t);
    }
    __device__ __forceinline__ uint64_t weight(float l) const { return (uint64_t)(share(l) * kOne + 0.5); }
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

// Cuts row.key / row.idx down to the shortest prefix whose count (BYW false) or
// weight reaches `target` (at least 1, and the kept elements reach it).
template <bool BYW>
__device__ void narrow(Row &row, uint64_t target, Shared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t hi = row.top, lo = row.key;
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
            if (k <= hi && k >= lo && row.kept(k, i)) {
                const uint32_t b = (hi - k) >> shift;
                atomicAdd(&sh.cnt[b], 1u);
                if (BYW) atomicAdd((unsigned long long *)&sh.wsum[b], (unsigned long long)row.weight(l));
            }
        }
        __syncthreads();
        // bins 2 tid and 2 tid + 1: the first whose running sum reaches the target
        uint64_t v0 = BYW ? sh.wsum[2 * tid] : sh.cnt[2 * tid], v1 = BYW ? sh.wsum[2 * tid + 1] : sh.cnt[2 * tid + 1];
        uint64_t in = v0 + v1;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
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
        if (pop <= kCand || lo == hi) {
            if (pop > kCand) break;
            // the candidates, each counting those before it
            for (int32_t i = tid; i < row.vocab; i += kThreads) {
                const float l = row.x[i];
                const uint32_t k = key_of(l);
                if (k <= hi && k >= lo && row.kept(k, i)) {
                    const uint32_t at = atomicAdd(&sh.n, 1u);
                    sh.ckey[at] = k;
                    sh.cidx[at] = i;
                    sh.cw[at] = BYW ? row.weight(l) : 1;
                }
            }
            __syncthreads();
            for (uint32_t c = tid; c < pop; c += kThreads) {
                const uint32_t k = sh.ckey[c], ix = sh.cidx[c];
                uint64_t s = above;
                for (uint32_t j = 0; j < pop; ++j)
                    if (sh.ckey[j] > k || (sh.ckey[j] == k && sh.cidx[j] < ix)) s += sh.cw[j];
                if (s < target && s + sh.cw[c] >= target) {
                    sh.key = k;
                    sh.idx = ix;
                }
            }
            __syncthreads();
            row.key = sh.key;
            row.idx = sh.idx;
            __syncthreads();
            return;
        }
    }
    // many equal logits: the border is the R-th of them in index order
    const float l = hi & 0x80000000u ? __builtin_bit_cast(float, hi & 0x7FFFFFFFu) : __builtin_bit_cast(float, ~hi);
    const uint64_t w = BYW ? row.weight(l) : 1;
    uint64_t left = (target - above + w - 1) / w;
    for (int32_t i0 = 0; i0 < row.vocab; i0 += kThreads) {
        const int32_t i = i0 + tid;
        const bool on = i < row.vocab && key_of(row.x[i]) == hi && row.kept(hi, i);
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
    row.key = hi;
    row.idx = sh.idx;
    __syncthreads();
}

// One block per row.
__global__ __launch_bounds__(kThreads) void sample_rows(const SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    Row row;
    row.x = a.logits + r * a.ld;
    row.vocab = a.vocab;

    // largest logit, first of equal ones
    uint64_t best = 0;
    for (int32_t i = tid; i < a.vocab; i += kThreads) {
        const uint64_t v = (uint64_t)key_of(row.x[i]) << 32 | (uint32_t)~i;
        best = best > v ? best : v;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_xor(best, d);
        best = best > o ? best : o;
    }
    if (lane == 0) sh.red[wave] = best;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) best = best > sh.red[i] ? best : sh.red[i];
    __syncthreads();
    row.top = (uint32_t)(best >> 32);
    const uint32_t arg = ~(uint32_t)best;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    if (row.top <= kNone || !(t > 0.0f)) {
        if (tid == 0) {
            const bool none = row.top <= kNone;
            a.tokens[r] = none ? -1 : (int32_t)arg;
            if (a.probs) a.probs[r] = none ? 0.0f : 1.0f;
        }
        return;
    }
    row.m = (double)row.x[arg];
    row.inv_t = row.m == INFINITY ? 1.0 : 1.0 / (double)t;
    row.key = kNone + 1;      // everything above -inf ...
    row.idx = 0xFFFFFFFFu;

    const int32_t k = a.top_k ? a.top_k[r] : 0;
    if (k > 0 && k < a.vocab) {
        uint64_t n = 0;       // elements above -inf
        for (int32_t i = tid; i < a.vocab; i += kThreads) n += key_of(row.x[i]) > kNone;
        n = block_sum64(n, sh);
        if ((uint64_t)k < n) narrow<false>(row, (uint64_t)k, sh);
    }
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    if (p < 1.0f) {
        uint64_t s = 0;
        for (int32_t i = tid; i < a.vocab; i += kThreads) {
            const float l = row.x[i];
            if (row.kept(key_of(l), i)) s += row.weight(l);
        }
        const double want = ceil((double)p * (double)block_sum64(s, sh));
        narrow<true>(row, want >= 1.0 ? (uint64_t)want : 1, sh);
    }
    // a weight below min_p is one of a logit below max + T log(min_p)
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    const double cut = mp > 0.0f ? log((double)mp) : -INFINITY;

    auto weight = [&](int32_t i) -> uint64_t {
        const float l = row.x[i];
        if (!row.kept(key_of(l), i) || ((double)l != row.m && ((double)l - row.m) * row.inv_t < cut)) return 0;
        return row.weight(l);
    };
    // sums of pieces of 256 elements, in index order
    const int32_t segs = (a.vocab + kSeg - 1) / kSeg;
    uint64_t all = 0;
    for (int32_t g = wave; g < segs; g += kWaves) {
        uint64_t s = 0;
        for (int j = 0; j < kSeg / 64; ++j) {
            const int32_t i = g * kSeg + j * 64 + lane;
            if (i < a.vocab) s += weight(i);
        }
        s = wave_sum64(s);
        if (lane == 0) sh.seg[g] = s;
        all += s;
    }
    if (lane == 0) sh.red[wave] = all;
    __syncthreads();
    uint64_t total = 0;
    for (int i = 0; i < kWaves; ++i) total += sh.red[i];
    if (wave != 0) return;
    float u = a.u[r];
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    uint64_t at = (uint64_t)((double)u * (double)total);      // below the total
    // the piece, then the element whose running sum passes `at`
    int32_t piece = -1;
    uint64_t run = 0;
    for (int32_t g0 = 0; piece < 0; g0 += 64) {
        uint64_t in = g0 + lane < segs ? sh.seg[g0 + lane] : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        const uint64_t over = __ballot(run + in > at);
        if (over) {
            const int f = __builtin_ctzll(over);
            piece = g0 + f;
            run += f ? __shfl(in, f - 1) : 0;
        } else {
            run += __shfl(in, 63);
            if (g0 + 64 >= segs) break;
        }
    }
    int32_t token = -1;
    for (int j = 0; j < kSeg / 64 && token < 0 && piece >= 0; ++j) {
        const int32_t i = piece * kSeg + j * 64 + lane;
        uint64_t in = i < a.vocab ? weight(i) : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        const uint64_t over = __ballot(run + in > at);
        if (over) token = piece * kSeg + j * 64 + __builtin_ctzll(over);
        else run += __shfl(in, 63);
    }
    if (lane == 0) {
        a.tokens[r] = token;
        if (a.probs) a.probs[r] = token < 0 ? 0.0f : (float)(row.share(row.x[token]) * (kOne / (double)total));
    }
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

hipError_t launch_sample(const SampleArgs &a, int64_t rows, hipStream_t s) {
    hipLaunchKernelGGL(sample_rows, dim3((unsigned)rows), dim3(kThreads), 0, s, a);
    return hipGetLastError();
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
