// tbh_beam.hip -- beam search: the best continuations of a request's beams over
// the whole vocabulary, and the paged cache reordered to follow them.
#include <algorithm>
#include <cmath>

#include "tbh_join.h"
#include "tbh_paged.h"
#include "tbh_wave.h"

namespace tbh {
namespace beam {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBeams = 64, kMaxPick = 64;
constexpr int64_t kMaxVocab = 1 << 20, kMaxRows = 1 << 20;
constexpr size_t kMaxPartials = (size_t)128 << 20;

struct SelectArgs {
    const float *logits;
    int64_t ld;
    const float *scores;
    const int32_t *done;
    int32_t *tokens, *parents, *done_out;
    float *scores_out;
    uint32_t *counters;     // [requests], then [rows]
    uint64_t *best;         // [rows][splits][k]: an element's key, largest first; 0: none
    double *sum;            // [rows][splits]: of exp(logit - most)
    float *most;            // [rows][splits]
    int vocab, splits, part, beams, k, eos;   // part: elements of a split
    int row0;               // the first row of the call's part
    bool vec;               // rows can be read four elements at a time
};

// (logit, index) as one number: the larger logit, then the lower index; 0 for what is never taken.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    const uint64_t key = (uint64_t)(u ^ ((int32_t)u < 0 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (0xFFFFFFFFu - i);
    return v > -HUGE_VALF ? key : 0;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, u ^ ((int32_t)u < 0 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// exp(d) for d in -700 .. 0: 2^n times 2^f for the fraction f of d / ln 2, |f| <= 1/2, by the
// polynomial of degree 8 that is 1 at 0 and of the least relative error, 1.1e-12.  (n from the low bits of
// a sum with 1.5 * 2^52, and into the exponent: conversions and scalings of 64-bit numbers
// are slower than their sums.)
constexpr double kLeastExp = -690.0;
__device__ __forceinline__ double exp_low(double d) {
    constexpr double kLog2E = 1.4426950408889634, kShift = 6755399441055744.0;
    const double u = __builtin_fma(d, kLog2E, kShift), f = __builtin_fma(d, kLog2E, -(u - kShift));
    double p = 1.33441836556714563e-06;
    p = __builtin_fma(p, f, 1.53142092288029329e-05);
    p = __builtin_fma(p, f, 1.54030982856375782e-04);
    p = __builtin_fma(p, f, 1.33334341575339402e-03);
    p = __builtin_fma(p, f, 9.61812955884047173e-03);
    p = __builtin_fma(p, f, 5.55041095922884711e-02);
    p = __builtin_fma(p, f, 2.40226506947425839e-01);
    p = __builtin_fma(p, f, 6.93147180541232699e-01);
    p = __builtin_fma(p, f, 1.0);
    u32x2 w = __builtin_bit_cast(u32x2, p);
    w[1] += __builtin_bit_cast(u32x2, u)[0] << 20;
    return __builtin_bit_cast(double, w);
}
// exp(v - most) of a v <= most, which is finite; below exp(kLeastExp) nothing counts, nor -inf and NaN
__device__ __forceinline__ double exp_below(float v, float most) {
    return exp_low(fmax((double)v - (double)most, kLeastExp));
}

template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v = dpp_add<wave::kXor1>(v);
    v = dpp_add<wave::kXor2>(v);
    v = dpp_add<wave::kHalfMirror>(v);
    v = dpp_add<wave::kRowMirror>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    auto row = [&](int l) { return __builtin_bit_cast(double, lane_key(u, l)); };
    return (row(0) + row(16)) + (row(32) + row(48));
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
    auto row = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return max(max(row(0), row(16)), max(row(32), row(48)));
}

// A running sum of exp(x - most); an infinite most counts the infinite x alone.
struct Total {
    float most;
    double sum;
    __device__ __forceinline__ void rescale(float to) {      // to >= most
        if (to > most) sum = to < HUGE_VALF && most > -HUGE_VALF ? sum * exp_below(most, to) : 0.0;
        most = to;
    }
};

// A list's length at which it is cut down to its k best, and elements that one step adds
// at most: fewer heads than few_heads pass as they are, of more at most k a wave.  W: waves
// of a block.
constexpr int kPer = 16, kLong = 128;
__host__ __device__ constexpr int few_heads(int W) { return 16 * W; }
__host__ __device__ constexpr int list_room(int k, int W) {
    return kLong + k + (W * k > few_heads(W) ? W * k : few_heads(W)) * kPer;
}

// Sum over each aligned group of 8 lanes, in all of them.
__device__ __forceinline__ int sum_of_8(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, wave::kXor1, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, wave::kXor2, 0xF, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, wave::kHalfMirror, 0xF, 0xF, false);
}

// Keeps the k largest of n distinct keys, in order (tmp: k keys).  Eight lanes find a key's rank.
template <int W>
__device__ __forceinline__ int prune(uint64_t *c, uint64_t *tmp, int n, int k) {
    const int part = threadIdx.x & 7;
    __syncthreads();
    for (int i = threadIdx.x >> 3; i < n; i += W * 8) {
        const uint64_t mine = c[i];
        int rank = 0;
#pragma unroll 4
        for (int o = part; o < n; o += 8) rank += c[o] > mine;
        rank = sum_of_8(rank);
        if (rank < k && part == 0) tmp[rank] = mine;
    }
    __syncthreads();
    n = min(n, k);
    for (int i = threadIdx.x; i < n; i += W * 64) c[i] = tmp[i];
    __syncthreads();
    return n;
}

// A key that k of a wave's 64 (one a lane, 0: none) are not below; 0 where there are fewer.
__device__ __forceinline__ uint64_t kth_of_wave(uint64_t key, int k) {
    int better = 0;
#pragma unroll
    for (int l = 0; l < 64; ++l) better += lane_key(key, l) > key;
    const uint64_t m = __ballot(key && better == k - 1);
    return m ? lane_key(key, (int)__builtin_ctzll(m)) : 0;
}

// A value that those of k of a wave's lanes are not below, as key_of's upper half; 0 where
// there are fewer.  Equal ones may make it more than k.
__device__ __forceinline__ uint32_t kth_value(uint32_t value, int k) {
    uint32_t most = 0;
    for (int left = k; left > 0;) {
        most = wave_most(value);
        const uint64_t m = __ballot(value == most);
        left -= __builtin_popcountll(m);
        if (!most) break;
        value = value == most ? 0 : value;
    }
    return most;
}

// Candidates of a request's rows, in LDS.
template <int N>
struct Candidates {
    double key[N];          // score + log probability
    uint64_t element[N];    // (logit, token) within the row; of equal keys the token counts
    int32_t row[N];
};

// Keeps the k first of n candidates, in order: the larger key, then the lower row, then the
// lower token.
template <int W, int N>
__device__ __forceinline__ int prune(Candidates<N> &c, Candidates<kMaxPick> &tmp, int n, int k) {
    const int part = threadIdx.x & 7;
    __syncthreads();
    for (int i = threadIdx.x >> 3; i < n; i += W * 8) {
        const double mine = c.key[i];
        int rank = 0, equal = 0;
#pragma unroll 4
        for (int o = part; o < n; o += 8) rank += c.key[o] > mine, equal += c.key[o] == mine;
        if (sum_of_8(equal) > 1)
            for (int o = part; o < n; o += 8)
                rank += c.key[o] == mine &&
                        (c.row[o] < c.row[i] || (c.row[o] == c.row[i] && (uint32_t)c.element[o] > (uint32_t)c.element[i]));
        rank = sum_of_8(rank);
        if (rank < k && part == 0) tmp.key[rank] = mine, tmp.element[rank] = c.element[i], tmp.row[rank] = c.row[i];
    }
    __syncthreads();
    n = min(n, k);
    for (int i = threadIdx.x; i < n; i += W * 64) c.key[i] = tmp.key[i], c.element[i] = tmp.element[i], c.row[i] = tmp.row[i];
    __syncthreads();
    return n;
}

// A wave's totals as one, in every lane.
__device__ __forceinline__ Total over_wave(Total t) {
    t.rescale(wave::max(t.most));
    t.sum = wave_sum(t.sum);
    return t;
}

// Everything of a block in LDS but its list, whose length depends on k.
template <int W>
struct Shared {
    Candidates<kMaxPick + 64 * W> held;
    Candidates<kMaxPick> tmp;
    Total wave_total[W];
    uint64_t wave_key[W];
    int heads[2][W];
    double total[kMaxBeams];      // log of the sum of exp(logit)
    int state[kMaxBeams];
    float score[kMaxBeams];
    int count;
    uint32_t seen;
};

// A candidate's score, from its row's and the logarithm of its row's sum.
__device__ __forceinline__ double score_of(float score, float logit, double total) {
    return (double)score + ((double)logit - total);
}

// The n candidates of a request with the tokens that they should have.  A row's list holds its
// largest logits, but where a score absorbs the difference of logits (they are tiny, or the
// score is huge) lower ones may be equal, at lower tokens.  Then the row is searched for its
// first ones of that score; how many of them there are is right as it is, since all that is
// above them is in the list.  No candidate of ordinary logits comes here.
template <int W>
__device__ __forceinline__ void take_lowest(const SelectArgs &a, int row0, int n, Shared<W> &sh) {
    constexpr int NT = 64 * W;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    bool absorbed = false;
    if (lane < n) {
        const int b = sh.held.row[lane] - row0;
        const float v = logit_of(sh.held.element[lane]);
        if (sh.state[b] == 1) {
            const float below = v == 0.0f ? -1.4e-45f : logit_of(sh.held.element[lane] - (1ull << 32));
            absorbed = score_of(sh.score[b], below, sh.total[b]) == sh.held.key[lane];
        }
    }
    const uint64_t some = __ballot(absorbed);      // the same in all waves
    if (!some) return;
    int turn = 0;          // of two sets of counts, which no two searches in a row share
    for (int i = 0; i < n;) {
        const double key = sh.held.key[i];
        const int row = sh.held.row[i], b = row - row0;
        int end = i + 1;
        while (end < n && sh.held.key[end] == key && sh.held.row[end] == row) ++end;
        const uint64_t group = (end < 64 ? 1ull << end : 0) - (1ull << i);
        if (some & group) {
            const float *x = a.logits + (int64_t)row * a.ld, score = sh.score[b];
            const double total = sh.total[b];
            int found = 0;
            for (int from = 0; from < a.vocab && found < end - i; from += NT, turn ^= 1) {
                const int j = from + tid;
                const float v = j < a.vocab ? x[j] : -HUGE_VALF;
                const bool equal = v > -HUGE_VALF && score_of(score, v, total) == key;
                const uint64_t lanes = __ballot(equal);
                if (lane == 0) sh.heads[turn][wave] = __builtin_popcountll(lanes);
                __syncthreads();
                int at = found + __builtin_popcountll(lanes & ((1ull << lane) - 1));
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    at += w < wave ? sh.heads[turn][w] : 0;
                    found += sh.heads[turn][w];
                }
                if (equal && i + at < end) sh.held.element[i + at] = key_of(v, (uint32_t)j);
            }
        }
        i = end;
    }
    __syncthreads();
}

// The request's last block: the lists of its rows joined.
template <int W>
__device__ __forceinline__ void join_rows(const SelectArgs &a, int request, Shared<W> &sh) {
    constexpr int NT = 64 * W;
    const int tid = threadIdx.x, row0 = request * a.beams, all = a.beams * a.k;
    // all rows' best first, then their next
    auto load = [&](int i) {
        return i < all ? handed_over(a.best + (int64_t)(row0 + i % a.beams) * a.splits * a.k + i / a.beams) : 0;
    };
    uint64_t next = load(tid);
    if (tid < a.beams) {
        const int row = row0 + tid;
        // (all loads before the first is used; a done row's sums are nothing)
        const float score = a.scores[row], most = handed_over(a.most + (int64_t)row * a.splits);
        const double sum = handed_over(a.sum + (int64_t)row * a.splits);
        // 1: goes on by its logits, 2: done, 3: as 1, by its infinite logits alone; 0: no candidates
        int st = a.done && a.done[row] ? 2 : 1;
        double total = 0.0;
        if (!(score > -HUGE_VALF && score < HUGE_VALF)) st = 0;
        if (st == 1) {
            st = !(most > -HUGE_VALF) ? 0 : most == HUGE_VALF ? 3 : 1;
            // infinite logits share all of the weight: the logarithm of their number
            total = (st == 1 ? (double)most : 0.0) + log(sum);
        }
        sh.state[tid] = st;
        sh.score[tid] = score;
        sh.total[tid] = total;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    int n = 0;
    for (int base = 0; base < all; base += NT) {
        const int i = base + tid, b = i % a.beams, level = i / a.beams;
        double key = 0.0;
        uint64_t element = next;
        bool in = false;
        if (base + NT < all) next = load(i + NT);
        if (i < all) {
            const int st = sh.state[b];
            const float score = sh.score[b];
            if (st == 1 || st == 3) {
                const float v = logit_of(element);
                key = score_of(score, st == 3 ? 0.0f : v, sh.total[b]);
                in = element && (st == 1 || v == HUGE_VALF);
            } else if (st == 2 && level == 0) {
                key = (double)score;
                element = 0xFFFFFFFFu - (uint32_t)a.eos;
                in = true;
            }
            // (one equal to the last held is sorted out by prune)
            if (in && n == a.k) in = key >= sh.held.key[a.k - 1];
        }
        if (in) {
            const int to = n + atomicAdd(&sh.count, 1);
            sh.held.key[to] = key, sh.held.element[to] = element, sh.held.row[to] = row0 + b;
        }
        __syncthreads();
        const int got = sh.count;
        if (got) n = prune<W>(sh.held, sh.tmp, n + got, a.k);
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
    }
    take_lowest<W>(a, row0, n, sh);
    const int64_t to = (int64_t)request * a.k;
    for (int i = tid; i < a.k; i += NT) {
        const bool some = i < n;
        const int32_t token = some ? (int32_t)(0xFFFFFFFFu - (uint32_t)sh.held.element[i]) : -1;
        a.tokens[to + i] = token;
        a.parents[to + i] = some ? sh.held.row[i] + a.row0 : -1;
        a.scores_out[to + i] = some ? (float)sh.held.key[i] : -HUGE_VALF;
        if (a.done_out) a.done_out[to + i] = some && (token == a.eos || sh.state[sh.held.row[i] - row0] == 2);
    }
}

// The row's last block: the lists and sums of its parts joined, to where its first part's stand.
template <int W>
__device__ __forceinline__ void join_parts(const SelectArgs &a, int row, uint64_t *list, Shared<W> &sh) {
    constexpr int NT = 64 * W;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t at = (int64_t)row * a.splits;
    uint64_t *best = a.best + at * a.k;
    const int all = a.splits * a.k;
    auto load = [&](int i) { return i < all ? handed_over(best + (int64_t)(i % a.splits) * a.k + i / a.splits) : 0; };
    uint64_t next = load(tid);
    Total t{-HUGE_VALF, 0.0};
    if (wave == 0) {
        for (int i = lane; i < a.splits; i += 64) {
            Total o{handed_over(a.most + at + i), handed_over(a.sum + at + i)};
            const float top = fmaxf(t.most, o.most);
            t.rescale(top), o.rescale(top);
            t.sum += o.sum;
        }
        t = over_wave(t);
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    int n = 0;
    uint64_t least = 0;
    for (int base = 0; base < all; base += NT) {       // all parts' best first, then their next
        const uint64_t key = next;
        if (base + NT < all) next = load(base + NT + tid);
        if (key > least) list[atomicAdd(&sh.count, 1)] = key;
        __syncthreads();
        n = sh.count;
        __syncthreads();
        if (n > kLong || base + NT >= all) {
            n = prune<W>(list, (uint64_t *)sh.tmp.key, n, a.k);
            if (n == a.k) least = list[a.k - 1];
            if (tid == 0) sh.count = n;
            __syncthreads();
        }
    }
    // every load of the parts is done
    for (int i = tid; i < a.k; i += NT) hand_over(best + i, i < n ? list[i] : 0);
    if (tid == 0) {
        hand_over(a.most + at, t.most);
        hand_over(a.sum + at, t.sum);
    }
}

// A part of a row, 16 elements a thread at a time: the largest logit, the sum of
// exp(logit - largest), and the k best elements, by a list of those that pass a
// key that k elements before them are not below.  The row's last
// block joins its parts, the request's last its rows (a counter takes some 70 ns an
// arrival, so that they are counted in two steps; all parts of four rows of 32000 counted
// and joined at once: 13.1 us against 13.5 in a graph, of 16 requests of them 18.4 against
// 15.2).  The sum decides which of two rows' candidates is the better, so that its terms have
// 64 bits, at some 16 64-bit operations each (with terms of 32 bits, off by up to 6e-7, 256 rows of
// 100000 took 30.5 us; with other orders of the same operations, or fewer of them, no less than so).
// Bound by the latency of one step, its
// ranking and the two joins for few rows (4 of 32000, k = 4: 11.7 us, of which the loads are
// 2), by these operations beside memory for many: 256 rows of 100000, k = 16 38.6 us, 2.65 TB/s.
template <int W>
__global__ __launch_bounds__(64 * W) void beam_select(SelectArgs a) {
    constexpr int NT = 64 * W, kChunk = NT * kPer;
    extern __shared__ uint64_t list[];       // [list_room]
    __shared__ Shared<W> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x, split = blockIdx.y, request = row / a.beams;
    const int64_t at = (int64_t)row * a.splits + split;
    const bool live = !a.done || !a.done[row];
    if (!live && split > 0) return;                // (a done row has one part)
    if (live) {
        const float *x = a.logits + (int64_t)row * a.ld;
        const int begin = split * a.part, end = min(a.vocab, begin + a.part);
        auto load = [&](int from, float (&v)[kPer]) {
#pragma unroll
            for (int j = 0; j < kPer / 4; ++j) {
                const int i = from + (j * NT + tid) * 4;
                if (a.vec && i + 4 <= end) {
                    const f32x4 q = *(const f32x4 *)(x + i);
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[4 * j + c] = q[c];
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[4 * j + c] = i + c < end ? x[i + c] : -HUGE_VALF;
                }
            }
        };
        Total t{-HUGE_VALF, 0.0};        // a thread's sum, on its wave's maximum
        uint64_t least = 0;
        auto index = [&](int from, int j) { return (uint32_t)(from + ((j / 4) * NT + tid) * 4 + j % 4); };
        // what of a step passes the list's threshold, by the whole block
        auto take = [&](const float (&v)[kPer], float top, int from) {
            // how many threads may have elements for the list (their places decide among equal ones)
            auto count_heads = [&](int *words) {
                const uint64_t lanes = __ballot(top > -HUGE_VALF && key_of(top, 0) > least);
                if (lane == 0) words[wave] = __builtin_popcountll(lanes);
                __syncthreads();
                int n = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) n += words[w];
                return n;
            };
            auto raise = [&](uint64_t key) { least = key > least + 1 ? key - 1 : least; };
            constexpr int kFew = few_heads(W);
            const int limit = max(W * a.k, kFew);
            if (count_heads(sh.heads[0]) > kFew) {
                const uint32_t best = (uint32_t)(key_of(top, 0) >> 32);
                // the least of the waves' (k / W)-th best: k elements are no smaller.  Some three
                // times as many pass as have to
                const uint32_t value = kth_value(best, (a.k + W - 1) / W);
                if (lane == 0) sh.wave_key[wave] = (uint64_t)value << 32;
                __syncthreads();
                uint64_t key = ~0ull;
#pragma unroll
                for (int w = 0; w < W; ++w) key = min(key, sh.wave_key[w]);
                raise(key);
                if (count_heads(sh.heads[1]) > limit) {
                    // unlike waves: the largest of their k-th best
                    const uint32_t kth = kth_value(best, a.k);
                    if (lane == 0) sh.wave_key[wave] = (uint64_t)kth << 32;
                    __syncthreads();
                    key = 0;
#pragma unroll
                    for (int w = 0; w < W; ++w) key = max(key, sh.wave_key[w]);
                    raise(key);
                    if (count_heads(sh.heads[0]) > limit) {
                        // many equal ones: by their places, too
                        uint32_t at = 0;
#pragma unroll
                        for (int j = kPer - 1; j >= 0; --j) at = v[j] == top ? index(from, j) : at;
                        const uint64_t exact = kth_of_wave(key_of(top, at), a.k);
                        if (lane == 0) sh.wave_key[wave] = exact;
                        __syncthreads();
                        key = 0;
#pragma unroll
                        for (int w = 0; w < W; ++w) key = max(key, sh.wave_key[w]);
                        raise(key);
                    }
                }
            }
            const float low = least ? logit_of(least) : -HUGE_VALF;
            if (top >= low) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (!(v[j] >= low)) continue;
                    const uint64_t key = key_of(v[j], index(from, j));
                    if (key > least) list[atomicAdd(&sh.count, 1)] = key;
                }
            }
            __syncthreads();
            const int n = sh.count;
            const int left = n > a.k ? prune<W>(list, (uint64_t *)sh.tmp.key, n, a.k) : n;
            if (left == a.k && n > a.k) least = list[a.k - 1];
            if (tid == 0) sh.count = left;
            __syncthreads();
        };
        // (NaN is in no comparison below, and in no maximum)
        auto largest = [&](const float (&v)[kPer]) {
            float top = -HUGE_VALF;
#pragma unroll
            for (int j = 0; j < kPer; ++j) top = fmaxf(top, v[j]);
            return top;
        };
        auto sum = [&](const float (&v)[kPer], float top) {
            const float wave_top = wave::max(top);
            if (wave_top > t.most) t.rescale(wave_top);
            if (t.most == HUGE_VALF) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) t.sum += v[j] == HUGE_VALF ? 1.0 : 0.0;
            } else {
                const float most = t.most > -HUGE_VALF ? t.most : 0.0f;
#pragma unroll
                for (int j = 0; j < kPer; ++j) t.sum += exp_below(v[j], most);
            }
        };
        float v[kPer], next[kPer];
        load(begin, v);
        if (tid == 0) sh.count = 0;
        if (begin + kChunk < end) load(begin + kChunk, next);
        // the first step's k best are the threshold for the others, which no barrier holds up: a wave
        // adds what passes to the list
        const float first = largest(v);
        take(v, first, begin);
        sum(v, first);
        const float low = least ? logit_of(least) : -HUGE_VALF;
        const int room = list_room(a.k, W);
        for (int from = begin + kChunk; from < end; from += kChunk) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = next[j];
            if (from + kChunk < end) load(from + kChunk, next);
            const float top = largest(v);
            if (__ballot(top >= low && top > -HUGE_VALF)) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (!__ballot(v[j] >= low)) continue;
                    const uint64_t key = key_of(v[j], index(from, j));
                    if (key > least) {
                        const int to = atomicAdd(&sh.count, 1);
                        if (to < room) list[to] = key;
                    }
                }
            }
            sum(v, top);
        }
        __syncthreads();
        if (sh.count > room) {
            // more than the list holds: the whole part again, step by step
            __syncthreads();
            if (tid == 0) sh.count = 0;
            least = 0;
            __syncthreads();
            for (int from = begin; from < end; from += kChunk) {
                load(from, v);
                const float top = largest(v);
                take(v, top, from);
            }
        }
        t.sum = wave_sum(t.sum);
        if (lane == 0) sh.wave_total[wave] = t;
        __syncthreads();
        const int n = prune<W>(list, (uint64_t *)sh.tmp.key, sh.count, a.k);
        for (int i = tid; i < a.k; i += NT) hand_over(a.best + at * a.k + i, i < n ? list[i] : 0);
        // (a lane a wave's: one after the other they took 2.7 us)
        if (wave == W - 1) {
            t = over_wave(lane < W ? sh.wave_total[lane] : Total{-HUGE_VALF, 0.0});
            if (lane == 0) {
                hand_over(a.most + at, t.most);
                hand_over(a.sum + at, t.sum);
            }
        }
        if (a.splits > 1) {
            if (!last_to_arrive(a.counters + gridDim.x / a.beams + row, (uint32_t)a.splits, &sh.seen)) return;
            join_parts<W>(a, row, list, sh);
        }
    }
    if (last_to_arrive(a.counters + request, (uint32_t)a.beams, &sh.seen)) join_rows<W>(a, request, sh);
}

// ---- reordering the cache ------------------------------------------------------
constexpr int kLayers = 24;          // of one launch

struct ReorderArgs {
    void *arrays[2 * kLayers];
    const int32_t *parents, *context, *shared;
    const int32_t *table;
    int32_t *table_out;
    int32_t *reordered;
    int rows, beams, most, num_blocks, shift, heads, count;   // count: arrays
    int row_bytes, steps;             // bytes of a position's head; blocks of the grid that part a row
};

// What becomes of the rows of a group: lane b of a wave learns it of row b.
struct Moves {
    int parent;        // in the group; -1: none
    int source;        // the row whose table row this row gets
    bool copy;         // whose contents are not the parent's yet
    bool ok;           // of the whole group: lengths and parents are as they should be
};

__device__ __forceinline__ Moves plan_moves(const ReorderArgs &a, int group) {
    const int lane = threadIdx.x & 63, first = group * a.beams;
    const bool in = lane < a.beams;
    int p = in ? a.parents[first + lane] : -1;
    const int len = in ? a.context[first + lane] : 0, len0 = __builtin_amdgcn_readfirstlane(len);
    Moves m;
    m.ok = __ballot(in && (p >= first + a.beams || (p >= 0 && p < first) || len != len0)) == 0;
    m.parent = m.source = lane;
    m.copy = false;
    if (!m.ok) return m;
    p = p < 0 ? -1 : p - first;
    const uint64_t stays = __ballot(in && p == lane);
    uint64_t chosen = 0;
    bool heir = false;
    for (int b = 0; b < a.beams; ++b) {
        const uint64_t c = __ballot(in && p == b);
        if (c) chosen |= 1ull << b;
        // the parent itself if it goes on, else its first child
        if (in && p == b) heir = (stays >> b & 1) ? lane == b : lane == __builtin_ctzll(c);
    }
    const uint64_t others = __ballot(in && !heir);
    uint64_t left = ~chosen & (a.beams == 64 ? ~0ull : (1ull << a.beams) - 1);   // as many as the others
    m.parent = p;
    m.source = p;
    if (in && !heir) {
        for (int turn = __builtin_popcountll(others & ((1ull << lane) - 1)); turn > 0; --turn) left &= left - 1;
        m.source = __builtin_ctzll(left);
        m.copy = p >= 0;
    }
    return m;
}

// Copies what a row does not inherit; V: the unit of a copy.  With a table of
// its own to write, the launch writes that too.  Every block works out its group's moves
// by itself (a few ballots), so that nothing is handed from launch to launch.  Bound by memory:
// eight groups of eight rows, 800 positions of 8 x 128 bf16 of two layers, 315 MB
// read and written, 64 to 69 us (4.8 TB/s, a large copy's rate; cache blocks of 32 and 64
// positions, of which one thread block copies each, 75 and 78); by its launch for one
// group of four: 4.8 us.
template <class V>
__global__ __launch_bounds__(256) void reorder_copy(ReorderArgs a) {
    const int row = blockIdx.x / a.steps, step = blockIdx.x % a.steps, group = row / a.beams;
    const int own = __builtin_amdgcn_readfirstlane(row - group * a.beams), first = group * a.beams;
    const Moves m = plan_moves(a, group);
    const int parent = __builtin_amdgcn_readlane(m.parent, own), source = __builtin_amdgcn_readlane(m.source, own);
    const bool copy = __builtin_amdgcn_readlane(m.copy, own);
    const int32_t *from = a.table + (int64_t)(first + max(parent, 0)) * a.most;
    const int32_t *to = a.table + (int64_t)(first + source) * a.most;
    if (blockIdx.y == 0 && a.table_out)
        for (int i = step * 256 + threadIdx.x; i < a.most; i += a.steps * 256)
            a.table_out[(int64_t)row * a.most + i] = to[i];
    if (blockIdx.y == 0 && step == 0 && own == 0 && threadIdx.x == 0 && a.reordered) a.reordered[group] = m.ok;
    if (!copy) return;
    const int bs = 1 << a.shift;
    const int len = min(max(a.context[row], 0), a.most << a.shift);
    const int begin = a.shared ? max(a.shared[group], 0) >> a.shift : 0;
    const int head_bytes = a.row_bytes << a.shift;
    for (int array = blockIdx.y; array < a.count; array += gridDim.y) {
        char *cache = (char *)a.arrays[array];
        for (int j = begin + step; j << a.shift < len; j += a.steps) {
            const int32_t s = from[j], d = to[j];
            if (s < 0 || d < 0 || s >= a.num_blocks || d >= a.num_blocks || s == d) continue;
            const int units = min(bs, len - (j << a.shift)) * a.row_bytes / (int)sizeof(V);   // of a head
            const char *sp = cache + (int64_t)s * a.heads * head_bytes;
            char *dp = cache + (int64_t)d * a.heads * head_bytes;
            for (int i = threadIdx.x; i < units * a.heads; i += 256) {
                const int h = i / units;
                const int64_t o = (int64_t)h * head_bytes + (int64_t)(i - h * units) * sizeof(V);
                *(V *)(dp + o) = *(const V *)(sp + o);
            }
        }
    }
}

// The table in place: a thread takes one column of a group, and holds it.  Some 3 to 8 us of a call
// (eight groups of eight rows 71.6 us, into a second table 63.6).
__global__ __launch_bounds__(64) void reorder_table(ReorderArgs a) {
    __shared__ int32_t column[kMaxBeams][64];
    __shared__ int source[kMaxBeams];
    const int group = blockIdx.x, first = group * a.beams, lane = threadIdx.x;
    const Moves m = plan_moves(a, group);
    if (lane < a.beams) source[lane] = m.source;
    __syncthreads();
    for (int i = lane; i < a.most; i += 64) {
        for (int b = 0; b < a.beams; ++b) column[b][lane] = a.table_out[(int64_t)(first + b) * a.most + i];
        for (int b = 0; b < a.beams; ++b)
            if (source[b] != b) a.table_out[(int64_t)(first + b) * a.most + i] = column[source[b]][lane];
    }
}

template <class V>
void launch_copy(const ReorderArgs &a, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((reorder_copy<V>), grid, dim3(256), 0, s, a);
}

// How a call's rows are parted.  Blocks of four waves, of 4096 elements at the least, until
// there are some four a CU; but a block of 16 waves a row, which ranks one list where the parts'
// lists would be ranked and joined, where each CU has a row and vocab * k is 2^20 or more.  Four
// waves / 16 in us: 256 rows of 100000, k = 16 49.1 / 42.1, k = 8 41.9 / 40.0, of 150000, k = 8
// 52.6 / 50.6, of 66000, k = 16 36.5 / 33.3; 512 of 50000, k = 16 45.1 / 52.6; 128 rows of 100000,
// k = 16 32.4 / 37.5; 1024 rows of 16000, k = 8 29.6 / 52.6, of 64000, k = 16 101 / 104, of 100000,
// k = 16 176 / 145; 4 rows of 32000, k = 4 11.7 / 16.7.
struct Parts {
    int waves, part, splits;
};
Parts parts_of(const tbh_device *dev, int64_t rows, int64_t vocab, int64_t k) {
    const int64_t cus = std::max(1, dev->cu_count);
    if (rows >= cus && vocab * k >= 1 << 20) return {16, (int)vocab, 1};
    const int64_t chunks = (vocab + 4095) / 4096, most = std::max<int64_t>(1, std::min(chunks, (4 * cus + rows - 1) / rows));
    const int64_t each = (chunks + most - 1) / most;
    return {4, (int)(each * 4096), (int)((chunks + each - 1) / each)};
}
size_t request_bytes(int64_t beams, int64_t splits, int64_t k) { return (size_t)(beams * splits) * (size_t)(k * 8 + 12); }
// requests of one part of a call
int64_t part_of(int64_t requests, int64_t beams, int64_t splits, int64_t k) {
    return std::max<int64_t>(1, std::min({requests, kCounters / (beams + 1), (int64_t)(kMaxPartials / request_bytes(beams, splits, k))}));
}

tbh_status check_select(const char *what, const tbh_device *dev, int64_t requests, int64_t beams, int64_t vocab, int64_t k) {
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!dev) return bad("NULL device");
    if (requests < 0) return bad("negative requests");
    if (beams < 1 || vocab < 1 || k < 1) return bad("beams, vocab and k must be positive");
    if (beams > kMaxBeams || k > kMaxPick || vocab > kMaxVocab || requests > kMaxRows / beams)
        return set_error(TBH_E_UNSUPPORTED,
                         std::string(what) + ": more than 64 beams or candidates, 2^20 rows or a vocabulary of 2^20");
    return TBH_OK;
}

}  // namespace
}  // namespace beam
}  // namespace tbh

using namespace tbh;
using namespace tbh::beam;

extern "C" {

tbh_status tbh_beam_select_workspace(tbh_device *dev, int64_t requests, int32_t beams, int64_t vocab, int32_t k,
                                     int64_t *bytes) {
    const char *what = "tbh_beam_select_workspace";
    const tbh_status st = check_select(what, dev, requests, beams, vocab, k);
    if (st != TBH_OK) return st;
    if (!bytes) return set_error(TBH_E_INVALID, std::string(what) + ": NULL pointer");
    const Parts p = parts_of(dev, requests * beams, vocab, k);
    *bytes = (int64_t)kCounterBytes;
    if (requests) *bytes += part_of(requests, beams, p.splits, k) * (int64_t)request_bytes(beams, p.splits, k);
    return TBH_OK;
}

tbh_status tbh_beam_select_device(tbh_device *dev, const float *logits, int64_t ld, int64_t requests, int32_t beams,
                                  int64_t vocab, const float *scores, const int32_t *done, int32_t eos, int32_t k,
                                  int32_t *tokens, int32_t *parents, float *scores_out, int32_t *done_out,
                                  void *workspace, int64_t workspace_bytes, void *stream) {
    const char *what = "tbh_beam_select";
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    tbh_status st = check_select(what, dev, requests, beams, vocab, k);
    if (st != TBH_OK) return st;
    if (requests == 0) return TBH_OK;
    if (!logits || !scores || !tokens || !parents || !scores_out) return bad("NULL pointer");
    if (ld < vocab && requests * beams > 1) return bad("ld is shorter than vocab");
    if (done && (eos < 0 || eos >= vocab)) return bad("done rows need an eos within the vocabulary");
    if (workspace && ((uintptr_t)workspace & 255)) return bad("the workspace must be 256-byte aligned");
    // What blocks read while others write.  (A request's scores are read by its last block alone,
    // before it writes.)
    const int64_t all_rows = requests * beams;
    const size_t in_bytes = (size_t)all_rows * 4, out_bytes = (size_t)(requests * k) * 4;
    if (done)
        for (const void *p : {(void *)tokens, (void *)parents, (void *)scores_out, (void *)done_out})
            if (p && overlap(Span(p, out_bytes), Span(done, in_bytes))) return bad("an output overlaps done");
    if ((k != beams || scores_out != scores) && overlap(Span(scores_out, out_bytes), Span(scores, in_bytes)))
        return bad("scores_out overlaps scores, and is not the same with k = beams");
    if (done_out) {
        const Span ended(done_out, out_bytes);
        if (overlap(ended, Span(scores, in_bytes)) || overlap(ended, Span(logits, vocab, ld, 4, all_rows)))
            return bad("done_out overlaps an input");
        for (const void *p : {(void *)tokens, (void *)parents, (void *)scores_out})
            if (overlap(ended, Span(p, out_bytes))) return bad("done_out overlaps another output");
    }
    const Parts p = parts_of(dev, requests * beams, vocab, k);
    const int64_t part = part_of(requests, beams, p.splits, k);
    const size_t need = (size_t)part * request_bytes(beams, p.splits, k);
    if (workspace && (workspace_bytes < 0 || (size_t)workspace_bytes < need + kCounterBytes))
        return bad("the workspace is too small");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    const auto held = hold_launches(dev, s);
    const Room room = room_of(dev, s, workspace, need);
    if (!room.counters)
        return set_error(TBH_E_OOM, std::string(what) + ": no workspace (a captured stream needs an earlier eager call, or a "
                                                        "workspace of the caller's)");
    hipError_t e = hipSuccess;
    for (int64_t at = 0; at < requests && e == hipSuccess; at += part) {
        const int64_t some = std::min(part, requests - at), rows = some * beams;
        SelectArgs a{};
        a.vocab = (int)vocab;
        a.splits = p.splits;
        a.part = p.part;
        a.beams = beams;
        a.k = k;
        a.eos = eos;
        a.row0 = (int)(at * beams);
        a.ld = ld;
        a.vec = (uintptr_t)logits % 16 == 0 && (requests * beams == 1 || ld % 4 == 0);
        a.logits = logits + at * beams * ld;
        a.scores = scores + at * beams;
        a.done = done ? done + at * beams : nullptr;
        a.tokens = tokens + at * k;
        a.parents = parents + at * k;
        a.scores_out = scores_out + at * k;
        a.done_out = done_out ? done_out + at * k : nullptr;
        a.counters = room.counters;
        a.sum = (double *)room.data;
        a.best = (uint64_t *)(a.sum + rows * a.splits);
        a.most = (float *)(a.best + rows * a.splits * k);
        const dim3 grid((unsigned)rows, (unsigned)a.splits);
        const size_t lds = (size_t)list_room(k, p.waves) * 8;
        if (p.waves == 16) hipLaunchKernelGGL((beam_select<16>), grid, dim3(1024), lds, s, a);
        else hipLaunchKernelGGL((beam_select<4>), grid, dim3(256), lds, s, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "beam select launch");
}

tbh_status tbh_paged_reorder_device(tbh_device *dev, const tbh_paged_layout *layout, int32_t beams,
                                    const int32_t *parents, const int32_t *context_lens, const int32_t *shared_lens,
                                    const int32_t *block_table, int32_t *table_out, int32_t layers,
                                    void *const *k_caches, void *const *v_caches, int32_t *reordered, void *stream) {
    const char *what = "tbh_paged_reorder";
    tbh_status st = paged::check_layout(what, dev, layout, true);
    if (st != TBH_OK) return st;
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (beams < 1 || beams > kMaxBeams) return bad("beams must be 1 .. 64");
    if (layout->max_requests % beams) return bad("max_requests must be a multiple of beams");
    if (layers < 0) return bad("negative layers");
    if (layers > 0 && (!k_caches || !v_caches)) return bad("NULL caches");
    for (int32_t l = 0; l < layers; ++l) {
        if (layout->num_blocks > 0 && (!k_caches[l] || !v_caches[l])) return bad("NULL cache");
        if (!paged::aligned(k_caches[l], 16) || !paged::aligned(v_caches[l], 16))
            return bad("the cache must be 16-byte aligned");
    }
    if (layout->max_requests == 0) return TBH_OK;
    if (!parents || !context_lens) return bad("NULL parents or context_lens");
    if (layout->max_blocks > 0 && (!block_table || !table_out)) return bad("NULL block_table");
    const uintptr_t t0 = (uintptr_t)block_table, t1 = (uintptr_t)table_out;
    if (t0 != t1 && (t0 < t1 ? t1 - t0 : t0 - t1) < (size_t)layout->max_requests * layout->max_blocks * 4)
        return bad("table_out overlaps block_table");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    ReorderArgs a{};
    a.parents = parents;
    a.context = context_lens;
    a.shared = shared_lens;
    a.table = block_table;
    a.table_out = table_out;
    a.reordered = reordered;
    a.rows = layout->max_requests;
    a.beams = beams;
    a.most = layout->max_blocks;
    a.num_blocks = layout->num_blocks;
    a.shift = __builtin_ctz((unsigned)layout->block_size);
    a.heads = layout->num_kv_heads;
    a.row_bytes = layout->head_dim * (int)paged::type_size(layout->type);
    const bool in_place = table_out == block_table;
    const auto held = hold_launches(dev, s);
    hipError_t e = hipSuccess;
    // at least one launch, for the table
    for (int32_t at = 0; (at < layers || at == 0) && e == hipSuccess; at += kLayers) {
        ReorderArgs b = a;
        b.count = 2 * std::min(kLayers, layers - at);
        for (int i = 0; i < b.count / 2; ++i) b.arrays[2 * i] = k_caches[at + i], b.arrays[2 * i + 1] = v_caches[at + i];
        if (in_place || at > 0) b.table_out = nullptr;
        if (at > 0) b.reordered = nullptr;
        // a row's blocks (here of 16) parted so that there are some thousands of thread blocks (1024, 2048,
        // 8192 or 32768 of them: the 64 rows above 103, 91, 64, 71 us, 64 rows of 100 positions 6.1,
        // 7.4, 8.8, 8.6; how much there is to copy is known on the device alone)
        const int64_t ys = std::max(1, b.count);
        const int64_t steps = std::max<int64_t>(1, std::min<int64_t>(a.most, 8192 / std::min<int64_t>(8192, a.rows * ys)));
        b.steps = (int)steps;
        // (rows of more blocks than one launch holds would need 2^20 requests)
        if (a.rows * steps > kMostBlocks) return set_error(TBH_E_UNSUPPORTED, std::string(what) + ": more than 2^20 rows");
        const dim3 grid((unsigned)(a.rows * steps), (unsigned)ys);
        if (a.row_bytes % 16 == 0) launch_copy<u32x4>(b, grid, s);
        else if (a.row_bytes % 4 == 0) launch_copy<uint32_t>(b, grid, s);
        else launch_copy<uint16_t>(b, grid, s);
        e = hipGetLastError();
    }
    if (e == hipSuccess && in_place && a.most > 0) {
        hipLaunchKernelGGL(reorder_table, dim3((unsigned)(a.rows / beams)), dim3(64), 0, s, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "paged reorder launch");
}

}  // extern "C"
