// tbh_paged.hip -- a step of many requests on one paged cache: the plan
// (blocks, slots and positions from the requests' lengths) and the store of
// new keys and values, with the rotary positions of keys and queries.
#include <algorithm>
#include <cmath>

#include "tbh_paged.h"

namespace tbh {
namespace {

using namespace paged;

struct PlanArgs {
    const int32_t *new_lens, *ctx, *free_count;
    int32_t *table, *free_blocks, *start, *granted, *ctx_out, *free_out, *slots, *positions;
    int32_t rows, most, num_blocks, shift;   // shift: log2 of the block size
    int64_t max_tokens;
};

constexpr int kPlanThreads = 1024;
// Tokens that plan_rows places itself (with at most 1024 requests): a launch of
// plan_tokens costs as much as four of its passes.  us of the plan of 64 requests
// and tokens: 14.4 in two launches, 7.8 in one.
constexpr int64_t kSoloTokens = 4096;

// Inclusive sum over a wave, lane by lane, of values whose sum fits 32 bits.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {   // 0 where no lane is that far down
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += shifted<0x111, 0xF>(v);    // row_shr 1, 2, 4, 8 within the 16-lane rows
    v += shifted<0x112, 0xF>(v);
    v += shifted<0x114, 0xF>(v);
    v += shifted<0x118, 0xF>(v);
    v += shifted<0x142, 0xA>(v);    // the last lane of rows 0 and 2 to rows 1 and 3,
    return v + shifted<0x143, 0xC>(v);   // of row 1 to rows 2 and 3
}

// Exclusive sum over the block's threads of values in 0 .. 2^31 - 1; total: over
// all of them.  red: one entry per wave.
__device__ __forceinline__ int64_t block_scan(int32_t v, int64_t *red, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // in halves of 16 bits, whose sums fit 32
    const int64_t in = ((int64_t)wave_scan((uint32_t)v >> 16) << 16) + wave_scan((uint32_t)v & 0xFFFFu);
    __syncthreads();
    if (lane == 63) red[wave] = in;
    __syncthreads();
    // lane i of every wave: the sum of the waves up to i
    int64_t w = lane < kPlanThreads / 64 ? red[lane] : 0;
#pragma unroll
    for (int d = 1; d < kPlanThreads / 64; d *= 2) {
        const int64_t o = __shfl_up(w, d);
        if (lane >= d) w += o;
    }
    total = __shfl(w, kPlanThreads / 64 - 1);
    const int64_t before = __shfl(w, max(wave - 1, 0));
    return (wave ? before : 0) + in - v;
}

__device__ __forceinline__ int32_t blocks_of(int64_t tokens, int shift) {
    return (int32_t)((tokens + (1 << shift) - 1) >> shift);
}

// First index whose value exceeds e, of n ascending values, the last of which does.
__device__ __forceinline__ int32_t first_above(const int32_t *v, int32_t n, int32_t e) {
    int32_t lo = 0, hi = n - 1;
    while (lo < hi) {
        const int32_t mid = (lo + hi) >> 1;
        if (v[mid] > e) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Rows of the plan: one block, a row per thread and tile of 1024 rows, its sums by
// block scans with a carry.  Bound by its chain of dependent steps: lengths, scan,
// blocks off the stack.  New blocks, and the tokens of a small step (solo), are
// dealt over all threads, each finding its row in the tile's sums (a row's own thread
// would walk a chunk's blocks alone).  7.8 us for 64 requests and tokens, 12 for 1000
// requests, whose scans over several blocks would need a launch more.
__global__ __launch_bounds__(kPlanThreads) void plan_rows(const PlanArgs a, bool solo) {
    __shared__ int64_t red[kPlanThreads / 64];
    __shared__ int32_t upto[kPlanThreads], have_[kPlanThreads];   // blocks asked for by the tile's rows up to this
    __shared__ int32_t end_[kPlanThreads], base_[kPlanThreads];   // tokens likewise; context, or -1: not granted
    __shared__ int32_t took;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t capacity = (int64_t)a.most << a.shift;
    int64_t height = min(max(a.free_count[0], 0), a.num_blocks);
    if (tid == 0) took = 0;

    // released rows push their blocks, a wave its own rows', one after another
    for (int32_t r0 = 0; r0 < a.rows; r0 += kPlanThreads) {
        const int32_t r = r0 + tid;
        const int32_t held =
            r < a.rows && a.new_lens[r] < 0 ? blocks_of(min((int64_t)max(a.ctx[r], 0), capacity), a.shift) : 0;
        if (!__syncthreads_or(held > 0)) continue;
        int64_t total;
        const int64_t at = height + block_scan(held, red, total);
        for (uint64_t m = __ballot(held > 0); m; m &= m - 1) {
            const int l = __builtin_ctzll(m);
            const int32_t n = __builtin_amdgcn_readlane(held, l);
            const int64_t to = __shfl(at, l);
            const int32_t *from = a.table + (int64_t)(r0 + (tid & ~63) + l) * a.most;
            for (int32_t j = lane; j < n; j += 64)
                if (to + j < a.num_blocks) a.free_blocks[to + j] = from[j];
        }
        height = min(height + total, (int64_t)a.num_blocks);
    }
    __syncthreads();   // the pushed ids are read below

    int64_t tokens = 0, asked = 0;
    for (int32_t r0 = 0; r0 < a.rows; r0 += kPlanThreads) {
        const int32_t r = r0 + tid, tile = min(kPlanThreads, a.rows - r0);
        const bool row = r < a.rows;
        const int32_t n = row ? a.new_lens[r] : 0, c = row ? max(a.ctx[r], 0) : 0;
        const int32_t more = max(n, 0);
        int64_t tile_tokens, tile_need;
        const int64_t first = tokens + block_scan(more, red, tile_tokens);
        // a token without an entry would get no slot, and its place be read unwritten
        const bool fits = more > 0 && (int64_t)c + more <= capacity && first + more <= a.max_tokens;
        const int32_t have = blocks_of(c, a.shift);
        const int32_t need = fits ? blocks_of((int64_t)c + more, a.shift) - have : 0;
        const int64_t before = asked + block_scan(need, red, tile_need);
        const bool ok = fits && (need == 0 || before + need <= height);
        if (row) {
            a.start[r] = (int32_t)min(first, (int64_t)INT32_MAX);
            a.granted[r] = ok ? n : 0;
            a.ctx_out[r] = n < 0 ? 0 : ok ? c + n : c;
        }
        upto[tid] = (int32_t)(before + need - asked);
        have_[tid] = have;
        end_[tid] = (int32_t)min(first + more, (int64_t)INT32_MAX);
        base_[tid] = ok ? c : -1;
        // rows that are given blocks come before those that are not: the highest
        // of a wave's has the most
        const uint64_t given = __ballot(ok && need > 0);
        if (given && lane == 63 - __builtin_clzll(given)) atomicMax(&took, (int32_t)(before + need));
        __syncthreads();
        const int32_t fresh = (int32_t)max(took - asked, (int64_t)0);   // this tile's
        for (int32_t e = tid; e < fresh; e += kPlanThreads) {
            const int32_t i = first_above(upto, tile, e);
            const int32_t j = e - (i ? upto[i - 1] : 0);
            a.table[(int64_t)(r0 + i) * a.most + have_[i] + j] = a.free_blocks[height - 1 - asked - e];
        }
        if (solo) {                               // one tile
            for (int32_t t = tid; t < a.max_tokens; t += kPlanThreads) {
                int32_t slot = -1, pos = -1;
                if (t < tile_tokens) {
                    const int32_t i = first_above(end_, tile, t), base = base_[i];
                    if (base >= 0) {
                        pos = base + t - (i ? end_[i - 1] : 0);
                        const int32_t j = (pos >> a.shift) - have_[i];
                        const int32_t id = j < 0 ? a.table[(int64_t)i * a.most + (pos >> a.shift)]
                                                 : a.free_blocks[height - 1 - (i ? upto[i - 1] : 0) - j];
                        if ((uint32_t)id < (uint32_t)a.num_blocks)
                            slot = (id << a.shift) + (pos & ((1 << a.shift) - 1));
                    }
                }
                a.slots[t] = slot;
                a.positions[t] = pos;
            }
        }
        __syncthreads();                          // the next tile writes the sums anew
        tokens += tile_tokens;
        asked += tile_need;
    }
    if (tid == 0) {
        a.start[a.rows] = (int32_t)min(tokens, (int64_t)INT32_MAX);
        a.free_out[0] = (int32_t)height - took;
    }
    if (solo && a.rows == 0)
        for (int32_t t = tid; t < a.max_tokens; t += kPlanThreads) a.slots[t] = a.positions[t] = -1;
}

// Last row whose start is at most t (the rows before it may be empty).
template <class F>
__device__ __forceinline__ int32_t row_of(int32_t t, int32_t rows, F start) {
    int32_t lo = 0, hi = rows;   // start(lo) <= t < start(hi + 1)
    while (lo < hi) {
        const int32_t mid = lo + ((hi - lo + 1) >> 1);
        if (start(mid) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Slots and positions of the step's tokens, one per thread, after plan_rows.  Bound
// by the latency of its search and look-ups: 4.4 us for 22000 tokens of 1000 requests.
__global__ __launch_bounds__(256) void plan_tokens(const PlanArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    const int32_t b = row_of((int32_t)t, a.rows, [&](int32_t i) { return a.start[i]; });
    int32_t slot = -1, pos = -1;
    if (b < a.rows) {
        const int32_t n = a.granted[b];
        if (n > 0) {
            pos = a.ctx_out[b] - n + ((int32_t)t - a.start[b]);
            const int32_t id = a.table[(int64_t)b * a.most + (pos >> a.shift)];
            if ((uint32_t)id < (uint32_t)a.num_blocks) slot = (id << a.shift) + (pos & ((1 << a.shift) - 1));
        }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
}

struct RowsArgs {
    tbh_paged_rows r;
    void *kc, *vc;
    int64_t slots_end;        // slots of the cache
    int32_t nkv, hd, shift;
    double rate;              // -2 log2(base) / head_dim
};

template <class T>
__device__ __forceinline__ float load1(const void *p, int64_t i) {
    return (float)((const T *)p)[i];
}

// The rows of one token.  The angle of pair i is position * base^(-2i / hd),
// formed in turns in double precision and reduced to (-1/2, 1/2] before the
// sine: at position 2^20 the reduced angle is off by 2^-31 turns.  A block per
// token, so that a pair's sine is formed once and shared by all heads through LDS;
// VEC: eight elements, four whole pairs, per load and store.  Bound by memory: 4096
// rows of 32 + 8 + 8 heads of 128 in bf16 17.5 us, 5.8 TB/s; by latency on few rows:
// 8 of fp32 4.0 us.
template <class XT, class CT, class QT, bool VEC>
__global__ __launch_bounds__(256) void append_rows(const RowsArgs a) {
    __shared__ float2 cs[kMaxHeadDim / 2];   // (cos, sin) per pair
    const tbh_paged_rows &r = a.r;
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, hd = a.hd;
    const bool rope = r.rope_base > 0.0f;
    if (rope) {
        const double pos = (double)max(r.positions[t], 0);
        for (int i = tid; i < hd / 2; i += 256) {
            double turns = pos * (exp2(a.rate * i) * 0.15915494309189535);   // 1 / (2 pi)
            turns -= rint(turns);
            float s, c;
            sincospif((float)(2.0 * turns), &s, &c);
            cs[i] = float2{c, s};
        }
        __syncthreads();
    }
    const int64_t slot = r.slots[t];
    const bool store = slot >= 0 && slot < a.slots_end;
    // place of key/value head 0 of the slot; heads are a block's size apart
    const int64_t hs = (int64_t)hd << a.shift;
    const int64_t at = (slot >> a.shift) * a.nkv * hs + (slot & ((1 << a.shift) - 1)) * hd;
    const int64_t nq = r.q ? (int64_t)r.num_heads * hd : 0, nk = (int64_t)a.nkv * hd;
    if constexpr (VEC) {
        for (int64_t e = (int64_t)tid * 8; e < nq + 2 * nk; e += 256 * 8) {
            const bool isq = e < nq, isk = !isq && e < nq + nk;
            const int64_t c = isq ? e : isk ? e - nq : e - nq - nk;
            if (!isq && !store) break;
            const XT *src = isq ? (const XT *)r.q + t * r.q_stride
                                : isk ? (const XT *)r.k + t * r.k_stride : (const XT *)r.v + t * r.v_stride;
            float x[8];
            unpack(*(const Vec8<XT> *)(src + c), x);
            const int h = (int)(c / hd), d = (int)(c % hd);
            if (rope && (isq || isk)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = cs[d / 2 + i];
                    const float x0 = x[2 * i], x1 = x[2 * i + 1];
                    x[2 * i] = x0 * p.x - x1 * p.y;
                    x[2 * i + 1] = x0 * p.y + x1 * p.x;
                }
            }
            if (isq) {
                Vec8<QT> o;
                pack(o, x);
                *(Vec8<QT> *)((QT *)r.q_out + t * r.q_out_stride + c) = o;
            } else {
                Vec8<CT> o;
                pack(o, x);
                *(Vec8<CT> *)((CT *)(isk ? a.kc : a.vc) + at + h * hs + d) = o;
            }
        }
    } else {
        // pairs (the last one of an odd head_dim is half)
        const int pairs = (hd + 1) / 2;
        const int64_t heads = (r.q ? r.num_heads : 0) + 2 * (int64_t)a.nkv;
        for (int64_t e = tid; e < heads * pairs; e += 256) {
            const int64_t hh = e / pairs;
            const int i = (int)(e % pairs), d = 2 * i;
            const int64_t qh = r.q ? r.num_heads : 0;
            const bool isq = hh < qh, isk = !isq && hh < qh + a.nkv, two = d + 1 < hd;
            const int64_t h = isq ? hh : isk ? hh - qh : hh - qh - a.nkv;
            if (!isq && !store) break;
            const void *src = isq ? r.q : isk ? r.k : r.v;
            const int64_t o = t * (isq ? r.q_stride : isk ? r.k_stride : r.v_stride) + h * hd + d;
            float x0 = load1<XT>(src, o), x1 = two ? load1<XT>(src, o + 1) : 0.0f;
            if (rope && (isq || isk)) {
                const float2 p = cs[i];
                const float y0 = x0 * p.x - x1 * p.y;
                x1 = x0 * p.y + x1 * p.x;
                x0 = y0;
            }
            if (isq) {
                QT *q = (QT *)r.q_out + t * r.q_out_stride + h * hd + d;
                q[0] = (QT)x0;
                if (two) q[1] = (QT)x1;
            } else {
                CT *c = (CT *)(isk ? a.kc : a.vc) + at + h * hs + d;
                c[0] = (CT)x0;
                if (two) c[1] = (CT)x1;
            }
        }
    }
}

template <class XT, class CT, class QT>
hipError_t launch_append(RowsArgs a, bool vec, hipStream_t s) {
    tbh_paged_rows &r = a.r;
    for (int64_t left = r.tokens;;) {
        const int64_t n = std::min(left, kMostBlocks);
        const dim3 grid((unsigned)n);
        if (vec) hipLaunchKernelGGL((append_rows<XT, CT, QT, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((append_rows<XT, CT, QT, false>), grid, dim3(256), 0, s, a);
        const hipError_t e = hipGetLastError();
        left -= n;
        if (e != hipSuccess || left == 0) return e;
        r.k = (const XT *)r.k + n * r.k_stride;
        r.v = (const XT *)r.v + n * r.v_stride;
        r.slots += n;
        if (r.positions) r.positions += n;
        if (!r.q) continue;
        r.q = (const XT *)r.q + n * r.q_stride;
        r.q_out = (QT *)r.q_out + n * r.q_out_stride;
    }
}

int log2_of(int32_t v) { return __builtin_ctz((unsigned)v); }

}  // namespace
}  // namespace tbh

using namespace tbh;

extern "C" {

tbh_status tbh_paged_plan_device(tbh_device *dev, const tbh_paged_layout *layout, const int32_t *new_lens,
                                 const int32_t *context_lens, int32_t *block_table, int32_t *free_blocks,
                                 const int32_t *free_count, int64_t max_tokens, int32_t *query_start,
                                 int32_t *granted, int32_t *context_out, int32_t *free_count_out,
                                 int32_t *slots, int32_t *positions, void *stream) {
    const char *what = "tbh_paged_plan";
    tbh_status st = check_layout(what, dev, layout, false);
    if (st != TBH_OK) return st;
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (max_tokens < 0 || max_tokens > INT32_MAX) return bad("max_tokens out of range");
    const int32_t B = layout->max_requests;
    if (!free_count || !query_start || !free_count_out) return bad("NULL pointer");
    if (B > 0 && (!new_lens || !context_lens || !granted || !context_out)) return bad("NULL pointer");
    if ((int64_t)B * layout->max_blocks > 0 && !block_table) return bad("NULL block_table");
    if (layout->num_blocks > 0 && !free_blocks) return bad("NULL free_blocks");
    if (max_tokens > 0 && (!slots || !positions)) return bad("NULL slots or positions");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    PlanArgs a{};
    a.new_lens = new_lens;
    a.ctx = context_lens;
    a.free_count = free_count;
    a.table = block_table;
    a.free_blocks = free_blocks;
    a.start = query_start;
    a.granted = granted;
    a.ctx_out = context_out;
    a.free_out = free_count_out;
    a.slots = slots;
    a.positions = positions;
    a.rows = B;
    a.most = layout->max_blocks;
    a.num_blocks = layout->num_blocks;
    a.shift = log2_of(layout->block_size);
    a.max_tokens = max_tokens;
    const hipStream_t s = (hipStream_t)stream;
    const bool solo = B <= kPlanThreads && max_tokens <= kSoloTokens;
    const auto held = hold_launches(dev, s);
    hipLaunchKernelGGL(plan_rows, dim3(1), dim3(kPlanThreads), 0, s, a, solo);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && max_tokens > 0 && !solo) {
        hipLaunchKernelGGL(plan_tokens, dim3((unsigned)((max_tokens + 255) / 256)), dim3(256), 0, s, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "paged plan launch");
}

tbh_status tbh_paged_append_device(tbh_device *dev, const tbh_paged_layout *layout, const tbh_paged_rows *rows,
                                   void *k_cache, void *v_cache, void *stream) {
    const char *what = "tbh_paged_append";
    tbh_status st = check_layout(what, dev, layout, true);
    if (st != TBH_OK) return st;
    auto bad = [&](const char *m) { return set_error(TBH_E_INVALID, std::string(what) + ": " + m); };
    if (!rows) return bad("rows is NULL");
    const tbh_paged_rows &r = *rows;
    if (r.tokens < 0 || r.tokens > INT32_MAX) return bad("tokens out of range");
    if (r.x_type != TBH_F32 && r.x_type != TBH_BF16) return bad("unknown x_type");
    if (r.q && (r.q_out_type != TBH_F32 && r.q_out_type != TBH_BF16)) return bad("unknown q_out_type");
    if (!(r.rope_base >= 0.0f) || std::isinf(r.rope_base)) return bad("rope_base must be finite and not negative");
    if (r.rope_base > 0.0f && layout->head_dim % 2) return bad("an odd head_dim cannot be rotated");
    const int64_t hd = layout->head_dim, nk = hd * layout->num_kv_heads;
    if (r.q && r.num_heads <= 0) return bad("num_heads must be positive");
    const int64_t nq = r.q ? hd * r.num_heads : 0;
    if (r.tokens == 0) return TBH_OK;
    if (!r.k || !r.v || !r.slots) return bad("NULL k, v or slots");
    if (r.q && !r.q_out) return bad("q_out is NULL");
    if (r.rope_base > 0.0f && !r.positions) return bad("positions are needed to rotate");
    if (layout->num_blocks > 0 && (!k_cache || !v_cache)) return bad("NULL cache");
    if (!aligned(k_cache, 16) || !aligned(v_cache, 16)) return bad("the cache must be 16-byte aligned");
    if (r.tokens > 1 && (r.k_stride < nk || r.v_stride < nk || (r.q && (r.q_stride < nq || r.q_out_stride < nq))))
        return bad("a stride is shorter than its row");
    if (r.q && r.q == r.q_out && (r.x_type != r.q_out_type || (r.tokens > 1 && r.q_stride != r.q_out_stride)))
        return bad("q_out may be q only with its type and stride");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    RowsArgs a{};
    a.r = r;
    a.kc = k_cache;
    a.vc = v_cache;
    a.nkv = layout->num_kv_heads;
    a.hd = (int32_t)hd;
    a.shift = log2_of(layout->block_size);
    a.slots_end = (int64_t)layout->num_blocks << a.shift;
    a.rate = r.rope_base > 0.0f ? -2.0 * std::log2((double)r.rope_base) / (double)hd : 0.0;
    const size_t xs = type_size(r.x_type), qs = type_size(r.q_out_type);
    auto rows16 = [](const void *p, int64_t stride, size_t size) {
        return aligned(p, 16) && (stride * (int64_t)size) % 16 == 0;
    };
    const bool vec = hd % 8 == 0 && rows16(r.k, r.k_stride, xs) && rows16(r.v, r.v_stride, xs) &&
                     (!r.q || (rows16(r.q, r.q_stride, xs) && rows16(r.q_out, r.q_out_stride, qs)));
    const hipStream_t s = (hipStream_t)stream;
    const int sel = (r.x_type == TBH_BF16) * 4 + (layout->type == TBH_BF16) * 2 + (r.q && r.q_out_type == TBH_BF16);
    hipError_t e;
    switch (sel) {
    case 0: e = launch_append<float, float, float>(a, vec, s); break;
    case 1: e = launch_append<float, float, __bf16>(a, vec, s); break;
    case 2: e = launch_append<float, __bf16, float>(a, vec, s); break;
    case 3: e = launch_append<float, __bf16, __bf16>(a, vec, s); break;
    case 4: e = launch_append<__bf16, float, float>(a, vec, s); break;
    case 5: e = launch_append<__bf16, float, __bf16>(a, vec, s); break;
    case 6: e = launch_append<__bf16, __bf16, float>(a, vec, s); break;
    default: e = launch_append<__bf16, __bf16, __bf16>(a, vec, s); break;
    }
    return e == hipSuccess ? TBH_OK : hip_error(e, "paged append launch");
}

}  // extern "C"
