// tbh_beam.hip -- beam search: the best continuations of a request's beams over
// the whole vocabulary, and the paged cache reordered to follow them.
#include <algorithm>
#include <cmath>

#include "tbh_paged.h"

namespace tbh {
namespace beam {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBeams = 64, kMaxPick = 64;
constexpr int64_t kMaxVocab = 1 << 20, kMaxRows = 1 << 20;
constexpr size_t kMaxPartials = (size_t)128 << 20;
constexpr int kPer = 16, kChunk = 256 * kPer;     // elements of a row that a block takes

struct SelectArgs {
    const float *logits;
    int64_t ld;
    const float *scores;
    const int32_t *done;
    int32_t *tokens, *parents, *done_out;
    float *scores_out;
    uint64_t *best;         // [rows][splits][k]: an element's key, largest first; 0: none
    float *most;            // [rows][splits]
    double *sum;            // [rows][splits]
    int vocab, splits, beams, k, eos;
    int row0;               // the first row of the call's part
};

// (logit, index) as one number: the larger logit, then the lower index.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return (uint64_t)(u ^ ((int32_t)u < 0 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, u ^ ((int32_t)u < 0 ? 0x80000000u : 0xFFFFFFFFu));
}

// A chunk of a row: its largest logit, the sum of exp(logit - largest) in 64
// bits, and its k best elements.
__global__ __launch_bounds__(256) void beam_chunk(SelectArgs a) {
    __shared__ uint64_t heads[256], found[kMaxPick * kPer];
    __shared__ uint64_t floor_key;
    __shared__ int count;
    __shared__ float wave_most[4];
    __shared__ double wave_sum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x, split = blockIdx.y;
    const int64_t at = (int64_t)row * a.splits + split;
    if (a.done && a.done[row]) return;       // its one candidate is no logit
    const float *x = a.logits + (int64_t)row * a.ld + (int64_t)split * kChunk;
    const int n = min(kChunk, a.vocab - split * kChunk);
    float v[kPer];
    float most = -HUGE_VALF;
    uint64_t head = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * 256 + tid;
        v[j] = i < n ? x[i] : -HUGE_VALF;
        if (v[j] != v[j]) v[j] = -HUGE_VALF;
        most = fmaxf(most, v[j]);
        const uint64_t key = v[j] > -HUGE_VALF ? key_of(v[j], (uint32_t)(split * kChunk + i)) : 0;
        head = key > head ? key : head;
    }
    heads[tid] = head;
    if (tid == 0) floor_key = 0, count = 0;
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    if (lane == 0) wave_most[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(wave_most[0], wave_most[1]), fmaxf(wave_most[2], wave_most[3]));
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (v[j] == most) s += most > -HUGE_VALF ? 1.0 : 0.0;
        else if (most < HUGE_VALF) s += exp((double)v[j] - (double)most);
    }
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) wave_sum[wave] = s;
    // the k-th largest of the threads' best: at least k elements are no smaller
    if (head) {
        int better = 0;
        for (int i = 0; i < 256; ++i) better += heads[i] > head;
        if (better == a.k - 1) floor_key = head;
    }
    __syncthreads();
    if (tid == 0) {
        a.most[at] = most;
        a.sum[at] = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    }
    const uint64_t least = floor_key;
    // threads whose best is below it have none; the k others at most all of theirs
    if (head && head >= least) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (!(v[j] > -HUGE_VALF)) continue;
            const uint64_t key = key_of(v[j], (uint32_t)(split * kChunk + j * 256 + tid));
            if (key >= least) found[atomicAdd(&count, 1)] = key;
        }
    }
    __syncthreads();
    uint64_t *best = a.best + at * a.k;
    const int c = count;
    for (int i = tid; i < c; i += 256) {
        const uint64_t key = found[i];
        int rank = 0;
        for (int o = 0; o < c; ++o) rank += found[o] > key;
        if (rank < a.k) best[rank] = key;
    }
    for (int i = c + tid; i < a.k; i += 256) best[i] = 0;
}

struct Candidate {
    double key;        // score + log probability
    uint64_t element;  // (logit, token) within the row
    int32_t row;
};
// in the order of the selection: ties to the lowest row, then token
__device__ __forceinline__ bool before(const Candidate &a, const Candidate &b) {
    if (a.key != b.key) return a.key > b.key;
    if (a.row != b.row) return a.row < b.row;
    return a.element > b.element;
}

constexpr int kRoom = kMaxPick + 256 + 64;

// Keeps the k first of n candidates, in order.
__device__ __forceinline__ int prune(Candidate *c, Candidate *tmp, int n, int k) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        int rank = 0;
        const Candidate mine = c[i];
        for (int o = 0; o < n; ++o) rank += before(c[o], mine);
        if (rank < k) tmp[rank] = mine;
    }
    __syncthreads();
    n = min(n, k);
    for (int i = threadIdx.x; i < n; i += 256) c[i] = tmp[i];
    __syncthreads();
    return n;
}

// A request: its chunks' lists joined, best elements of all lists first.
__global__ __launch_bounds__(256) void beam_join(SelectArgs a) {
    __shared__ Candidate held[kRoom], tmp[kMaxPick];
    __shared__ double total[kMaxBeams];       // log of the sum of exp(logit)
    __shared__ int alive[kMaxBeams];          // 1: continued by its logits, 2: done, 0: neither
    __shared__ int fresh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row0 = blockIdx.x * a.beams;
    for (int b = wave; b < a.beams; b += 4) {
        const int row = row0 + b;
        const float score = a.scores[row];
        int state = a.done && a.done[row] ? 2 : 1;
        if (!(score > -HUGE_VALF && score < HUGE_VALF)) state = 0;
        double sum = 0.0;
        float most = -HUGE_VALF;
        if (state == 1) {
            const float *m = a.most + (int64_t)row * a.splits;
            const double *s = a.sum + (int64_t)row * a.splits;
            for (int i = lane; i < a.splits; i += 64) most = fmaxf(most, m[i]);
            for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
            for (int i = lane; i < a.splits; i += 64)
                if (m[i] > -HUGE_VALF) sum += m[i] == most ? s[i] : most < HUGE_VALF ? s[i] * exp((double)m[i] - (double)most) : 0.0;
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
            if (!(most > -HUGE_VALF)) state = 0;
        }
        if (lane == 0) {
            alive[b] = state;
            // infinite logits share all of the weight: total holds their log count
            total[b] = state == 1 ? (most < HUGE_VALF ? (double)most : 0.0) + log(sum) : 0.0;
        }
    }
    if (tid == 0) fresh = 0;
    __syncthreads();
    int n = 0;
    const int lists = a.beams * a.splits;
    for (int level = 0; level < a.k; ++level) {
        bool more = false;
        for (int base = 0; base < lists; base += 256) {
            const int i = base + tid, b = i / a.splits, split = i - b * a.splits;
            Candidate c{};
            bool in = false;
            if (i < lists) {
                const int row = row0 + b;
                c.row = row;
                if (alive[b] == 1) {
                    c.element = a.best[((int64_t)row * a.splits + split) * a.k + level];
                    if (c.element) {
                        const float v = logit_of(c.element);
                        // beside infinite logits a finite one weighs nothing
                        const bool inf = v == HUGE_VALF, infs = a.most[(int64_t)row * a.splits + split] == HUGE_VALF;
                        c.key = (double)a.scores[row] + ((inf ? 0.0 : (double)v) - total[b]);
                        in = inf || !infs;
                        if (in && !inf)
                            for (int o = 0; o < a.splits && in; ++o) in = a.most[(int64_t)row * a.splits + o] < HUGE_VALF;
                    }
                } else if (alive[b] == 2 && level == 0 && split == 0) {
                    c.key = (double)a.scores[row];
                    c.element = 0xFFFFFFFFu - (uint32_t)a.eos;
                    in = true;
                }
                if (in && n == a.k) in = before(c, held[a.k - 1]);
            }
            if (in) held[n + atomicAdd(&fresh, 1)] = c;
            __syncthreads();
            const int got = fresh;
            __syncthreads();
            if (tid == 0) fresh = 0;
            if (got) {
                more = true;
                n = prune(held, tmp, n + got, a.k);
            } else {
                __syncthreads();
            }
        }
        // lists go down: where no list's next element is among the best, none behind it is
        if (!more) break;
    }
    const int64_t to = (int64_t)blockIdx.x * a.k;
    for (int i = tid; i < a.k; i += 256) {
        const bool some = i < n;
        const int32_t token = some ? (int32_t)(0xFFFFFFFFu - (uint32_t)held[i].element) : -1;
        a.tokens[to + i] = token;
        a.parents[to + i] = some ? held[i].row + a.row0 : -1;
        a.scores_out[to + i] = some ? (float)held[i].key : -HUGE_VALF;
        if (a.done_out) a.done_out[to + i] = some && (token == a.eos || alive[held[i].row - row0] == 2);
    }
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
// its own to write, the launch writes that too.
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

// The table in place: a thread takes one column of a group, and holds it.
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

int64_t splits_of(int64_t vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t request_bytes(int64_t beams, int64_t vocab, int64_t k) {
    return (size_t)(beams * splits_of(vocab)) * (size_t)(k * 8 + 16);
}
// requests of one part of a call
int64_t part_of(int64_t requests, int64_t beams, int64_t vocab, int64_t k) {
    return std::max<int64_t>(1, std::min<int64_t>(requests, (int64_t)(kMaxPartials / request_bytes(beams, vocab, k))));
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
    *bytes = requests ? part_of(requests, beams, vocab, k) * (int64_t)request_bytes(beams, vocab, k) : 0;
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
    const int64_t part = part_of(requests, beams, vocab, k);
    const size_t need = (size_t)part * request_bytes(beams, vocab, k);
    if (workspace && (workspace_bytes < 0 || (size_t)workspace_bytes < need)) return bad("the workspace is too small");
    if ((st = use_device(dev->ordinal)) != TBH_OK) return st;
    const hipStream_t s = (hipStream_t)stream;
    const auto held = hold_launches(dev, s);
    char *room = (char *)(workspace ? workspace : stream_workspace(dev, s, need));
    if (!room)
        return set_error(TBH_E_OOM, std::string(what) + ": no workspace (a captured stream needs an earlier eager call, or a "
                                                        "workspace of the caller's)");
    hipError_t e = hipSuccess;
    for (int64_t at = 0; at < requests && e == hipSuccess; at += part) {
        const int64_t some = std::min(part, requests - at), rows = some * beams;
        SelectArgs a{};
        a.vocab = (int)vocab;
        a.splits = (int)splits_of(vocab);
        a.beams = beams;
        a.k = k;
        a.eos = eos;
        a.row0 = (int)(at * beams);
        a.ld = ld;
        a.logits = logits + at * beams * ld;
        a.scores = scores + at * beams;
        a.done = done ? done + at * beams : nullptr;
        a.tokens = tokens + at * k;
        a.parents = parents + at * k;
        a.scores_out = scores_out + at * k;
        a.done_out = done_out ? done_out + at * k : nullptr;
        a.sum = (double *)room;
        a.best = (uint64_t *)(a.sum + rows * a.splits);
        a.most = (float *)(a.best + rows * a.splits * k);
        hipLaunchKernelGGL(beam_chunk, dim3((unsigned)rows, (unsigned)a.splits), dim3(256), 0, s, a);
        if ((e = hipGetLastError()) != hipSuccess) break;
        hipLaunchKernelGGL(beam_join, dim3((unsigned)some), dim3(256), 0, s, a);
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
        // a row's blocks parted so that there are some thousands of thread blocks
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
