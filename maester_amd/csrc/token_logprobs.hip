// Log-probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// With y_j = cap(x_j) / T, cap(x) = c tanh(x / c) (or x), per row of logits x and target t:
//   m = max_j y_j,  l = sum_j exp(y_j - m),  s = sum_j (y_j - m) exp(y_j - m)
//   logp = (y_t - m) - log l,   entropy = log l - s / l
// and for gradients a of logp and b of the entropy, log p_j = (y_j - m) - log l:
//   dx_j = (a ([j = t] - p_j) - b p_j (log p_j + entropy)) (1 - tanh(x_j / c)^2) / T.
// Everything is fp32; m, l and s run together over one pass (a larger maximum rescales l and s), so the
// row is read once.  exp(y - m) is taken as exp2((y - m) log2e): the difference first, so that a row of
// the type's lowest value does not overflow; for the same reason the gradient is handed m and log l and
// not their sum, which would absorb log l there.
#include <hip/hip_runtime.h>

#include "common.h"
#include "logprobs.h"
#include "rowio.h"

#define MA_TRY(expr)            \
    do {                        \
        int rc__ = (expr);      \
        if (rc__) return rc__;  \
    } while (0)

namespace ma {

namespace {

constexpr int kLpThreads = 512;       // >= 8 * MA_LOGPROBS_MAX_TOP: the waves' best keys, one a thread
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpMaxParts = 64;       // of a row: a lane each in the join

// A row in groups of 8 elements whose full groups start on a 16-byte boundary wherever the row itself
// starts: group g holds elements [8 g - shift, 8 g - shift + 8) cut to [0, vocab).
template <typename T>
struct Row {
    const T* p;
    int shift, vocab, groups;
    __device__ __forceinline__ Row(const T* row, int n) : p(row), vocab(n) {
        shift = (int)(((uintptr_t)row / sizeof(T)) % (16 / sizeof(T)));
        groups = (vocab + shift + 7) / 8;
    }
    __device__ __forceinline__ int first(int g) const { return g * 8 - shift; }
    __device__ __forceinline__ bool whole(int g) const { return first(g) >= 0 && first(g) + 8 <= vocab; }
    // elements outside the row come back as -inf, which adds nothing to any sum
    __device__ __forceinline__ void load(int g, float* v) const {
        const int j = first(g);
        if (whole(g)) {
            ld8<T>(p + j, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = j + i >= 0 && j + i < vocab ? ld1<T>(p + j + i) : -INFINITY;
        }
    }
    // -inf again for what lies outside the row, after a cap has made it finite
    __device__ __forceinline__ void exclude(int g, float* v) const {
        if (whole(g)) return;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first(g) + i < 0 || first(g) + i >= vocab) v[i] = -INFINITY;
    }
};

// the statistics of the whole workgroup, in every thread; box: one slot per wave
__device__ __forceinline__ LpStats workgroup_stats(LpStats t, float inv_temp, LpStats* box) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        t = lp_merged(t, lp_shuffled(t, off), inv_temp);
    }
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = t;
    __syncthreads();
    t = box[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) t = lp_merged(t, box[w], inv_temp);
    return t;
}

// ---- order of the alternatives ------------------------------------------------------------------------
// A candidate is one 64-bit key, unique in its row: the logit's bits made monotone above, the complement
// of the index below, so that larger is better and equal logits go to the lower index.  -0 equals +0 (made
// so on the bits: the build's math flags drop an addition of 0), NaN ranks with -inf.  0 is no key.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t a = __float_as_uint(x == x ? x : -INFINITY), b = a == 0x80000000u ? 0u : a;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t key_of(float x, int index) { return (uint64_t)ordered(x) << 32 | (uint32_t)~index; }

__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)k, off, 64);
        k = o > k ? o : k;
    }
    return k;
}

// 64 keys of a wave, one a lane, into descending order
__device__ __forceinline__ uint64_t wave_sort_descending(uint64_t k) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1) {
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)k, stride, 64);
            const bool larger = ((lane & size) == 0) == ((lane & stride) == 0);   // this lane keeps the larger key
            k = (o > k) == larger ? o : k;
        }
    }
    return k;
}

// LDS of the selection: keys (one slot a thread), the number of them that are in use
struct Selection {
    alignas(16) uint64_t key[kLpThreads];
    int count;
};
// Number of the n keys in LDS that are larger than `key`: its rank, as keys are unique.
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* keys, int n) {
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += keys[i] > key ? 1 : 0;
    return rank;
}
// The `want` largest of the workgroup's per-thread keys (0: none), best first, in sel.key; returns how many there are
// (fewer than `want` if not enough threads have a key).  Every wave sorts its own 64, the waves' best are ranked by
// counting.  Ends with a barrier.
__device__ __forceinline__ int best_of_threads(uint64_t key, int want, Selection& sel) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    key = wave_sort_descending(key);
    if (threadIdx.x == 0) sel.count = 0;
    __syncthreads();
    if (lane < want) sel.key[wave * want + lane] = key;
    if (lane < want && key) atomicAdd(&sel.count, 1);
    __syncthreads();
    const int n = kLpWaves * want, have = sel.count < want ? sel.count : want;
    uint64_t mine = 0;
    int rank = kLpThreads;
    if ((int)threadIdx.x < n) {
        mine = sel.key[threadIdx.x];
        if (mine) rank = rank_of(mine, sel.key, n);
    }
    __syncthreads();
    if (rank < want) sel.key[rank] = mine;
    __syncthreads();
    return have;
}

// ---- forward --------------------------------------------------------------------------------------------
// A row is cut into `parts` runs of groups, one workgroup each, so that a few rows fill the chip as well; part 0..parts-1
// of every row leave their statistics and their best keys in the workspace for token_logprobs_join_kernel (parts == 1:
// the outputs are written here).
//
// The alternatives do not need the row again: while a thread streams its groups it remembers the best group of its own
// (larger maximum, then lower index).  The k largest elements lie in the k threads whose best is largest, since any
// other thread's elements are below k distinct ones; those threads' groups, k / 512 of the part, are read once more (from
// cache) and what is not below the k-th best thread's maximum, a little over k elements, is ranked by counting.  If
// those threads hold more than 512 such elements the k largest are taken one after another.  Against a pass over the row
// per alternative: 4096 rows of 262208 bf16 logits with 8 alternatives 4.26 -> 0.42 ms (5.1 TB/s, a large copy moves
// 4.8), one such row with 20 alternatives, cut into 64 parts, 909 -> 18 us in the two kernels.
//
// With a soft cap the arithmetic bounds it, not the bytes: an element takes 25 instructions more (tanh 18, two of them at
// a quarter of the rate) than the 11 of the sums.  4096 x 262208 bf16 473 us without and 865 with a cap, 2047 x 128257 114 and
// 239 (fp32: 197 and 257), 48 x 262208 fp32 rows 16.7 and 23.5 in this kernel.
struct Outputs {
    float *logp, *entropy, *stats;
    int64_t* top_ids;
    float* top_logp;
};
struct Workspace {
    LpStats* stats;      // [rows, parts]
    uint64_t* keys;    // [rows, parts, top_k]
};

template <typename T, bool CAP>
__device__ __forceinline__ void write_row(const Row<T>& r, int64_t row, int64_t target, bool valid, const LpShape& sh, const LpStats& t,
                                          const Outputs& out) {
    const float log_l = log2f(t.l) * kLpLn2;
    const float y = valid ? lp_capped<CAP>(ld1<T>(r.p + target), sh) : 0.f;
    out.logp[row] = valid ? (y - t.m) * sh.inv_temp - log_l : 0.f;
    out.entropy[row] = valid ? log_l - t.s / t.l : 0.f;
    if (out.stats) *(float2*)(out.stats + 2 * row) = make_float2(t.m, log_l);
}
template <bool CAP>
__device__ __forceinline__ void write_alternative(uint64_t key, int64_t at, const LpShape& sh, const LpStats& t, const Outputs& out) {
    out.top_ids[at] = (int64_t)(int)~(uint32_t)key;
    out.top_logp[at] = (lp_capped<CAP>(unordered((uint32_t)(key >> 32)), sh) - t.m) * sh.inv_temp - log2f(t.l) * kLpLn2;
}

template <typename T, bool CAP, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_fwd_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                        const int64_t* __restrict__ targets, int vocab,
                                                                        int64_t ignore_index, LpShape sh, int top_k, int parts,
                                                                        Workspace ws, Outputs out) {
    __shared__ LpStats s_box[kLpWaves];
    __shared__ Selection s_sel;
    __shared__ alignas(16) uint64_t s_found[kLpThreads];
    __shared__ uint64_t s_key[kLpWaves];
    __shared__ int s_found_n;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const Row<T> r(logits + row * pitch, vocab);
    const int64_t target = targets[row];
    const bool valid = target != ignore_index && target >= 0 && target < vocab;
    // groups [g0, g1) of this part; the last parts of a short row may be empty
    const int per = (r.groups + parts - 1) / parts;
    const int g0 = min(part * per, r.groups), g1 = min(g0 + per, r.groups);

    if (!TOP && !valid) {     // nothing of this row is asked for: it is not read
        if (tid == 0) {
            if (parts > 1) {
                ws.stats[blockIdx.x] = {0.f, 1.f, 0.f};
            } else {
                out.logp[row] = out.entropy[row] = 0.f;
                if (out.stats) *(float2*)(out.stats + 2 * row) = make_float2(0.f, 0.f);
            }
        }
        return;
    }
    LpStats t = {-INFINITY, 0.f, 0.f};
    float best = -INFINITY;
    int best_g = g0 + tid;
    auto take = [&](int g, float* v) {
        if (TOP) {
            float vm = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
            vm = fmaxf(vm, fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
            if (vm > best) {
                best = vm;
                best_g = g;
            }
        }
        if (CAP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = lp_capped<CAP>(v[i], sh);
            r.exclude(g, v);
        }
        lp_fold<8>(v, sh.inv_temp, t);
    };
    // Four groups' loads at a time, then one: with a single load in flight per thread a row of 128257 comes at 3.3 TB/s.
    // Only a row's first and last group can be cut, and only those go through the guarded load.
    const int w0 = g0 + (g0 < g1 && !r.whole(g0) ? 1 : 0), w1 = g1 - (g1 > w0 && !r.whole(g1 - 1) ? 1 : 0);
    int g = g0 + tid;
    float v[4][8];
    if (g < w0) {
        r.load(g, v[0]);
        take(g, v[0]);
        g += kLpThreads;
    }
    for (; g + 3 * kLpThreads < w1; g += 4 * kLpThreads) {
#pragma unroll
        for (int n = 0; n < 4; ++n) ld8<T>(r.p + r.first(g + n * kLpThreads), v[n]);
#pragma unroll
        for (int n = 0; n < 4; ++n) take(g + n * kLpThreads, v[n]);
    }
    for (; g < w1; g += kLpThreads) {
        ld8<T>(r.p + r.first(g), v[0]);
        take(g, v[0]);
    }
    if (g < g1) {
        r.load(g, v[0]);
        take(g, v[0]);
    }
    t = workgroup_stats(t, sh.inv_temp, s_box);
    if (tid == 0) {
        if (parts == 1)
            write_row<T, CAP>(r, row, target, valid, sh, t, out);
        else
            ws.stats[blockIdx.x] = t;
    }
    if (!TOP) return;

    const int threads = best_of_threads(g0 + tid < g1 ? key_of(best, best_g) : 0, top_k, s_sel);
    // (maximum, group) of the last of the best threads; with fewer threads than top_k every element of theirs counts
    const uint64_t bar = threads == top_k ? s_sel.key[threads - 1] : 0;
    if (tid == 0) s_found_n = 0;
    __syncthreads();
    // their groups, each thread's `rounds` of them in a row
    const int rounds = (g1 - g0 + kLpThreads - 1) / kLpThreads;
    auto each = [&](auto&& f) {
        for (int c = tid; c < threads * rounds; c += kLpThreads) {
            const int owner = ((int)~(uint32_t)s_sel.key[c / rounds] - g0) % kLpThreads;
            const int g = g0 + owner + (c % rounds) * kLpThreads;
            if (g >= g1) continue;
            float v[8];
            r.load(g, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = r.first(g) + i;
                if (j >= 0 && j < vocab && key_of(v[i], g) >= bar) f(key_of(v[i], j));
            }
        }
    };
    each([&](uint64_t key) {
        const int n = atomicAdd(&s_found_n, 1);
        if (n < kLpThreads) s_found[n] = key;
    });
    __syncthreads();
    const int found = s_found_n;
    if (found <= kLpThreads) {
        if (tid < found) {
            const int rank = rank_of(s_found[tid], s_found, found);
            if (rank < top_k) {
                if (parts == 1)
                    write_alternative<CAP>(s_found[tid], row * top_k + rank, sh, t, out);
                else
                    ws.keys[(int64_t)blockIdx.x * top_k + rank] = s_found[tid];
            }
        }
        if (parts > 1 && tid >= found && tid < top_k) ws.keys[(int64_t)blockIdx.x * top_k + tid] = 0;
        return;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top_k; ++k) {
        uint64_t top = 0;
        each([&](uint64_t key) {
            if (key < last && key > top) top = key;
        });
        top = wave_max_key(top);
        __syncthreads();
        if ((tid & 63) == 0) s_key[tid >> 6] = top;
        __syncthreads();
        for (int w = 0; w < kLpWaves; ++w) top = s_key[w] > top ? s_key[w] : top;
        last = top;
        if (tid == 0) {
            if (parts == 1)
                write_alternative<CAP>(top, row * top_k + k, sh, t, out);
            else
                ws.keys[(int64_t)blockIdx.x * top_k + k] = top;
        }
    }
}

// The same without alternatives: a wave per row, a part a lane.
template <typename T, bool CAP>
__global__ __launch_bounds__(256) void token_logprobs_join_stats_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                        const int64_t* __restrict__ targets, int64_t rows, int vocab,
                                                                        int64_t ignore_index, LpShape sh, int parts, Workspace ws,
                                                                        Outputs out) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    LpStats t = {-INFINITY, 0.f, 0.f};
    if (lane < parts) t = ws.stats[row * parts + lane];
    for (int off = 1; off < parts; off <<= 1) t = lp_merged(t, lp_shuffled(t, off), sh.inv_temp);
    if (lane) return;
    const int64_t target = targets[row];
    write_row<T, CAP>(Row<T>(logits + row * pitch, vocab), row, target, target != ignore_index && target >= 0 && target < vocab, sh, t, out);
}

// One workgroup per row of several parts: at most kLpMaxParts statistics and kLpMaxParts * 64 keys, 8 a thread.
template <typename T, bool CAP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                         const int64_t* __restrict__ targets, int vocab,
                                                                         int64_t ignore_index, LpShape sh, int top_k, int parts,
                                                                         Workspace ws, Outputs out) {
    __shared__ LpStats s_box[kLpWaves];
    __shared__ Selection s_sel;
    __shared__ alignas(16) uint64_t s_found[kLpThreads];
    __shared__ int s_found_n;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    LpStats t = {-INFINITY, 0.f, 0.f};
    if (tid < parts) t = ws.stats[row * parts + tid];
    t = workgroup_stats(t, sh.inv_temp, s_box);
    if (tid == 0) {
        const int64_t target = targets[row];
        write_row<T, CAP>(Row<T>(logits + row * pitch, vocab), row, target, target != ignore_index && target >= 0 && target < vocab, sh, t, out);
    }
    const uint64_t* keys = ws.keys + row * parts * top_k;
    const int n = parts * top_k;
    uint64_t best = 0;
    for (int i = tid; i < n; i += kLpThreads) best = keys[i] > best ? keys[i] : best;
    const int threads = best_of_threads(best, top_k, s_sel);
    const uint64_t bar = threads == top_k ? s_sel.key[threads - 1] : 0;
    if (tid == 0) s_found_n = 0;
    __syncthreads();
    // only the best threads have keys at or above the bar, so at most 64 * 8 of them
    for (int i = tid; i < n; i += kLpThreads)
        if (keys[i] && keys[i] >= bar) s_found[atomicAdd(&s_found_n, 1)] = keys[i];
    __syncthreads();
    if (tid < s_found_n) {
        const int rank = rank_of(s_found[tid], s_found, s_found_n);
        if (rank < top_k) write_alternative<CAP>(s_found[tid], row * top_k + rank, sh, t, out);
    }
}

// ---- gradient -------------------------------------------------------------------------------------------
constexpr int kLpBwdThreads = 256, kLpBwdGroups = 4;      // groups of 8 per thread
template <typename T, bool CAP>
__global__ __launch_bounds__(kLpBwdThreads) void token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                           const int64_t* __restrict__ targets, int vocab,
                                                                           int64_t ignore_index, LpShape sh,
                                                                           const float* __restrict__ stats,
                                                                           const float* __restrict__ entropy_in,
                                                                           const float* __restrict__ dlogp,
                                                                           const float* __restrict__ dentropy, T* __restrict__ dlogits,
                                                                           int64_t dpitch, int chunks) {
    const int64_t row = blockIdx.x / chunks;
    const int chunk = blockIdx.x % chunks;
    const Row<T> in(logits + row * pitch, vocab), out(dlogits + row * dpitch, vocab);   // groups follow the output's alignment
    T* dst = dlogits + row * dpitch;
    const int64_t target = targets[row];
    const bool valid = target != ignore_index && target >= 0 && target < vocab;
    const float a = valid && dlogp ? dlogp[row] : 0.f, b = valid && dentropy ? dentropy[row] : 0.f;
    const float top = stats[2 * row], log_l = stats[2 * row + 1], h = entropy_in[row];
    const bool same = in.shift == out.shift;
#pragma unroll
    for (int n = 0; n < kLpBwdGroups; ++n) {
        const int g = (chunk * kLpBwdGroups + n) * kLpBwdThreads + threadIdx.x;
        if (g >= out.groups) break;
        const int j = out.first(g);
        float d[8];
        if (!valid) {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = 0.f;
        } else {
            float v[8];
            if (same) {
                in.load(g, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = j + i >= 0 && j + i < vocab ? ld1<T>(in.p + j + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float th = CAP ? lp_tanh(v[i] * sh.inv_cap) : 0.f;
                const float lp = fmaf((CAP ? sh.cap * th : v[i]) - top, sh.inv_temp, -log_l);
                const float p = __builtin_amdgcn_exp2f(lp * kLpLog2e);        // (0 below -150: no product with a larger lp)
                d[i] = -p * fmaf(b, fmaxf(lp, -200.f) + h, a);
                if (j + i == target) d[i] += a;
                d[i] *= CAP ? (1.f - th * th) * sh.inv_temp : sh.inv_temp;
            }
        }
        if (out.whole(g)) {
            st8<T>(dst + j, d);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i >= 0 && j + i < vocab) st1<T>(dst + j + i, d[i]);
        }
    }
}

}  // namespace

// Parts that a row is cut into, none with fewer than 512 groups (a group per thread): few rows to two workgroups a compute
// unit, as a part ends with some 10 us of selection (48 fp32 rows: 26 us, with 4096 workgroups 41); many rows to four
// rounds of the 1024 resident ones, so that the last round is a small part of them all.
int token_logprobs_parts(int64_t rows, int64_t vocab) {
    const int64_t want = rows >= 1024 ? (4096 + rows - 1) / rows : 512 / rows, most = (vocab / 8 + kLpThreads - 1) / kLpThreads;
    const int64_t parts = want < most ? want : most;
    return (int)(parts < 1 ? 1 : parts > kLpMaxParts ? kLpMaxParts : parts);
}
static size_t stats_bytes(int64_t rows, int parts) { return ((size_t)rows * parts * sizeof(LpStats) + 15) & ~(size_t)15; }
size_t token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_k) {
    const int parts = token_logprobs_parts(rows, vocab);
    return parts == 1 ? 0 : stats_bytes(rows, parts) + (size_t)rows * parts * top_k * sizeof(uint64_t);
}

// workgroups per row of the gradient kernel, for a row that starts anywhere
int token_logprobs_bwd_chunks(int64_t vocab) {
    const int per = kLpBwdThreads * kLpBwdGroups;
    return (int)(((vocab + 14) / 8 + per - 1) / per);
}

namespace {

template <typename T, bool CAP>
int fwd(const TokenLogprobsArgs& a, hipStream_t st) {
    const LpShape sh = lp_shape(a.softcap, a.temperature);
    const int parts = token_logprobs_parts(a.rows, a.vocab);
    const Workspace ws = {(LpStats*)a.ws, (uint64_t*)((char*)a.ws + stats_bytes(a.rows, parts))};
    const Outputs out = {a.logp, a.entropy, a.stats, a.top_ids, a.top_logp};
    auto kernel = a.top_k ? token_logprobs_fwd_kernel<T, CAP, true> : token_logprobs_fwd_kernel<T, CAP, false>;
    kernel<<<(unsigned)(a.rows * parts), kLpThreads, 0, st>>>((const T*)a.logits, a.pitch, a.targets, (int)a.vocab, a.ignore_index, sh,
                                                              a.top_k, parts, ws, out);
    if (parts > 1) {
        MA_TRY(check_launch("token_logprobs_fwd_kernel"));
        if (a.top_k)
            token_logprobs_join_kernel<T, CAP><<<(unsigned)a.rows, kLpThreads, 0, st>>>((const T*)a.logits, a.pitch, a.targets, (int)a.vocab,
                                                                                         a.ignore_index, sh, a.top_k, parts, ws, out);
        else
            token_logprobs_join_stats_kernel<T, CAP><<<(unsigned)((a.rows + 3) / 4), 256, 0, st>>>(
                (const T*)a.logits, a.pitch, a.targets, a.rows, (int)a.vocab, a.ignore_index, sh, parts, ws, out);
    }
    return check_launch("token_logprobs_fwd_kernel");
}
template <typename T>
int bwd(const TokenLogprobsArgs& a, hipStream_t st) {
    const LpShape sh = lp_shape(a.softcap, a.temperature);
    const int chunks = token_logprobs_bwd_chunks(a.vocab);
    const dim3 grid((unsigned)(a.rows * chunks));
    auto kernel = a.softcap > 0.f ? token_logprobs_bwd_kernel<T, true> : token_logprobs_bwd_kernel<T, false>;
    kernel<<<grid, kLpBwdThreads, 0, st>>>((const T*)a.logits, a.pitch, a.targets, (int)a.vocab, a.ignore_index, sh, a.stats, a.entropy,
                                           a.dlogp, a.dentropy, (T*)a.dlogits, a.dpitch, chunks);
    return check_launch("token_logprobs_bwd_kernel");
}

}  // namespace

int launch_token_logprobs_fwd(const TokenLogprobsArgs& a, int dtype, hipStream_t st) {
    if (a.softcap > 0.f) return dtype == MA_DTYPE_BF16 ? fwd<uint16_t, true>(a, st) : fwd<float, true>(a, st);
    return dtype == MA_DTYPE_BF16 ? fwd<uint16_t, false>(a, st) : fwd<float, false>(a, st);
}
int launch_token_logprobs_bwd(const TokenLogprobsArgs& a, int dtype, hipStream_t st) {
    return dtype == MA_DTYPE_BF16 ? bwd<uint16_t>(a, st) : bwd<float>(a, st);
}

}  // namespace ma
