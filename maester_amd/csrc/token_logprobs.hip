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
#include "rowio.h"

#pragma clang fp reassociate(off)

namespace ma {

namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWaves = kLpThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float ld1(const T* p);
template <>
__device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ld1<uint16_t>(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
template <typename T>
__device__ __forceinline__ void st1(T* p, float v);
template <>
__device__ __forceinline__ void st1<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void st1<uint16_t>(uint16_t* p, float v) {
    const __bf16 b = (__bf16)v;
    *p = *(const uint16_t*)&b;
}

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
};

struct Shape {
    float cap, inv_cap, inv_temp;
};
template <bool CAP>
__device__ __forceinline__ float capped(float x, const Shape& s) { return CAP ? s.cap * tanhf(x * s.inv_cap) : x; }

// running maximum (in units of the capped logits), sum of exponentials and of (y - m) exp(y - m)
struct Stats {
    float m, l, s;
};
__device__ __forceinline__ Stats merged(const Stats& a, const Stats& b, float inv_temp) {
    const float m = fmaxf(a.m, b.m);
    const float base = m == -INFINITY ? 0.f : m;
    const float da = fmaxf((a.m - base) * inv_temp, -1e30f), db = fmaxf((b.m - base) * inv_temp, -1e30f);
    const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    return {m, a.l * fa + b.l * fb, fa * (a.s + da * a.l) + fb * (b.s + db * b.l)};
}
// 8 capped logits.  A NaN among them (or +inf, as inf - inf) makes l NaN, and with it every output.
__device__ __forceinline__ void fold8(const float* y, float inv_temp, Stats& t) {
    float vm = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    vm = fmaxf(vm, fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    const float m = fmaxf(t.m, vm);
    const float base = m == -INFINITY ? 0.f : m;    // nothing but -inf so far: l and s stay 0
    const float dt = fmaxf((t.m - base) * inv_temp, -1e30f);
    const float f = __builtin_amdgcn_exp2f(dt * kLog2e);
    float l = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = (y[i] - base) * inv_temp;
        const float e = __builtin_amdgcn_exp2f(d * kLog2e);
        l += e;
        s = fmaf(fmaxf(d, -1e30f), e, s);           // 0 * -inf would be NaN: a term of weight 0 adds nothing
    }
    t.s = f * (t.s + dt * t.l) + s;
    t.l = t.l * f + l;
    t.m = m;
}

// the statistics of the whole workgroup, in every thread; box: one slot per wave
__device__ __forceinline__ Stats workgroup_stats(Stats t, float inv_temp, Stats* box) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const Stats o = {__shfl_xor(t.m, off, 64), __shfl_xor(t.l, off, 64), __shfl_xor(t.s, off, 64)};
        t = merged(t, o, inv_temp);
    }
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = t;
    __syncthreads();
    t = box[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) t = merged(t, box[w], inv_temp);
    return t;
}

// ---- order of the alternatives ------------------------------------------------------------------------
// A candidate is one 64-bit key, unique in its row: the logit's bits made monotone above, the complement
// of the index below, so that larger is better and equal logits go to the lower index.  -0 equals +0,
// NaN ranks with -inf.  0 is no key.
__device__ __forceinline__ uint32_t ordered(float x) {
    x = x == x ? x + 0.f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
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

template <typename T, bool CAP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_fwd_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                        const int64_t* __restrict__ targets, int vocab,
                                                                        int64_t ignore_index, Shape sh, int top_k,
                                                                        float* __restrict__ logp_out, float* __restrict__ entropy_out,
                                                                        float* __restrict__ stats_out, int64_t* __restrict__ top_ids,
                                                                        float* __restrict__ top_logp) {
    __shared__ Stats s_box[kLpWaves];
    __shared__ uint64_t s_key[kLpWaves];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Row<T> r(logits + row * pitch, vocab);
    const int64_t target = targets[row];
    const bool valid = target != ignore_index && target >= 0 && target < vocab;

    Stats t = {-INFINITY, 0.f, 0.f};
    for (int g = tid; g < r.groups; g += kLpThreads) {
        float v[8];
        r.load(g, v);
        if (CAP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = capped<CAP>(v[i], sh);
        }
        fold8(v, sh.inv_temp, t);
    }
    t = workgroup_stats(t, sh.inv_temp, s_box);
    const float log_l = log2f(t.l) * kLn2;
    if (tid == 0) {
        const float y = valid ? capped<CAP>(ld1<T>(r.p + target), sh) : 0.f;
        logp_out[row] = valid ? (y - t.m) * sh.inv_temp - log_l : 0.f;
        entropy_out[row] = valid ? log_l - t.s / t.l : 0.f;
        if (stats_out) *(float2*)(stats_out + 2 * row) = make_float2(t.m, log_l);
    }
    // the alternatives, best first: each round takes the largest key below the last round's
    uint64_t last = ~0ull;
    for (int k = 0; k < top_k; ++k) {
        uint64_t best = 0;
        for (int g = tid; g < r.groups; g += kLpThreads) {
            float v[8];
            r.load(g, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = r.first(g) + i;
                const uint64_t key = key_of(v[i], j);
                if (j >= 0 && j < vocab && key < last && key > best) best = key;
            }
        }
        best = wave_max_key(best);
        __syncthreads();
        if ((tid & 63) == 0) s_key[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < kLpWaves; ++w) best = s_key[w] > best ? s_key[w] : best;
        last = best;
        if (tid == 0) {
            top_ids[row * top_k + k] = (int64_t)(int)~(uint32_t)best;
            top_logp[row * top_k + k] = (capped<CAP>(unordered((uint32_t)(best >> 32)), sh) - t.m) * sh.inv_temp - log_l;
        }
    }
}

// ---- gradient -------------------------------------------------------------------------------------------
constexpr int kLpBwdThreads = 256, kLpBwdGroups = 4;      // groups of 8 per thread
template <typename T, bool CAP>
__global__ __launch_bounds__(kLpBwdThreads) void token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t pitch,
                                                                           const int64_t* __restrict__ targets, int vocab,
                                                                           int64_t ignore_index, Shape sh,
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
                const float th = CAP ? tanhf(v[i] * sh.inv_cap) : 0.f;
                const float lp = fmaf((CAP ? sh.cap * th : v[i]) - top, sh.inv_temp, -log_l);
                const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
                d[i] = -p * fmaf(b, fmaxf(lp, -1e30f) + h, a);
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

// workgroups per row of the gradient kernel, for a row that starts anywhere
int token_logprobs_bwd_chunks(int64_t vocab) {
    const int per = kLpBwdThreads * kLpBwdGroups;
    return (int)(((vocab + 14) / 8 + per - 1) / per);
}

namespace {

Shape shape_of(float softcap, float temperature) {
    return {softcap, softcap > 0.f ? 1.f / softcap : 0.f, 1.f / temperature};
}

template <typename T>
int fwd(const TokenLogprobsArgs& a, hipStream_t st) {
    const Shape sh = shape_of(a.softcap, a.temperature);
    const dim3 grid((unsigned)a.rows);
    auto kernel = a.softcap > 0.f ? token_logprobs_fwd_kernel<T, true> : token_logprobs_fwd_kernel<T, false>;
    kernel<<<grid, kLpThreads, 0, st>>>((const T*)a.logits, a.pitch, a.targets, (int)a.vocab, a.ignore_index, sh, a.top_k, a.logp,
                                        a.entropy, a.stats, a.top_ids, a.top_logp);
    return check_launch("token_logprobs_fwd_kernel");
}
template <typename T>
int bwd(const TokenLogprobsArgs& a, hipStream_t st) {
    const Shape sh = shape_of(a.softcap, a.temperature);
    const int chunks = token_logprobs_bwd_chunks(a.vocab);
    const dim3 grid((unsigned)(a.rows * chunks));
    auto kernel = a.softcap > 0.f ? token_logprobs_bwd_kernel<T, true> : token_logprobs_bwd_kernel<T, false>;
    kernel<<<grid, kLpBwdThreads, 0, st>>>((const T*)a.logits, a.pitch, a.targets, (int)a.vocab, a.ignore_index, sh, a.stats, a.entropy,
                                           a.dlogp, a.dentropy, (T*)a.dlogits, a.dpitch, chunks);
    return check_launch("token_logprobs_bwd_kernel");
}

}  // namespace

int launch_token_logprobs_fwd(const TokenLogprobsArgs& a, int dtype, hipStream_t st) {
    return dtype == MA_DTYPE_BF16 ? fwd<uint16_t>(a, st) : fwd<float>(a, st);
}
int launch_token_logprobs_bwd(const TokenLogprobsArgs& a, int dtype, hipStream_t st) {
    return dtype == MA_DTYPE_BF16 ? bwd<uint16_t>(a, st) : bwd<float>(a, st);
}

}  // namespace ma
