// One AdamW step (decoupled weight decay) over many tensors in one launch, states in 32 or 8 bits, with the global
// norm of the gradients and clipping by it.
//
// Per element, with c the clip factor min(1, max_norm / (norm + 1e-6)), t the step after this one's increment:
//   g = c g;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit states: m and r = sqrt(v) are kept as e4m3 codes with one power-of-two scale per 128 consecutive elements, the
// smallest that brings the block's largest magnitude to 448 or less.  r and not v: its range is v's with half the
// exponent, and 17 binades below the block's maximum is what e4m3 holds.  Codes are rounded stochastically: with
// round-to-nearest a moment that changes by less than half a code a step (3 % at best; (1 - b2) of it changes) would
// never move.  The 16 random bits per rounding come from a hash of (seed, t, tensor, element), so a step is a function of
// its inputs.  A nonzero r is never rounded to zero: m / (0 + eps) would be a jump of any size.  Scaling by powers of two
// is exact, and the file is compiled without contraction or reassociation, square roots are rounded correctly (roots8), so
// that the states, in 32 and in 8 bits, are those of the formula in IEEE single precision, operation by operation.  A
// parameter's quotient alone is a product with the hardware's reciprocal, a last place off at most (step8).
#include <hip/hip_runtime.h>

#include "common.h"
#include "rowio.h"

namespace ma {

namespace {

constexpr int kAwThreads = 256;
constexpr int kAwChunk = kAwThreads * 8;          // elements per workgroup
constexpr int kAwBatch = 48;                      // tensors per launch: their descriptors travel as kernel arguments
constexpr int kNormGroups = 2048;                 // workgroups of a norm launch, one partial sum each

struct Batch {
    ma_adamw_tensor t[kAwBatch];
    int first[kAwBatch + 1];      // first chunk of every tensor, then the number of chunks
    int count, ordinal;           // ordinal: number of t[0] in the whole list (the hash goes by it)
};

// what a step's elements share, left in device memory by adamw_prepare_kernel
struct Scalars {
    float clip, decay, step_size, inv_root_bc, b1, one_b1, b2, one_b2, eps;
    uint32_t key;
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ int tensor_of(const Batch& b, int chunk) {
    int lo = 0, hi = b.count;     // first[lo] <= chunk < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (b.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// 8 elements from i, n of them inside the tensor (whole: all 8, and 16-byte aligned)
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t i, int n, bool whole, float* v) {
    if (whole) {
        ld8<T>(p + i, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? ld1<T>(p + i + e) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t i, int n, bool whole, const float* v) {
    if (whole) {
        st8<T>(p + i, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) st1<T>(p + i + e, v[e]);
    }
}

// ---- 8-bit states ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void load_codes(const uint8_t* p, int64_t i, int n, bool whole, uint32_t* w) {
    if (whole) {
        const uint2 q = *(const uint2*)(p + i);
        w[0] = q.x;
        w[1] = q.y;
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) w[e >> 2] |= (uint32_t)p[i + e] << (8 * (e & 3));
    }
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t i, int n, bool whole, const uint32_t* w) {
    if (whole) {
        *(uint2*)(p + i) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[i + e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
}
__device__ __forceinline__ void decode(const uint32_t* w, float scale, float* v) {
    v[0] = __builtin_amdgcn_cvt_f32_fp8(w[0], 0) * scale;
    v[1] = __builtin_amdgcn_cvt_f32_fp8(w[0], 1) * scale;
    v[2] = __builtin_amdgcn_cvt_f32_fp8(w[0], 2) * scale;
    v[3] = __builtin_amdgcn_cvt_f32_fp8(w[0], 3) * scale;
    v[4] = __builtin_amdgcn_cvt_f32_fp8(w[1], 0) * scale;
    v[5] = __builtin_amdgcn_cvt_f32_fp8(w[1], 1) * scale;
    v[6] = __builtin_amdgcn_cvt_f32_fp8(w[1], 2) * scale;
    v[7] = __builtin_amdgcn_cvt_f32_fp8(w[1], 3) * scale;
}
// exponent field of the block's scale from its largest magnitude: 2^k, the smallest with top <= 448 * 2^k = 1.75 * 2^(k + 8)
__device__ __forceinline__ int scale_field(float top) {
    if (top == 0.f) return 127;
    const int k = (int)((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8;
    return k < 1 ? 1 : k;
}
// the largest of a block's 128 magnitudes, 8 in each of 16 neighbouring lanes; NaN if one is
__device__ __forceinline__ float block_top(const float* v) {
    uint32_t m = 0;      // magnitudes compare as integers, NaN above all
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
    return __uint_as_float(m);
}
// Codes of y = |x| * 2^-k: the 20 bits below a code's last are rounded up with probability their value (r: 20 random
// bits).  From 2^-6 on a code is the float's own exponent and first three mantissa bits (less 120 << 3: e4m3's exponent
// starts at 2^-7); below, multiples of 2^-9.  The second kind costs twice as much and is rare (a code there is less than
// 3.5e-5 to 7e-5 of its block's largest), so a wave without one leaves it out.
template <bool POSITIVE>
__device__ __forceinline__ void encode(const float* v, const uint32_t* h, uint32_t* w, float& scale) {
    const float top = block_top(v);
    const bool finite = top < INFINITY;
    const int k = scale_field(top);
    scale = finite ? __uint_as_float((uint32_t)k << 23) : NAN;     // a block with an inf or a NaN is NaN from here on
    const float inv = __uint_as_float((uint32_t)(254 - k) << 23);
    float y[8];
    uint32_t c[8], r[8];
    float least = INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        y[e] = fabsf(v[e]) * inv;
        least = fminf(least, y[e]);
        r[e] = ((POSITIVE ? h[e] >> 12 : h[e] << 4) & 0xffff0u) | 8u;
        c[e] = (__float_as_uint(y[e]) + (r[e] - (960u << 20))) >> 20;
    }
    if (__any(least < 0.015625f)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t small = ((uint32_t)(y[e] * 536870912.f) + r[e]) >> 20;
            c[e] = y[e] >= 0.015625f ? c[e] : small;
            if (POSITIVE) c[e] = max(c[e], min(__float_as_uint(v[e]), 1u));
        }
    }
    w[0] = w[1] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (!POSITIVE) c[e] |= (__float_as_uint(v[e]) >> 24) & 0x80u;
        w[e >> 2] |= c[e] << (8 * (e & 3));
    }
    w[0] = finite ? w[0] : 0u;
    w[1] = finite ? w[1] : 0u;
}

// sqrt of 8 values, correctly rounded: the hardware's root (one step off at most) and one correction with its exact
// residual, taken one step lower, as the root's curvature lies below its tangent (without that 4^k (1 - 2^-24), whose root
// lies 2^-51 beside a midpoint, comes out a step high; with it every float of seven binades agrees with the fp64 root).  Residuals of values near the end of the exponent range would underflow, and infinity has none:
// those waves take the library's root.
__device__ __forceinline__ void roots8(const float* v, float* r) {
    uint32_t low = 0xffffffffu, high = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float s = __builtin_amdgcn_sqrtf(v[e]);
        const float half = 0.5f * __builtin_amdgcn_rcpf(fmaxf(s, 1e-30f));
        const float left = fmaf(-s, s, v[e]);
        r[e] = fmaf(fmaf(-fabsf(left), 0x1p-23f, left), half, s);
        low = min(low, __float_as_uint(v[e]) - 1u);          // (zero, whose residual is zero, wraps to the top)
        high = max(high, __float_as_uint(v[e]));
    }
    if (__any(low < 0x0f800000u || high >= 0x7f800000u)) {   // 2^-96
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = sqrtf(v[e]);
    }
}

// ---- the step ------------------------------------------------------------------------------------------------
template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void step8(const ma_adamw_tensor& t, int64_t i, uint32_t key, const Scalars& s) {
    const int64_t left = t.n - i;
    const int n = left < 0 ? 0 : left < 8 ? (int)left : 8;
    const bool whole = n == 8 && t.aligned;
    float p[8], g[8], m[8], v[8], r[8];
    P* param = (P*)t.param;
    float* master = (float*)t.master;
    load8<G>((const G*)t.grad, i, n, whole, g);
    if (MASTER) load8<float>(master, i, n, whole, p);
    else load8<P>(param, i, n, whole, p);
    const int64_t block = i >> 7;
    if (BITS == 32) {
        load8<float>((const float*)t.exp_avg, i, n, whole, m);
        load8<float>((const float*)t.exp_avg_sq, i, n, whole, v);
    } else {
        uint32_t wm[2], wr[2];
        load_codes((const uint8_t*)t.exp_avg, i, n, whole, wm);
        load_codes((const uint8_t*)t.exp_avg_sq, i, n, whole, wr);
        const float sm = n > 0 ? t.exp_avg_scale[block] : 0.f, sr = n > 0 ? t.exp_avg_sq_scale[block] : 0.f;
        decode(wm, sm, m);
        decode(wr, sr, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * v[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float ge = g[e] * s.clip;
        m[e] = m[e] * s.b1 + ge * s.one_b1;
        v[e] = v[e] * s.b2 + ge * ge * s.one_b2;
    }
    roots8(v, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // (the reciprocal is one step off at most, of an update that is a fraction of the weight)
        const float update = s.step_size * (m[e] * __builtin_amdgcn_rcpf(r[e] * s.inv_root_bc + s.eps));
        p[e] = p[e] * s.decay - update;
    }
    if (BITS == 32) {
        store8<float>((float*)t.exp_avg, i, n, whole, m);
        store8<float>((float*)t.exp_avg_sq, i, n, whole, v);
    } else {
        // every lane of a block's 16 takes part in its maximum; elements past the tensor's end count as 0
        uint32_t h[8], wm[2], wr[2];
        float sm, sr;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = mix((uint32_t)i * 0x9E3779B9u + (e * 0x9E3779B9u + key));
            if (e >= n) m[e] = r[e] = 0.f;
        }
        encode<false>(m, h, wm, sm);
        encode<true>(r, h, wr, sr);
        store_codes((uint8_t*)t.exp_avg, i, n, whole, wm);
        store_codes((uint8_t*)t.exp_avg_sq, i, n, whole, wr);
        if ((i & 127) == 0 && n > 0) {
            t.exp_avg_scale[block] = sm;
            t.exp_avg_sq_scale[block] = sr;
        }
    }
    if (MASTER) store8<float>(master, i, n, whole, p);
    store8<P>(param, i, n, whole, p);
}

// Eight elements a thread, every array read and written once in 8 to 32 bytes a lane: bound by memory.  189 M bf16
// parameters with fp32 masters and states 1.08 ms (5.3 GB, 4.9 TB/s; a large copy reaches 4.8), with 8-bit states 0.40 ms
// (1.9 GB, 4.8 TB/s), 671 M with 8-bit states 1.41 ms (6.8 GB, 4.8 TB/s).  With 8-bit states the arithmetic of the codes (two
// roundings, a square root and a hash an element) takes about as long as the bytes.
template <int BITS>
__global__ __launch_bounds__(kAwThreads) void adamw_kernel(const Batch b, const Scalars* __restrict__ scalars) {
    const int at = tensor_of(b, blockIdx.x);
    const ma_adamw_tensor t = b.t[at];
    const Scalars s = *scalars;
    const int64_t i = (int64_t)(blockIdx.x - b.first[at]) * kAwChunk + (int64_t)threadIdx.x * 8;
    const uint32_t key = s.key + (uint32_t)(b.ordinal + at) * 0xBB67AE85u;
    const bool pb = t.param_dtype == MA_DTYPE_BF16, gb = t.grad_dtype == MA_DTYPE_BF16;
    if (t.master) {
        if (gb) step8<uint16_t, uint16_t, true, BITS>(t, i, key, s);
        else step8<uint16_t, float, true, BITS>(t, i, key, s);
    } else if (pb) {
        if (gb) step8<uint16_t, uint16_t, false, BITS>(t, i, key, s);
        else step8<uint16_t, float, false, BITS>(t, i, key, s);
    } else {
        if (gb) step8<float, uint16_t, false, BITS>(t, i, key, s);
        else step8<float, float, false, BITS>(t, i, key, s);
    }
}

// ---- norm ------------------------------------------------------------------------------------------------------
// Sums of squares in fp64 (exact products of fp32 values), every partial sum over the same elements in every run.
template <typename G>
__device__ __forceinline__ double squares8(const ma_adamw_tensor& t, int64_t i) {
    const int64_t left = t.n - i;
    const int n = left < 0 ? 0 : left < 8 ? (int)left : 8;
    float g[8];
    load8<G>((const G*)t.grad, i, n, n == 8 && t.aligned, g);
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fma((double)g[e], (double)g[e], s);
    return s;
}
__device__ __forceinline__ double workgroup_sum(double x, double* box) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = x;
    __syncthreads();
    x = box[0];
    for (int w = 1; w < (int)blockDim.x / 64; ++w) x += box[w];
    return x;
}
// (sums in 64 bits, in an order that depends on the sizes alone; bound by reading the gradients)
__global__ __launch_bounds__(kAwThreads) void grad_norm_kernel(const Batch b, double* __restrict__ partial) {
    __shared__ double s_box[kAwThreads / 64];
    double sum = 0.0;
    for (int chunk = blockIdx.x; chunk < b.first[b.count]; chunk += gridDim.x) {
        const int at = tensor_of(b, chunk);
        const ma_adamw_tensor& t = b.t[at];
        const int64_t i = (int64_t)(chunk - b.first[at]) * kAwChunk + (int64_t)threadIdx.x * 8;
        sum += t.grad_dtype == MA_DTYPE_BF16 ? squares8<uint16_t>(t, i) : squares8<float>(t, i);
    }
    sum = workgroup_sum(sum, s_box);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// ---- scalars ---------------------------------------------------------------------------------------------------
struct Hyper {
    double lr, b1, b2, eps, weight_decay, max_norm;
    uint32_t seed;
    int want_norm;
};
// One workgroup: finishes the norm (partials of all norm launches) and, unless `scalars` is NULL, counts the step and leaves
// what its elements share.
__global__ __launch_bounds__(1024) void adamw_prepare_kernel(const double* __restrict__ partial, int n_partial, Hyper h,
                                                             const float* __restrict__ lr_device, const float* __restrict__ clip_in,
                                                             int64_t* __restrict__ step, float* __restrict__ norm_out,
                                                             float* __restrict__ clip_out, Scalars* __restrict__ scalars) {
    __shared__ double s_box[16];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 1024) sum += partial[i];
    sum = workgroup_sum(sum, s_box);
    if (threadIdx.x != 0) return;
    float clip = clip_in ? *clip_in : 1.f;
    if (h.want_norm) {
        const float norm = (float)sqrt(sum);
        if (norm_out) *norm_out = norm;
        double c = h.max_norm / ((double)norm + 1e-6);
        if (c > 1.0) c = 1.0;
        if (h.max_norm >= 0.0) clip = (float)c;
        if (clip_out) *clip_out = clip;
    }
    if (!scalars) return;
    const int64_t t = *step + 1;
    *step = t;
    const double lr = lr_device ? (double)*lr_device : h.lr;
    Scalars s;
    s.clip = clip;
    s.decay = (float)(1.0 - lr * h.weight_decay);
    s.step_size = (float)(lr / (1.0 - pow(h.b1, (double)t)));
    s.inv_root_bc = (float)(1.0 / sqrt(1.0 - pow(h.b2, (double)t)));
    s.b1 = (float)h.b1;
    s.one_b1 = (float)(1.0 - h.b1);
    s.b2 = (float)h.b2;
    s.one_b2 = (float)(1.0 - h.b2);
    s.eps = (float)h.eps;
    s.key = mix((uint32_t)t * 0x9E3779B9u + h.seed);
    *scalars = s;
}

// the next launch's tensors from list[at ..]; returns how many
int fill(Batch& b, const ma_adamw_tensor* list, int count, int at, int chunk) {
    b.count = count - at < kAwBatch ? count - at : kAwBatch;
    b.ordinal = at;
    int64_t first = 0;
    for (int i = 0; i < b.count; ++i) {
        ma_adamw_tensor& t = b.t[i];
        t = list[at + i];
        const uintptr_t any = (uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq | (uintptr_t)t.master;
        t.aligned = (any & 15) == 0;
        b.first[i] = (int)first;
        first += (list[at + i].n + chunk - 1) / chunk;
        if (first >= (int64_t)1 << 24) {     // a launch has fewer than 2^32 threads: this tensor opens the next one
            b.count = i;
            break;
        }
        b.first[i + 1] = (int)first;
    }
    return b.count;
}

}  // namespace

// A launch ends with its 48th tensor or before the one that would bring it to 2^24 workgroups; of the latter kind there are
// at most 2 * 2^37 / (2^24 * kAwChunk) + 1 <= 9 with MA_ADAMW_MAX_ELEMENTS in all.
size_t adamw_workspace_bytes(int count) { return 256 + (size_t)(count / kAwBatch + 16) * kNormGroups * sizeof(double); }
static_assert(MA_ADAMW_MAX_ELEMENTS / kAwChunk / ((int64_t)1 << 24) <= 4, "workspace of the norm's launches");
static_assert(MA_ADAMW_MAX_TENSOR / kAwChunk < ((int64_t)1 << 24), "one tensor fits a launch");
static_assert(sizeof(Batch) + 16 <= 4096, "kernel arguments");

int launch_grad_norm(const ma_adamw_tensor* list, int count, double* partial, int* n_partial, hipStream_t st) {
    Batch b;
    for (int at = 0; at < count; at += b.count) {
        fill(b, list, count, at, kAwChunk);
        const int chunks = b.first[b.count], grid = chunks < kNormGroups ? chunks : kNormGroups;
        if (grid == 0) continue;
        grad_norm_kernel<<<grid, kAwThreads, 0, st>>>(b, partial + *n_partial);
        *n_partial += grid;
        const int rc = check_launch("grad_norm_kernel");
        if (rc) return rc;
    }
    return MA_OK;
}

int launch_adamw(const AdamwArgs& a, hipStream_t st) {
    Scalars* scalars = (Scalars*)a.ws;
    double* partial = (double*)((char*)a.ws + 256);
    int n_partial = 0;
    if (a.want_norm) {
        const int rc = launch_grad_norm(a.list, a.count, partial, &n_partial, st);
        if (rc) return rc;
    }
    const Hyper h = {a.lr, a.b1, a.b2, a.eps, a.weight_decay, a.max_norm, a.seed, a.want_norm};
    adamw_prepare_kernel<<<1, 1024, 0, st>>>(partial, n_partial, h, a.lr_device, a.clip_in, a.step, a.norm_out, a.clip_out,
                                             a.step ? scalars : nullptr);
    int rc = check_launch("adamw_prepare_kernel");
    if (rc || !a.step) return rc;
    Batch b;
    for (int at = 0; at < a.count; at += b.count) {
        fill(b, a.list, a.count, at, kAwChunk);
        const int chunks = b.first[b.count];
        if (chunks == 0) continue;
        if (a.state_bits == 8) adamw_kernel<8><<<chunks, kAwThreads, 0, st>>>(b, scalars);
        else adamw_kernel<32><<<chunks, kAwThreads, 0, st>>>(b, scalars);
        rc = check_launch("adamw_kernel");
        if (rc) return rc;
    }
    return MA_OK;
}

}  // namespace ma
