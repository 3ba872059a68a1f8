// What the two forms of the token log-probabilities share: the softmax statistics of a row and how they join.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

// (y - m) has to be formed as it stands: distributed over the factors that follow it would overflow
#pragma clang fp reassociate(off)

namespace ma {

constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLn2 = 0.6931471805599453f;

struct LpShape {
    float cap, inv_cap, inv_temp;
};
inline LpShape lp_shape(float softcap, float temperature) { return {softcap, softcap > 0.f ? 1.f / softcap : 0.f, 1.f / temperature}; }
// tanh: its series up to 0.35 (six terms; the seventh is below 2^-26 of the value there), 1 - 2 / (exp(2 |z|) + 1) above
// (off by 2^-23 at most); 18 instructions and no branch.
__device__ __forceinline__ float lp_tanh(float z) {
    const float a = fabsf(z), q = z * z;
    const float big = fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a * (2.f * kLpLog2e)) + 1.f), 1.f);
    float t = fmaf(q, -1382.f / 155925.f, 62.f / 2835.f);
    t = fmaf(q, t, -17.f / 315.f);
    t = fmaf(q, t, 2.f / 15.f);
    t = fmaf(q, t, -1.f / 3.f);
    t = fmaf(a * q, t, a);
    return copysignf(a < 0.35f ? t : big, z);
}
template <bool CAP>
__device__ __forceinline__ float lp_capped(float x, const LpShape& s) { return CAP ? s.cap * lp_tanh(x * s.inv_cap) : x; }

// running maximum (in units of the capped logits), sum of exp((y - m) / T) and of (y - m) / T * exp((y - m) / T)
struct LpStats {
    float m, l, s;
};
__device__ __forceinline__ LpStats lp_merged(const LpStats& a, const LpStats& b, float inv_temp) {
    const float m = fmaxf(a.m, b.m);
    const float base = m == -INFINITY ? 0.f : m;
    const float da = fmaxf((a.m - base) * inv_temp, -1e30f), db = fmaxf((b.m - base) * inv_temp, -1e30f);
    const float fa = __builtin_amdgcn_exp2f(da * kLpLog2e), fb = __builtin_amdgcn_exp2f(db * kLpLog2e);
    return {m, a.l * fa + b.l * fb, fa * (a.s + da * a.l) + fb * (b.s + db * b.l)};
}
// what (m, l, s) are relative to a larger maximum m
__device__ __forceinline__ void lp_rescale(LpStats& t, float m, float inv_temp) {
    const float base = m == -INFINITY ? 0.f : m;
    const float d = fmaxf((t.m - base) * inv_temp, -1e30f);
    const float f = __builtin_amdgcn_exp2f(d * kLpLog2e);
    t.s = f * (t.s + d * t.l);
    t.l = t.l * f;
    t.m = m;
}
// one capped logit at or below t.m
__device__ __forceinline__ void lp_add(LpStats& t, float y, float inv_temp) {
    const float base = t.m == -INFINITY ? 0.f : t.m;    // nothing but -inf so far: l and s stay 0
    const float d = (y - base) * inv_temp;
    const float e = __builtin_amdgcn_exp2f(d * kLpLog2e);
    t.l += e;
    t.s = fmaf(fmaxf(d, -1e30f), e, t.s);               // 0 * -inf would be NaN: a term of weight 0 adds nothing
}
// N capped logits.  A NaN among them (or +inf, as inf - inf) makes l NaN, and with it every output.
template <int N>
__device__ __forceinline__ void lp_fold(const float* y, float inv_temp, LpStats& t) {
    float m = t.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, y[i]);
    lp_rescale(t, m, inv_temp);
    LpStats one = {m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) lp_add(one, y[i], inv_temp);
    t.l += one.l;
    t.s += one.s;
}
// The same in units of log2 for logits that are sums of products: scale = log2 e / T, m holds the reference max(y) scale
// as it was rounded, s is sum x 2^x with x = y scale - m, one multiply-add.  All terms have to refer to the very number
// m: a reference rounded anew at every use would weigh the parts of a row 2^-24 |m| apart, which showed in the entropy
// (3e-6 relative, ten times an fp32 softmax's).  Logits whose product with the scale overflows come out NaN.
__device__ __forceinline__ LpStats lp2_merged(const LpStats& a, const LpStats& b) {
    const float m = fmaxf(a.m, b.m);
    const float base = m == -INFINITY ? 0.f : m;
    const float da = fmaxf(a.m - base, -1e30f), db = fmaxf(b.m - base, -1e30f);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    return {m, a.l * fa + b.l * fb, fa * (a.s + da * a.l) + fb * (b.s + db * b.l)};
}
template <int N>
__device__ __forceinline__ void lp2_fold(const float* y, float scale, LpStats& t) {
    float top = y[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, y[i]);
    const float m = fmaxf(t.m, top * scale);
    const float base = m == -INFINITY ? 0.f : m;
    const float d = fmaxf(t.m - base, -1e30f);
    const float f = __builtin_amdgcn_exp2f(d);
    float l = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = fmaf(y[i], scale, -base);
        const float e = __builtin_amdgcn_exp2f(x);
        l += e;
        s = fmaf(fmaxf(x, -1e30f), e, s);
    }
    t.s = f * (t.s + d * t.l) + s;
    t.l = t.l * f + l;
    t.m = m;
}
__device__ __forceinline__ LpStats lp_shuffled(const LpStats& t, int off) {
    return {__shfl_xor(t.m, off, 64), __shfl_xor(t.l, off, 64), __shfl_xor(t.s, off, 64)};
}

}  // namespace ma
