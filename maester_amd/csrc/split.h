// fp32 products on the bf16 matrix instructions.  An fp32 value is the exact sum of three bf16 values, x = h + m + l: its first
// 8 mantissa bits, cut off; the next 8, rounded to the nearest; what is left.  |m| <= 2^-7 |x| and |l| <= 2^-16 |x|, l of either
// sign.  Of the nine products of two such sums six are formed, h h + m m, h m + m h and h l + l h; what is left out, m l + l m +
// l l, is at most 2^-22 of the product and 0 on average.  Products are exact and summed in fp32, as with the fp32 instructions.
// (With m cut off too, l has the sign of x and is twice as large: up to 2^-21 were left out, 2^-24.6 on average and always towards
// zero.  With h rounded as well 2^-23 are left out, but fp32's largest magnitudes have no h, unless it is clamped: 3 % of the time.)
//
// v_mfma_f32_32x32x16_bf16 takes 8 values a lane: the four values of an fp32 fragment fill it with two of the six products,
// so a fragment pair is three instructions (96 cycles) where v_mfma_f32_32x32x2_f32 needs four of 64 (256), and the sums
// run over 8 indices at a time instead of 2.  Cutting a fragment up costs some 25 vector operations, done while the matrix
// unit works on earlier ones.  Measured (us, before and after): 2048 x 32000, 4096 rows, statistics 3821 -> 2379 (226 TFLOP/s);
// 640 x 32003, 300 rows, statistics and gradients 520 -> 407, their error against 64 bits 9.2e-7 -> 7.3e-7 of their size.
//
// Magnitudes up to fp32's largest have parts (a product above 2^128 (1 - 2^-17) may overflow, as h + m may round up to 2^128).
// An infinity has none: it makes NaN of the sums that it takes part in.  Parts below 2^-126 may count as zero: values below
// 2^-103 may lose their last bits, below 2^-110 their third part, below 2^-118 the second.
#pragma once

#include "mfma.h"

namespace ma {

struct SplitA {
    u32x4 hm, hl;
};
struct SplitB {
    u32x4 hm, mh, lh;
};

__device__ __forceinline__ uint32_t nearest_pair(float x0, float x1) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 p = __builtin_convertvector(f32x2{x0, x1}, bf16x2);
    return *(const uint32_t*)&p;
}
__device__ __forceinline__ void split_pair(uint32_t x0, uint32_t x1, uint32_t& h, uint32_t& m, uint32_t& l) {
    constexpr uint32_t kHigh = 0xffff0000u, kHalves = 0x07060302u;       // the upper halves of two words
    const float r0 = __uint_as_float(x0) - __uint_as_float(x0 & kHigh), r1 = __uint_as_float(x1) - __uint_as_float(x1 & kHigh);
    h = __builtin_amdgcn_perm(x1, x0, kHalves);
    m = nearest_pair(r0, r1);
    // (8 bits: the upper halves are all there is)
    const float s0 = r0 - __uint_as_float(m << 16), s1 = r1 - __uint_as_float(m & kHigh);
    l = __builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), kHalves);
}
__device__ __forceinline__ SplitA split_a(u32x4 x) {
    uint32_t h[2], m[2], l[2];
    split_pair(x[0], x[1], h[0], m[0], l[0]);
    split_pair(x[2], x[3], h[1], m[1], l[1]);
    return {{h[0], h[1], m[0], m[1]}, {h[0], h[1], l[0], l[1]}};
}
__device__ __forceinline__ SplitB split_b(u32x4 x) {
    uint32_t h[2], m[2], l[2];
    split_pair(x[0], x[1], h[0], m[0], l[0]);
    split_pair(x[2], x[3], h[1], m[1], l[1]);
    return {{h[0], h[1], m[0], m[1]}, {m[0], m[1], h[0], h[1]}, {l[0], l[1], h[0], h[1]}};
}
__device__ __forceinline__ f32x16 mac_split(const SplitA& a, const SplitB& b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)&a.hm, *(const bf16x8*)&b.hm, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)&a.hm, *(const bf16x8*)&b.mh, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)&a.hl, *(const bf16x8*)&b.lh, c, 0, 0, 0);
}

// The fragments of a wave's MT x NT tiles as the matrix instructions take them.  bf16: the fragments as they are.  fp32: split,
// both of A's buffers and the two columns of B that are in use.
template <typename T, int MT, int NT>
struct Fragments {
    u32x4 a[2][MT], b[2][NT];
    static constexpr bool kSplit = sizeof(T) == 4;
    SplitA sa[2][kSplit ? MT : 1];
    SplitB sb[2];

    __device__ __forceinline__ static constexpr int column(int buf, int j) { return (j + (NT & 1) * buf) & 1; }
    // after the first fragments have been read
    __device__ __forceinline__ void begin() {
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < MT; ++i) sa[0][i] = split_a(a[0][i]);
            sb[0] = split_b(b[0][0]);
        }
    }
    // product STEP of MT * NT of buffer `buf` and what is to be cut up in its shadow: B's next column in the first product
    // of a column, the next fragments (read during the first half) in the second half
    template <int STEP>
    __device__ __forceinline__ void product(int buf, f32x16 (&acc)[MT][NT]) {
        constexpr int i = STEP % MT, j = STEP / MT, P = MT * NT, H = P / 2;
        if constexpr (kSplit) {
            acc[i][j] = mac_split(sa[buf][i], sb[column(buf, j)], acc[i][j]);
            if constexpr (i == 0 && j + 1 < NT) sb[column(buf, j + 1)] = split_b(b[buf][j + 1]);
            if constexpr (STEP >= H) {
                static_for<(STEP - H) * MT / (P - H), (STEP - H + 1) * MT / (P - H)>([&](auto k) {
                    sa[buf ^ 1][decltype(k)::value] = split_a(a[buf ^ 1][decltype(k)::value]);
                });
                if constexpr (STEP == P - 1) sb[column(buf ^ 1, 0)] = split_b(b[buf ^ 1][0]);
            }
        } else {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)&a[buf][i], *(const bf16x8*)&b[buf][j], acc[i][j], 0, 0, 0);
        }
    }
};

}  // namespace ma
