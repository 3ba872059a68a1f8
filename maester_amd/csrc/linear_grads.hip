// The two products that end the backward of linear_token_logprobs, from the gradient x [rows, vocab] of the logits:
//   de [rows, K] = x c        (contraction over the vocabulary, cut into ranges whose fp32 sums are joined afterwards)
//   dc [vocab, K] = x^T e     (contraction over the rows)
// with c [vocab, K] and e [rows, K] as they lie in memory: no transposed copies.  Both are computed transposed, M = K and
// N = rows or vocabulary, so that a lane ends up with runs of four of an output row.
//
// The loop is that of linear_logprobs.hip (256 x 256 tiles, four waves of 128 x 128, five LDS slots of one operand's step,
// counted waits, one barrier a step); what differs is that an operand may have the contraction along its ROWS: c and e
// always, x for dc.  A step of such an operand is 64 (fp32: 32) rows of 256 columns, and a fragment, which wants
// consecutive contraction indices in a lane, is read through ds_read_b64_tr_b16 (four rows by sixteen columns exchanged
// among 16 lanes; fp32: four single words).  Its 16-byte chunks are stored exchanged, chunk c of row r in place c ^ 4 (r % 4)
// (fp32: c ^ 8 (r / 4 % 2)), so that the rows that are read together lie in different banks.
//
// What bounds it: the matrix units (70 to 77 % busy in bf16, at the chip's power limit), below some 100 rows the bytes of c
// and dc.  2560 x 262208 in bf16: 2047 rows de 2.16 ms, dc 2.22 (1.27 and 1.24 PFLOP/s; a large library product that reads its
// operands along their rows reaches 1.38), 8 rows 0.26 ms each (5.2 TB/s).
//
// Workgroups are persistent, one a compute unit, and walk a list of units (N block, M tile, range) in an order in which the
// 32 of an XCD are on 8 N blocks x 4 M tiles of one range at a time and share both operands through its L2.
#include <hip/hip_runtime.h>

#include "common.h"
#include "mfma.h"
#include "split.h"

namespace ma {

namespace {

constexpr int kSlot = 32 * 1024;         // one operand's step
constexpr int kSlots = 5;

struct GradArgs {
    const char *a, *x;                   // a: c or e, rows of K
    int64_t a_stride, x_stride;          // bytes between rows
    int m, n, contraction;               // K; rows or vocab; vocab or rows
    int m_tiles, n_blocks, ranges, range_steps, units;
    void* out;
    int64_t out_stride, range_stride;    // elements between rows, between the ranges' results
};

enum Output { kInput, kStored, kAdded };      // in the operands' type; fp32, stored; fp32, added to what is there

// One operand: how its step lies in a slot, which bytes a lane loads, where a lane reads its fragments.
// ROWS: the contraction runs along its rows; otherwise its rows are those of the tile, 128 bytes of contraction a step.
template <typename T, bool ROWS, int EDGE>
struct Operand {
    static constexpr int kElt = sizeof(T), kDeep = 128 / kElt;               // contraction indices per step
    static constexpr int kPitch = ROWS ? EDGE * kElt : 128;                  // bytes of a slot's row
    static constexpr int kRunRows = 1024 / kPitch, kChunks = kPitch / 16;
    static constexpr int kRuns = EDGE / 32, kBlocks = EDGE / 64;             // 1 KB loads of a wave and step, 32-blocks of a wave
    static constexpr int kOffs = ROWS ? kBlocks : 4;
    uint32_t off[kRuns], lane_off[kOffs];
    int chunk[2];                        // fetched by this lane in its even / odd runs
    // load side: next step
    uint64_t at;
    int64_t stride;
    uint32_t lds, past[2];
    int left, width;                     // contraction indices of the unit still to load; ROWS: bytes of a row inside the matrix
    int rows;                            // otherwise: rows of the tile inside the matrix
    u32x4 rsrc;

    static __device__ __forceinline__ int swap_of(int row) {
        if (!ROWS) return (row >> 1) & 7;
        return kElt == 2 ? (row & 3) << 2 : ((row >> 2) & 1) << 3;
    }
    __device__ __forceinline__ void init(int64_t row_stride, int w, int lane, int wave_at) {
        stride = row_stride;
#pragma unroll
        for (int p = 0; p < kRuns; ++p) {
            const int row = (w + 4 * p) * kRunRows + lane / kChunks, c = (lane % kChunks) ^ swap_of(row);
            off[p] = (uint32_t)row * (uint32_t)row_stride + c * 16;
            if (p < 2) chunk[p] = c;     // (the exchange repeats every second run of a wave, or sooner)
        }
        const int r = lane & 31, hh = lane >> 5, i = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
        for (int q = 0; q < kOffs; ++q) {
            if (!ROWS) lane_off[q] = (wave_at + r) * 128 + (((2 * q + hh) ^ swap_of(r)) << 4);                 // q: 32 bytes of the step
            else if (kElt == 2)                                                                                // q: 32 columns
                lane_off[q] = (8 * hh + (i >> 2)) * kPitch + (((wave_at / 32 + q) ^ (i >> 2)) << 6) + (g << 5) + ((i & 3) << 3);
            else lane_off[q] = 4 * hh * kPitch + (((wave_at / 4 + 8 * q + r / 4) ^ (hh << 3)) << 4) + (r & 3) * 4;
        }
    }
    // fragment of 32 rows / columns (block) and 32 bytes (16 or 8 indices) of the contraction (sub)
    template <int BLOCK, int SUB>
    __device__ __forceinline__ u32x4 read(lds_ptr slot) const {
        if constexpr (!ROWS) {
            return *(MA_LDS u32x4*)(slot + lane_off[SUB] + BLOCK * 32 * 128);
        } else if constexpr (kElt == 2) {
            const lds_ptr at_ = slot + lane_off[BLOCK] + SUB * 16 * kPitch;
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((MA_LDS bf16x4*)at_);
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((MA_LDS bf16x4*)(at_ + 4 * kPitch));
            const bf16x8 f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return *(const u32x4*)&f;
        } else {
            const lds_ptr at_ = slot + lane_off[BLOCK] + SUB * 8 * kPitch;
            u32x4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = *(MA_LDS uint32_t*)(at_ + j * kPitch);
            return f;
        }
    }
    // a unit: `count` contraction indices from `first`, tile columns / rows from `edge` of `edges`
    __device__ __forceinline__ void open(const char* base, int64_t first, int count, int edge, int edges) {
        left = count;
        if (ROWS) {
            at = (uint64_t)base + (uint64_t)(first * stride) + (uint64_t)edge * kElt;
            width = (min(EDGE, edges - edge) * kElt + 15) & ~15;         // (whole chunks: rows are padded to them)
        } else {
            at = (uint64_t)base + (uint64_t)((int64_t)edge * stride) + (uint64_t)first * kElt;
            rows = min(EDGE, edges - edge);
        }
    }
    // count 0 (no unit left): nothing is in range
    __device__ __forceinline__ void begin(uint32_t lds_at) {
        uint32_t bytes;
        if (ROWS) {
            bytes = left > 0 ? (uint32_t)((min(kDeep, left) - 1) * stride) + width : 0u;
            past[0] = chunk[0] * 16 < width ? 0u : 0x80000000u;
            past[1] = chunk[1] * 16 < width ? 0u : 0x80000000u;
        } else {
            bytes = left > 0 ? (uint32_t)((rows - 1) * stride) + ((min(kDeep, left) * kElt + 15) & ~15) : 0u;
            past[0] = past[1] = chunk[0] * 16 < left * kElt ? 0u : 0x80000000u;
        }
        rsrc = uniform_rsrc(at, bytes);
        lds = __builtin_amdgcn_readfirstlane(lds_at);
    }
    template <int P>
    __device__ __forceinline__ void load() const {
        buffer_to_lds_run_at<P * 4096>(rsrc, off[P] | past[ROWS && kElt == 4 ? P & 1 : 0], lds);
    }
    // true: the unit has no steps left
    __device__ __forceinline__ bool advance() {
        at += ROWS ? (uint64_t)(kDeep * stride) : 128u;
        left -= kDeep;
        return left <= 0;
    }
};

template <typename T, bool X_ROWS, Output OUT, int BM, int BN>
__global__ __launch_bounds__(256, 1) void linear_grads_kernel(const GradArgs a) {
    extern __shared__ __align__(16) char smem_raw[];
    const lds_ptr smem = (lds_ptr)smem_raw;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hh = lane >> 5, wm = (w & 1) * (BM / 2), wn = (w >> 1) * (BN / 2);
    constexpr int kDeep = 128 / sizeof(T), MT = BM / 64, NT = BN / 64, kA = BM / 32, kX = BN / 32;

    // this workgroup's units: XCD x has the x-th eighth of the list, its workgroups take turns in it
    const int xcd = blockIdx.x % kXcds, mine = blockIdx.x / kXcds, team = gridDim.x / kXcds;
    const int u0 = (int)((int64_t)a.units * xcd / kXcds), u1 = (int)((int64_t)a.units * (xcd + 1) / kXcds);
    const int count = u0 + mine < u1 ? (u1 - u0 - mine + team - 1) / team : 0;
    if (count == 0) return;
    // unit -> (range, N block, M tile): ranges outermost, then groups of 8 N blocks, in a group M tiles
    auto unit = [&](int t, int& range, int& nb, int& mt) {
        const int u = u0 + mine + t * team, per = a.n_blocks * a.m_tiles;
        const int rg = u / per, in = u - rg * per, group = in / (8 * a.m_tiles), at = in - group * 8 * a.m_tiles;
        const int height = min(8, a.n_blocks - group * 8);
        range = __builtin_amdgcn_readfirstlane(rg);
        mt = __builtin_amdgcn_readfirstlane(at / height);
        nb = __builtin_amdgcn_readfirstlane(group * 8 + at % height);
    };
    auto indices = [&](int range, int& first) {       // contraction indices of a range
        first = range * a.range_steps * kDeep;
        return min(a.range_steps * kDeep, a.contraction - first);
    };

    Operand<T, true, BM> ca;
    Operand<T, X_ROWS, BN> cx;
    ca.init(a.a_stride, w, lane, wm);
    cx.init(a.x_stride, w, lane, wn);
    int a_unit = 0, x_unit = 0;
    auto open_a = [&]() {
        int range = 0, nb = 0, mt = 0, first = 0;
        if (a_unit < count) unit(a_unit, range, nb, mt);
        const int n = a_unit < count ? indices(range, first) : 0;
        ca.open(a.a, first, n, mt * BM, a.m);
    };
    auto open_x = [&]() {
        int range = 0, nb = 0, mt = 0, first = 0;
        if (x_unit < count) unit(x_unit, range, nb, mt);
        const int n = x_unit < count ? indices(range, first) : 0;
        cx.open(a.x, first, n, nb * BN, a.n);
    };
    auto next_a = [&]() {
        if (ca.advance()) {
            ++a_unit;
            open_a();
        }
    };
    auto next_x = [&]() {
        if (cx.advance()) {
            ++x_unit;
            open_x();
        }
    };
    open_a();
    open_x();

    const uint32_t lds0 = lds_addr(smem) + w * 1024;
    Fragments<T, MT, NT> frags;
    f32x16 acc[MT][NT];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x16(0.f);
    };
    auto read_one = [&](int buf, lds_ptr slot_a, lds_ptr slot_x, auto sub, auto which) {
        constexpr int SUB = decltype(sub)::value, i = decltype(which)::value;
        if constexpr (i < MT) frags.a[buf][i] = ca.template read<i, SUB>(slot_a);
        else frags.b[buf][i - MT] = cx.template read<i - MT, SUB>(slot_x);
    };
    auto load_run = [&](auto run) {                   // 0 .. kA - 1: a, the others x
        constexpr int p = decltype(run)::value;
        if constexpr (p < kA) ca.template load<p>();
        else cx.template load<p - kA>();
    };
    // products of 32 bytes of the contraction, between them the reads of the next 32 (sub SUB of the given slots) and loads
    // FIRST .. LAST - 1
    auto part = [&](int buf, lds_ptr slot_a, lds_ptr slot_x, auto sub, auto first, auto last) {
        constexpr int P = MT * NT, H = P / 2, R = MT + NT, W0 = decltype(first)::value, W = decltype(last)::value - W0;
        static_for<0, P>([&](auto step) {
            constexpr int i = decltype(step)::value;
            if constexpr (i < H) static_for<i * R / H, (i + 1) * R / H>([&](auto k) { read_one(buf ^ 1, slot_a, slot_x, sub, k); });
            else static_for<W0 + (i - H) * W / (P - H), W0 + (i - H + 1) * W / (P - H)>([&](auto k) { load_run(k); });
            frags.template product<i>(buf, acc);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    const auto barrier = [] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // slots as in linear_logprobs.hip: a of step t, x of step t, a of t + 1, x of t + 1, a of t + 2
    clear();
    ca.begin(lds0);
    static_for<0, kA>(load_run);
    next_a();
    cx.begin(lds0 + kSlot);
    static_for<kA, kA + kX>(load_run);
    next_x();
    ca.begin(lds0 + 2 * kSlot);
    static_for<0, kA>(load_run);
    next_a();
    cx.begin(lds0 + 3 * kSlot);
    static_for<kA, kA + kX / 2>(load_run);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kA + kX / 2) : "memory");
    barrier();
    static_for<0, MT + NT>([&](auto k) { read_one(0, smem, smem + kSlot, std::integral_constant<int, 0>{}, k); });
    frags.begin();
    int slot = 0;
    const auto slot_at = [](int i) { return (i >= kSlots ? i - kSlots : i) * kSlot; };
    for (int t = 0; t < count; ++t) {
        int range, nb, mt, first;
        unit(t, range, nb, mt);
        const int steps = (indices(range, first) + kDeep - 1) / kDeep;
        int k = 0;
        do {
            const lds_ptr sa = smem + slot_at(slot), sx = smem + slot_at(slot + 1);
            part(0, sa, sx, std::integral_constant<int, 1>{}, std::integral_constant<int, kA + kX / 2>{}, std::integral_constant<int, kA + kX>{});
            next_x();
            ca.begin(lds0 + slot_at(slot + 4));
            part(1, sa, sx, std::integral_constant<int, 2>{}, std::integral_constant<int, 0>{}, std::integral_constant<int, kA / 2>{});
            part(0, sa, sx, std::integral_constant<int, 3>{}, std::integral_constant<int, kA / 2>{}, std::integral_constant<int, kA>{});
            next_a();
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kA) : "memory");       // all but a of step t + 2
            barrier();
            cx.begin(lds0 + slot_at(slot));
            slot = slot + 2 >= kSlots ? slot + 2 - kSlots : slot + 2;
            part(1, smem + slot_at(slot), smem + slot_at(slot + 1), std::integral_constant<int, 0>{}, std::integral_constant<int, kA>{},
                 std::integral_constant<int, kA + kX / 2>{});
        } while (++k < steps);
        // lane: rows n of the output, fours of columns m; what lies outside the output lies outside the descriptor
        constexpr int kOut = OUT == kInput ? (int)sizeof(T) : 4;
        const int n0 = nb * BN, m0 = mt * BM;
        const int64_t start = (int64_t)range * a.range_stride + (int64_t)n0 * a.out_stride + m0;
        const auto out = __builtin_amdgcn_make_buffer_rsrc((char*)a.out + start * kOut, 0,
                                                           (int)(((int64_t)(min(BN, a.n - n0) - 1) * a.out_stride + a.m - m0) * kOut), 0x00020000);
        const uint32_t pitch = (uint32_t)a.out_stride * kOut, left = (uint32_t)(a.m - m0);
        if constexpr (kOut == 2) {
            // Through the slot that is free until the next step's second part, a wave by itself in the runs that only it
            // loads into, so that whole rows of the tile are stored (as they are, a lane has 8 bytes of a row and an
            // instruction 32 rows: dc of 2560 x 262208 took 426 us so with 8 rows and 2357 with 2047, now 256 and 2220): 32 rows
            // at a time, 16-byte chunk c of row r in place c ^ r % kChunks.
            constexpr int kChunks = BM / 16, kRows = 1024 / BM;
            const lds_ptr mine = smem + slot_at(slot + 4) + w * 1024;
            const auto row_at = [&](int row) { return mine + (row / kRows) * 4096 + (row % kRows) * BM; };
            const lds_ptr put = row_at(r) + 8 * hh;
            const int chunk = lane % kChunks;
            static_for<0, NT>([&](auto column) {
                constexpr int j = decltype(column)::value;
                static_for<0, MT>([&](auto block) {
                    constexpr int i = decltype(block)::value;
                    // (an accumulator at a time, in the accumulation registers until then: not all of them copied first)
                    __builtin_amdgcn_sched_barrier(0);
                    asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        bf16x4 o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = (__bf16)acc[i][j][4 * q + e];
                        *(MA_LDS bf16x4*)(put + (((4 * i + q) ^ (r % kChunks)) << 4)) = o;
                    }
                });
                asm volatile("" ::: "memory");
#pragma unroll
                for (int k = 0; k < 32 / kRows; ++k) {
                    const int row = k * kRows + lane / kChunks;
                    const u32x4 v = *(MA_LDS u32x4*)(row_at(row) + ((chunk ^ (row % kChunks)) << 4));
                    const uint32_t m = wm + 8 * chunk;
                    __builtin_amdgcn_raw_buffer_store_b128(v, out, (uint32_t)(wn + 32 * j + row) * pitch + m * kOut + (m < left ? 0u : 0x80000000u), 0, 0);
                }
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            });
        } else {
            const uint32_t row0 = (uint32_t)(wn + r) * pitch;
            static_for<0, MT * NT>([&](auto tile) {
                constexpr int i = decltype(tile)::value % MT, j = decltype(tile)::value / MT;
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t m = wm + 32 * i + 8 * q + 4 * hh;
                    const uint32_t at = (row0 + 32 * j * pitch + m * kOut) + (m < left ? 0u : 0x80000000u);
                    f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if constexpr (OUT == kAdded) {
                        const u32x4 before = __builtin_amdgcn_raw_buffer_load_b128(out, at, 0, 0);
                        v += *(const f32x4*)&before;
                    }
                    __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4*)&v, out, at, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        clear();
    }
    // the last loads (of steps that do not exist) must not land in LDS that another workgroup has been given
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

// de = sum of the shares of a result (its ranges, its rows' parts), rounded once
template <typename T>
__global__ __launch_bounds__(256) void linear_grads_join_kernel(const float* __restrict__ part, int shares, int64_t n, T* __restrict__ out) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 v = *(const f32x4*)(part + i);
    for (int r = 1; r < shares; ++r) v += *(const f32x4*)(part + (int64_t)r * n + i);
    if constexpr (sizeof(T) == 4) {
        *(f32x4*)(out + i) = v;
    } else {
        bf16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (__bf16)v[e];
        *(bf16x4*)(out + i) = o;
    }
}

// e's rows as the contraction over them takes them: zeros for a token that does not count, since its x is 0 but its hidden
// state may be anything, and 0 * NaN is NaN; `copies` times, one for each part of x.  A wave a row, 16 bytes a lane.
__global__ __launch_bounds__(256) void linear_counted_rows_kernel(const char* __restrict__ e, int64_t stride, const int64_t* __restrict__ targets,
                                                                  int64_t rows, int64_t vocab, int64_t ignore_index, int bytes, int copies,
                                                                  char* __restrict__ out) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int64_t target = targets[row];
    const bool valid = target != ignore_index && target >= 0 && target < vocab;
    for (int at = (threadIdx.x & 63) * 16; at < bytes; at += 64 * 16) {
        const u32x4 v = valid ? *(const u32x4*)(e + row * stride + at) : u32x4{0, 0, 0, 0};
        for (int c = 0; c < copies; ++c) *(u32x4*)(out + (c * rows + row) * bytes + at) = v;
    }
}

template <typename T, bool X_ROWS, Output OUT, int BM, int BN>
int start(const GradArgs& a, hipStream_t st) {
    auto kernel = linear_grads_kernel<T, X_ROWS, OUT == kInput && sizeof(T) == 4 ? kStored : OUT, BM, BN>;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kSlots * kSlot);
    if (e != hipSuccess) return fail(MA_ERR_LAUNCH, "linear_grads_kernel: %s", hipGetErrorString(e));
    const int cus = compute_units() / kXcds * kXcds;
    int grid = (a.units + kXcds - 1) / kXcds * kXcds;
    if (grid > cus) grid = cus < kXcds ? kXcds : cus;
    kernel<<<grid, 256, kSlots * kSlot, st>>>(a);
    return check_launch("linear_grads_kernel");
}

// Tile and number of ranges of a product [n, m] over `steps` steps, from its time in us: rounds of the chip's workgroups
// times the steps of a unit and what its results take, and the results of more than one range, written and joined.  The
// larger tiles do more per byte that they read; the smaller ones leave less of the chip idle and of a tile empty.  Measured
// with 256 x 256, 128 x 256 and 128 x 128 alone (us, de and dc): bf16, 2560 x 262208, 2047 rows 2157 + 2365, 3077 + 2709,
// 4103 + 3408; 128 x 2051, 257 rows 21 + 14, 19 + 11, 13 + 7; fp32, 2048 x 32000, 4096 rows 2456 + 2468, 2767 + 2988,
// 3388 + 3323, and 640 x 32003, 300 rows 123 + 104, 115 + 93, 107 + 94.
constexpr int kTiles[3][2] = {{256, 256}, {128, 256}, {128, 128}};          // M, N
struct Cut {
    int tile, ranges;
};
Cut cut(int64_t n, int64_t m, int64_t steps, bool bf16, int most) {
    static const double step_us[2][3] = {{5.1, 2.9, 1.75}, {1.7, 1.2, 0.8}};
    Cut best = {0, 1};
    double least = 1e300;
    for (int t = 0; t < 3; ++t) {
        const int64_t tiles = ((m + kTiles[t][0] - 1) / kTiles[t][0]) * ((n + kTiles[t][1] - 1) / kTiles[t][1]);
        const double store = kTiles[t][0] * kTiles[t][1] * (bf16 ? 0.7e-4 : 1.5e-4);
        for (int r = 1; r <= most && r <= steps; ++r) {
            const double cost = (double)((tiles * r + 255) / 256) * ((double)((steps + r - 1) / r) * step_us[bf16][t] + store) +
                                (r == 1 ? 0.0 : 4.0 + (double)r * n * m * 8.0 / 4.5e6);
            if (cost < least) {
                least = cost;
                best = {t, r};
            }
            if (tiles * r > 4096) break;
        }
    }
    const int64_t per = (steps + best.ranges - 1) / best.ranges;            // (no range is empty)
    best.ranges = (int)((steps + per - 1) / per);
    return best;
}

constexpr int kMostRanges = 128;

int64_t steps_of(int64_t contraction, bool bf16) { return (contraction * (bf16 ? 2 : 4) + 127) / 128; }

template <typename T, bool X_ROWS, Output OUT>
int start_cut(GradArgs& a, const Cut& how, hipStream_t st) {
    const int64_t steps = steps_of(a.contraction, sizeof(T) == 2);
    a.ranges = how.ranges;
    a.range_steps = (int)((steps + how.ranges - 1) / how.ranges);
    a.m_tiles = (a.m + kTiles[how.tile][0] - 1) / kTiles[how.tile][0];
    a.n_blocks = (a.n + kTiles[how.tile][1] - 1) / kTiles[how.tile][1];
    a.units = a.m_tiles * a.n_blocks * a.ranges;
    if (how.tile == 0) return start<T, X_ROWS, OUT, 256, 256>(a, st);
    if (how.tile == 1) return start<T, X_ROWS, OUT, 128, 256>(a, st);
    return start<T, X_ROWS, OUT, 128, 128>(a, st);
}

template <typename T>
int launch(const LinearGradsArgs& p, hipStream_t st) {
    constexpr bool bf16 = sizeof(T) == 2;
    GradArgs a = {};
    a.x = (const char*)p.x;
    a.x_stride = p.x_stride * sizeof(T);
    a.m = (int)p.dim;
    a.out_stride = p.dim;
    if (p.de) {
        a.a = (const char*)p.c;
        a.a_stride = p.c_stride * sizeof(T);
        a.n = (int)p.rows;
        a.contraction = (int)p.vocab;
        a.range_stride = p.rows * p.dim;
        const Cut how = cut(p.rows, p.dim, steps_of(p.vocab, bf16), bf16, kMostRanges);
        const int shares = how.ranges * p.parts;             // of a result: ranges, and in each the parts' rows
        a.out = shares == 1 ? p.de : p.ws;
        const int rc = bf16 && shares == 1 ? start_cut<T, false, kInput>(a, how, st) : start_cut<T, false, kStored>(a, how, st);
        if (rc) return rc;
        if (shares > 1) {
            const int64_t n = p.rows / p.parts * p.dim;
            linear_grads_join_kernel<T><<<(unsigned)((n / 4 + 255) / 256), 256, 0, st>>>((const float*)p.ws, shares, n, (T*)p.de);
            const int joined = check_launch("linear_grads_join_kernel");
            if (joined) return joined;
        }
    }
    if (p.dc) {
        a.a = (const char*)p.e;
        a.a_stride = p.e_stride * sizeof(T);
        a.n = (int)p.vocab;
        a.contraction = (int)p.rows;
        a.out = p.dc;
        a.range_stride = 0;
        const Cut how = cut(p.vocab, p.dim, steps_of(p.rows, bf16), bf16, 1);
        return p.dc_added ? start_cut<T, true, kAdded>(a, how, st) : start_cut<T, true, kInput>(a, how, st);
    }
    return MA_OK;
}

}  // namespace

size_t linear_grads_workspace_bytes(int64_t rows, int64_t vocab, int64_t dim, int parts, int dtype) {
    const bool bf16 = dtype == MA_DTYPE_BF16;
    const Cut how = cut(rows, dim, steps_of(vocab, bf16), bf16, kMostRanges);
    return how.ranges * parts == 1 ? 0 : (size_t)how.ranges * rows * dim * sizeof(float);
}

int launch_linear_counted_rows(const void* e, int64_t e_stride, const int64_t* targets, int64_t rows, int64_t vocab, int64_t dim,
                               int64_t ignore_index, int copies, void* out, int dtype, hipStream_t st) {
    const int elt = dtype == MA_DTYPE_BF16 ? 2 : 4;
    linear_counted_rows_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>((const char*)e, e_stride * elt, targets, rows, vocab, ignore_index,
                                                                           (int)dim * elt, copies, (char*)out);
    return check_launch("linear_counted_rows_kernel");
}

int launch_linear_grads(const LinearGradsArgs& p, int dtype, hipStream_t st) {
    return dtype == MA_DTYPE_BF16 ? launch<uint16_t>(p, st) : launch<float>(p, st);
}

}  // namespace ma
