// Log-probabilities of given tokens and entropy from hidden states e [rows, K] and the classifier c [vocab, K],
// without the [rows, vocab] logits x = e c^T: a matrix product whose epilogue keeps, per row, the running maximum and
// sums of token_logprobs.hip in registers.  The same product with another epilogue forms d loss / d x a block of rows
// at a time for the two gradient products.
//
// Tiles are computed transposed, x^T = c e^T (M: vocabulary, N: tokens), because of where the matrix instruction
// leaves its result: a lane of a 32 x 32 tile holds 16 rows of ONE column, so with the vocabulary along the rows a
// lane folds its logits of one token without talking to another lane; lanes, waves and workgroups that share a token
// join their statistics once at the end of a workgroup's whole vocabulary range.
//
// A workgroup of four waves owns BN tokens and a range of the vocabulary that it walks in tiles of 256.  Both operands are
// brought in steps of 128 bytes of K, global memory -> LDS without registers; rows past the end of the range or of the
// tokens lie outside the loads' descriptors and arrive as zeros.  A row of a step is 8 chunks of 16 bytes, chunk c of row r
// stored in place c ^ (r / 2 % 8): the 16 lanes that read together (16 rows, one chunk each) then touch all 64 banks once.
// Which chunk a lane of a load fetches is decided on the global side, so the exchange costs nothing.  With BN = 256 the LDS
// holds five slots of one operand's step each, with fewer tokens three stages of both; either way one barrier a step is
// enough, and the reads and loads are issued one or two to a product, in its shadow.
//
// What bounds it, in bf16: the matrix units from some 128 tokens on, the classifier's bytes below.  2560 x 262208: 8192
// tokens 8.7 ms (1.26 PFLOP/s; a library product of these sizes that only stores its result 7.95), 1433 tokens 1.56 ms,
// 8 tokens 0.24 ms (5.6 TB/s).  fp32 (split.h), 2048 x 32000, 4096 tokens 2.38 ms (226 TFLOP/s; the library's fp32
// products reach 139, and this kernel on the fp32 instructions took 3.82), 640 x 32003, 210 tokens 71 us.  A soft cap's tanh
// is arithmetic of the epilogue, which nothing hides: 8192 tokens 8.6 -> 9.7 ms, 2047 tokens 2.2 -> 2.4 and the gradient of
// their logits 2.3 -> 2.6, 300 fp32 tokens of 640 x 32003 111 -> 118 us.
#include <hip/hip_runtime.h>

#include "common.h"
#include "logprobs.h"
#include "mfma.h"
#include "rowio.h"
#include "split.h"

namespace ma {

namespace {

constexpr int kBM = 256;                     // vocabulary rows of a tile

struct LinArgs {
    const char *e, *c;
    int64_t e_stride, c_stride;              // bytes between rows
    int rows, vocab, k_bytes;
    int row_blocks, splits, span;            // workgroups: row_blocks * splits, each `span` of the vocabulary
    LpShape sh;
    const int64_t* targets;
    int64_t ignore_index;
    LpStats* part;                           // forward: [splits, rows], in units of log2
    float* picked;                           // forward: [rows], the target's capped logit
    const float *stats, *entropy, *dlogp, *dentropy;   // gradient
    void* dlogits;
    int64_t pitch;                           // elements between its rows
    int64_t second;                          // elements from a row to what its rounding left (0: not kept)
};

template <int BN>
struct Tiling {
    static constexpr int kWaveM = BN >= 128 ? 128 : 64, kWaveN = BN >= 128 ? BN / 2 : BN;
    static constexpr int kMT = kWaveM / 32, kNT = kWaveN / 32;
    static constexpr bool kRing = BN == 256;                           // five slots of one operand, or stages of both
    static constexpr int kStep = 128, kStages = 3;                     // bytes of K per step and row
    static constexpr int kSubs = kStep / 32, kChunks = kStep / 16, kRunRows = 1024 / kStep;
    static constexpr int kARuns = kBM / kRunRows / 4, kBRuns = BN / kRunRows / 4;       // 1 KB loads per wave and step
    static constexpr int kStage = (kBM + BN) * kStep;
    // place of chunk c of row r of a stage: c ^ key(r)
    static constexpr __host__ __device__ int key(int r) { return (r >> 1) & 7; }
    static constexpr int kLds = kRing ? 5 * kBM * kStep : kStage * kStages;
    static_assert(kLds <= 160 * 1024, "LDS");
};

// workgroup -> (row block, split).  Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of the order
// below, groups of 8 row blocks times all splits, so that the workgroups of one XCD share both operands through its L2:
// 32 of them then read 8 blocks of e and 4 of c.
__device__ __forceinline__ bool place(const LinArgs& a, int& rb, int& split) {
    const int total = a.row_blocks * a.splits, per = (total + kXcds - 1) / kXcds;
    const int j = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
    if (j >= total) return false;
    const int super = j / (8 * a.splits), in = j - super * 8 * a.splits;
    const int height = min(8, a.row_blocks - super * 8);
    // (integer division runs on the vector ALU: the results go back to scalar registers, where descriptors live)
    split = __builtin_amdgcn_readfirstlane(in / height);
    rb = __builtin_amdgcn_readfirstlane(super * 8 + in % height);
    return true;
}

template <typename T, int BN, bool CAP, bool GRAD>
__global__ __launch_bounds__(256, 1) void linear_logprobs_kernel(const LinArgs a) {
    using L = Tiling<BN>;
    constexpr int MT = L::kMT, NT = L::kNT, STAGES = L::kStages;
    extern __shared__ __align__(16) char smem_raw[];
    const lds_ptr smem = (lds_ptr)smem_raw;
    int rb, split;
    if (!place(a, rb, split)) return;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hh = lane >> 5;
    const int wm = BN >= 128 ? (w & 1) * L::kWaveM : w * L::kWaveM, wn = BN >= 128 ? (w >> 1) * L::kWaveN : 0;
    const int n0 = rb * BN, v0 = split * a.span, v1 = min(v0 + a.span, a.vocab);
    const int tiles = (v1 - v0 + kBM - 1) / kBM, ksteps = (a.k_bytes + L::kStep - 1) / L::kStep;

    // ---- loads: run t of kRunRows rows, of which this lane fetches one chunk of one row (key(row) is the same for all
    // runs of a wave, which are four apart)
    const int run_row = lane / L::kChunks, chunk = (lane % L::kChunks) ^ L::key(w * L::kRunRows + run_row);
    uint32_t a_off[L::kARuns], b_off[L::kBRuns];
#pragma unroll
    for (int p = 0; p < L::kARuns; ++p) a_off[p] = (uint32_t)((w + 4 * p) * L::kRunRows + run_row) * (uint32_t)a.c_stride + chunk * 16;
#pragma unroll
    for (int p = 0; p < L::kBRuns; ++p) b_off[p] = (uint32_t)((w + 4 * p) * L::kRunRows + run_row) * (uint32_t)a.e_stride + chunk * 16;
    const uint32_t lds0 = lds_addr(smem) + w * 1024;
    // the next step of an operand to load: address and bytes in range move on by a step's bytes and start over with the
    // next tile's rows; past the last tile nothing is in range
    struct Feed {
        uint64_t at;
        uint32_t bytes, past, lds;
        int left, tile;
        u32x4 rsrc;
    } feed[2];                                // c, e
    auto open = [&](Feed& f, bool is_c) {
        const int rows = f.tile >= tiles ? 0 : is_c ? min(kBM, v1 - v0 - f.tile * kBM) : min(BN, a.rows - n0);
        const int64_t stride = is_c ? a.c_stride : a.e_stride;
        f.at = is_c ? (uint64_t)a.c + (uint64_t)(v0 + f.tile * kBM) * stride : (uint64_t)a.e + (uint64_t)n0 * stride;
        f.bytes = rows ? (uint32_t)((rows - 1) * stride) + a.k_bytes : 0u;
        f.left = a.k_bytes;
    };
    feed[0].tile = feed[1].tile = 0;
    open(feed[0], true);
    open(feed[1], false);
    auto begin = [&](Feed& f, uint32_t lds) {
        f.rsrc = uniform_rsrc(f.at, f.bytes);
        // chunks past the end of a row are the next row's first: out of any descriptor's range
        f.past = chunk * 16 < f.left ? 0u : 0x80000000u;
        f.lds = __builtin_amdgcn_readfirstlane(lds0 + lds);
    };
    auto advance = [&](Feed& f, bool is_c) {
        f.at += L::kStep;
        f.bytes = f.bytes ? f.bytes - L::kStep : 0u;      // (the last step of a tile may wrap: it is opened anew)
        f.left -= L::kStep;
        if (f.left <= 0) {
            ++f.tile;
            open(f, is_c);
        }
    };
    // runs 0 .. kARuns - 1 of a step are c's, the others e's
    constexpr int kRuns = L::kARuns + L::kBRuns;
    auto load_run = [&](auto run) {
        constexpr int p = decltype(run)::value, q = p - L::kARuns;
        if constexpr (q < 0) buffer_to_lds_run_at<p * 4096>(feed[0].rsrc, a_off[p] | feed[0].past, feed[0].lds);
        else buffer_to_lds_run_at<q * 4096>(feed[1].rsrc, b_off[q] | feed[1].past, feed[1].lds);
    };

    // ---- fragments: 32 rows, chunks 2 s and 2 s + 1 of a step
    uint32_t frag[L::kSubs];
#pragma unroll
    for (int s = 0; s < L::kSubs; ++s) frag[s] = r * L::kStep + (((2 * s + hh) ^ L::key(r)) << 4);
    Fragments<T, MT, NT> frags;
    auto read_one = [&](int buf, lds_ptr at_c, lds_ptr at_e, auto which) {
        constexpr int i = decltype(which)::value;
        if constexpr (i < MT) frags.a[buf][i] = *(MA_LDS u32x4*)(at_c + (wm + 32 * i) * L::kStep);
        else frags.b[buf][i - MT] = *(MA_LDS u32x4*)(at_e + (wn + 32 * (i - MT)) * L::kStep);
    };
    f32x16 acc[MT][NT];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x16(0.f);
    };
    // The products of a step's 32 bytes on fragments `buf`, with the reads of the next 32's fragments (into the other
    // buffer) and runs FIRST .. LAST - 1 of a later step's loads between them, an instruction or two to each product: a
    // wave has its SIMD to itself, and what it issues between two products runs in their shadow.
    auto part = [&](int buf, lds_ptr next_c, lds_ptr next_e, auto first, auto last) {
        constexpr int P = MT * NT, H = P / 2, R = MT + NT, W0 = decltype(first)::value, W = decltype(last)::value - W0;
        static_for<0, P>([&](auto step) {
            constexpr int i = decltype(step)::value;
            // the reads in the first half: what the next part begins with has arrived by then
            if constexpr (i < H) static_for<i * R / H, (i + 1) * R / H>([&](auto k) { read_one(buf ^ 1, next_c, next_e, k); });
            else static_for<W0 + (i - H) * W / (P - H), W0 + (i - H + 1) * W / (P - H)>([&](auto k) { load_run(k); });
            frags.template product<i>(buf, acc);
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    // ---- this lane's tokens
    const float scale = a.sh.inv_temp * kLpLog2e;
    int target[NT];
    LpStats run[NT];
    float ga[NT], gb[NT], gc[NT], top[NT], log_l[NT];       // d x = p (gb log2 p + gc), at the target + ga
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = n0 + wn + 32 * j + r;
        const int64_t t = n < a.rows ? a.targets[n] : -1;
        const bool valid = t != a.ignore_index && t >= 0 && t < a.vocab;
        target[j] = valid ? (int)t : -1;
        run[j] = {-INFINITY, 0.f, 0.f};
        if (GRAD) {
            const float g = valid && a.dlogp ? a.dlogp[n] : 0.f, h = valid && a.dentropy ? a.dentropy[n] : 0.f;
            ga[j] = g * a.sh.inv_temp;
            gb[j] = -h * kLpLn2 * a.sh.inv_temp;
            gc[j] = -fmaf(h, valid ? a.entropy[n] : 0.f, g) * a.sh.inv_temp;
            top[j] = valid ? a.stats[2 * n] : 0.f;
            log_l[j] = valid ? a.stats[2 * n + 1] : 0.f;
        }
    }

    // this lane's rows of a tile: m0 + row_of(16 i + v) + 4 hh for accumulator i's register v
    auto row_of = [](int i) constexpr { return 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4; };
    auto finish_tile = [&](int m0, auto is_partial) __attribute__((always_inline)) {
        constexpr bool PARTIAL = decltype(is_partial)::value;
        // (unrolled by hand where an accumulator is named: past a size the compiler leaves a loop and moves them to memory)
        static_for<0, NT>([&](auto column) __attribute__((always_inline)) {
            constexpr int j = decltype(column)::value;
            const int t = target[j] - m0 - 4 * hh;     // the target's row of this tile, if it is one of this lane's
            const bool here = t >= 0 && t < L::kWaveM && (t & 4) == 0 && target[j] >= 0;
            if (!GRAD) {
                // two accumulators of one token's column at a time: the others stay where they are
                static_for<0, MT / 2>([&](auto half) {
                    constexpr int i0 = decltype(half)::value * 32;
                    __builtin_amdgcn_sched_barrier(0);
                    asm volatile("" : "+a"(acc[i0 / 16][j]), "+a"(acc[i0 / 16 + 1][j]));
                    float y[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = lp_capped<CAP>(acc[(i0 + i) / 16][j][i % 16], a.sh);
                    if constexpr (PARTIAL) {
                        const int left = v1 - m0 - 4 * hh;
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = row_of(i0 + i) < left ? y[i] : -INFINITY;
                    }
                    if (__any(here)) {
                        float x = 0.f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) x = row_of(i0 + i) == t ? y[i] : x;
                        // (a target past v1 belongs to the next range's workgroup)
                        if (here && t / 64 == decltype(half)::value && target[j] < v1) a.picked[n0 + wn + 32 * j + r] = x;
                    }
                    lp2_fold<32>(y, scale, run[j]);
                    // done here, not where the sums are next needed (which would keep every column's logits in registers)
                    asm volatile("" : "+v"(run[j].m), "+v"(run[j].l), "+v"(run[j].s));
                    __builtin_amdgcn_sched_barrier(0);
                });
            } else {
                const int n = n0 + wn + 32 * j + r;
                T* out = (T*)a.dlogits + (int64_t)n * a.pitch;
                // (the row's padding up to the next eight columns is written too, zeros: the products that follow read it)
                const int m_end = v1 == a.vocab ? (v1 + 7) & ~7 : v1;
                const auto store = [&](auto is_here) __attribute__((always_inline)) {
                    static_for<0, MT>([&](auto block) __attribute__((always_inline)) {
                        constexpr int i = decltype(block)::value;
                        // (an accumulator at a time, in the accumulation registers until then)
                        __builtin_amdgcn_sched_barrier(0);
                        asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int m = m0 + 32 * i + 8 * q + 4 * hh;
                            float d[4];
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const float x = acc[i][j][4 * q + v];
                                const float th = CAP ? lp_tanh(x * a.sh.inv_cap) : 0.f;
                                const float lp = fmaf(CAP ? a.sh.cap * th : x, scale, -top[j]) - log_l[j];      // log2 p
                                const float p = __builtin_amdgcn_exp2f(lp);        // (0 below -150: no product with a larger lp)
                                d[v] = p * fmaf(gb[j], fmaxf(lp, -200.f), gc[j]);
                                if constexpr (decltype(is_here)::value) d[v] += here && 32 * i + 8 * q + v == t ? ga[j] : 0.f;
                                if (CAP) d[v] *= 1.f - th * th;
                                if (target[j] < 0) d[v] = 0.f;
                                if (PARTIAL && m + v >= a.vocab) d[v] = 0.f;
                            }
                            if (n < a.rows && (!PARTIAL || m < m_end)) {
                                if constexpr (sizeof(T) == 2) {
                                    // Rounded as the products' instructions take it: as large as the results' own rounding, but
                                    // alike for all results of a row's largest coefficient.  Few rows, among which that does
                                    // not average out, are kept in two parts (the products are then bound by memory anyway).
                                    bf16x4 o;
#pragma unroll
                                    for (int v = 0; v < 4; ++v) o[v] = (__bf16)d[v];
                                    *(bf16x4*)(out + m) = o;
                                    if constexpr (BN <= kLinearPartsRows) {
                                        if (a.second) {
#pragma unroll
                                            for (int v = 0; v < 4; ++v) o[v] = (__bf16)(d[v] - (float)o[v]);
                                            *(bf16x4*)(out + a.second + m) = o;
                                        }
                                    }
                                } else {
                                    *(float4*)(out + m) = make_float4(d[0], d[1], d[2], d[3]);
                                }
                            }
                        }
                    });
                };
                if (__any(here)) store(std::true_type{});
                else store(std::false_type{});
            }
        });
    };

    const auto close_tile = [&](int tile) __attribute__((always_inline)) {
        const int m0 = v0 + tile * kBM + wm;
        if (m0 + L::kWaveM > v1) finish_tile(m0, std::integral_constant<bool, true>{});
        else finish_tile(m0, std::integral_constant<bool, false>{});
        clear();
    };
    const auto barrier = [] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    clear();
    if constexpr (L::kRing) {
        // Five slots of one operand's step each, c and e in turn: while step t is computed from two of them, e of step t + 1
        // and c of step t + 2 arrive in two others and c of step t + 1 has arrived or is about to.  After the barrier of
        // step t, e of step t + 2 goes where c of step t was and c of step t + 3 where its e was.
        static_assert(L::kSubs == 4 && L::kARuns == 8 && L::kBRuns == 8, "four parts, four loads each");
        constexpr int kSlot = kBM * L::kStep;
        begin(feed[0], 0);
        static_for<0, 8>([&](auto k) { load_run(k); });
        advance(feed[0], true);
        begin(feed[1], kSlot);
        static_for<8, 16>([&](auto k) { load_run(k); });
        advance(feed[1], false);
        begin(feed[0], 2 * kSlot);
        static_for<0, 8>([&](auto k) { load_run(k); });
        advance(feed[0], true);
        begin(feed[1], 3 * kSlot);
        static_for<8, 12>([&](auto k) { load_run(k); });
        asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
        barrier();
        static_for<0, MT + NT>([&](auto k) { read_one(0, smem + frag[0], smem + kSlot + frag[0], k); });
        frags.begin();
        int slot = 0;                         // of this step's c; e of it and the units after it follow
        const auto slot_at = [](int i) { return (i >= 5 ? i - 5 : i) * kSlot; };
        for (int tile = 0; tile < tiles; ++tile) {
            for (int k = 0; k < ksteps; ++k) {
                const lds_ptr c = smem + slot_at(slot), e = smem + slot_at(slot + 1);
                part(0, c + frag[1], e + frag[1], std::integral_constant<int, 12>{}, std::integral_constant<int, 16>{});
                advance(feed[1], false);
                begin(feed[0], slot_at(slot + 4));
                part(1, c + frag[2], e + frag[2], std::integral_constant<int, 0>{}, std::integral_constant<int, 4>{});
                part(0, c + frag[3], e + frag[3], std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
                advance(feed[0], true);
                asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");   // all but c of step t + 2
                barrier();
                begin(feed[1], slot_at(slot));
                slot = slot + 2 >= 5 ? slot - 3 : slot + 2;
                part(1, smem + slot_at(slot) + frag[0], smem + slot_at(slot + 1) + frag[0], std::integral_constant<int, 8>{},
                     std::integral_constant<int, 12>{});
            }
            close_tile(tile);
        }
    } else {
        // Stages of both operands' step.  A step's loads go out in as many groups as it has parts: the first in the last part
        // of a step, when its stage has become free, the others in the first parts of the next step.
        constexpr int kInFlight = (STAGES - 2) * kRuns;      // loads in flight when a step's operands must have landed
        constexpr auto group = [](int g) constexpr { return g * kRuns / L::kSubs; };
        const auto begin_both = [&](int stage) {
            begin(feed[0], stage * L::kStage);
            begin(feed[1], stage * L::kStage + kBM * L::kStep);
        };
        const auto advance_both = [&]() {
            advance(feed[0], true);
            advance(feed[1], false);
        };
        for (int s = 0; s < STAGES - 1; ++s) {
            begin_both(s);
            static_for<0, kRuns>([&](auto k) { load_run(k); });
            advance_both();
        }
        begin_both(STAGES - 1);
        static_for<0, group(1)>([&](auto k) { load_run(k); });
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kInFlight + group(1)) : "memory");
        barrier();
        const auto e_of = [&](lds_ptr c) { return c + kBM * L::kStep; };
        static_for<0, MT + NT>([&](auto k) { read_one(0, smem + frag[0], e_of(smem + frag[0]), k); });
        frags.begin();
        int stage = 0;
        for (int tile = 0; tile < tiles; ++tile) {
            for (int k = 0; k < ksteps; ++k) {
                const lds_ptr at = smem + stage * L::kStage;
                static_for<0, L::kSubs - 1>([&](auto s) {
                    constexpr int i = decltype(s)::value;
                    part(i & 1, at + frag[i + 1], e_of(at + frag[i + 1]), std::integral_constant<int, group(i + 1)>{},
                         std::integral_constant<int, group(i + 2)>{});
                });
                advance_both();
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kInFlight) : "memory");
                barrier();
                begin_both(stage);
                stage = stage + 1 == STAGES ? 0 : stage + 1;
                const lds_ptr next = smem + stage * L::kStage + frag[0];
                part(1, next, e_of(next), std::integral_constant<int, 0>{}, std::integral_constant<int, group(1)>{});
            }
            close_tile(tile);
        }
    }
    // the last loads (of steps that do not exist) must not land in LDS that is used again
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (GRAD) return;
    // lanes l and l + 32 share a token, and so do the waves along the vocabulary
    constexpr int kMWaves = BN >= 128 ? 2 : 4;
    MA_LDS LpStats* box = (MA_LDS LpStats*)smem;       // [kMWaves][BN]
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const LpStats t = lp2_merged(run[j], lp_shuffled(run[j], 32));
        if (hh == 0) {
            MA_LDS LpStats* at = box + (BN >= 128 ? (w & 1) : w) * BN + wn + 32 * j + r;
            at->m = t.m;
            at->l = t.l;
            at->s = t.s;
        }
    }
    __syncthreads();
    for (int n = tid; n < BN && n0 + n < a.rows; n += 256) {
        LpStats t = {box[n].m, box[n].l, box[n].s};
#pragma unroll
        for (int m = 1; m < kMWaves; ++m) {
            MA_LDS LpStats* o = box + m * BN + n;
            t = lp2_merged(t, {o->m, o->l, o->s});
        }
        a.part[(int64_t)split * a.rows + n0 + n] = t;
    }
}

// a wave per token joins the splits
__global__ __launch_bounds__(256) void linear_logprobs_join_kernel(const LinArgs a, float* __restrict__ logp, float* __restrict__ entropy,
                                                                   float* __restrict__ stats) {
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (n >= a.rows) return;
    LpStats t = {-INFINITY, 0.f, 0.f};
    for (int s = lane; s < a.splits; s += 64) t = lp2_merged(t, a.part[(int64_t)s * a.rows + n]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) t = lp2_merged(t, lp_shuffled(t, off));
    if (lane) return;
    const int64_t target = a.targets[n];
    const bool valid = target != a.ignore_index && target >= 0 && target < a.vocab;
    const float log_l = log2f(t.l);
    logp[n] = valid ? (fmaf(a.picked[n], a.sh.inv_temp * kLpLog2e, -t.m) - log_l) * kLpLn2 : 0.f;
    entropy[n] = valid ? (log_l - t.s / t.l) * kLpLn2 : 0.f;
    if (stats) *(float2*)(stats + 2 * (int64_t)n) = make_float2(t.m, log_l);      // both in units of log2
}

// Tokens per block and splits of the vocabulary.  A tile of 256 x BN takes (us, of 2560 bytes of K and per 1000 rows' run on
// the full chip) 67, 39, 30, 26 in bf16 and 161, 82, 43, 24 in fp32 for BN = 256, 128, 64, 32: narrow blocks cost more per
// token, wide ones leave compute units without work or rows without tokens when there are few rows.  The plan is the one
// with the least of (rounds of 256 workgroups) * (tiles of a range) * (that weight).  Ranges are whole tiles, or for the
// two narrow blocks, bound by reading c, multiples of 32 so that it is shared out evenly.  Measured at 262208 x 2560 bf16:
// 48 tokens 248 us in one block of 64 against 309 in two of 32, 384 tokens 549 in three of 128 against 583 in two of 256;
// at 32003 x 640 fp32, 210 tokens 71 us in two of 128 against 100 in one of 256 and 83 in four of 64, 300 tokens 107 in two of
// 256 against 118 in five of 64.
int plan(LinArgs& a, int dtype) {
    constexpr int kWidths[4] = {32, 64, 128, 256};
    constexpr double kWeight[2][4] = {{0.22, 0.41, 0.60, 1.0}, {0.39, 0.45, 0.58, 1.0}};     // MA_DTYPE_F32, MA_DTYPE_BF16
    constexpr int kUnits = 256;                        // compute units
    const int most = (a.vocab + kBM - 1) / kBM;
    double best = 1e300;
    int width = 256;
    for (int w = 0; w < 4; ++w) {
        const int blocks = (a.rows + kWidths[w] - 1) / kWidths[w], unit = w < 2 ? 32 : kBM;
        for (int splits = 1; splits <= most && splits <= kUnits; ++splits) {
            const int span = ((a.vocab + splits - 1) / splits + unit - 1) / unit * unit;
            const int64_t rounds = ((int64_t)blocks * splits + kUnits - 1) / kUnits;
            const double cost = (double)rounds * span * kWeight[dtype == MA_DTYPE_BF16][w];
            if (cost < best) {
                best = cost;
                width = kWidths[w];
                a.row_blocks = blocks;
                a.span = span;
            }
        }
    }
    a.splits = (a.vocab + a.span - 1) / a.span;        // none of them empty
    return width;
}

LinArgs args_of(const LinearLogprobsArgs& p, int dtype, int& width) {
    LinArgs a = {};
    const int elt = dtype == MA_DTYPE_BF16 ? 2 : 4;
    a.e = (const char*)p.e;
    a.c = (const char*)p.c;
    a.e_stride = p.e_stride * elt;
    a.c_stride = p.c_stride * elt;
    a.rows = (int)p.rows;
    a.vocab = (int)p.vocab;
    a.k_bytes = (int)p.dim * elt;
    a.sh = lp_shape(p.softcap, p.temperature);
    a.targets = p.targets;
    a.ignore_index = p.ignore_index;
    width = plan(a, dtype);
    return a;
}

template <typename T, int BN, bool CAP, bool GRAD>
int start(const LinArgs& a, hipStream_t st) {
    auto kernel = linear_logprobs_kernel<T, BN, CAP, GRAD>;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, Tiling<BN>::kLds);
    if (e != hipSuccess) return fail(MA_ERR_LAUNCH, "linear_logprobs_kernel: %s", hipGetErrorString(e));
    const int grid = (a.row_blocks * a.splits + kXcds - 1) / kXcds * kXcds;
    kernel<<<grid, 256, Tiling<BN>::kLds, st>>>(a);
    return check_launch("linear_logprobs_kernel");
}
template <typename T, bool CAP, bool GRAD>
int by_width(const LinArgs& a, int width, hipStream_t st) {
    switch (width) {
        case 32: return start<T, 32, CAP, GRAD>(a, st);
        case 64: return start<T, 64, CAP, GRAD>(a, st);
        case 128: return start<T, 128, CAP, GRAD>(a, st);
        default: return start<T, 256, CAP, GRAD>(a, st);
    }
}
template <bool GRAD>
int by_type(const LinArgs& a, int width, int dtype, hipStream_t st) {
    const bool bf16 = dtype == MA_DTYPE_BF16;
    if (a.sh.cap > 0.f) return bf16 ? by_width<uint16_t, true, GRAD>(a, width, st) : by_width<float, true, GRAD>(a, width, st);
    return bf16 ? by_width<uint16_t, false, GRAD>(a, width, st) : by_width<float, false, GRAD>(a, width, st);
}

}  // namespace

// picked [rows] (rounded up to 16 bytes), then part [splits, rows] for at most 256 splits of 256 or more
size_t linear_logprobs_workspace_bytes(int64_t rows, int64_t vocab) {
    int64_t splits = (vocab + kBM - 1) / kBM;
    if (splits > 256) splits = 256;
    return (((size_t)rows * 4 + 15) & ~(size_t)15) + (size_t)splits * rows * sizeof(LpStats);
}

int launch_linear_logprobs_fwd(const LinearLogprobsArgs& p, int dtype, hipStream_t st) {
    int width = 0;
    LinArgs a = args_of(p, dtype, width);
    a.picked = (float*)p.ws;
    a.part = (LpStats*)((char*)p.ws + (((size_t)p.rows * 4 + 15) & ~(size_t)15));
    const int rc = by_type<false>(a, width, dtype, st);
    if (rc) return rc;
    linear_logprobs_join_kernel<<<(unsigned)((p.rows + 3) / 4), 256, 0, st>>>(a, p.logp, p.entropy, p.stats);
    return check_launch("linear_logprobs_join_kernel");
}

int launch_linear_logprobs_dlogits(const LinearLogprobsArgs& p, int dtype, hipStream_t st) {
    int width = 0;
    LinArgs a = args_of(p, dtype, width);
    a.stats = p.stats;
    a.entropy = p.entropy;
    a.dlogp = p.dlogp;
    a.dentropy = p.dentropy;
    a.dlogits = p.dlogits;
    a.pitch = p.pitch;
    if (p.parts == 2) {
        if (width > kLinearPartsRows) return fail(MA_ERR_UNSUPPORTED, "linear_logprobs: two parts of %d rows", a.rows);
        a.second = p.rows * p.pitch;
    }
    return by_type<true>(a, width, dtype, st);
}

}  // namespace ma
