// Gradient products in bf16, 256 x 256 tiles of four waves on gfx950:
//   dX [M][K] = dP [M][N] W [N][K]        sums over N
//   dW [N][K] = dP^T X,  dP [M][N], X [M][K]   sums over M
// C[r][c] = sum over d of A(r, d) B(d, c) in both: B's rows are the sum's
// index (K-major: as W and X lie), A is row-major for dX and K-major for dW.
//
//  * wave (wm, wn) of four owns 128 x 128 outputs, 4 x 4 blocks of
//    v_mfma_f32_32x32x16_bf16 in AGPRs (16x16x32, twice the instructions and,
//    with their wait states, nearly every issue slot: dX / dW of M = N = 4096, K =
//    7168 199 / 205 us, now 194 / 197);
//    a K-tile is 64 deep, so a row of a row-major operand is 128 bytes and a
//    K-major stage 64 rows of 512 bytes; 32 KB per operand and stage, two
//    stages of both in LDS;
//  * the wave's rows of a K-tile sit in registers as four halves (A rows
//    0 - 63 / 64 - 127, B columns likewise); a K-tile runs as four quadrants in
//    Gray-code order over (A half, B half), rotating by one per K-tile, so a
//    half's registers are free for the next K-tile as soon as its last
//    quadrant has issued, and the LDS reads run under the MFMAs;
//  * barrier B1 (all of K-tile t has been read) frees t's stage for the DMA of
//    t + 2, spread over the next three quadrants; B2 waits for t + 1's DMA only;
//  * K-major operands are transposed by ds_read_b64_tr_b16: within 16 lanes,
//    lane 4j + c addresses columns 4c .. 4c + 3 of row j, and lane i receives
//    column i of the four rows.  Two of them (rows 8g .. 8g + 3, + 4) give lane
//    (g, r) of a 32 x 16 operand block the eight k = 8g .. 8g + 7 of column r,
//    which is what a row-major operand's 16-byte chunk g of row r holds;
//  * swizzles: row-major chunk ^ (row >> 1 & 7); K-major 32-byte granule ^ 2 (k &
//    3), which puts the four rows and two granules that half a wave touches on
//    eight different places: all 64 banks;
//  * every load's descriptor ends with its operand, so rows past the sum's end
//    read as zeros.  A row-major A has its rows padded with zeros to whole
//    K-tiles (a following row's NaN times 0 would be NaN).  Columns past an
//    operand's width hold its next row's: they reach only outputs that are
//    not stored.
#pragma once
#include <type_traits>
#include <utility>

#include "act_grad.hpp"
#include "common.hpp"

namespace qg {

struct GradProduct {
    const uint16_t* a;       // row-major [rows][lda], or (a_km) K-major [depth][lda]
    const uint16_t* b;       // [depth][ldb]
    uint16_t* c;             // bf16 [rows][ldc], rows on 16 bytes, cols a multiple of 8
    float* ws;               // splitk > 1: planes [splitk][rows][cols]
    int rows, cols, depth;   // depth: the sum's length; a row-major A holds zeros from there to the next multiple of 64
    int tiles_m, tiles_n, group_m;
    int splitk, kt_per_split;
    int a_km;
    long long lda, ldb, ldc; // elements
    long long a_bytes, b_bytes;
    __host__ __device__ int blocks() const { return tiles_m * tiles_n * splitk; }
};

// One launch of one or two products, the one with the longer tiles first: its
// last, partial round of workgroups leaves CUs that the other's tiles take.
// M = 2048, N = K = 4096 (128 tiles of 64 K-tiles and 256 of 32): 112 us, against
// 64 + 14 (a split of dX and its sum) + 59 in a launch each.
struct GradArgs {
    GradProduct p[2];
    int n;
    // the bias's gradient from its partial rows, by workgroups after the
    // products' (they run beside the last tiles; a launch of their own took 5 us
    // of linear 129 and 27 us backward calls); parts 0: none
    PartialSumArgs bias;
};

namespace grad {
constexpr int kDeep = 64;    // K-tile
constexpr int qa(int g) { return (g & 3) >= 2 ? 1 : 0; }
constexpr int qb(int g) { return ((g & 3) == 1 || (g & 3) == 2) ? 1 : 0; }
// the half that quadrants k and k + 1 of the K-tile in phase P share: {is it A's, which}
constexpr bool shared_a(int P, int k) { return qa((k + P) & 3) == qa((k + 1 + P) & 3); }
constexpr int shared_half(int P, int k) { return shared_a(P, k) ? qa((k + P) & 3) : qb((k + P) & 3); }
template <int V>
struct I {
    static constexpr int value = V;
};
template <class F, int... K>
__device__ __forceinline__ void each_impl(F&& f, std::integer_sequence<int, K...>) {
    (f(I<K>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_impl(f, std::make_integer_sequence<int, N>{});
}
// acc += B A with the accumulator in AGPRs: left to the register allocator, 256
// of them beside 128 operand registers move through VGPRs.  The two wait
// states are what an MFMA needs after a VALU write of an operand, which the
// compiler does not insert for inline asm; they pass under the MFMA before.
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ void mfma(f32x16& acc, const i32x4& b, const i32x4& a) {
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}
}  // namespace grad

constexpr int kGradStage = 256 * 128;

// Workgroup `id` of product p.  AKM: A is K-major.  A split product writes fp32
// planes for splitk_reduce_kernel.
template <bool AKM>
__device__ __forceinline__ void grad_tile(const GradProduct& p, int id, uint8_t (&lA0)[kGradStage],
                                          uint8_t (&lA1)[kGradStage], uint8_t (&lB0)[kGradStage],
                                          uint8_t (&lB1)[kGradStage]) {
    constexpr int BM = 256;

    // tile: an XCD's workgroups (blockIdx % 8) take neighbouring tiles, in groups of group_m rows
    const int T = p.tiles_m * p.tiles_n;
    const int sk = id / T;
    int bid = id - sk * T;
    if ((T & 7) == 0) bid = (bid & 7) * (T >> 3) + (bid >> 3);
    const int gfull = p.group_m * p.tiles_n;
    const int gi = bid / gfull;
    const int first_m = gi * p.group_m;
    const int gm = min(p.tiles_m - first_m, p.group_m);
    const int within = bid - gi * gfull;
    const int m0 = (first_m + within % gm) * BM, n0 = (within / gm) * BM;
    const int kt0 = sk * p.kt_per_split;
    const int nk = min((p.depth + grad::kDeep - 1) / grad::kDeep, kt0 + p.kt_per_split) - kt0;

    // an opaque copy: the two forms in one kernel share no lane offsets, which would
    // stay live from before the branch
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), L = tid & 63;
    const int wm = w >> 1, wn = w & 1;
    const int g = L >> 5, l32 = L & 31, l16 = L & 15;
    const int M = p.rows, N = p.cols;

    // DMA t of wave w: 8 rows of a row-major operand (lane L: row + L/8, chunk
    // L%8), or 2 rows of a K-major one (lane L: row + L/32, chunk L%32)
    int aoff[8], boff[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const int r = (w * 8 + t) * 8 + (L >> 3);
        const int kr = (w * 8 + t) * 2 + (L >> 5);
        const int kc = (((((L & 31) >> 1) ^ ((kr & 3) << 1)) << 1) | (L & 1)) * 16;
        if constexpr (AKM) aoff[t] = kr * (int)p.lda * 2 + kc;
        else aoff[t] = (min(m0 + r, M - 1) - m0) * (int)p.lda * 2 + ((L & 7) ^ ((r >> 1) & 7)) * 16;
        boff[t] = kr * (int)p.ldb * 2 + kc;
    }
    const uint8_t* A = (const uint8_t*)p.a;
    const uint8_t* B = (const uint8_t*)p.b;
    auto rsrc = [](const uint8_t* base, long long off, long long bytes) __attribute__((always_inline)) {
        const long long left = bytes - off;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + off), 0,
                                                 (int)(left < 0 ? 0 : min(left, 0x7fffffffLL)), 0x00020000);
    };
    // K-tile kt of the slice; past the slice an empty range (zeros, no reads)
    auto src_a = [&](int kt) __attribute__((always_inline)) {
        const long long x = kt0 + kt;
        const long long off = AKM ? x * (grad::kDeep * 2) * p.lda + 2ll * m0 : 2ll * m0 * p.lda + x * (grad::kDeep * 2);
        return rsrc(A, off, kt < nk ? p.a_bytes : 0);
    };
    auto src_b = [&](int kt) __attribute__((always_inline)) {
        const long long x = kt0 + kt;
        return rsrc(B, x * (grad::kDeep * 2) * p.ldb + 2ll * n0, kt < nk ? p.b_bytes : 0);
    };

    QG_LDS uint8_t* pA0 = (QG_LDS uint8_t*)lA0;
    QG_LDS uint8_t* pA1 = (QG_LDS uint8_t*)lA1;
    QG_LDS uint8_t* pB0 = (QG_LDS uint8_t*)lB0;
    QG_LDS uint8_t* pB1 = (QG_LDS uint8_t*)lB1;

    // operand read offsets: chunk 2s + g of row l32 (step s of 16); K-major k = 8g + j (lane 4j + c of 16),
    // columns 4c .. of granule 0 or, for the upper 16 columns of a block, 1
    const int rsw = (l32 >> 1) & 7;
    const int krow = (8 * g + (l16 >> 2)) * 512 + ((((l16 >> 2) << 1) ^ (l32 >> 4)) << 5) + (l16 & 3) * 8;
    // (opaque: as plain lane arithmetic the compiler loses track of which LDS
    // array the reads hit and waits for every DMA in flight before them)
    int tra = krow + wm * 256, trb = krow + wn * 256;
    asm("" : "+v"(tra));
    asm("" : "+v"(trb));

    grad::f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    i32x4 ah[2][2][4], bh[2][2][4];    // [half][32-row block][step of 16]

    // unit x (0 .. 3) of half h: steps 2 (x % 2) and + 1 of block x / 2
    auto read_one = [&](bool is_a, int h, int x, const QG_LDS uint8_t* sA,
                        const QG_LDS uint8_t* sB) __attribute__((always_inline)) {
        i32x4(&dst)[2][2][4] = is_a ? ah : bh;
        const int blk = 2 * h + (x >> 1);
#pragma unroll
        for (int s = 2 * (x & 1); s < 2 * (x & 1) + 2; ++s) {
            if (is_a && !AKM) {
                const QG_LDS uint8_t* row = sA + (wm * 128 + blk * 32 + l32) * 128;
                dst[h][x >> 1][s] = *(const QG_LDS i32x4*)(row + (((2 * s + g) ^ rsw) << 4));
            } else {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                const QG_LDS uint8_t* st = (is_a ? sA : sB) + ((is_a ? tra : trb) ^ (blk << 6)) + s * 16 * 512;
                const i32x2 lo =
                    __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((QG_LDS s16x4*)st));
                const i32x2 hi =
                    __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((QG_LDS s16x4*)(st + 4 * 512)));
                dst[h][x >> 1][s] = i32x4{lo[0], lo[1], hi[0], hi[1]};
            }
        }
    };
    // 16 MFMAs, the four steps outermost (no two in a row on one accumulator);
    // after each one fill(k) issues a share of the LDS reads and DMAs, in this order
    auto quadrant = [&](int ha, int hb, auto&& fill) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int s = k >> 2, i = (k >> 1) & 1, j = k & 1;
            grad::mfma(acc[2 * ha + i][2 * hb + j], bh[hb][j][s], ah[ha][i][s]);
            __builtin_amdgcn_sched_barrier(0);
            fill(k);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto dma_all = [&](int kt, QG_LDS uint8_t* sA, QG_LDS uint8_t* sB) __attribute__((always_inline)) {
        const auto ra = src_a(kt), rb = src_b(kt);
#pragma unroll
        for (int t = 0; t < 8; ++t) dma16_buf(ra, sA + (w * 8 + t) * 1024, aoff[t], 0);
#pragma unroll
        for (int t = 0; t < 8; ++t) dma16_buf(rb, sB + (w * 8 + t) * 1024, boff[t], 0);
    };

    // K-tile t in phase P = t % 4 (stage P & 1 holds t, then t + 2)
    auto ktile = [&](auto PC, int t) __attribute__((always_inline)) {
        constexpr int P = decltype(PC)::value;
        QG_LDS uint8_t* sA = (P & 1) ? pA1 : pA0;
        QG_LDS uint8_t* sB = (P & 1) ? pB1 : pB0;
        QG_LDS uint8_t* nA = (P & 1) ? pA0 : pA1;
        QG_LDS uint8_t* nB = (P & 1) ? pB0 : pB1;
        constexpr bool r0a = grad::shared_a(P, 0), r1a = grad::shared_a(P, 1), r2a = grad::shared_a(P, 2);
        constexpr int r0 = grad::shared_half(P, 0), r1 = grad::shared_half(P, 1), r2 = grad::shared_half(P, 2);
        __builtin_amdgcn_sched_barrier(0);
        quadrant(grad::qa(P), grad::qb(P), [&](int k) __attribute__((always_inline)) {
            if (k < 4) read_one(r1a, r1, k, sA, sB);
            else if (k < 8) read_one(r2a, r2, k - 4, sA, sB);
        });
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // B1
        const auto ra = src_a(t + 2), rb = src_b(t + 2);
        auto dma_op = [&](int d) __attribute__((always_inline)) {
            if (d < 8) dma16_buf(ra, sA + (w * 8 + d) * 1024, aoff[d], 0);
            else dma16_buf(rb, sB + (w * 8 + d - 8) * 1024, boff[d - 8], 0);
        };
        quadrant(grad::qa(P + 1), grad::qb(P + 1), [&](int k) __attribute__((always_inline)) {
            if (k % 3 == 0) dma_op(k / 3);
        });
        asm volatile("s_waitcnt vmcnt(6)\n\ts_barrier" ::: "memory");      // B2
        quadrant(grad::qa(P + 2), grad::qb(P + 2), [&](int k) __attribute__((always_inline)) {
            if (k % 3 == 2) dma_op(6 + k / 3);
            if (k < 8 && (k & 1) == 0) read_one(r0a, r0, k >> 1, nA, nB);
        });
        quadrant(grad::qa(P + 3), grad::qb(P + 3), [&](int k) __attribute__((always_inline)) {
            if (k % 3 == 1) dma_op(11 + k / 3);
            if (k < 4) read_one(r1a, r1, k, nA, nB);
        });
    };

    dma_all(0, pA0, pB0);
    dma_all(1, pA1, pB1);
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        read_one(grad::shared_a(0, 3), grad::shared_half(0, 3), x, pA0, pB0);
        read_one(grad::shared_a(0, 0), grad::shared_half(0, 0), x, pA0, pB0);
    }
    int t = 0;
    for (; t + 4 <= nk; t += 4)
        grad::each<4>([&](auto pc) __attribute__((always_inline)) { ktile(pc, t + decltype(pc)::value); });
    grad::each<3>([&](auto pc) __attribute__((always_inline)) {
        if (t + decltype(pc)::value < nk) ktile(pc, t + decltype(pc)::value);
    });
    wait_vmcnt<0>();
    // the compiler does not see the inline-asm MFMAs' latency before the reads of their results
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");

    // accumulator element 4 v4 + e of block (i, j): row 32i + l32, column 32j + 8 v4 + 4g + e
    const int mw = m0 + wm * 128, nw = n0 + wn * 128;
    // block row i stays in AGPRs up to here: otherwise all 256 values are copied
    // to VGPRs before the branch, and spill
    auto row_of = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+a"(acc[i][j]));
    };
    if (p.splitk > 1) {
        float* plane = p.ws + (long long)sk * M * N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = mw + 32 * i + l32;
            row_of(i);
            if (m < M) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int v4 = 0; v4 < 4; ++v4) {
                        const int n = nw + 32 * j + 8 * v4 + 4 * g;
                        const grad::f32x16& a = acc[i][j];
                        // (the width is a multiple of 8)
                        if (n < N)
                            *(f32x4*)(plane + (long long)m * N + n) =
                                f32x4{a[4 * v4], a[4 * v4 + 1], a[4 * v4 + 2], a[4 * v4 + 3]};
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return;
    }
    // through the wave's own 32 KB stage, so that stores write whole rows of 256 bytes
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    QG_LDS uint8_t* img = w == 0 ? pA0 : w == 1 ? pA1 : w == 2 ? pB0 : pB1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        row_of(i);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4) {
                const int r = 32 * i + l32, cbyte = 2 * (32 * j + 8 * v4 + 4 * g);
                const grad::f32x16& a = acc[i][j];
                *(QG_LDS u32x2*)(img + r * 256 + (((cbyte >> 4) ^ (r & 15)) << 4) + (cbyte & 15)) =
                    u32x2{pack_bf16x2(a[4 * v4], a[4 * v4 + 1]), pack_bf16x2(a[4 * v4 + 2], a[4 * v4 + 3])};
            }
        __builtin_amdgcn_sched_barrier(0);
    }
    const int rr = L >> 4, cc = L & 15;
    const int n = nw + cc * 8;
    if (n >= N) return;    // N is a multiple of 8
#pragma unroll 8
    for (int u = 0; u < 32; ++u) {
        const int r = u * 4 + rr, m = mw + r;
        const i32x4 v = *(const QG_LDS i32x4*)(img + r * 256 + ((cc ^ (r & 15)) << 4));
        if (m < M) __builtin_nontemporal_store(v, (i32x4*)(p.c + m * p.ldc + n));
    }
}

}  // namespace qg
