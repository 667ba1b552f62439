// The epilogues of a product's C tile, in fp32 before the one rounding:
//   linear: p = c + bias;  y = act(p) + residual
//   gated:  B's rows alternate, 16 of a gate and 16 of an up projection, so
//           that columns n and n + 16 (n % 32 < 16) of c meet in one lane:
//           g, u = c + bias at n and n + 16;  h[16 (n / 32) + n % 16] = act(g) u
// both with p, or g and u, stored as bf16 on request (what a backward pass
// reads; stored before the activation, from the same fp32 values).
//
// The tile kernels' accumulators hold 4 columns of a row per lane, 16 rows
// apart in 16-lane groups; a tile goes through LDS in fp32 and leaves it by
// rows, 8 consecutive columns per lane: 16-byte stores and residual loads, a
// lane's columns the same in every row (bias in registers), and the code of
// the activations once in a loop rather than once per accumulator.
#pragma once
#include <climits>

#include "layer_math.hpp"
#include "tile_args.hpp"

namespace qg {

struct EpiArgs {
    const void* bias;          // [rows of B] or NULL
    const void* residual;      // [M][ld_res] or NULL (linear only)
    uint16_t* pre;             // [M][ld_pre] bf16, as wide as C's columns before the gating, or NULL
    void* out;                 // [M][ld_out]
    long long ld_res, ld_pre, ld_out;
    int m, n;                  // rows; columns of `out`: N, or the features of a gated block
    int act, gated;
    int bias_type, res_type, out_type;
};

// a tile launch with an epilogue
struct TileEpiArgs : TileArgs {
    EpiArgs e;
};

namespace epi {

// Rows start on any element, and global memory takes vector accesses at any
// element's address, so there is one path for every alignment.  Element by
// element, rows off the 16 bytes were bound by the issue of their stores (MXFP4
// M = 6092, N = 15945, K = 2560: 272 us, now 163; MXFP8 M = 2048, N = 4091,
// K = 4096, silu and residual: 54, now 45; the aligned N = 4096: 38), and one
// column per lane, 128 bytes per store, by more of them (485, 66).

// the first `left` (0 to 7) of eight bf16 columns
__device__ __forceinline__ void store_head(uint16_t* p, u32x4 w, int left) {
    uint32_t a = w[0], b = w[1];
    if (left & 4) {
        *(u32x2_any*)p = u32x2{a, b};
        p += 4;
        a = w[2];
        b = w[3];
    }
    if (left & 2) {
        __builtin_memcpy(p, &a, 4);
        p += 2;
        a = b;
    }
    if (left & 1) *p = (uint16_t)a;
}

// V columns at element `at`: vector accesses when `whole`, else the first `left` of them
template <int V>
__device__ __forceinline__ void store_cols(void* p, long long at, int type, const float (&v)[V], bool whole, int left) {
    if (whole) {
        if (type == kTypeBf16) {
            uint16_t* c = static_cast<uint16_t*>(p) + at;
            if constexpr (V == 8)
                *(u32x4_any*)c = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                       pack_bf16x2(v[6], v[7])};
            else if constexpr (V == 1)
                *c = bf16_bits(v[0]);
            else
                *(u32x2_any*)c = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        } else {
            float* c = static_cast<float*>(p) + at;
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                if constexpr (V == 1) c[e] = v[e];
                else *(f32x4_any*)(c + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (e >= left) break;
        if (type == kTypeBf16) static_cast<uint16_t*>(p)[at + e] = bf16_bits(v[e]);
        else static_cast<float*>(p)[at + e] = v[e];
    }
}
// A residual's V columns, loaded apart from their use so that the loads of
// several rows are in flight together; held as loaded
template <int V>
struct Residual {
    uint32_t w[V];
    // EDGE: the columns may end inside these V
    template <bool EDGE>
    __device__ __forceinline__ void load(const EpiArgs& e, int m, int n) {
        if (!e.residual || m >= e.m || (EDGE && n >= e.n)) return;
        const long long at = m * e.ld_res + n;
        if (V == 1 || (EDGE && e.n - n < V)) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                w[i] = n + i < e.n ? __float_as_uint(load_f32(e.residual, at + i, e.res_type)) : 0u;
        } else if (e.res_type == kTypeF32) {
#pragma unroll
            for (int i = 0; i < V; i += 4) *(u32x4*)(w + i) = *(const u32x4_any*)((const float*)e.residual + at + i);
        } else if constexpr (V == 8) {
            *(u32x4*)w = *(const u32x4_any*)((const uint16_t*)e.residual + at);
        } else if constexpr (V == 4) {
            *(u32x2*)w = *(const u32x2_any*)((const uint16_t*)e.residual + at);
        }
    }
    template <bool EDGE>
    __device__ __forceinline__ void add(const EpiArgs& e, int n, float (&v)[V]) const {
        if (!e.residual) return;
        if (V == 1 || e.res_type == kTypeF32 || (EDGE && e.n - n < V)) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                v[2 * i] += bf16_lo(w[i]);
                v[2 * i + 1] += bf16_hi(w[i]);
            }
        }
    }
};
// bias of columns n .. n + V - 1 (0 past `cols`)
template <int V>
__device__ __forceinline__ void bias_cols(const EpiArgs& e, int n, int cols, float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = e.bias && i < cols - n ? load_f32(e.bias, n + i, e.bias_type) : 0.f;
}

// columns n .. n + V - 1 of row m, accumulators v, biases b, residual r
template <int V>
__device__ __forceinline__ void linear(const EpiArgs& e, int m, int n, float (&v)[V], const float (&b)[V],
                                       const Residual<V>& r) {
    if (m >= e.m || n >= e.n) return;
    const int left = e.n - n;
    const bool whole = left >= V;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += b[i];
    if (e.pre) store_cols<V>(e.pre, m * e.ld_pre + n, kTypeBf16, v, whole, left);
    activate<V>(e.act, v);
    r.template add<true>(e, n, v);
    store_cols<V>(e.out, m * e.ld_out + n, e.out_type, v, whole, left);
}
// gate columns n .. n + V - 1 (in B's row order) of row m in g, the up columns 16 further on in u
template <int V>
__device__ __forceinline__ void gated(const EpiArgs& e, int m, int n, float (&g)[V], float (&u)[V],
                                      const float (&bg)[V], const float (&bu)[V]) {
    const int f = (n >> 5) * 16 + (n & 15);
    if (m >= e.m || f >= (e.n + 15) / 16 * 16) return;    // B has whole groups of 16
#pragma unroll
    for (int i = 0; i < V; ++i) {
        g[i] += bg[i];
        u[i] += bu[i];
    }
    if (e.pre) {
        store_cols<V>(e.pre, m * e.ld_pre + n, kTypeBf16, g, true, V);
        store_cols<V>(e.pre, m * e.ld_pre + n + 16, kTypeBf16, u, true, V);
    }
    activate<V>(e.act, g);
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] *= u[i];
    store_cols<V>(e.out, m * e.ld_out + f, e.out_type, g, e.n - f >= V, e.n - f);
}

// A tile of COLS fp32 columns in LDS, rows of COLS * 4 bytes whose 16-byte
// chunks are XORed with the row, so that both the accumulators' writes (16
// rows at a time) and the row reads meet different banks.
template <int COLS>
__device__ __forceinline__ int image_at(int r, int chunk) {
    return r * COLS * 4 + ((chunk ^ (r & (COLS / 4 - 1))) << 4);
}

template <int COLS>
__device__ __forceinline__ void read8(const QG_LDS uint8_t* img, int r, int c, float (&v)[8]) {
    const f32x4 a = *(const QG_LDS f32x4*)(img + image_at<COLS>(r, c >> 2));
    const f32x4 b = *(const QG_LDS f32x4*)(img + image_at<COLS>(r, (c >> 2) + 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}
template <bool EDGE>
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8], int left) {
    const u32x4 w{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    if (!EDGE || left >= 8) *(u32x4_any*)p = w;
    else if (left > 0) store_head(p, w, left);
}

// 64 image rows, row 0 being row m0 and column 0 column n0 of C (in B's row
// order), by one wave, bf16 out; EDGE: the columns may end inside the tile.  One
// loop for each activation, four rows at a time without a branch between their
// LDS reads: with the general code below in their place (every activation and
// edge case inside the row loop) an epilogue took the time of its instruction
// fetches, ~15 us of a 256 x 256 tile's ~115 (MXFP8 M = 8192, N = 7168, K = 8192, no activation 397 us).  Now that is 348, the product
// without an epilogue 340; with a bias 355, with gelu too 393, with a residual 385:
// its tile is read by all CUs at once, and touching its lines over the last K-tiles
// instead slowed those by more (422).  Gated, M = 4096, 8192 features, K = 7168: product
// 326, silu 334, pre-activations saved too 355.
template <int COLS, int ACT, bool EDGE>
__device__ __forceinline__ void bf16_rows(const EpiArgs& e, const QG_LDS uint8_t* img, int L, int m0, int n0) {
    constexpr int U = 4;
    if (e.gated) {
        constexpr int LPR = COLS / 16, RPI = 64 / LPR;
        const int cc = L % LPR, c = (cc >> 1) * 32 + (cc & 1) * 8, n = n0 + c;
        const int f = (n >> 5) * 16 + (n & 15);
        float bg[8], bu[8];
        const int cols = EDGE ? (e.n + 15) / 16 * 32 : INT_MAX;    // B has whole groups of 16
        bias_cols<8>(e, n, cols, bg);
        bias_cols<8>(e, n + 16, cols, bu);
#pragma unroll 1
        for (int r0 = L / LPR; r0 < 64; r0 += 2 * RPI) {
            float g[2][8], u[2][8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                read8<COLS>(img, r0 + x * RPI, c, g[x]);
                read8<COLS>(img, r0 + x * RPI, c + 16, u[x]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int m = m0 + r0 + x * RPI;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    g[x][i] += bg[i];
                    u[x][i] += bu[i];
                }
                if (e.pre && m < e.m && (!EDGE || n < cols)) {
                    store8<false>(e.pre + m * e.ld_pre + n, g[x], 8);
                    store8<false>(e.pre + m * e.ld_pre + n + 16, u[x], 8);
                }
                activate<8>(ACT, g[x]);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[x][i] *= u[x][i];
                if (m < e.m) store8<EDGE>(static_cast<uint16_t*>(e.out) + m * e.ld_out + f, g[x], e.n - f);
            }
        }
        return;
    }
    constexpr int LPR = COLS / 8, RPI = 64 / LPR;
    const int c = (L % LPR) * 8, n = n0 + c;
    float b[8];
    bias_cols<8>(e, n, EDGE ? e.n : INT_MAX, b);
    // a group of U rows' residuals is loaded while the group before is computed
    Residual<8> res[2][U];
    auto load = [&](int k, int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) res[k][u].template load<EDGE>(e, m0 + r0 + u * RPI, n);
    };
    auto group = [&](int k, int r0) __attribute__((always_inline)) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) read8<COLS>(img, r0 + u * RPI, c, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] += b[i];
        if (e.pre) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int m = m0 + r0 + u * RPI;
                if (m < e.m) store8<EDGE>(e.pre + m * e.ld_pre + n, v[u], e.n - n);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) activate<8>(ACT, v[u]);
        if (e.residual) {
#pragma unroll
            for (int u = 0; u < U; ++u) res[k][u].template add<EDGE>(e, n, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int m = m0 + r0 + u * RPI;
            if (m < e.m) store8<EDGE>(static_cast<uint16_t*>(e.out) + m * e.ld_out + n, v[u], e.n - n);
        }
    };
    constexpr int STEP = U * RPI;
    if (!e.residual) {    // half the code to fetch
#pragma unroll 1
        for (int r0 = L / LPR; r0 < 64; r0 += STEP) group(0, r0);
        return;
    }
    load(0, L / LPR);
#pragma unroll 1
    for (int r0 = L / LPR; r0 < 64; r0 += 2 * STEP) {
        load(1, r0 + STEP);
        group(0, r0);
        if (r0 + 2 * STEP < 64) load(0, r0 + 2 * STEP);
        group(1, r0 + STEP);
    }
}

template <int COLS, bool EDGE>
__device__ __forceinline__ void bf16_rows_of(const EpiArgs& e, const QG_LDS uint8_t* img, int L, int m0, int n0) {
    switch (e.act) {
    case kActRelu: return bf16_rows<COLS, kActRelu, EDGE>(e, img, L, m0, n0);
    case kActSilu: return bf16_rows<COLS, kActSilu, EDGE>(e, img, L, m0, n0);
    case kActGelu: return bf16_rows<COLS, kActGelu, EDGE>(e, img, L, m0, n0);
    case kActGeluTanh: return bf16_rows<COLS, kActGeluTanh, EDGE>(e, img, L, m0, n0);
    default: return bf16_rows<COLS, kActNone, EDGE>(e, img, L, m0, n0);
    }
}

template <int COLS>
__device__ __forceinline__ void rows_out(const EpiArgs& e, const QG_LDS uint8_t* img, int L, int m0, int n0) {
    if (e.out_type == kTypeBf16) {
        const int last = e.gated ? (n0 + COLS) / 2 : n0 + COLS;    // whole tiles of a gated block are whole pairs
        return last <= e.n ? bf16_rows_of<COLS, false>(e, img, L, m0, n0) : bf16_rows_of<COLS, true>(e, img, L, m0, n0);
    }
    // fp32 out
    if (e.gated) {
        constexpr int LPR = COLS / 16, RPI = 64 / LPR;
        const int cc = L % LPR, c = (cc >> 1) * 32 + (cc & 1) * 8;
        const int cols = (e.n + 15) / 16 * 32;
        float bg[8], bu[8];
        bias_cols<8>(e, n0 + c, cols, bg);
        bias_cols<8>(e, n0 + c + 16, cols, bu);
#pragma unroll 1
        for (int r = L / LPR; r < 64; r += RPI) {
            float g[8], u[8];
            read8<COLS>(img, r, c, g);
            read8<COLS>(img, r, c + 16, u);
            gated<8>(e, m0 + r, n0 + c, g, u, bg, bu);
        }
    } else {
        constexpr int LPR = COLS / 8, RPI = 64 / LPR;
        const int c = (L % LPR) * 8;
        float b[8];
        bias_cols<8>(e, n0 + c, e.n, b);
#pragma unroll 1
        for (int r = L / LPR; r < 64; r += RPI) {
            Residual<8> res;
            float v[8];
            res.template load<true>(e, m0 + r, n0 + c);
            read8<COLS>(img, r, c, v);
            linear<8>(e, m0 + r, n0 + c, v, b, res);
        }
    }
}

}  // namespace epi

// The slice sum of a K split with an epilogue (epilogue.hip): fp32 planes
// [splitk][M][n_cols] in slice order, n_cols = rows of B.
struct EpiReduceArgs {
    EpiArgs e;
    const float* ws;
    int n_cols, splitk;
};

}  // namespace qg
