// Layer norm, forward and backward.
//
// forward, per row of n:  mean = sum x / n,  var = sum (x - mean)^2 / n,
//   rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd w + b
// backward, g = dy w, xh = (x - mean) rstd:
//   dx = rstd (g - sum g / n - xh (sum g xh) / n)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and
// writes dx, once each.  T threads hold a row in registers (E values each, 16
// bytes per load where pitch and base allow), so the squared deviations are
// summed about the mean itself; a workgroup walks rows with its share of w and
// b in registers and the next row's loads issued before the sums of the
// current one.
//
// dw and db: every workgroup keeps fp32 sums of its rows in registers and
// writes one partial row; a second launch adds the partial rows in order, so
// results do not depend on timing.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "act_grad.hpp"
#include "launch.hpp"
#include "layer_math.hpp"
#include "norm.hpp"

// fused where written: the variants of a kernel give the same bits
#pragma clang fp contract(off)

namespace qg {
namespace {

// V consecutive elements as loaded: 16 bytes where n and the rows' starts are
// multiples of them, else one element (V = 1), which costs little: consecutive
// lanes read consecutive elements and the stores are two bytes a lane, yet M =
// 16384, N = 7167 bf16 takes 100 us forward, 144 backward, N = 7168 100 and 139.
// Vectors at any address in their place took 120 and 180.
template <bool F32, int V>
struct Raw;
template <>
struct Raw<true, 4> {
    f32x4 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = *(const f32x4*)((const float*)p + i); }
    __device__ __forceinline__ void to(float (&f)[4]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = v[e];
    }
};
template <>
struct Raw<false, 8> {
    u32x4 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = *(const u32x4*)((const uint16_t*)p + i); }
    __device__ __forceinline__ void to(float (&f)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = bf16_lo(v[e]);
            f[2 * e + 1] = bf16_hi(v[e]);
        }
    }
};
template <>
struct Raw<true, 1> {
    float v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = ((const float*)p)[i]; }
    __device__ __forceinline__ void to(float (&f)[1]) const { f[0] = v; }
};
template <>
struct Raw<false, 1> {
    uint16_t v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = ((const uint16_t*)p)[i]; }
    __device__ __forceinline__ void to(float (&f)[1]) const { f[0] = bf16_to_f32(v); }
};

template <bool F32, int V>
__device__ __forceinline__ void store(void* p, long long i, const float (&f)[V]) {
    if constexpr (F32 && V == 4) {
        *(f32x4*)((float*)p + i) = f32x4{f[0], f[1], f[2], f[3]};
    } else if constexpr (F32) {
        ((float*)p)[i] = f[0];
    } else if constexpr (V == 8) {
        *(u32x4*)((uint16_t*)p + i) =
            u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    } else {
        ((uint16_t*)p)[i] = bf16_bits(f[0]);
    }
}

// Sums of K values over the T threads of a row, the same in all of them.
// Calls alternate between the two halves of `lds`: a thread that writes a
// half again has passed the barrier of the call between, which every thread
// reaches after its reads of that half.
template <int T, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* lds, int& half) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        float* h = lds + half * (2 * W);
        half ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) h[k * W + (threadIdx.x >> 6)] = v[k];
        }
        __syncthreads();
        // the W sums by lanes, not one by one: a row's fixed cost counts beside
        // its 8 - 16 values per thread (M = 16384, N = 7168: forward 101 -> 95 us,
        // with the divisions below)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = first_lanes_sum<W>(h[k * W + (threadIdx.x & (W - 1))]);
    }
}

// s / len with the correctly rounded quotient's first correction (r = 1 / len):
// a constant row's mean is its value
__device__ __forceinline__ float mean_of(float s, float len, float r) {
    const float q = s * r;
    return __builtin_fmaf(__builtin_fmaf(-q, len, s), r, q);
}

// T threads per row (T = 64: a row per wave, four to a workgroup), E values
// per thread in pieces of V.  M = 16384, N = 7168 bf16: 95 us, 4.9 TB/s; a copy
// of as many bytes runs 5.1 - 5.9 TB/s by its grid.
template <bool F32, int V, int T, int E>
__global__ __launch_bounds__(T == 64 ? 256 : T) void norm_kernel(const NormArgs a) {
    constexpr int P = E / V, RPB = T == 64 ? 4 : 1;
    __shared__ float lds[T > 64 ? 4 * (T / 64) : 1];
    const int tid = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int step = gridDim.x * RPB;
    long long row = blockIdx.x * RPB + (T == 64 ? threadIdx.x >> 6 : 0);
    int col[P];
    bool in[P];
    float w[P][V], b[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        col[p] = (p * T + tid) * V;
        in[p] = col[p] < a.n;    // V divides n
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[p][e] = a.weight && in[p] ? load_f32(a.weight, col[p] + e, a.w_type) : 1.f;
            b[p][e] = a.bias && in[p] ? load_f32(a.bias, col[p] + e, a.w_type) : 0.f;
        }
    }
    Raw<F32, V> next[P];
    auto fetch = [&](long long r) __attribute__((always_inline)) {
        if (r >= a.rows) return;
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (in[p]) next[p].load(a.x, r * a.ldx + col[p]);
    };
    fetch(row);
    const float len = (float)a.n, inv = 1.0f / len;
    int half = 0;
    for (; row < a.rows; row += step) {
        float x[P][V], s[1] = {0.f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!in[p]) continue;
            next[p].to(x[p]);
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += x[p][e];
        }
        fetch(row + step);
        row_sums<T, 1>(s, lds, half);
        const float mean = mean_of(s[0], len, inv);
        s[0] = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!in[p]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[p][e] -= mean;
                s[0] = __builtin_fmaf(x[p][e], x[p][e], s[0]);
            }
        }
        row_sums<T, 1>(s, lds, half);
        const float rstd = rsqrtf(__builtin_fmaf(s[0], inv, a.eps));
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!in[p]) continue;
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = __builtin_fmaf(x[p][e] * rstd, w[p][e], b[p][e]);
            store<F32, V>(a.y, row * a.ldy + col[p], y);
        }
        if (a.mean && tid == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// Rows past the registers: three passes over the row (the second and third
// from cache), 1024 threads, one element at a time.  M = 2048 bf16: N = 16400 68
// us, N = 40000 204 (a pass over memory would be 56 at the copy's 5.9 TB/s); backward
// 194 and 571.  A thread adds up to 64 elements in 32 bits and those sums in 64
// (2^21 fp32 additions of one sign would lose 1e-3; 64 bits throughout took 1 - 5%
// longer).  n may be up to 2^31 - 1, past which a signed column counter would go.
template <class Body, class Flush>
__device__ __forceinline__ void long_row(unsigned n, Body&& body, Flush&& flush) {
    for (unsigned c0 = threadIdx.x; c0 < n; c0 += 64 * 1024) {
        const unsigned end = min(n, c0 + 64 * 1024);
        for (unsigned c = c0; c < end; c += 1024) body(c);
        flush();
    }
}
__global__ __launch_bounds__(1024) void norm_long_kernel(const NormArgs a) {
    __shared__ float lds[64];
    int half = 0;
    const unsigned n = a.n;
    const float len = (float)a.n, inv = 1.0f / len;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long x0 = row * a.ldx, y0 = row * a.ldy;
        double sum = 0.0;
        float part = 0.f;
        const auto flush = [&]() __attribute__((always_inline)) {
            sum += part;
            part = 0.f;
        };
        long_row(n, [&](unsigned c) __attribute__((always_inline)) { part += load_f32(a.x, x0 + c, a.x_type); }, flush);
        float s[1] = {(float)sum};
        row_sums<1024, 1>(s, lds, half);
        const float mean = mean_of(s[0], len, inv);
        sum = 0.0;
        long_row(n, [&](unsigned c) __attribute__((always_inline)) {
            const float d = load_f32(a.x, x0 + c, a.x_type) - mean;
            part = __builtin_fmaf(d, d, part);
        }, flush);
        s[0] = (float)sum;
        row_sums<1024, 1>(s, lds, half);
        const float rstd = rsqrtf(__builtin_fmaf(s[0], inv, a.eps));
        for (unsigned c = threadIdx.x; c < n; c += 1024) {
            const float w = a.weight ? load_f32(a.weight, c, a.w_type) : 1.f;
            const float b = a.bias ? load_f32(a.bias, c, a.w_type) : 0.f;
            const float y = __builtin_fmaf((load_f32(a.x, x0 + c, a.x_type) - mean) * rstd, w, b);
            if (a.x_type == kTypeF32) static_cast<float*>(a.y)[y0 + c] = y;
            else static_cast<uint16_t*>(a.y)[y0 + c] = bf16_bits(y);
        }
        if (a.mean && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// T, E, V as in norm_kernel.  SUMS: partial rows of dw and db too.
template <bool F32, int V, int T, int E, int D, bool SUMS>
__global__ __launch_bounds__(T == 64 ? 256 : T) void norm_grad_kernel(const NormGradArgs a) {
    constexpr int P = E / V, RPB = T == 64 ? 4 : 1;
    __shared__ float lds[T > 64 ? 4 * (T / 64) : 1];
    const int tid = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int step = gridDim.x * RPB;
    long long row = blockIdx.x * RPB + (T == 64 ? threadIdx.x >> 6 : 0);
    int col[P];
    bool in[P];
    float w[P][V], dw[P][V], db[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        col[p] = (p * T + tid) * V;
        in[p] = col[p] < a.n;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[p][e] = a.weight && in[p] ? load_f32(a.weight, col[p] + e, a.w_type) : 1.f;
            dw[p][e] = db[p][e] = 0.f;
        }
    }
    Raw<F32, V> nx[D][P], ny[D][P];
    float nmean[D], nrstd[D];
    auto fetch = [&](int d, long long r) __attribute__((always_inline)) {
        if (r >= a.rows) return;
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (in[p]) {
                nx[d][p].load(a.x, r * a.ldx + col[p]);
                ny[d][p].load(a.dy, r * a.lddy + col[p]);
            }
        nmean[d] = a.mean[r];
        nrstd[d] = a.rstd[r];
    };
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(d, row + (long long)d * step);
    const float inv = 1.0f / (float)a.n;
    int half = 0;
    while (row < a.rows) {
#pragma unroll
        for (int d = 0; d < D; ++d, row += step) {
            if (row >= a.rows) break;
            // the row stays as loaded and is converted again for dx: half the registers of two fp32 copies
            const float mean = nmean[d], rstd = nrstd[d];
            auto piece = [&](int p, float(&xh)[V], float(&dy)[V]) __attribute__((always_inline)) {
                nx[d][p].to(xh);
                ny[d][p].to(dy);
#pragma unroll
                for (int e = 0; e < V; ++e) xh[e] = (xh[e] - mean) * rstd;
            };
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if (!in[p]) continue;
                float xh[V], dy[V];
                piece(p, xh, dy);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (SUMS) {
                        dw[p][e] = __builtin_fmaf(dy[e], xh[e], dw[p][e]);
                        db[p][e] += dy[e];
                    }
                    const float g = dy[e] * w[p][e];
                    s[0] += g;
                    s[1] = __builtin_fmaf(g, xh[e], s[1]);
                }
            }
            row_sums<T, 2>(s, lds, half);
            const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if (!in[p]) continue;
                float xh[V], dy[V];
                piece(p, xh, dy);
#pragma unroll
                for (int e = 0; e < V; ++e) dy[e] = rstd * __builtin_fmaf(-xh[e], c1, dy[e] * w[p][e] - c0);
                store<F32, V>(a.dx, row * a.lddx + col[p], dy);
            }
            fetch(d, row + (long long)D * step);
        }
    }
    if constexpr (SUMS) {
        if constexpr (T == 64) {    // the workgroup's four rows of sums meet in wave order
            __shared__ float part[3][2][E][64];
            const int wave = threadIdx.x >> 6;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (wave) {
                        part[wave - 1][0][p * V + e][tid] = dw[p][e];
                        part[wave - 1][1][p * V + e][tid] = db[p][e];
                    }
            __syncthreads();
            if (wave) return;
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dw[p][e] += part[k][0][p * V + e][tid];
                        db[p][e] += part[k][1][p * V + e][tid];
                    }
        }
        float* out = a.partials + 2ll * blockIdx.x * a.n;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!in[p]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                out[col[p] + e] = dw[p][e];
                out[a.n + col[p] + e] = db[p][e];
            }
        }
    }
}

// Long rows: dx in two passes over x and dy ...
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(const NormGradArgs a) {
    __shared__ float lds[64];
    int half = 0;
    const unsigned n = a.n;
    const float inv = 1.0f / (float)a.n;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long x0 = row * a.ldx, g0 = row * a.lddy, d0 = row * a.lddx;
        const float mean = a.mean[row], rstd = a.rstd[row];
        double sg = 0.0, sgx = 0.0;
        float pg = 0.f, pgx = 0.f;
        long_row(n, [&](unsigned c) __attribute__((always_inline)) {
            const float xh = (load_f32(a.x, x0 + c, a.x_type) - mean) * rstd;
            const float g = load_f32(a.dy, g0 + c, a.x_type) * (a.weight ? load_f32(a.weight, c, a.w_type) : 1.f);
            pg += g;
            pgx = __builtin_fmaf(g, xh, pgx);
        }, [&]() __attribute__((always_inline)) {
            sg += pg;
            sgx += pgx;
            pg = pgx = 0.f;
        });
        float s[2] = {(float)sg, (float)sgx};
        row_sums<1024, 2>(s, lds, half);
        const float c0 = s[0] * inv, c1 = s[1] * inv;
        for (unsigned c = threadIdx.x; c < n; c += 1024) {
            const float xh = (load_f32(a.x, x0 + c, a.x_type) - mean) * rstd;
            const float g = load_f32(a.dy, g0 + c, a.x_type) * (a.weight ? load_f32(a.weight, c, a.w_type) : 1.f);
            const float d = rstd * __builtin_fmaf(-xh, c1, g - c0);
            if (a.x_type == kTypeF32) static_cast<float*>(a.dx)[d0 + c] = d;
            else static_cast<uint16_t*>(a.dx)[d0 + c] = bf16_bits(d);
        }
    }
}
// ... and partial rows of dw and db by columns: block y takes every
// gridDim.y-th row.
__global__ __launch_bounds__(256) void norm_grad_cols_kernel(const NormGradArgs a) {
    const long long n = a.n, c = blockIdx.x * 256ll + threadIdx.x;    // 2 n columns pass 32 bits
    if (c >= n) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float xh = (load_f32(a.x, row * a.ldx + c, a.x_type) - a.mean[row]) * a.rstd[row];
        const float g = load_f32(a.dy, row * a.lddy + c, a.x_type);
        dw = __builtin_fmaf(g, xh, dw);
        db += g;
    }
    float* out = a.partials + 2 * blockIdx.y * n;
    out[c] = dw;
    out[n + c] = db;
}

// Adds partial rows, 64 columns per workgroup: wave g of 16 adds rows g,
// g + 16, ... in order, then the 16 sums meet in wave order.
__global__ __launch_bounds__(1024) void partial_sum_kernel(const PartialSumArgs a, long long first) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long long c = first + blockIdx.x * 64ll + lane;
    float s = 0.f;
    if (c < a.width) {
        int r = g;
        for (; r + 112 < a.parts; r += 128) {    // eight loads in flight
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = a.partials[(r + 16 * u) * a.width + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; r < a.parts; r += 16) s += a.partials[r * a.width + c];
    }
    lds[g][lane] = s;
    __syncthreads();
    if (g != 0 || c >= a.width) return;
#pragma unroll
    for (int u = 1; u < 16; ++u) s += lds[u][lane];
    void* out = c < a.split ? a.out0 : a.out1;
    const long long i = c < a.split ? c : c - a.split;
    if (!out) return;
    if (a.type == kTypeF32) static_cast<float*>(out)[i] = s;
    else static_cast<uint16_t*>(out)[i] = bf16_bits(s);
}

bool aligned16(const void* p, long long ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem) % 16 == 0;
}

// PER workgroups per CU walk the rows.  The threads of a row, its values per
// thread and PER were timed over T = 64 - 1024, E = 8 - 32, PER = 1 - 8 at
// M = 16384 bf16 (us): N = 7168 T 1024 E 8 PER 2 94.9, PER 1 108, 3 104, T 512
// E 16 PER 3 95.8, 4 125, T 256 E 32 133 at best; N = 2048 T 256 E 8 PER 4 25.3,
// PER 2 28.2, 6 26.2; N = 1024 T 64 E 16 16.4 (T 256 22.5); M = 8192, N = 16384
// T 1024 E 16 PER 1 110 (2 115, T 512 E 32 137).
template <bool F32, int V, int T, int E, int PER>
hipError_t go(const NormArgs& a, int cus, hipStream_t s) {
    constexpr int rpb = T == 64 ? 4 : 1, threads = T == 64 ? 256 : T;
    const int blocks = std::min(a.rows / rpb + (a.rows % rpb != 0), cus * PER);
    norm_kernel<F32, V, T, E><<<blocks, threads, 0, s>>>(a);
    trace_launch("norm<%s,x%d,t%d,e%d>", F32 ? "fp32" : "bf16", V, T, E);
    return hipGetLastError();
}

template <bool F32, int V>
hipError_t by_length(const NormArgs& a, int cus, hipStream_t s) {
    if (a.n <= 512) return go<F32, V, 64, 8, 2>(a, cus, s);
    if (a.n <= 1024) return go<F32, V, 64, 16, 2>(a, cus, s);
    if (a.n <= 2048) return go<F32, V, 256, 8, 4>(a, cus, s);
    if (a.n <= 4096) return go<F32, V, 512, 8, 3>(a, cus, s);
    if (a.n <= 8192) return go<F32, V, 1024, 8, 2>(a, cus, s);
    return go<F32, V, 1024, 16, 1>(a, cus, s);
}

// The same for the gradients, D rows of loads in flight: each workgroup more
// costs a partial row to write and add.  M = 8192 bf16 (us, kernel + sum):
// N = 7168 T 1024 E 8 PER 1 D 2 75.2 + 2.7 (D 1 77.7, PER 2 86.4 + 3.2, T 512
// E 16 75.1); N = 4096 T 512 E 8 D 2 38.0 (PER 2 38.7 + 3.1); N = 2048 T 256 E 8
// PER 2 23.3 + 3.1 (PER 1 30.8, 4 27.7 + 4.1; with few rows PER 1: M = 777, N =
// 1537 fp32 12.8 -> 12.2 a pass); M = 4096, N = 16384 T 1024 E 16 D 1 100 (D 2 spills: 182).
int grad_per(int rows, int n, int cus) { return n <= 2048 && rows >= 8 * cus ? 2 : 1; }

template <bool F32, int V, int T, int E, int D>
hipError_t grad_go(const NormGradArgs& a, int parts, hipStream_t s) {
    constexpr int threads = T == 64 ? 256 : T;
    const bool sums = a.dweight || a.dbias;
    if (sums) norm_grad_kernel<F32, V, T, E, D, true><<<parts, threads, 0, s>>>(a);
    else norm_grad_kernel<F32, V, T, E, D, false><<<parts, threads, 0, s>>>(a);
    trace_launch("norm_grad<%s,x%d,t%d,e%d%s>", F32 ? "fp32" : "bf16", V, T, E, sums ? ",sums" : "");
    return hipGetLastError();
}

template <bool F32, int V>
hipError_t grad_by_length(const NormGradArgs& a, int parts, hipStream_t s) {
    if (a.n <= 512) return grad_go<F32, V, 64, 8, 1>(a, parts, s);
    if (a.n <= 2048) return grad_go<F32, V, 256, 8, 1>(a, parts, s);
    if (a.n <= 4096) return grad_go<F32, V, 512, 8, 2>(a, parts, s);
    if (a.n <= 8192) return grad_go<F32, V, 1024, 8, 2>(a, parts, s);
    return grad_go<F32, V, 1024, 16, 1>(a, parts, s);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int cus, hipStream_t s) {
    if (a.n > kNormRegs) {
        norm_long_kernel<<<std::min(a.rows, 2 * cus), 1024, 0, s>>>(a);
        trace_launch("norm_long<%s>", a.x_type == kTypeF32 ? "fp32" : "bf16");
        return hipGetLastError();
    }
    const int elem = a.x_type == kTypeF32 ? 4 : 2;
    const bool vec = a.n % (16 / elem) == 0 && aligned16(a.x, a.ldx, elem) && aligned16(a.y, a.ldy, elem);
    if (a.x_type == kTypeF32) return vec ? by_length<true, 4>(a, cus, s) : by_length<true, 1>(a, cus, s);
    return vec ? by_length<false, 8>(a, cus, s) : by_length<false, 1>(a, cus, s);
}

int norm_grad_partials(int rows, int n, int cus) {
    const int blocks = n <= 512 ? rows / 4 + (rows % 4 != 0) : rows;    // a row per wave, or per workgroup
    return std::min(blocks, grad_per(rows, n, cus) * cus);
}

hipError_t launch_norm_grad(const NormGradArgs& a, int cus, hipStream_t s) {
    const int parts = norm_grad_partials(a.rows, a.n, cus);
    const bool sums = a.dweight || a.dbias;
    hipError_t st;
    if (a.n > kNormRegs) {
        norm_grad_long_kernel<<<std::min(a.rows, 2 * cus), 1024, 0, s>>>(a);
        trace_launch("norm_grad_long<%s>", a.x_type == kTypeF32 ? "fp32" : "bf16");
        st = hipGetLastError();
        if (st != hipSuccess || !sums) return st;
        norm_grad_cols_kernel<<<dim3((unsigned)((a.n + 255ll) / 256), parts), 256, 0, s>>>(a);
        trace_launch("norm_grad_cols");
        st = hipGetLastError();
    } else {
        const int elem = a.x_type == kTypeF32 ? 4 : 2;
        const bool vec = a.n % (16 / elem) == 0 && aligned16(a.x, a.ldx, elem) && aligned16(a.dy, a.lddy, elem) &&
                         aligned16(a.dx, a.lddx, elem);
        if (a.x_type == kTypeF32) st = vec ? grad_by_length<true, 4>(a, parts, s) : grad_by_length<true, 1>(a, parts, s);
        else st = vec ? grad_by_length<false, 8>(a, parts, s) : grad_by_length<false, 1>(a, parts, s);
    }
    if (st != hipSuccess || !sums) return st;
    return launch_partial_sum({a.partials, parts, 2ll * a.n, a.n, a.dweight, a.dbias, a.w_type}, s);
}

hipError_t launch_partial_sum(const PartialSumArgs& a, hipStream_t s) {
    const long long blocks = (a.width + 63) / 64;
    if (blocks <= 0) return hipErrorInvalidValue;
    constexpr long long kMost = (1 << 22) - 1;    // workgroups of a launch: its threads fit 32 bits
    for (long long b = 0; b < blocks; b += kMost) {
        partial_sum_kernel<<<(unsigned)std::min(blocks - b, kMost), 1024, 0, s>>>(a, 64 * b);
        trace_launch("partial_sum");
        const hipError_t st = hipGetLastError();
        if (st != hipSuccess) return st;
    }
    return hipSuccess;
}

}  // namespace qg
