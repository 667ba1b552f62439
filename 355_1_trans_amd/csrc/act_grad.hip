// The elementwise half of a linear layer's or gated block's backward pass:
//   linear  dp = dy act'(p)
//   gated   dg = dh u act'(g),  du = dh act(g), in B's row order (16 g, 16 u)
// as bf16 rows padded with zeros to whole 64-deep K-tiles for the products
// that read them, and the column sums of the fp32 values (the bias's
// gradient) as partial rows.  One pass over memory: a wave reads 1 KB of a row,
// 8 columns per lane (gated: 8 features, 16 columns), and walks every fourth
// row of its workgroup's, so that column sums stay in registers; the four
// waves' sums meet in LDS, in wave order.
// The rounding to bf16 is the products' choice: fp32 operands have a sixteenth of
// the bf16 matrix rate, and a second bf16 term of dp would double both products.
// It moves dx and dw by 0.0015 of their norm (0.0023 off in all, their own rounding
// 0.0017).  M = 2048, N = 4096: 12 us, 4.1 TB/s; gated, M = 4096, 2048 features: 19.
#include <algorithm>

#include "act_grad.hpp"
#include "launch.hpp"
#include "layer_math.hpp"

namespace qg {
namespace {

// 8 bf16 values from column c on, zeros from column `cols` on; rows start on any
// element (by elements off the 16 bytes, a call of M = 4096, N = 4092, K = 1024
// took 123 us, now 107)
__device__ __forceinline__ void load8(const uint16_t* p, int c, int cols, float (&v)[8]) {
    if (c + 8 <= cols) {
        const u32x4 r = *(const u32x4_any*)(p + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = bf16_lo(r[e]);
            v[2 * e + 1] = bf16_hi(r[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? bf16_to_f32(p[c + e]) : 0.f;
    }
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
    *(u32x4*)p = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// WRITE: dp is wanted (else only the sums)
template <bool GATED, bool WRITE>
__global__ __launch_bounds__(256) void act_grad_kernel(const ActGradArgs a) {
    constexpr int S = GATED ? 16 : 8;                         // sums per lane
    __shared__ float lds[3][S][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int f = (blockIdx.x * 64 + lane) * 8;               // the columns of dy
    const int n = GATED ? (f >> 4) * 32 + (f & 15) : f;       // of p and dp
    const bool in_row = n < a.ldp;
    float s0[8], s1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s0[e] = s1[e] = 0.f;
    for (long long row = blockIdx.y * 4 + wave; in_row && row < a.rows; row += gridDim.y * 4) {
        float d[8], g[8], y[8];
        load8(a.dy + row * a.lddy, f, a.cols, d);
        if constexpr (GATED) {
            float u[8];
            const uint16_t* pre = a.pre + row * a.ldpre;
            load8(pre, n, a.n, g);
            load8(pre, n + 16, a.n, u);
            activate_slope<8>(a.act, g, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] *= d[e];
                d[e] *= u[e];
            }
            through<8>(a.act, g, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // padding features have no dy: 0, whatever p holds there
                const bool in = f + e < a.cols;
                g[e] = in ? d[e] : 0.f;
                u[e] = in ? y[e] : 0.f;
                s0[e] += g[e];
                s1[e] += u[e];
            }
            if constexpr (WRITE) {
                store8(a.dp + row * a.ldp + n, g);
                store8(a.dp + row * a.ldp + n + 16, u);
            }
        } else {
            if (a.act != kActNone) {
                load8(a.pre + row * a.ldpre, n, a.n, g);
                activate_slope<8>(a.act, g, y);
                through<8>(a.act, g, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = f + e < a.cols ? d[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s0[e] += d[e];
            if constexpr (WRITE) store8(a.dp + row * a.ldp + n, d);
        }
    }
    if (!a.partials) return;
    if (wave) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lds[wave - 1][e][lane] = s0[e];
            if (GATED) lds[wave - 1][S - 8 + e][lane] = s1[e];
        }
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s0[e] += lds[w][e][lane];
            if (GATED) s1[e] += lds[w][S - 8 + e][lane];
        }
    float* out = a.partials + (long long)blockIdx.y * a.n;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (n + e < a.n) out[n + e] = s0[e];
        if (GATED && n + 16 + e < a.n) out[n + 16 + e] = s1[e];
    }
}

}  // namespace

// Workgroups per strip of 64 x 8 columns of dy: with bias sums four per CU in all,
// so that a wave walks a few rows (more only add partial rows), else eight.
int act_grad_parts(int rows, int ldp, bool gated, bool sums, int cus) {
    const int strips = (ldp / (gated ? 16 : 8) + 63) / 64;
    return std::max(1, std::min(rows / 4 + (rows % 4 != 0), (sums ? 4 : 8) * cus / strips));
}

hipError_t launch_act_grad(const ActGradArgs& a, bool write, int cus, hipStream_t s) {
    const dim3 grid((a.ldp / (a.gated ? 16 : 8) + 63) / 64,
                    act_grad_parts(a.rows, a.ldp, a.gated, a.partials != nullptr, cus));
    if (a.gated) act_grad_kernel<true, true><<<grid, 256, 0, s>>>(a);
    else if (write) act_grad_kernel<false, true><<<grid, 256, 0, s>>>(a);
    else act_grad_kernel<false, false><<<grid, 256, 0, s>>>(a);
    trace_launch("act_grad<%s%s>", a.gated ? "gated" : "linear", a.partials ? ",sums" : "");
    return hipGetLastError();
}

}  // namespace qg
