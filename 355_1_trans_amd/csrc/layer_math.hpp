// Arithmetic shared by the kernels of the layer around the products: sums over
// a wave, activations and their slopes, bf16 loads.
#pragma once
#include "common.hpp"

namespace qg {

// vectors at any element's address: global memory takes them
using u32x4_any = u32x4 __attribute__((aligned(2)));
using u32x2_any = u32x2 __attribute__((aligned(2)));
using f32x4_any = f32x4 __attribute__((aligned(4)));

// Element types of activations and weights (QGEMM_IN_* in qgemm.h).
enum : int { kTypeF32 = 0, kTypeBf16 = 1 };

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float load_f32(const void* p, long long i, int type) {
    return type == kTypeF32 ? static_cast<const float*>(p)[i] : bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// v + the lanes that a DPP control selects (0 where it selects none)
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Sum over the 64 lanes, the same in every lane: prefix sums within rows of
// 16 (row_shr 1, 2, 4, 8), row totals passed on (row_bcast 15 and 31), then
// lane 63's value.
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0x111>(v);
    v = dpp_add<0x112>(v);
    v = dpp_add<0x114>(v);
    v = dpp_add<0x118>(v);
    v = dpp_add<0x142>(v);
    v = dpp_add<0x143>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sum over lanes 0 .. W - 1 (W = 4, 8 or 16) of a value that repeats every W
// lanes, the same in every lane: rotations within rows of 16
template <int W>
__device__ __forceinline__ float first_lanes_sum(float v) {
    static_assert(W == 4 || W == 8 || W == 16, "within one DPP row");
    v = dpp_add<0x121>(v);                              // row_ror:1
    v = dpp_add<0x122>(v);                              // row_ror:2
    if constexpr (W > 4) v = dpp_add<0x124>(v);
    if constexpr (W > 8) v = dpp_add<0x128>(v);
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// Activations (QGEMM_ACT_* in qgemm.h)
enum : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4, kActCount = 5 };

// 1 / (1 + e^-x): e^-x overflows to infinity for large -x, and 1 / inf = 0
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// gelu_tanh: 0.5 v (1 + tanh z) = v sigmoid(2 z), z = sqrt(2 / pi) (v + 0.044715 v^3)
constexpr float kGeluC = 0.79788456080286535588f, kGeluA = 0.044715f;
// 1 / sqrt(2 pi): the normal density at 0
constexpr float kPhi0 = 0.39894228040143267794f;

// The normal distribution function Phi(v) by its upper tail Q(|v|) = e^(-v^2 / 2)
// g(|v|), g(x) = e^(x^2 / 2) Q(x), which falls from 1/2 like 1 / x: g = t P(t), t =
// 1 / (1 + 0.3 x), P the polynomial of degree 7 with the least largest relative
// error over x <= 13.6 (reweighted least squares in 64 bits), 1.5e-7; 6e-7 with
// the fp32 steps.  So a negative v's Phi is right relative to itself: beside that
// 6e-7 it has the exponential's error, about v^2 2^-24.  (An approximation of erfc
// within an absolute 1.5e-7 takes three steps less and is 5e-5 off at v = -3, 1.6e-3
// at -5; the library's erff, 1 + erf aside, takes about twice the instructions.)
// Past 13.1 e^(-v^2 / 2) leaves fp32's normal range.  e: e^(-v^2 / 2).
__device__ __forceinline__ float normal_cdf(float v, float e) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, fabsf(v), 1.0f));
    float p = 0.0358798530f;
    p = __builtin_fmaf(p, t, -0.1580590818f);
    p = __builtin_fmaf(p, t, 0.2078313338f);
    p = __builtin_fmaf(p, t, -0.0550468021f);
    p = __builtin_fmaf(p, t, 0.1292845613f);
    p = __builtin_fmaf(p, t, 0.0996938194f);
    p = __builtin_fmaf(p, t, 0.1207892620f);
    p = __builtin_fmaf(p, t, 0.1196269884f);
    const float q = p * t * e;
    return v < 0.f ? q : 1.0f - q;
}
__device__ __forceinline__ float normal_exp(float v) { return __expf(-0.5f * v * v); }

// v[i] = act(v[i]); `act` is uniform, so the branch is outside the elements
template <int E>
__device__ __forceinline__ void activate(int act, float (&v)[E]) {
    switch (act) {
    case kActRelu:
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];    // NaN stays
        break;
    case kActSilu:
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] *= sigmoid(v[i]);
        break;
    case kActGelu:
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] *= normal_cdf(v[i], normal_exp(v[i]));
        break;
    case kActGeluTanh:
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] *= sigmoid(2.0f * kGeluC * (v[i] + kGeluA * v[i] * v[i] * v[i]));
        break;
    default:
        break;
    }
}

// y[i] = act(v[i]), v[i] = act'(v[i])
template <int E>
__device__ __forceinline__ void activate_slope(int act, float (&v)[E], float (&y)[E]) {
    switch (act) {
    case kActRelu:
#pragma unroll
        for (int i = 0; i < E; ++i) {
            y[i] = v[i] < 0.f ? 0.f : v[i];
            v[i] = v[i] <= 0.f ? 0.f : 1.f;    // NaN is active, as in y
        }
        break;
    case kActSilu:
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float s = sigmoid(v[i]);
            y[i] = v[i] * s;
            v[i] = s * (1.0f + v[i] * (1.0f - s));
        }
        break;
    case kActGelu:
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float e = normal_exp(v[i]), cdf = normal_cdf(v[i], e);
            y[i] = v[i] * cdf;
            v[i] = cdf + v[i] * kPhi0 * e;
        }
        break;
    case kActGeluTanh:
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // bounded: past |v| = 1.8e19 the square would be infinite, and s (1 - s) = 0 times it NaN
            const float x2 = fminf(v[i] * v[i], 1e30f);
            const float s = sigmoid(2.0f * kGeluC * v[i] * (1.0f + kGeluA * x2));
            y[i] = v[i] * s;
            v[i] = s + v[i] * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * x2);
        }
        break;
    default:
#pragma unroll
        for (int i = 0; i < E; ++i) {
            y[i] = v[i];
            v[i] = 1.f;
        }
        break;
    }
}

// dy[i] act'(v[i]) from the slopes; relu passes dy on or stops it, also an infinite
// or NaN one (a choice per element inside one loop for all activations cost 1 us of
// a call's 125)
template <int E>
__device__ __forceinline__ void through(int act, const float (&slope)[E], float (&dy)[E]) {
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < E; ++i) dy[i] = slope[i] != 0.f ? dy[i] : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) dy[i] *= slope[i];
    }
}

}  // namespace qg
