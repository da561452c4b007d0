// Activations and 16-byte element vectors shared by the layer kernels (gs_conv.cu, gs_norm.cu,
// gs_linear.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gs_common.cuh"

// GELU(x) = 0.5 x (1 + erf(x / sqrt 2)) with erf from the rational approximation of Abramowitz &
// Stegun, Handbook of Mathematical Functions, formula 7.1.26: for z >= 0,
// erf(z) = 1 - t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-z^2), t = 1 / (1 + p z), |error| <= 1.5e-7.
// 1 + erf(x / sqrt 2) is formed as 2 - q (x >= 0) or q (x < 0), q = t (...) exp(-z^2), so the negative
// tail keeps its relative accuracy.  In fp32 the GELU error stays below 7e-7 absolute over [-12, 12],
// far under the bf16 rounding of the stored activation.
__device__ __forceinline__ float gs_erfc_as(float x, float &e) {  // q above; e = exp(-x^2 / 2)
    const float z = fabsf(x) * 0.70710678118654752f;
    const float t = gs_rcp(fmaf(0.3275911f, z, 1.0f));
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    e = gs_ex2(-(z * z) * 1.4426950408889634f);
    return q * (t * e);
}
__device__ __forceinline__ float gs_gelu(float x) {
    float e;
    const float q = gs_erfc_as(x, e);
    return 0.5f * x * (x >= 0.f ? 2.0f - q : q);
}
// d GELU / dx = Phi(x) + x phi(x): the same exponential serves both terms
__device__ __forceinline__ float gs_gelu_slope(float x) {
    float e;
    const float q = gs_erfc_as(x, e);
    return fmaf(x * 0.39894228040143268f, e, 0.5f * (x >= 0.f ? 2.0f - q : q));
}
// SiLU(x) = x s, s = 1 / (1 + exp(-x)); slope s + x s (1 - s)
__device__ __forceinline__ float gs_sigmoid(float x) { return gs_rcp(1.0f + gs_ex2(-1.4426950408889634f * x)); }

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_SILU = 2 };  // gs_activation

template <int ACT>
__device__ __forceinline__ float gs_act(float x) {
    if (ACT == ACT_GELU) return gs_gelu(x);
    if (ACT == ACT_SILU) return x * gs_sigmoid(x);
    return x;
}
template <int ACT>
__device__ __forceinline__ float gs_act_slope(float x) {
    if (ACT == ACT_GELU) return gs_gelu_slope(x);
    if (ACT == ACT_SILU) {
        const float s = gs_sigmoid(x);
        return fmaf(x * s, 1.0f - s, s);
    }
    return 1.0f;
}
// activation and slope together; the activation has gs_act's bits
template <int ACT>
__device__ __forceinline__ float gs_act_both(float x, float &slope) {
    if (ACT == ACT_GELU) {
        float e;
        const float q = gs_erfc_as(x, e), c = x >= 0.f ? 2.0f - q : q;
        slope = fmaf(x * 0.39894228040143268f, e, 0.5f * c);
        return 0.5f * x * c;
    }
    if (ACT == ACT_SILU) {
        const float s = gs_sigmoid(x), y = x * s;
        slope = fmaf(y, 1.0f - s, s);
        return y;
    }
    slope = 1.0f;
    return x;
}

// ---- element types: fp32, bf16, fp16 (gs_dtype); a vector is 16 bytes
template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half &o) { o = __float2half_rn(v); }

// two packed 16-bit elements <-> two floats
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<__half2 *>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &p, float *v) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpack2(w[i], T());
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void unpack16<float>(const uint4 &p, float *v) {
    v[0] = __uint_as_float(p.x);
    v[1] = __uint_as_float(p.y);
    v[2] = __uint_as_float(p.z);
    v[3] = __uint_as_float(p.w);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float *v) {
    return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
}
template <>
__device__ __forceinline__ uint4 pack16<float>(const float *v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
