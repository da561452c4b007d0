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
// ---- the layer kernels' forms, on pairs (fma.rn.f32x2: the FMA pipe's rate at half the issue slots)
using f2 = float2;
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ f2 both(float v) { return {v, v}; }

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_SILU = 2 };  // gs_activation

// GELU from the same formula 7.1.26, arranged for eleven FMA-pipe operations and two MUFU an element:
//   x Phi(x) = max(x, 0) - |x| q / 2,  q = erfc(|x| / sqrt 2) = t poly(t) e,  e = exp(-x^2 / 2)
// and d/dx = Phi(x) + x phi(x), whose exponential is e.  SiLU: x s, s = 1 / (1 + exp(-x)), slope
// s + x s (1 - s).  Both below 7e-7 (1 + |x|) of the exact values; the activation has the same bits with
// and without its slope.
//
// The pair instructions take constants only from register pairs: an Act keeps them there for the kernel's
// whole loop (made opaque, or the compiler forms them anew at every use).
__device__ __forceinline__ f2 pinned(float v) {
    f2 k = both(v);
    asm volatile("" : "+f"(k.x), "+f"(k.y));
    return k;
}
__device__ __forceinline__ float gelu_abs(float x) {  // |x|, at most 16 (q is 0 from there on), NaN kept
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(x)), "f"(16.0f));
    return r;
}
__device__ __forceinline__ float with_sign(float mag, float sgn) {
    return __uint_as_float((__float_as_uint(mag) & 0x7fffffffu) | (__float_as_uint(sgn) & 0x80000000u));
}

template <int ACT, bool SLOPE = false>
struct Act {  // no activation
    __device__ __forceinline__ f2 operator()(f2 x) const { return x; }
    __device__ __forceinline__ f2 operator()(f2 x, f2 &slope) const {
        slope = both(1.0f);
        return x;
    }
};
template <bool SLOPE>
struct Act<ACT_GELU, SLOPE> {
    // |x| scaled to s = |x| sqrt(log2(e) / 2), so e = 2^-(s^2); the polynomial divided by its leading a5
    static constexpr float S = 0.84932180028801905f, A5 = 1.061405429f;
    f2 s_, p, one, b4, b3, b2, b1, h, w, half, f;
    __device__ __forceinline__ Act() {
        s_ = pinned(S);
        p = pinned(0.3275911f * 0.70710678118654752f / S);
        one = pinned(1.0f);
        b4 = pinned(-1.453152027f / A5);
        b3 = pinned(1.421413741f / A5);
        b2 = pinned(-0.284496736f / A5);
        b1 = pinned(0.254829592f / A5);
        h = pinned(-0.5f * A5 / S);
        if (SLOPE) {
            w = pinned(-0.5f * A5);
            half = pinned(0.5f);
            f = pinned(0.39894228040143268f);
        }
    }
    __device__ __forceinline__ f2 value(f2 x, f2 &q, f2 &e) const {
        const f2 s = mul2({gelu_abs(x.x), gelu_abs(x.y)}, s_);
        const f2 d = fma2(s, p, one), m = mul2(s, s);
        const f2 t = {gs_rcp(d.x), gs_rcp(d.y)};
        e = {gs_ex2(-m.x), gs_ex2(-m.y)};
        q = add2(t, b4);
        q = fma2(q, t, b3);
        q = fma2(q, t, b2);
        q = fma2(q, t, b1);
        q = mul2(q, mul2(t, e));  // q / a5
        return fma2(mul2(s, h), q, {fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)});
    }
    __device__ __forceinline__ f2 operator()(f2 x) const {
        f2 q, e;
        return value(x, q, e);
    }
    // Phi(x) = 1/2 + sign(x) (1/2 - q / 2)
    __device__ __forceinline__ f2 operator()(f2 x, f2 &slope) const {
        f2 q, e;
        const f2 y = value(x, q, e), c = fma2(q, w, half);
        slope = fma2(mul2(x, f), e, add2({with_sign(c.x, x.x), with_sign(c.y, x.y)}, half));
        return y;
    }
};
template <bool SLOPE>
struct Act<ACT_SILU, SLOPE> {
    f2 l, one, neg;
    __device__ __forceinline__ Act() {
        l = pinned(-1.4426950408889634f);
        one = pinned(1.0f);
        if (SLOPE) neg = pinned(-1.0f);
    }
    __device__ __forceinline__ f2 sigmoid(f2 x) const {
        const f2 m = mul2(x, l), d = add2({gs_ex2(m.x), gs_ex2(m.y)}, one);
        return {gs_rcp(d.x), gs_rcp(d.y)};
    }
    __device__ __forceinline__ f2 operator()(f2 x) const { return mul2(x, sigmoid(x)); }
    __device__ __forceinline__ f2 operator()(f2 x, f2 &slope) const {
        const f2 s = sigmoid(x), y = mul2(x, s);
        slope = fma2(y, fma2(s, neg, one), s);
        return y;
    }
};

// ---- element types: fp32, bf16, fp16 (gs_dtype); a vector is eight elements
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half &o) { o = __float2half_rn(v); }

// two packed 16-bit elements <-> a pair of floats
__device__ __forceinline__ f2 unpack2(uint32_t w, __nv_bfloat16) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
__device__ __forceinline__ f2 unpack2(uint32_t w, __half) {
    const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&w));
    return {f.x, f.y};
}
__device__ __forceinline__ uint32_t pack2(f2 v, __nv_bfloat16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(f2 v, __half) {
    __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<uint32_t *>(&h);
}
// 16 bytes <-> pairs: four of 16-bit elements, two of fp32
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &p, f2 *v) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = unpack2(w[i], T());
}
template <>
__device__ __forceinline__ void unpack16<float>(const uint4 &p, f2 *v) {
    v[0] = {__uint_as_float(p.x), __uint_as_float(p.y)};
    v[1] = {__uint_as_float(p.z), __uint_as_float(p.w)};
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const f2 *v) {
    return make_uint4(pack2(v[0], T()), pack2(v[1], T()), pack2(v[2], T()), pack2(v[3], T()));
}
template <>
__device__ __forceinline__ uint4 pack16<float>(const f2 *v) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
}
// eight elements as they lie in memory
template <typename T>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, f2 *v) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; k++) unpack16<T>(r.q[k], v + 2 * k);
}
template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const f2 *v) {
    Raw8<T> r;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; k++) r.q[k] = pack16<T>(v + 2 * k);
    return r;
}
// element i of a vector of pairs
__device__ __forceinline__ float &at(f2 *v, int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }
__device__ __forceinline__ float at(const f2 *v, int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }

// ---- launches of one call that follow each other (programmatic dependent launch): the first lets its follower
// be set up early, the follower waits here until the kernel before it has finished and its writes are visible.
// Every block of a follower waits, so a chain's end implies its beginning.
__device__ __forceinline__ void gs_let_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void gs_wait_leader() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// launches kern; follows: as the follower of the launch before it on the stream; cluster: CTAs per cluster
template <typename K, typename... A>
inline void gs_launch(K kern, dim3 grid, int threads, size_t smem, cudaStream_t s, bool follows, int cluster,
                      const A &...args) {
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    c.attrs = at;
    if (follows) {
        at[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[c.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[c.numAttrs].val.clusterDim.x = (unsigned)cluster;
        at[c.numAttrs].val.clusterDim.y = at[c.numAttrs].val.clusterDim.z = 1;
        c.numAttrs++;
    }
    cudaLaunchKernelEx(&c, kern, args...);
}
