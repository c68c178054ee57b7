// Element types of activations (fp32, bf16, fp16) and the scalar activation functions, shared by the norm and the
// int4 product kernels.  Every value is widened to fp32 on load and rounded once on store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "common.cuh"

namespace forge {

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float to_f(float v) { return v; }
    static __device__ __forceinline__ float from_f(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
};

// eight consecutive elements, 16-byte aligned (two accesses for fp32)
template <typename T> __device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 raw = *reinterpret_cast<const uint4 *>(p);
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(e[i]);
    }
}
// the same eight elements as they are in memory, for loads that run ahead of their use
template <typename T> struct Raw8 {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const T *e = reinterpret_cast<const T *>(q);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(e[i]);
    }
};
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 raw;
        T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_f(v[i]);
        *reinterpret_cast<uint4 *>(p) = raw;
    }
}

// 1 / (1 + exp(-z)) from the hardware's exponential and reciprocal: about 2^-21 relative (2^-24 |z| from the exponent's
// rounding), against the 2^-9 or 2^-12 of the 16-bit result; 0 where the exact value is below 2^-126.
__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// Phi(z), given e = exp(-z^2 / 2):  Phi(-x) = e t p(t) for x >= 0, t = 1 / (1 + 0.3 x), p the polynomial of degree 7 whose
// largest relative error over x in [0, 14] is least (weighted least squares, fitted for this file: 2^-22.7; 2^-21.1 when it is
// evaluated in fp32, 2^-16.5 with the exponential's own error at x = 8).  1 + erf(z / sqrt 2) loses its bits where z is
// negative, all of them at -5.5.  2048 x 2048 values of dz take 10.0 us (15.0 with erfcf, 11.4 with erff).
__device__ __forceinline__ float normal_cdf(float z, float e) {
    const float t = __fdividef(1.0f, fmaf(0.3f, fabsf(z), 1.0f));
    float p = 0.03567478805780411f;
    p = fmaf(p, t, -0.1572030484676361f);
    p = fmaf(p, t, 0.2063533067703247f);
    p = fmaf(p, t, -0.05368337780237198f);
    p = fmaf(p, t, 0.12856145203113556f);
    p = fmaf(p, t, 0.09991355985403061f);
    p = fmaf(p, t, 0.1207539513707161f);
    p = fmaf(p, t, 0.11962930113077164f);
    const float q = e * (t * p);
    return z < 0.0f ? q : 1.0f - q;
}

template <int ACT> __device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == FORGE_ACT_RELU) return z < 0.0f ? 0.0f : z;      // NaN passes through
    if constexpr (ACT == FORGE_ACT_SILU) return z * sigmoid_fast(z);
    if constexpr (ACT == FORGE_ACT_GELU) return z * normal_cdf(z, __expf(-0.5f * z * z));
    return z;
}
template <int ACT> __device__ __forceinline__ float act_bwd(float z) {
    if constexpr (ACT == FORGE_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == FORGE_ACT_SILU) {
        const float s = sigmoid_fast(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if constexpr (ACT == FORGE_ACT_GELU) {
        const float e = __expf(-0.5f * z * z);
        return normal_cdf(z, e) + z * e * 0.39894228040143268f;
    }
    return 1.0f;
}
__device__ __forceinline__ float act_fwd_rt(int act, float z) {
    switch (act) {
        case FORGE_ACT_RELU: return act_fwd<FORGE_ACT_RELU>(z);
        case FORGE_ACT_SILU: return act_fwd<FORGE_ACT_SILU>(z);
        case FORGE_ACT_GELU: return act_fwd<FORGE_ACT_GELU>(z);
        default: return z;
    }
}

}  // namespace forge
