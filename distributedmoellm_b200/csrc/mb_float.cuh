// Shared by the float experts' kernels: element types, scales and rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "mb_common.cuh"

constexpr int kScaleBlock = MB_SCALE_BLOCK;

// The scale of a group whose largest magnitude is m: m / 448, and 1 where that is 0 (a group of zeros, or of values so
// small that the quotient underflows), as mb_encode_rows does for int8.  NaN counts as no value: m, a maximum by fmaxf, is
// NaN only for a group of nothing else, which has scale 1 then.
__device__ __forceinline__ float e4m3_scale(float m)
{
    m = fmaxf(m, 0.0f);
    const float r = 1.0f / 448.0f, q = m * r;              // see Quotient
    const float s = m > 0x1p-100f && m < 0x1p120f ? fmaf(fmaf(-q, 448.0f, m), r, q) : __fdiv_rn(m, 448.0f);
    return s == 0.0f ? 1.0f : s;
}

// x / s, correctly rounded, for many x and one s: r = 1 / s correctly rounded, then one correction of x * r by its
// remainder x - q s (Markstein, IBM J. Res. Dev. 34, 1990), which has to be exact.  It is a multiple of ulp(q) ulp(s); for
// quotients q from 2^-20 on, ulp(q) >= 2^-43, and s >= 2^-80 has ulp(s) >= 2^-103: at least 2^-146, which f32 holds, as a
// subnormal if need be.  Smaller quotients round to e4m3's zero whatever their last bits.  Scales outside `fast` divide.
struct Quotient {
    float s, r;
    bool fast;
    __device__ __forceinline__ explicit Quotient(float scale)
        : s(scale), r(1.0f / scale), fast(scale > 0x1p-80f && scale < 0x1p100f)
    {
    }
};

// x[i] / s for four values, two at a time in packed arithmetic.
__device__ __forceinline__ void quotient4(float (&x)[4], float s, float r)
{
    uint64_t s2, r2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(-s));
    asm("mov.b64 %0, {%1, %1};" : "=l"(r2) : "f"(r));
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        uint64_t v, q, e;
        float lo, hi;
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x[i]), "f"(x[i + 1]));
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(v), "l"(r2));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(q), "l"(s2), "l"(v));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(e), "l"(r2), "l"(q));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(q));
        x[i] = copysignf(lo, x[i]);                        // the correction turns -0 into +0
        x[i + 1] = copysignf(hi, x[i + 1]);
    }
}

// Nearest e4m3 (ties to even) of two values, as bytes lo, hi.  Saturation matters only where s is subnormal: x / s may
// then round to above 448.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// out[i] = v, rounded once (to nearest even) to the type; not e4m3.
template <int TYPE>
__device__ __forceinline__ void store_out(void* out, int64_t i, float v)
{
    if (TYPE == MB_T_F32)
        reinterpret_cast<float*>(out)[i] = v;
    else if (TYPE == MB_T_BF16)
        reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
    else
        reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
}
