// fp8_common.cuh — e4m3 values with one scale per block of 128: the arithmetic every kernel of the
// 8-bit layers shares.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "exl3_internal.h"

namespace exl3b {
namespace fp8 {

constexpr int kBlock = 128;                     // columns (and weight rows) that share a scale
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxMin = 5.421010862427522e-20f;      // 2^-64: the block maximum a scale is made from is at least this

// The scale of a block whose largest magnitude is `amax`: amax / 448, or the least power of two s with
// amax <= 448 s.  NaN and inf go through (a block that holds one has no finite values).
__device__ __forceinline__ float block_scale(float amax, bool pow2)
{
    amax = amax < kAmaxMin ? kAmaxMin : amax;
    if (!pow2) return __fdiv_rn(amax, kE4m3Max);
    const uint32_t u = __float_as_uint(amax);
    if (u >= 0x7f800000u) return amax;
    // 448 = 1.75 * 2^8; amax = f * 2^p with 1 <= f < 2: 2^(p-8) while f <= 1.75, else 2^(p-7)
    const uint32_t e = (u >> 23) - 8u + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
    return __uint_as_float(e << 23);
}

// x / scale as a float that rounds to the same e4m3 value as the exact quotient does.  A plain rounded
// quotient can land on the border between two e4m3 values that the exact one only comes near; where
// the division is inexact its last bit is made odd, towards the exact quotient (borders have an even one).
static __device__ __noinline__ float quotient_sticky(float x, float scale)
{
    const float q = __fdiv_rn(x, scale);
    const float r = __fmaf_rn(-q, scale, x);                // exact: the sign of what the rounding lost
    uint32_t u = __float_as_uint(q);
    if (r != 0.0f && !(u & 1u) && (u & 0x7fffffffu) < 0x7f800000u && u << 1)
    {
        const bool grow = (r > 0.0f) == (x > 0.0f);         // the exact quotient is further from zero
        u += grow ? 1u : 0xffffffffu;
    }
    return __uint_as_float(u);
}

// The same, cheaply: x * inv is within 2 units in the last place of the quotient, so only products that
// close to a border between e4m3 values (normal ones: their low 20 bits near 0x80000) need the division.
// Below 2^-6 the spacing is that of e4m3's subnormals, with borders elsewhere: those are always divided.
__device__ __forceinline__ float quotient(float x, float scale, float inv)
{
    const float v = x * inv;
    const uint32_t u = __float_as_uint(v);
    const bool border = ((u + 4u - 0x80000u) & 0xfffffu) <= 8u;
    const bool small = (u & 0x7fffffffu) < 0x3c800000u && x != 0.0f;
    return border || small ? quotient_sticky(x, scale) : v;
}

// Two floats to e4m3 (round to nearest even), a in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// silu(min(g, L)) * clamp(u, -L, L) in fp32; NaN goes through.
__device__ __forceinline__ float clamped_swiglu(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
    return __fdividef(g, 1.0f + __expf(-g)) * u;
}

}  // namespace fp8
}  // namespace exl3b
