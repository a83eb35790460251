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
    const uint32_t u = __float_as_uint(amax);
    if (u >= 0x7f800000u) return amax;
    if (!pow2)
    {
        // amax / 448 rounded, as a product with the rounded 1 / 448 corrected by its remainder
        constexpr float r = 1.0f / kE4m3Max;
        const float s = amax * r;
        return __fmaf_rn(__fmaf_rn(-s, kE4m3Max, amax), r, s);
    }
    // 448 = 1.75 * 2^8; amax = f * 2^p with 1 <= f < 2: 2^(p-8) while f <= 1.75, else 2^(p-7)
    const uint32_t e = (u >> 23) - 8u + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
    return __uint_as_float(e << 23);
}

// 1 / s to a unit or so in the last place (s is normal, inf or NaN): quotient() corrects what it is used for.
__device__ __forceinline__ float reciprocal(float s)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return r;
}

// x / scale as a float that rounds to the same e4m3 value as the exact quotient, with inv near 1 / scale.  The product is
// corrected once by its remainder, which makes it the rounded quotient; that can still land on the border between
// two e4m3 values (an even float) when the exact one only comes near, so where a remainder is left the last
// bit is made odd, towards the exact quotient.  Seven cheap operations: testing for borders first cost more, since with
// 16-bit inputs every seventh block (a maximum whose bits are a multiple of 7, as 448 is) has exact ties.
__device__ __forceinline__ float quotient(float x, float scale, float inv)
{
    float v = x * inv;
    v = __fmaf_rn(__fmaf_rn(-v, scale, x), inv, v);
    const float rest = __fmaf_rn(-v, scale, x);             // exact: the sign of what the rounding lost
    const uint32_t u = __float_as_uint(v);
    const uint32_t odd = (u + (uint32_t) ((int32_t) (u ^ __float_as_uint(rest)) >> 31)) | 1u;
    return __uint_as_float(rest != 0.0f ? odd : u);
}

// Programmatic dependent launch.  Every kernel of the 8-bit layers lets the next launch of its stream start at once and, before
// it touches what an earlier launch wrote (or what one may still read), waits until all of them have ended; launched
// with launch_after() it is set up while its predecessor runs.
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... Params, class... Args>
int launch_after(const char* what, void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                 const Args&... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (err != cudaSuccess) return set_cuda_error(what, err);
    return check_launch(what);
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

// silu(min(g, L)) * clamp(u, -L, L) in fp32; NaN goes through.  silu(g) = g / (1 + 2^(-g log2 e)) with the approximate
// power and reciprocal (2^-22 each, and the rounding of the argument): the sum is at least 1, so nothing needs scaling, and where
// the power overflows the quotient is the zero that it should be.
__device__ __forceinline__ float clamped_swiglu(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
    return g * reciprocal(1.0f + e) * u;
}

}  // namespace fp8
}  // namespace exl3b
