// Exponentials and maxima of the attention kernels.
#pragma once

#include "common.cuh"

namespace lyraq {
namespace attn {

__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x of two values on the FMA and ALU pipes: x = n + f with n an integer and f in [-1/2, 1/2]; 2^f from its minimax polynomial of
// degree 5 (Remez exchange on the relative error: 7.5e-8 in exact arithmetic, 2.1e-7 evaluated in fp32, which is what ex2.approx
// has), and n added to the exponent.  x of -127 and below gives the smallest subnormal, which both 16-bit types round to a weight of zero,
// as ex2.approx.ftz does: such a key adds nothing to O, whatever its value row holds.  (Between -126 and -127 the result is some subnormal.)
// NaN and infinity do not come through: the caller looks for them in the row's maximum.
__device__ __forceinline__ float2 ex2_poly(float2 x)
{
    const float  magic = 12582912.0f;   // 1.5 * 2^23: the sum's low mantissa bits are n
    x                  = make_float2(fmaxf(x.x, -127.0f), fmaxf(x.y, -127.0f));
    const float2 t     = add_f32x2(x, make_float2(magic, magic));
    const float2 n     = add_f32x2(t, make_float2(-magic, -magic));
    const float2 f     = fma_f32x2(n, make_float2(-1.0f, -1.0f), x);
    auto two = [](float v) { return make_float2(v, v); };
    float2 q = fma_f32x2(two(0.0013276472454890609f), f, two(0.009675540961325169f));
    q        = fma_f32x2(q, f, two(0.05550713092088699f));
    q        = fma_f32x2(q, f, two(0.24022120237350464f));
    q        = fma_f32x2(q, f, two(0.6931469440460205f));
    q        = fma_f32x2(q, f, two(1.0000001192092896f));
    return make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + __float_as_uint(q.x)), __uint_as_float((__float_as_uint(t.y) << 23) + __float_as_uint(q.y)));
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

}  // namespace attn
}  // namespace lyraq
