// The 8-bit values of a paged cache (e4m3: a sign, four bits of exponent, three of mantissa, no infinities) and their scales.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>

namespace mk {

// The least power of two s with most <= 448 s, at least 2^-100; most: the bits of a finite fp32 magnitude.
// 448 = 1.75 * 2^8, so of most = f 2^e it is 2^(e - 8) where f <= 1.75, else the next one.
__device__ __forceinline__ float scale_of(uint32_t most)
{
    const int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)((e < -100 ? -100 : e) + 127) << 23);
}

// Two numbers, rounded to nearest even; the first in the low byte. What is no finite number becomes 0x7f, which stands for NaN.
__device__ __forceinline__ uint32_t codes2(float x, float y)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
    return r;
}

__device__ __forceinline__ uint32_t codes4(const float (&x)[8], int at, float by)
{
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = x[at + i] * by;
        if (isinf(y[i])) // (it would be taken for 448)
            y[i] = __int_as_float(0x7fc00000);
    }
    return codes2(y[0], y[1]) | codes2(y[2], y[3]) << 16;
}

// Two codes, as fp16 (which holds all of them exactly).
__device__ __forceinline__ uint32_t halves_of(uint32_t codes)
{
    uint32_t r;
    asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes));
    return r;
}

// Four codes, as two pairs of fp16.
__device__ __forceinline__ uint2 halves_of4(uint32_t codes)
{
    uint2 r;
    asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, low;\n\tcvt.rn.f16x2.e4m3x2 %1, high;\n\t}"
        : "=r"(r.x), "=r"(r.y)
        : "r"(codes));
    return r;
}

// Four codes, each times a power of two.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float by)
{
    const uint32_t low = halves_of(codes & 0xffffu), high = halves_of(codes >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&low)), y = __half22float2(*reinterpret_cast<const __half2*>(&high));
    return codes2(x.x * by, x.y * by) | codes2(y.x * by, y.y * by) << 16;
}

} // namespace mk
