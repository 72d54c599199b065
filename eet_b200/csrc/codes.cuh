// 8-bit codes of a paged cache: a row of head_dim values y is kept as codes c and one fp32 scale s, and stands for c * s.
//   int8   c in [-127, 127], s = max |y| / 127
//   e4m3   1 sign, 4 exponent (bias 7), 3 mantissa bits, c in [-448, 448], s = max |y| / 448
// s is 1 for a row of zeros, at least the smallest normal number otherwise, and NaN for a row with a NaN or an infinity, whose
// codes stand for nothing (of e4m3 they are zeros): whoever reads it gets NaN.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace eet {

namespace {

template<typename T, int kCodes>
struct PagedCode {
    using type = uint8_t;
};
template<typename T>
struct PagedCode<T, 0> {
    using type = T;
};

template<int kCodes>
constexpr float kMostCode = kCodes == kCodesInt8 ? 127.0f : 448.0f;

// The scale of a row whose largest magnitude has these bits.
template<int kCodes>
__device__ __forceinline__ float code_scale(uint32_t top)
{
    if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    if (top == 0) return 1.0f;
    return fmaxf(__fdiv_rn(__uint_as_float(top), kMostCode<kCodes>), 1.17549435e-38f);
}

// Codes of 16 values: y / scale rounded once, to nearest, ties to even.  A quotient rounded to 24 bits may fall on the border of two
// codes when the true one lies beside it, which 16-bit values over a scale made from one of them often do (0.2 % of e4m3 codes were
// off by a step).  So the quotient is rounded to odd: where it is not exact, its last bit is set, on the side of the true one, and the
// second rounding cannot be misled.  `inverse` times y, with one step of Newton's iteration, is within an ulp.
template<int kCodes>
__device__ __forceinline__ void quantize16(const float (&y)[16], float scale, uint32_t (&codes)[4])
{
    const float inverse = __fdiv_rn(1.0f, scale);
    float z[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float m = fabsf(y[e]);
        float q = m * inverse;
        q = fmaf(fmaf(-q, scale, m), inverse, q);
        const float rest = fmaf(-q, scale, m);
        uint32_t bits = __float_as_uint(q);
        if (rest != 0.f && !(bits & 1)) bits += rest > 0.f ? 1u : 0xffffffffu;
        z[e] = __uint_as_float(bits | (__float_as_uint(y[e]) & 0x80000000u));
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (kCodes == kCodesInt8) {
            codes[w] = 0;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                // (whole numbers, in two's complement, as the low bits of a sum with 1.5 2^23)
                const uint32_t lo = __float_as_uint(z[4 * w + e] + 12582912.0f), hi = __float_as_uint(z[4 * w + e + 1] + 12582912.0f);
                codes[w] = e == 0 ? __byte_perm(lo, hi, 0x0040) : __byte_perm(codes[w], __byte_perm(lo, hi, 0x0040), 0x5410);
            }
        }
        else {
            uint16_t lo, hi;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(z[4 * w + 1]), "f"(z[4 * w]));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(z[4 * w + 3]), "f"(z[4 * w + 2]));
            // (zeros beside a scale of NaN: a code of NaN would reach rows of a tile that do not see it)
            codes[w] = scale == scale ? (uint32_t)lo | ((uint32_t)hi << 16) : 0u;
        }
    }
}

// Four codes as fp16 pairs {c0, c1}, {c2, c3}, exactly.
//   int8   under the exponent pattern 0x64 a byte b reads as 1024 + b; b is the code + 128
//   e4m3   an instruction for two (with shifts and masks instead, eight instructions for four codes, two sequences of 60000 to 100000
//          positions took 104 us)
template<int kCodes>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    if (kCodes == kCodesInt8) {
        cvt_u8x4_to_f16x4(w ^ 0x80808080u, lo, hi);
    }
    else {
        asm("{\n"
            ".reg .b16 a, b;\n"
            "mov.b32 {a, b}, %2;\n"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n"
            "}\n"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

template<int kCodes>
__device__ __forceinline__ void dequantize16(const uint4& x, float scale, float (&y)[16])
{
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[2];
        codes_to_half<kCodes>(w[i], h[0], h[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            y[4 * i + 2 * e] = f.x * scale;
            y[4 * i + 2 * e + 1] = f.y * scale;
        }
    }
}

// ------------------------------------------------------------------------------------------------ shared memory
// (of a size of zero nothing is read, and zeros are written)
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

}  // namespace

}  // namespace eet
