// The 16-bit and MX (block-scaled 8- and 4-bit) element formats of the serving kernels, and the warp-level products
// that consume them.  An MX block is 32 consecutive elements that share one float8_e8m0 scale byte (value
// 2^(byte - 127), 255 = NaN), elements float8_e4m3fn or float4_e2m1: the format of the MX GEMM's operands.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace pto_b200 {

enum KvFormat : int { kKvF16 = 0, kKvBf16 = 1, kKvMxFp8 = 2, kKvMxFp4 = 3 };

// bytes of a cached row of `d` elements
__host__ __device__ constexpr int kv_row_bytes(int fmt, int d)
{
    return fmt == kKvMxFp8 ? d : (fmt == kKvMxFp4 ? d / 2 : 2 * d);
}

// D (16 x 8 fp32) += A (16 x 16) * B (16 x 8), 16-bit operands in registers
template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1)
{
    if constexpr (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// the same with the accumulator starting at zero
template <bool kBf16>
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                uint32_t b1)
{
    if constexpr (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_16x2(float lo, float hi)
{
    uint32_t d;
    if constexpr (kBf16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    }
    return d;
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack_16x2(uint32_t v)
{
    if constexpr (kBf16) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t mul_16x2(uint32_t a, uint32_t b)
{
    uint32_t d;
    if constexpr (kBf16) {
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    } else {
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    }
    return d;
}

// four e4m3 codes -> two float16 pairs, eight e2m1 codes -> four, the lower code in the low half (exact); the conversions
// take a byte or half of the register where it is
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t &p0, uint32_t &p1)
{
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
}

__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&p)[4])
{
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
        : "r"(w));
}

// two scale bytes (the low 16 bits) as fp32, 255: NaN
__device__ __forceinline__ float2 e8m0x2_to_f32(uint32_t v)
{
    uint32_t d;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, a;\n\t}" : "=r"(d) : "r"(v));
    return make_float2(__uint_as_float(d << 16), __uint_as_float(d & 0xffff0000u));
}

// Scale byte of a block with largest magnitude `amax` (finite): the smallest power of two with amax <= limit * 2^e,
// limit = 448 = 1.75 * 2^8 (e4m3) or 6 = 1.5 * 2^2 (e2m1), so that no element saturates.  e stays in
// [-127, 119] (e4m3) / [-127, 125] (e2m1): above that the largest code's value would leave bfloat16's range.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax, bool fp4)
{
    const uint32_t bits = __float_as_uint(amax);
    const int field = static_cast<int>(bits >> 23); // biased exponent, 0 for subnormals: those end at byte 0
    const uint32_t mant = bits & 0x7fffffu;
    int byte = fp4 ? field - 2 + (mant > 0x400000u ? 1 : 0) : field - 8 + (mant > 0x600000u ? 1 : 0);
    const int most = fp4 ? 252 : 246;
    byte = field == 0 || byte < 0 ? 0 : byte;
    return static_cast<uint32_t>(byte > most ? most : byte);
}

// 2^-e for a scale byte that mx_scale_byte gave
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte)
{
    return __uint_as_float((254u - byte) << 23);
}

} // namespace pto_b200
