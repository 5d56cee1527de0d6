// Four-bit blocks: conversions shared by the quantiser and the products.
//
// A row of d values is held as E2M1 codes (sign, two exponent bits, one mantissa bit: 0, 0.5,
// 1, 1.5, 2, 3, 4, 6), two a byte with the even value in the low half, and one scale byte per
// block; rows are padded with zero codes to a multiple of 32 values, so that they start on 16
// bytes.
//   mxfp4  blocks of 32, scale 2^(byte - 127); byte 255 = NaN (a block that held NaN or
//          infinity)
//   nvfp4  blocks of 16, scale E4M3 (byte) times a power of two of the row (fp32; NaN if the
//          row held NaN or infinity)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "pa_common.cuh"

namespace pa {
namespace fp4 {

__host__ __device__ constexpr int block_of(int method) { return method == PA_MXFP4 ? 32 : 16; }
__host__ __device__ constexpr int64_t padded(int64_t d) { return (d + 31) / 32 * 32; }

// eight values -> eight codes, value i in bits [4 i, 4 i + 4); nearest, ties to even, largest 6
__device__ __forceinline__ uint32_t codes_of(const float (&v)[8]) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

__device__ __forceinline__ uint8_t e4m3_of(float v) {  // nearest even; callers keep v <= 448
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
    return static_cast<uint8_t>(r & 0xffu);
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {  // exact
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(byte)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(r & 0xffffu)));
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    if (byte == 255u) return CUDART_NAN_F;
    return __uint_as_float(byte == 0u ? 1u << 22 : byte << 23);  // 2^-127 is subnormal
}

}  // namespace fp4
}  // namespace pa
