// Rows of values to 4-bit blocks (fp4.cuh has the formats) and back.
//
// mxfp4: the scale of a block is 2^(floor(log2 max|v|) - 2), the largest E2M1 exponent being
// 2; dividing by it is exact, values above 6 saturate.  nvfp4: the row's scale s is the least
// power of two with max|v| <= 6 * 448 s, a block's is max|v| / (6 s) rounded to E4M3.  s is a
// power of two so that no rounding of it decides how a value next to a border is coded: the
// quotients are those of the definition, up to fp32's own half step.  Rows are independent of
// one another: a query's codes do not depend on the batch it comes in.
#include "fp4.cuh"
#include "grouped.cuh"

namespace pa {
namespace fp4 {

constexpr int kWarps = 8;  // rows per CTA, a warp each

// A lane has eight consecutive values of a chunk of 256, a block is four lanes (mxfp4) or two;
// CHUNKS (1 to 4) chunks are loaded before any is worked on.  Rows are read once where they fit
// those registers (or the method needs no maximum of the row), else a second time from the caches.
// Eight values as they are in memory: 32 bytes of fp32, 16 of the others.
template <typename T> struct Raw { uint32_t w[2 * sizeof(T)]; };

template <typename T>
__device__ __forceinline__ void load8(Raw<T> &raw, const T *row, int64_t at, int64_t d, bool vec) {
    if (vec && at + 8 <= d) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(row + at) + i);
            raw.w[4 * i] = a.x; raw.w[4 * i + 1] = a.y; raw.w[4 * i + 2] = a.z; raw.w[4 * i + 3] = a.w;
        }
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            raw.w[j] = at + j < d ? __ldg(reinterpret_cast<const uint32_t *>(row) + at + j) : 0u;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h =
                at + j < d ? __ldg(reinterpret_cast<const uint16_t *>(row) + at + j) : 0u;
            raw.w[j / 2] = j % 2 ? raw.w[j / 2] | (h << 16) : h;
        }
    }
}

__device__ __forceinline__ void values8(float (&v)[8], const Raw<float> &raw) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw.w[j]);
}
__device__ __forceinline__ void values8(float (&v)[8], const Raw<__nv_bfloat16> &raw) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(raw.w[j] << 16);
        v[2 * j + 1] = __uint_as_float(raw.w[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void values8(float (&v)[8], const Raw<__half> &raw) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&raw.w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
}

// Bits of the largest magnitude, as fp32: magnitudes order like their bits in every type, NaN above
// infinity above the rest, so 16-bit ones are compared two at a time.
__device__ __forceinline__ uint32_t top_bits(const Raw<float> &raw) {
    uint32_t t = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = max(t, raw.w[j] & 0x7fffffffu);
    return t;
}
template <typename T> __device__ __forceinline__ uint32_t top_bits(const Raw<T> &raw) {
    uint32_t t = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) t = __vmaxu2(t, raw.w[j] & 0x7fff7fffu);
    t = max(t & 0xffffu, t >> 16);
    if (grouped::is_bf16<T>()) return t << 16;
    const float f = __half2float(__ushort_as_half(static_cast<unsigned short>(t)));
    return __float_as_uint(f);
}

// v / step as codes.  fp32 values are divided.  16-bit ones have at most 11 significant bits and
// step has four, so that a quotient is a border between two codes (a multiple of 1/4) exactly or at
// least 2^-13 away from it: a product with the reciprocal, off by 2^-22 of its value, is rounded
// to a multiple of 2^-14 by adding and subtracting 768, which lands on the border in the first
// case and stays off it in the other, for two instructions a value.  The subtraction makes a +0 of what
// becomes 0; signs come from the values, so that codes do not depend on their type.
__device__ __forceinline__ uint32_t signs_of(const Raw<float> &) { return 0; }  // not lost
template <typename T> __device__ __forceinline__ uint32_t signs_of(const Raw<T> &raw) {
    // high bytes of the even and the odd values
    const uint32_t a = __byte_perm(raw.w[0], raw.w[1], 0x7351),
                   b = __byte_perm(raw.w[2], raw.w[3], 0x7351);
    const uint32_t even = __byte_perm(a, b, 0x5410), odd = __byte_perm(a, b, 0x7632);
    return (even >> 4 & 0x08080808u) | (odd & 0x80808080u);
}
template <typename T>
__device__ __forceinline__ uint32_t codes_by(float (&v)[8], float step, const Raw<T> &raw) {
    if (sizeof(T) == 2 && step >= 1.1754944e-38f) {  // a reciprocal that does not overflow
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));  // step < 2^126
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(__fmaf_rn(v[j], inv, 768.0f), -768.0f);
        return codes_of(v) | signs_of(raw);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = step > 0.0f ? __fdiv_rn(v[j], step) : 0.0f;
    return codes_of(v);
}

// E4M3 of top / 6: borders have five significant bits, so the same holds of a product with 1 / 6,
// here rounded to 18 bits behind the leading one
template <typename T> __device__ __forceinline__ uint32_t scale_of(float top) {
    float ratio;
    if (sizeof(T) == 2)
        ratio = __uint_as_float((__float_as_uint(__fmul_rn(top, 1.0f / 6.0f)) + 16u) & ~31u);
    else
        ratio = __fdiv_rn(top, 6.0f);
    return e4m3_of(fminf(ratio, 448.0f));
}

template <typename T, int METHOD, int CHUNKS>
__global__ void __launch_bounds__(32 * kWarps)
quantize_kernel(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                float *__restrict__ row_scale, const T *__restrict__ x, int64_t rows, int64_t d,
                int64_t ldx, bool vec) {
    const int lane = threadIdx.x & 31;
    const int64_t r = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const T *row = x + r * ldx;
    const int64_t dp = padded(d);
    constexpr int kLanes = METHOD == PA_MXFP4 ? 4 : 2;  // lanes of a block
    uint32_t *to = reinterpret_cast<uint32_t *>(codes + r * (dp / 2)) + lane;
    uint8_t *to_scale = scales + r * (dp / (8 * kLanes)) + lane / kLanes;
    Raw<T> raw[CHUNKS];
    float s = 1.0f, s_inv = 1.0f;
    if (METHOD == PA_NVFP4) {
        uint32_t top = 0;
        for (int64_t a0 = 0; a0 < dp; a0 += 256 * CHUNKS) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) load8(raw[c], row, a0 + 256 * c + 8 * lane, d, vec);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) top = max(top, top_bits(raw[c]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        // 6 * 448 = 1.3125 * 2^11; the power is in [-126, 117]
        const int power = max(static_cast<int>(top >> 23) - 127 - 11 + ((top & 0x7fffffu) > 0x280000u),
                              -126);
        const bool fine = top < 0x7f800000u;
        s = fine ? __uint_as_float(static_cast<uint32_t>(power + 127) << 23) : CUDART_NAN_F;
        s_inv = fine ? __uint_as_float(static_cast<uint32_t>(127 - power) << 23) : CUDART_NAN_F;
        if (lane == 0) row_scale[r] = s;
    }
    for (int64_t a0 = 0; a0 < dp; a0 += 256 * CHUNKS) {
        if (METHOD == PA_MXFP4 || dp > 256 * CHUNKS) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) load8(raw[c], row, a0 + 256 * c + 8 * lane, d, vec);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t at = a0 + 256 * c + 8 * lane;
            if (a0 + 256 * c >= dp) break;  // uniform
            uint32_t top = top_bits(raw[c]);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            float v[8];
            values8(v, raw[c]);
            uint32_t byte, code;
            if (METHOD == PA_MXFP4) {
                const uint32_t e = top >> 23;
                byte = e > 2u ? e - 2u : 0u;
                const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], inv);
                code = codes_of(v);
                if (e == 255u) { byte = 255u; code = 0u; }
            } else {
                byte = scale_of<T>(__fmul_rn(__uint_as_float(top), s_inv));
                code = codes_by(v, __fmul_rn(e4m3_value(byte), s), raw[c]);
                if (!(s > 0.0f)) { byte = 0u; code = 0u; }  // NaN: the row's scale says it
            }
            if (at < dp) {
                to[(a0 + 256 * c) / 8] = code;
                if (lane % kLanes == 0) to_scale[(a0 + 256 * c) / (8 * kLanes)] = byte;
            }
        }
    }
}

// four codes -> four values of their block (exact: two significant bits times at most four)
__device__ __forceinline__ float4 values_of(uint32_t code, float scale) {
    uint32_t lo, hi;
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %2;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(code));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)),
                 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return make_float4(__fmul_rn(a.x, scale), __fmul_rn(a.y, scale), __fmul_rn(b.x, scale),
                       __fmul_rn(b.y, scale));
}

// A warp has a row; it loads 256 codes (4 bytes a lane) at a time and hands them around so that
// the lanes store 16 bytes side by side.
template <int METHOD, int CHUNKS>
__global__ void __launch_bounds__(32 * kWarps)
dequantize_kernel(float *__restrict__ out, const uint8_t *__restrict__ codes,
                  const uint8_t *__restrict__ scales, const float *__restrict__ row_scale,
                  int64_t rows, int64_t d, bool vec) {
    const int lane = threadIdx.x & 31;
    const int64_t r = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int64_t dp = padded(d);
    constexpr int kLanes = METHOD == PA_MXFP4 ? 4 : 2;
    const uint32_t *from = reinterpret_cast<const uint32_t *>(codes + r * (dp / 2)) + lane;
    const uint8_t *from_scale = scales + r * (dp / (8 * kLanes)) + lane / kLanes;
    const float s = METHOD == PA_NVFP4 ? row_scale[r] : 1.0f;
    float *to = out + r * d + 4 * lane;
    for (int64_t a0 = 0; a0 < d; a0 += 256 * CHUNKS) {
        uint32_t code[CHUNKS], byte[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t a = a0 + 256 * c;
            const bool live = a + 8 * lane < dp;
            code[c] = live ? __ldg(from + a / 8) : 0u;
            byte[c] = live ? __ldg(from_scale + a / (8 * kLanes)) : 0u;
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t a = a0 + 256 * c;
            if (a >= d) break;  // uniform
            const float scale = METHOD == PA_MXFP4 ? e8m0_value(byte[c]) : e4m3_value(byte[c]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int src = 16 * k + lane / 2;
                const uint32_t mine = __shfl_sync(0xffffffffu, code[c], src) >> (16 * (lane & 1));
                const float by = __shfl_sync(0xffffffffu, scale, src);
                float4 v = values_of(mine, by);
                if (METHOD == PA_NVFP4) {
                    v.x = __fmul_rn(v.x, s); v.y = __fmul_rn(v.y, s);
                    v.z = __fmul_rn(v.z, s); v.w = __fmul_rn(v.w, s);
                }
                const int64_t at = a + 128 * k + 4 * lane;
                float *p = to + a + 128 * k;
                if (vec && at < d) {
                    *reinterpret_cast<float4 *>(p) = v;
                } else {
                    if (at < d) p[0] = v.x;
                    if (at + 1 < d) p[1] = v.y;
                    if (at + 2 < d) p[2] = v.z;
                    if (at + 3 < d) p[3] = v.w;
                }
            }
        }
    }
}

// chunks of 256 values a row has, at most 4
int chunks_of(int64_t d) { return static_cast<int>(d > 768 ? 4 : (d + 255) / 256); }

template <typename T>
int quantize_launch(uint8_t *codes, uint8_t *scales, float *row_scale, const void *x, int64_t rows,
                    int64_t d, int64_t ldx, int method, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
    const bool vec = aligned16(x) && ldx * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    auto go = [&](auto kernel) {
        kernel<<<grid, 32 * kWarps, 0, s>>>(codes, scales, row_scale, static_cast<const T *>(x),
                                            rows, d, ldx, vec);
    };
    const int chunks = chunks_of(d);
    if (method == PA_MXFP4)
        chunks == 1   ? go(quantize_kernel<T, PA_MXFP4, 1>)
        : chunks == 2 ? go(quantize_kernel<T, PA_MXFP4, 2>)
        : chunks == 3 ? go(quantize_kernel<T, PA_MXFP4, 3>)
                      : go(quantize_kernel<T, PA_MXFP4, 4>);
    else
        chunks == 1   ? go(quantize_kernel<T, PA_NVFP4, 1>)
        : chunks == 2 ? go(quantize_kernel<T, PA_NVFP4, 2>)
        : chunks == 3 ? go(quantize_kernel<T, PA_NVFP4, 3>)
                      : go(quantize_kernel<T, PA_NVFP4, 4>);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

int check_table(int64_t rows, int64_t d, int method) {
    PA_REQUIRE(rows >= 0 && rows <= PA_MAX_ROWS, "rows out of range");
    PA_REQUIRE(d >= 1 && d <= PA_MAX_WIDTH, "d must be in [1, %d]", PA_MAX_WIDTH);
    PA_REQUIRE(method == PA_MXFP4 || method == PA_NVFP4, "unknown 4-bit method %d", method);
    return PA_OK;
}

}  // namespace fp4
}  // namespace pa

extern "C" int pa_quantize_fp4(uint8_t *codes, uint8_t *scales, float *row_scale, const void *x,
                               int64_t rows, int d, int64_t ldx, int dtype, int method,
                               void *stream) {
    using namespace pa;
    int rc = fp4::check_table(rows, d, method);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(ldx >= d, "row stride must cover the row");
    PA_REQUIRE(dtype == PA_F32 || dtype == PA_BF16 || dtype == PA_F16, "unknown dtype %d", dtype);
    if (rows == 0) return PA_OK;
    PA_REQUIRE(codes && scales && x && (row_scale || method == PA_MXFP4), "null pointer");
    PA_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
    PA_REQUIRE(aligned_to(x, dtype == PA_F32 ? 4 : 2) && aligned_to(row_scale, 4),
               "x and row_scale must be aligned to their values");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PA_F32)
        return fp4::quantize_launch<float>(codes, scales, row_scale, x, rows, d, ldx, method, s);
    if (dtype == PA_BF16)
        return fp4::quantize_launch<__nv_bfloat16>(codes, scales, row_scale, x, rows, d, ldx,
                                                   method, s);
    return fp4::quantize_launch<__half>(codes, scales, row_scale, x, rows, d, ldx, method, s);
}

extern "C" int pa_dequantize_fp4(float *out, const uint8_t *codes, const uint8_t *scales,
                                 const float *row_scale, int64_t rows, int d, int method,
                                 void *stream) {
    using namespace pa;
    int rc = fp4::check_table(rows, d, method);
    if (rc != PA_OK) return rc;
    if (rows == 0) return PA_OK;
    PA_REQUIRE(out && codes && scales && (row_scale || method == PA_MXFP4), "null pointer");
    PA_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
    PA_REQUIRE(aligned_to(out, 4) && aligned_to(row_scale, 4),
               "out and row_scale must be aligned to their values");
    const unsigned grid = static_cast<unsigned>((rows + fp4::kWarps - 1) / fp4::kWarps);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool vec = aligned16(out) && d % 4 == 0;
    auto go = [&](auto kernel) {
        kernel<<<grid, 32 * fp4::kWarps, 0, s>>>(out, codes, scales, row_scale, rows, d, vec);
    };
    const int chunks = fp4::chunks_of(d);
    if (method == PA_MXFP4)
        chunks == 1   ? go(fp4::dequantize_kernel<PA_MXFP4, 1>)
        : chunks == 2 ? go(fp4::dequantize_kernel<PA_MXFP4, 2>)
        : chunks == 3 ? go(fp4::dequantize_kernel<PA_MXFP4, 3>)
                      : go(fp4::dequantize_kernel<PA_MXFP4, 4>);
    else
        chunks == 1   ? go(fp4::dequantize_kernel<PA_NVFP4, 1>)
        : chunks == 2 ? go(fp4::dequantize_kernel<PA_NVFP4, 2>)
        : chunks == 3 ? go(fp4::dequantize_kernel<PA_NVFP4, 3>)
                      : go(fp4::dequantize_kernel<PA_NVFP4, 4>);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}
