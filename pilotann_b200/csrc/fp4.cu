// Rows of values to 4-bit blocks (fp4.cuh has the formats) and back.
//
// mxfp4: the scale of a block is 2^(floor(log2 max|v|) - 2), the largest E2M1 exponent being
// 2; dividing by it is exact, values above 6 saturate.  nvfp4: the row's scale s is the least
// power of two with max|v| <= 6 * 448 s, a block's is max|v| / (6 s) rounded to E4M3.  s is a
// power of two so that no rounding of it decides how a value next to a border is coded: the
// quotients are those of the definition, up to fp32's own half step.  Rows are independent of
// one another: a query's codes do not depend on the batch it comes in.
#include "fp4.cuh"

namespace pa {
namespace fp4 {

constexpr int kWarps = 8;  // rows per CTA, a warp each

// A lane has eight consecutive values of a chunk of 256, a block is four lanes (mxfp4) or two;
// kChunks chunks are loaded before any is worked on.  Rows are read once where they fit those
// registers (or the method needs no maximum of the row), else a second time from the caches.
constexpr int kChunks = 4;

__device__ __forceinline__ void unpack8(float (&v)[8], const float *p) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)),
                 b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void unpack8(float (&v)[8], const __nv_bfloat16 *p) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack8(float (&v)[8], const __half *p) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
}
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T *row, int64_t at, int64_t d, bool vec) {
    if (vec && at + 8 <= d) {
        unpack8(v, row + at);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = at + j < d ? load_f32(row + at + j) : 0.0f;
    }
}

__device__ __forceinline__ uint32_t top_bits(const float (&v)[8]) {
    uint32_t t = 0;  // magnitudes order like their bits; NaN above infinity above the rest
#pragma unroll
    for (int j = 0; j < 8; ++j) t = max(t, __float_as_uint(v[j]) & 0x7fffffffu);
    return t;
}

// v / step as codes.  fp32 values are divided.  16-bit ones have at most 11 significant bits and
// step has four, so that a quotient is a border between two codes exactly or at least 2^-12 of
// its value away from it: a product with the reciprocal (off by 2^-23), rounded to 18 bits
// behind the leading one, lands on the border in the first case and stays off it in the other,
// at a third of the instructions.
template <typename T>
__device__ __forceinline__ uint32_t codes_by(float (&v)[8], float step) {
    if (sizeof(T) == 2 && step >= 1.1754944e-38f) {  // a reciprocal that does not overflow
        const float inv = __frcp_rn(step);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __uint_as_float((__float_as_uint(__fmul_rn(v[j], inv)) + 16u) & ~31u);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = step > 0.0f ? __fdiv_rn(v[j], step) : 0.0f;
    }
    return codes_of(v);
}

template <typename T, int METHOD>
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
    float v[kChunks][8];
    float s = 1.0f, s_inv = 1.0f;
    if (METHOD == PA_NVFP4) {
        uint32_t top = 0;
        for (int64_t a0 = 0; a0 < dp; a0 += 256 * kChunks) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) load8(v[c], row, a0 + 256 * c + 8 * lane, d, vec);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) top = max(top, top_bits(v[c]));
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
    for (int64_t a0 = 0; a0 < dp; a0 += 256 * kChunks) {
        if (METHOD == PA_MXFP4 || dp > 256 * kChunks) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) load8(v[c], row, a0 + 256 * c + 8 * lane, d, vec);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = a0 + 256 * c + 8 * lane;
            if (a0 + 256 * c >= dp) break;  // uniform
            uint32_t top = top_bits(v[c]);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            uint32_t byte, code;
            if (METHOD == PA_MXFP4) {
                const uint32_t e = top >> 23;
                byte = e > 2u ? e - 2u : 0u;
                const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = __fmul_rn(v[c][j], inv);
                code = codes_of(v[c]);
                if (e == 255u) { byte = 255u; code = 0u; }
            } else {
                const float ratio = __fdiv_rn(__fmul_rn(__uint_as_float(top), s_inv), 6.0f);
                byte = e4m3_of(fminf(ratio, 448.0f));
                code = codes_by<T>(v[c], __fmul_rn(e4m3_value(byte), s));
                if (!(s > 0.0f)) { byte = 0u; code = 0u; }  // NaN: the row's scale says it
            }
            if (at < dp) {
                to[(a0 + 256 * c) / 8] = code;
                if (lane % kLanes == 0) to_scale[(a0 + 256 * c) / (8 * kLanes)] = byte;
            }
        }
    }
}

// eight codes -> eight values of their block (exact: two significant bits times at most four)
__device__ __forceinline__ void values_of(float (&v)[8], uint32_t code, float scale) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t h;
        asm("{\n"
            ".reg .b8 b;\n"
            "cvt.u8.u32 b, %1;\n"
            "cvt.rn.f16x2.e2m1x2 %0, b;\n"
            "}\n"
            : "=r"(h)
            : "r"((code >> (8 * j)) & 0xffu));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        v[2 * j] = __fmul_rn(f.x, scale);
        v[2 * j + 1] = __fmul_rn(f.y, scale);
    }
}

template <int METHOD>
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
    float *to = out + r * d + 8 * lane;
    for (int64_t a0 = 0; a0 < d; a0 += 256 * kChunks) {
        uint32_t code[kChunks], byte[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t a = a0 + 256 * c;
            const bool live = a + 8 * lane < d;
            code[c] = live ? __ldg(from + a / 8) : 0u;
            byte[c] = live ? __ldg(from_scale + a / (8 * kLanes)) : 0u;
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t a = a0 + 256 * c, at = a + 8 * lane;
            if (at >= d) break;
            float v[8];
            if (METHOD == PA_MXFP4) {
                values_of(v, code[c], e8m0_value(byte[c]));
            } else {
                values_of(v, code[c], e4m3_value(byte[c]));
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], s);
            }
            if (vec) {
                *reinterpret_cast<float4 *>(to + a) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(to + a + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at + j < d) to[a + j] = v[j];
            }
        }
    }
}

template <typename T>
int quantize_launch(uint8_t *codes, uint8_t *scales, float *row_scale, const void *x, int64_t rows,
                    int64_t d, int64_t ldx, int method, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
    const bool vec = aligned16(x) && ldx * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    if (method == PA_MXFP4)
        quantize_kernel<T, PA_MXFP4><<<grid, 32 * kWarps, 0, s>>>(
            codes, scales, row_scale, static_cast<const T *>(x), rows, d, ldx, vec);
    else
        quantize_kernel<T, PA_NVFP4><<<grid, 32 * kWarps, 0, s>>>(
            codes, scales, row_scale, static_cast<const T *>(x), rows, d, ldx, vec);
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
    const unsigned grid = static_cast<unsigned>((rows + fp4::kWarps - 1) / fp4::kWarps);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool vec = aligned16(out) && d % 8 == 0;
    if (method == PA_MXFP4)
        fp4::dequantize_kernel<PA_MXFP4><<<grid, 32 * fp4::kWarps, 0, s>>>(out, codes, scales,
                                                                           row_scale, rows, d, vec);
    else
        fp4::dequantize_kernel<PA_NVFP4><<<grid, 32 * fp4::kWarps, 0, s>>>(out, codes, scales,
                                                                           row_scale, rows, d, vec);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}
