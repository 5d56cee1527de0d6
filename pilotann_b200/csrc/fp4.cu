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

// A lane has eight consecutive values, a warp 256; a block is four lanes (mxfp4) or two.
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T *row, int64_t at, int64_t d) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at + j < d ? load_f32(row + at + j) : 0.0f;
}

__device__ __forceinline__ uint32_t top_bits(const float (&v)[8]) {
    uint32_t t = 0;  // magnitudes order like their bits; NaN above infinity above the rest
#pragma unroll
    for (int j = 0; j < 8; ++j) t = max(t, __float_as_uint(v[j]) & 0x7fffffffu);
    return t;
}

template <typename T, int METHOD>
__global__ void __launch_bounds__(32 * kWarps)
quantize_kernel(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                float *__restrict__ row_scale, const T *__restrict__ x, int64_t rows, int64_t d,
                int64_t ldx) {
    const int lane = threadIdx.x & 31;
    const int64_t r = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const T *row = x + r * ldx;
    const int64_t dp = padded(d);
    float s = 1.0f;
    if (METHOD == PA_NVFP4) {
        uint32_t top = 0;
        for (int64_t at = 8 * lane; at < dp; at += 256) {
            float v[8];
            load8(v, row, at, d);
            top = max(top, top_bits(v));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        // 6 * 448 = 1.3125 * 2^11
        const int power = static_cast<int>(top >> 23) - 127 - 11 + ((top & 0x7fffffu) > 0x280000u);
        s = top >= 0x7f800000u ? CUDART_NAN_F
                               : __uint_as_float(static_cast<uint32_t>(max(power, -126) + 127) << 23);
        if (lane == 0) row_scale[r] = s;
    }
    constexpr int kLanes = METHOD == PA_MXFP4 ? 4 : 2;  // lanes of a block
    for (int64_t a0 = 0; a0 < dp; a0 += 256) {
        const int64_t at = a0 + 8 * lane;
        float v[8];
        load8(v, row, at, d);
        uint32_t top = top_bits(v);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
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
            const float most = __uint_as_float(top);
            byte = e4m3_of(fminf(__fdiv_rn(__fdiv_rn(most, s), 6.0f), 448.0f));
            const float step = __fmul_rn(e4m3_value(byte), s);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = step > 0.0f ? __fdiv_rn(v[j], step) : 0.0f;
            code = codes_of(v);
            if (!(s > 0.0f)) { byte = 0u; code = 0u; }  // NaN: the row's scale says it
        }
        if (at < dp) {
            *reinterpret_cast<uint32_t *>(codes + r * (dp / 2) + at / 2) = code;
            if (lane % kLanes == 0) scales[r * (dp / (8 * kLanes)) + at / (8 * kLanes)] = byte;
        }
    }
}

template <int METHOD>
__global__ void __launch_bounds__(32 * kWarps)
dequantize_kernel(float *__restrict__ out, const uint8_t *__restrict__ codes,
                  const uint8_t *__restrict__ scales, const float *__restrict__ row_scale,
                  int64_t rows, int64_t d) {
    const int lane = threadIdx.x & 31;
    const int64_t r = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int64_t dp = padded(d);
    const float s = METHOD == PA_NVFP4 ? row_scale[r] : 1.0f;
    for (int64_t at = 8 * lane; at < d; at += 256) {
        const uint32_t code = *reinterpret_cast<const uint32_t *>(codes + r * (dp / 2) + at / 2);
        const uint32_t byte = scales[r * (dp / block_of(METHOD)) + at / block_of(METHOD)];
        const float b = METHOD == PA_MXFP4 ? e8m0_value(byte) : e4m3_value(byte);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = __fmul_rn(code_value((code >> (4 * j)) & 15u), b);
            if (METHOD == PA_NVFP4) v = __fmul_rn(v, s);
            if (at + j < d) out[r * d + at + j] = v;
        }
    }
}

template <typename T>
int quantize_launch(uint8_t *codes, uint8_t *scales, float *row_scale, const void *x, int64_t rows,
                    int64_t d, int64_t ldx, int method, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
    if (method == PA_MXFP4)
        quantize_kernel<T, PA_MXFP4><<<grid, 32 * kWarps, 0, s>>>(
            codes, scales, row_scale, static_cast<const T *>(x), rows, d, ldx);
    else
        quantize_kernel<T, PA_NVFP4><<<grid, 32 * kWarps, 0, s>>>(
            codes, scales, row_scale, static_cast<const T *>(x), rows, d, ldx);
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
    if (method == PA_MXFP4)
        fp4::dequantize_kernel<PA_MXFP4><<<grid, 32 * fp4::kWarps, 0, s>>>(out, codes, scales,
                                                                           row_scale, rows, d);
    else
        fp4::dequantize_kernel<PA_NVFP4><<<grid, 32 * fp4::kWarps, 0, s>>>(out, codes, scales,
                                                                           row_scale, rows, d);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}
