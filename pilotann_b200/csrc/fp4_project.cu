// Products of 4-bit rows with a 4-bit table, dense or with one table per group of rows:
//   out[i, n] = sum_k q(i, k) t(g, n, k)
// fp32 sums; the segments of rows are those of grouped.cu.
#include "fp4.cuh"
#include "grouped.cuh"

namespace pa {
namespace fp4 {

using grouped::edge;
using grouped::from_f32;

constexpr int kT = 64, kK = 32;

template <int METHOD>
__device__ __forceinline__ void load_slice(float (*t_s)[kT + 4], const uint8_t *codes,
                                           const uint8_t *scales, int64_t r0, int n_r, int64_t k0,
                                           int64_t dp) {
    // 64 rows x 32 values; a thread has eight of one row
    const int r = threadIdx.x >> 2, k = 8 * (threadIdx.x & 3);
    uint32_t code = 0;
    float b = 0.0f;
    if (r < n_r) {
        code = *reinterpret_cast<const uint32_t *>(codes + (r0 + r) * (dp / 2) + (k0 + k) / 2);
        const uint32_t byte = scales[(r0 + r) * (dp / block_of(METHOD)) + (k0 + k) / block_of(METHOD)];
        b = METHOD == PA_MXFP4 ? e8m0_value(byte) : e4m3_value(byte);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) t_s[k + j][r] = r < n_r ? code_value((code >> (4 * j)) & 15u) * b : 0.0f;
}

template <int METHOD, typename O>
__global__ void __launch_bounds__(256)
project_kernel(O *__restrict__ out, const uint8_t *__restrict__ q_codes,
               const uint8_t *__restrict__ q_scales, const float *__restrict__ q_row_scale,
               const uint8_t *__restrict__ t_codes, const uint8_t *__restrict__ t_scales,
               const float *__restrict__ t_row_scale, const int64_t *__restrict__ offsets,
               int64_t rows, int n_groups, int d, int64_t d_out) {
    __shared__ __align__(16) float p_s[kK][kT + 4], q_s[kK][kT + 4];
    const int64_t dp = padded(d), slot = blockIdx.y;
    int64_t lo = 0, hi = rows, r0 = slot * kT;
    int seg = 1;
    if (offsets != nullptr) {
        int below = 0;
        for (int i0 = 0; i0 < n_groups + 2; i0 += 256) {
            const int i = i0 + threadIdx.x;
            below += __syncthreads_count(i < n_groups + 2 &&
                                         edge(offsets, n_groups, rows, i) / kT + i <= slot);
        }
        seg = below - 1;
        lo = edge(offsets, n_groups, rows, seg);
        hi = edge(offsets, n_groups, rows, seg + 1);
        r0 = lo + (slot - (lo / kT + seg)) * kT;
    }
    if (r0 < lo || r0 >= hi) return;
    const int n_r = static_cast<int>(min(static_cast<int64_t>(kT), hi - r0));
    const int64_t c0 = blockIdx.x * static_cast<int64_t>(kT);
    const int n_c = static_cast<int>(min(static_cast<int64_t>(kT), d_out - c0));
    const bool grouped_row = seg >= 1 && seg <= n_groups;
    const int64_t t0 = (seg - 1) * d_out + c0;  // first table row of this tile
    float acc[4][4] = {};
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int64_t k0 = 0; grouped_row && k0 < dp; k0 += kK) {
        load_slice<METHOD>(p_s, q_codes, q_scales, r0, n_r, k0, dp);
        load_slice<METHOD>(q_s, t_codes, t_scales, t0, n_c, k0, dp);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kK; ++t) {
            const float4 a = *reinterpret_cast<const float4 *>(&p_s[t][4 * ty]);
            const float4 b = *reinterpret_cast<const float4 *>(&q_s[t][4 * tx]);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = 4 * ty + i, c = 4 * tx + j;
            if (r < n_r && c < n_c) {
                float v = acc[i][j];
                if (METHOD == PA_NVFP4 && grouped_row) v *= q_row_scale[r0 + r] * t_row_scale[t0 + c];
                out[(r0 + r) * d_out + c0 + c] = from_f32<O>(v);
            }
        }
}

template <int METHOD, typename O>
int project_launch(void *out, const uint8_t *q_codes, const uint8_t *q_scales,
                   const float *q_row_scale, const uint8_t *t_codes, const uint8_t *t_scales,
                   const float *t_row_scale, const int64_t *offsets, int64_t rows, int n_groups,
                   int d, int64_t d_out, cudaStream_t s) {
    const int64_t slots = offsets ? rows / kT + n_groups + 2 : (rows + kT - 1) / kT;
    PA_REQUIRE(slots <= 65535, "too many rows for one call");
    dim3 grid(static_cast<unsigned>((d_out + kT - 1) / kT), static_cast<unsigned>(slots));
    project_kernel<METHOD, O><<<grid, 256, 0, s>>>(static_cast<O *>(out), q_codes, q_scales,
                                                   q_row_scale, t_codes, t_scales, t_row_scale,
                                                   offsets, rows, n_groups, d, d_out);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

}  // namespace fp4
}  // namespace pa

extern "C" int pa_project_fp4(void *out, const uint8_t *query_codes, const uint8_t *query_scales,
                              const float *query_row_scale, const uint8_t *codes,
                              const uint8_t *scales, const float *row_scale,
                              const int64_t *offsets, int64_t rows, int n_groups, int d,
                              int64_t d_out, int out_dtype, int method, void *stream) {
    using namespace pa;
    PA_REQUIRE(rows >= 0 && rows <= PA_MAX_ROWS, "rows out of range");
    PA_REQUIRE(d >= 1 && d <= PA_MAX_WIDTH, "d must be in [1, %d]", PA_MAX_WIDTH);
    PA_REQUIRE(method == PA_MXFP4 || method == PA_NVFP4, "unknown 4-bit method %d", method);
    PA_REQUIRE(out_dtype == PA_F32 || out_dtype == PA_BF16 || out_dtype == PA_F16,
               "unknown dtype %d", out_dtype);
    PA_REQUIRE(n_groups >= 1 && n_groups <= PA_MAX_GROUPS, "n_groups must be in [1, %d]",
               PA_MAX_GROUPS);
    PA_REQUIRE(offsets || n_groups == 1, "several groups need offsets");
    PA_REQUIRE(d_out >= 0 && d_out * n_groups <= 0x7fffffff, "table rows out of range");
    if (rows == 0 || d_out == 0) return PA_OK;
    PA_REQUIRE(out && query_codes && query_scales && codes && scales, "null pointer");
    PA_REQUIRE(method == PA_MXFP4 || (query_row_scale && row_scale), "nvfp4 needs row scales");
    PA_REQUIRE(aligned16(query_codes) && aligned16(codes), "codes must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define PA_GO(M, O)                                                                              \
    return fp4::project_launch<M, O>(out, query_codes, query_scales, query_row_scale, codes,     \
                                     scales, row_scale, offsets, rows, n_groups, d, d_out, s)
    if (method == PA_MXFP4) {
        if (out_dtype == PA_F32) PA_GO(PA_MXFP4, float);
        if (out_dtype == PA_BF16) PA_GO(PA_MXFP4, __nv_bfloat16);
        PA_GO(PA_MXFP4, __half);
    }
    if (out_dtype == PA_F32) PA_GO(PA_NVFP4, float);
    if (out_dtype == PA_BF16) PA_GO(PA_NVFP4, __nv_bfloat16);
    PA_GO(PA_NVFP4, __half);
#undef PA_GO
}
