// The segments of grouped rows, and what the products share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pa_common.cuh"

namespace pa {
namespace grouped {

template <typename T> __device__ __forceinline__ T from_f32(float v);  // round to nearest even
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) {
    return __float2bfloat16_rn(v);
}

template <typename T> constexpr bool is_bf16() { return false; }
template <> constexpr bool is_bf16<__nv_bfloat16>() { return true; }

// The rows as n_groups + 2 segments: those before the first group, the groups, those behind
// the last.  Edge i (0 .. n_groups + 2) is where segment i starts.
__device__ __forceinline__ int64_t edge(const int64_t *offsets, int n_groups, int64_t rows, int i) {
    if (i == 0) return 0;
    if (i == n_groups + 2) return rows;
    const int64_t e = offsets[i - 1];
    return e < 0 ? 0 : (e > rows ? rows : e);
}

// grouped_mma.cu: 16-bit values on the tensor cores, rows on 16 bytes
template <typename T>
int rows_mma(void *out, const void *in, const void *w, const int64_t *offsets, int64_t rows,
             int n_groups, int d_sum, int d_out, int64_t ldi, int64_t ldw, int64_t ldo,
             bool transposed,
             cudaStream_t s);
template <typename T>
int matrices_mma(void *dw, const void *dy, const void *x, const int64_t *offsets, int64_t rows,
                 int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s);

}  // namespace grouped
}  // namespace pa
