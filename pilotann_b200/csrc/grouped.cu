// Products of rows with the matrix of their group.  Rows of a group are contiguous:
// group g has rows [offsets[g], offsets[g + 1]).
//   forward   y[i, n]     = sum_k x[i, k]  w[g, n, k]
//   rows      dx[i, k]    = sum_n dy[i, n] w[g, n, k]
//   matrices  dw[g, n, k] = sum_{i in g} dy[i, n] x[i, k]
// Rows before offsets[0] and from offsets[n_groups] on belong to no group: y and dx are zero
// there.  Offsets are clamped to [0, rows], so that none of them makes an access leave the
// tensors, whatever they hold.
#include "grouped.cuh"

namespace pa {

namespace grouped {

constexpr int kT = 64;   // output tile, both ways
constexpr int kK = 16;   // slice of the summed axis

// 64 x 64 outputs, 256 threads with 4 x 4 each, fp32 fma along the summed axis.
//   C[r, c] = sum_t P(r, t) Q(c, t), P(r, t) = p[r * pr + t * pt], Q likewise
template <typename T, bool P_T_FAST, bool Q_T_FAST>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], const T *p, int64_t pr, int64_t pt,
                                             int n_r, const T *q, int64_t qc, int64_t qt, int n_c,
                                             int64_t n_t, float (*p_s)[kT + 4],
                                             float (*q_s)[kT + 4]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int64_t t0 = 0; t0 < n_t; t0 += kK) {
#pragma unroll
        for (int i = threadIdx.x; i < kT * kK; i += 256) {
            const int r = P_T_FAST ? i / kK : i % kT, t = P_T_FAST ? i % kK : i / kT;
            p_s[t][r] = r < n_r && t0 + t < n_t ? to_f32(p[r * pr + (t0 + t) * pt]) : 0.0f;
        }
#pragma unroll
        for (int i = threadIdx.x; i < kT * kK; i += 256) {
            const int c = Q_T_FAST ? i / kK : i % kT, t = Q_T_FAST ? i % kK : i / kT;
            q_s[t][c] = c < n_c && t0 + t < n_t ? to_f32(q[c * qc + (t0 + t) * qt]) : 0.0f;
        }
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
}

// Rows side: forward (W_T_FAST: w's last axis is summed) and the gradient of the rows.
// blockIdx.x = a slot of 64 rows.  Segment i owns the slots from floor(edge_i / 64) + i on, which
// are enough for its tiles of 64 rows wherever it starts; a slot without rows returns.
template <typename T, bool W_T_FAST>
__global__ void __launch_bounds__(256)
rows_kernel(T *__restrict__ out, const T *__restrict__ x, const T *__restrict__ w,
            const int64_t *__restrict__ offsets, int64_t rows, int n_groups, int d_sum, int d_out,
            int64_t ldx, int64_t ldo) {
    __shared__ __align__(16) float p_s[kK][kT + 4], q_s[kK][kT + 4];
    const int64_t slot = blockIdx.x;
    int below = 0;  // segments that start at or before this slot
    for (int i0 = 0; i0 < n_groups + 2; i0 += 256) {
        const int i = i0 + threadIdx.x;
        below += __syncthreads_count(i < n_groups + 2 &&
                                     edge(offsets, n_groups, rows, i) / kT + i <= slot);
    }
    const int seg = below - 1;
    const int64_t lo = edge(offsets, n_groups, rows, seg),
                  hi = edge(offsets, n_groups, rows, seg + 1);
    const int64_t r0 = lo + (slot - (lo / kT + seg)) * kT;
    if (r0 < lo || r0 >= hi) return;
    const int n_r = static_cast<int>(min(static_cast<int64_t>(kT), hi - r0));
    const int c0 = blockIdx.y * kT, n_c = min(kT, d_out - c0);
    float acc[4][4] = {};
    if (seg >= 1 && seg <= n_groups) {
        const T *wg = w + static_cast<int64_t>(seg - 1) * d_sum * d_out;
        if (W_T_FAST)
            tile_product<T, true, true>(acc, x + r0 * ldx, ldx, 1, n_r,
                                        wg + static_cast<int64_t>(c0) * d_sum, d_sum, 1, n_c, d_sum,
                                        p_s, q_s);
        else
            tile_product<T, true, false>(acc, x + r0 * ldx, ldx, 1, n_r, wg + c0, 1, d_out, n_c,
                                         d_sum, p_s, q_s);
    }
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = 4 * ty + i, c = 4 * tx + j;
            if (r < n_r && c < n_c) out[(r0 + r) * ldo + c0 + c] = from_f32<T>(acc[i][j]);
        }
}

// Gradient of the matrices: one 64 x 64 tile of one group per CTA, summed over its rows.
template <typename T>
__global__ void __launch_bounds__(256)
matrices_kernel(T *__restrict__ dw, const T *__restrict__ dy, const T *__restrict__ x,
                const int64_t *__restrict__ offsets, int64_t rows, int n_groups, int d, int d_out,
                int64_t ldy, int64_t ldx) {
    __shared__ __align__(16) float p_s[kK][kT + 4], q_s[kK][kT + 4];
    const int g = blockIdx.z;
    const int n0 = blockIdx.y * kT, k0 = blockIdx.x * kT;
    const int n_n = min(kT, d_out - n0), n_k = min(kT, d - k0);
    const int64_t lo = edge(offsets, n_groups, rows, g + 1),
                  hi = edge(offsets, n_groups, rows, g + 2);
    float acc[4][4] = {};
    tile_product<T, false, false>(acc, dy + lo * ldy + n0, 1, ldy, n_n, x + lo * ldx + k0, 1, ldx,
                                  n_k, hi - lo, p_s, q_s);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = 4 * ty + i, k = 4 * tx + j;
            if (n < n_n && k < n_k)
                dw[(static_cast<int64_t>(g) * d_out + n0 + n) * d + k0 + k] =
                    from_f32<T>(acc[i][j]);
        }
}

// ---- 16-bit operands that a bulk-tensor copy cannot read --------------------------
// Rows that do not start on 16 bytes (an odd width, a slice of a wider tensor) are copied into
// the workspace with a pitch of whole 16 bytes first; the products then run on that.  A copy
// reads and writes the operand once (of the matrices only those whose group has rows), which the
// tensor cores win back many times over plain loads: 4099 rows x 13 matrices of 333 x 200, all
// gradients, 178 us with the 64 x 64 tiles above.
constexpr int kCopyRows = 32;  // per CTA

__global__ void __launch_bounds__(256)
repitch_kernel(uint4 *__restrict__ out, const uint16_t *__restrict__ in, int64_t rows, int width,
               int64_t ld, const int64_t *__restrict__ offsets, int n_groups, int64_t n_rows) {
    const int pieces = (width + 7) / 8, g = blockIdx.y;
    if (offsets && edge(offsets, n_groups, n_rows, g + 1) >= edge(offsets, n_groups, n_rows, g + 2))
        return;
    out += g * rows * pieces;
    in += g * rows * ld;
    const int64_t r0 = blockIdx.x * static_cast<int64_t>(kCopyRows);
    const int n = static_cast<int>(min(static_cast<int64_t>(kCopyRows), rows - r0)) * pieces;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int r = i / pieces, p = i - r * pieces;
        const uint16_t *src = in + (r0 + r) * ld + 8 * p;
        // aligned words that hold one of the piece's values, shifted by half a word if need be
        const uint32_t half = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src) >> 1) & 1u;
        const uint32_t *base = reinterpret_cast<const uint32_t *>(src - half);
        const int have = min(8, width - 8 * p) + half;  // 16-bit values from base on
        uint32_t w[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) w[j] = 2 * j < have ? __ldg(base + j) : 0u;
        uint4 v;
        v.x = __funnelshift_r(w[0], w[1], 16 * half);
        v.y = __funnelshift_r(w[1], w[2], 16 * half);
        v.z = __funnelshift_r(w[2], w[3], 16 * half);
        v.w = __funnelshift_r(w[3], w[4], 16 * half);
        out[(r0 + r) * pieces + p] = v;
    }
}

int64_t pitched(int width) { return (width + 7) / 8 * 8; }

// rows of 16-bit values that a bulk-tensor copy can start at
bool rows_ok(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }
int64_t copy_bytes(const void *p, int64_t rows, int width, int64_t ld) {
    return rows_ok(p, ld) ? 0 : rows * pitched(width) * 2;
}

int repitch(uint8_t *to, const void *p, int64_t ld, int64_t rows, int width, int n_groups,
            const int64_t *offsets, int64_t n_rows, cudaStream_t s) {
    dim3 grid(static_cast<unsigned>((rows + kCopyRows - 1) / kCopyRows),
              static_cast<unsigned>(n_groups));
    repitch_kernel<<<grid, 256, 0, s>>>(reinterpret_cast<uint4 *>(to),
                                        static_cast<const uint16_t *>(p), rows, width, ld, offsets,
                                        n_groups, n_rows);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

// *p and *ld on exit: the operand itself, or its copy, with *ws moved behind it
int rows_make_ok(const void **p, int64_t *ld, int64_t rows, int width, uint8_t **ws,
                 cudaStream_t s) {
    if (rows_ok(*p, *ld)) return PA_OK;
    int rc = repitch(*ws, *p, *ld, rows, width, 1, nullptr, 0, s);
    *p = *ws;
    *ld = pitched(width);
    *ws += rows * pitched(width) * 2;
    return rc;
}

int matrices_make_ok(const void **w, int64_t *ld, int n_groups, int d, int d_out,
                     const int64_t *offsets, int64_t n_rows, uint8_t **ws, cudaStream_t s) {
    if (rows_ok(*w, *ld)) return PA_OK;
    int rc = repitch(*ws, *w, *ld, d_out, d, n_groups, offsets, n_rows, s);
    *w = *ws;
    *ld = pitched(d);
    *ws += static_cast<int64_t>(n_groups) * d_out * pitched(d) * 2;
    return rc;
}

int rows_f32(float *out, const float *x, const float *w, const int64_t *offsets, int64_t rows,
             int n_groups, int d_sum, int d_out, int64_t ldx, int64_t ldo, bool transposed,
             cudaStream_t s) {
    dim3 grid(static_cast<unsigned>(rows / kT + n_groups + 2),
              static_cast<unsigned>((d_out + kT - 1) / kT));
    if (transposed)
        rows_kernel<float, false><<<grid, 256, 0, s>>>(out, x, w, offsets, rows, n_groups, d_sum,
                                                       d_out, ldx, ldo);
    else
        rows_kernel<float, true><<<grid, 256, 0, s>>>(out, x, w, offsets, rows, n_groups, d_sum,
                                                      d_out, ldx, ldo);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

int matrices_f32(float *dw, const float *dy, const float *x, const int64_t *offsets, int64_t rows,
                 int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s) {
    dim3 grid(static_cast<unsigned>((d + kT - 1) / kT), static_cast<unsigned>((d_out + kT - 1) / kT),
              static_cast<unsigned>(n_groups));
    matrices_kernel<float><<<grid, 256, 0, s>>>(dw, dy, x, offsets, rows, n_groups, d, d_out, ldy,
                                                ldx);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

int check(int64_t rows, int n_groups, int d, int d_out, int dtype) {
    PA_REQUIRE(rows >= 0 && rows <= PA_MAX_ROWS, "rows out of range");
    PA_REQUIRE(n_groups >= 1 && n_groups <= PA_MAX_GROUPS, "n_groups must be in [1, %d]",
               PA_MAX_GROUPS);
    PA_REQUIRE(d >= 1 && d <= PA_MAX_WIDTH && d_out >= 1 && d_out <= PA_MAX_WIDTH,
               "d and d_out must be in [1, %d]", PA_MAX_WIDTH);
    PA_REQUIRE(dtype == PA_F32 || dtype == PA_BF16 || dtype == PA_F16, "unknown dtype %d", dtype);
    return PA_OK;
}

// forward, or with `transposed` the gradient of the rows, of 16-bit values
int rows_16(void *out, const void *in, int64_t ldi, const void *w, int64_t ldw,
            const int64_t *offsets, int64_t rows, int n_groups, int d_sum, int d_out, int64_t ldo,
            int dtype, bool transposed, cudaStream_t s) {
    if (dtype == PA_BF16)
        return rows_mma<__nv_bfloat16>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi, ldw,
                                       ldo, transposed, s);
    return rows_mma<__half>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi, ldw, ldo,
                            transposed, s);
}

}  // namespace grouped
}  // namespace pa

extern "C" int64_t pa_project_grouped_workspace_bytes(const void *query, const void *VT,
                                                      int64_t rows, int n_groups, int d, int d_out,
                                                      int64_t ld_query, int dtype) {
    using namespace pa::grouped;
    if (dtype == PA_F32) return 0;
    return copy_bytes(query, rows, d, ld_query) +
           copy_bytes(VT, static_cast<int64_t>(n_groups) * d_out, d, d);
}

extern "C" int pa_project_grouped(void *out, const void *query, const void *VT,
                                  const int64_t *offsets, int64_t rows, int n_groups, int d,
                                  int d_out, int64_t ld_query, int64_t ld_out, int dtype,
                                  void *workspace, void *stream) {
    using namespace pa;
    int rc = grouped::check(rows, n_groups, d, d_out, dtype);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(ld_query >= d && ld_out >= d_out, "row strides must cover the rows");
    if (rows == 0) return PA_OK;
    PA_REQUIRE(out && query && VT && offsets, "null pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PA_F32)
        return grouped::rows_f32(static_cast<float *>(out), static_cast<const float *>(query),
                                 static_cast<const float *>(VT), offsets, rows, n_groups, d, d_out,
                                 ld_query, ld_out, false, s);
    PA_REQUIRE(workspace || !pa_project_grouped_workspace_bytes(query, VT, rows, n_groups, d, d_out,
                                                               ld_query, dtype),
               "workspace missing (pa_project_grouped_workspace_bytes)");
    PA_REQUIRE(aligned16(workspace), "workspace must be 16-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    int64_t ldw = d;
    rc = grouped::rows_make_ok(&query, &ld_query, rows, d, &ws, s);
    if (rc != PA_OK) return rc;
    rc = grouped::matrices_make_ok(&VT, &ldw, n_groups, d, d_out, offsets, rows, &ws, s);
    if (rc != PA_OK) return rc;
    return grouped::rows_16(out, query, ld_query, VT, ldw, offsets, rows, n_groups, d, d_out,
                            ld_out, dtype, false, s);
}

extern "C" int64_t pa_project_grouped_backward_workspace_bytes(
    const void *grad, const void *query, const void *VT, int64_t rows, int n_groups, int d,
    int d_out, int64_t ld_grad, int64_t ld_query, int dtype, int want_query, int want_VT) {
    using namespace pa::grouped;
    if (dtype == PA_F32) return 0;
    return copy_bytes(grad, rows, d_out, ld_grad) +
           (want_query ? copy_bytes(VT, static_cast<int64_t>(n_groups) * d_out, d, d) : 0) +
           (want_VT ? copy_bytes(query, rows, d, ld_query) : 0);
}

extern "C" int pa_project_grouped_backward(void *grad_query, void *grad_VT, const void *grad,
                                           const void *query, const void *VT,
                                           const int64_t *offsets, int64_t rows, int n_groups,
                                           int d, int d_out, int64_t ld_grad, int64_t ld_query,
                                           int64_t ld_grad_query, int dtype, void *workspace,
                                           void *stream) {
    using namespace pa;
    int rc = grouped::check(rows, n_groups, d, d_out, dtype);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(ld_grad >= d_out, "row strides must cover the rows");
    PA_REQUIRE(!grad_query || ld_grad_query >= d, "row strides must cover the rows");
    PA_REQUIRE(!grad_VT || ld_query >= d, "row strides must cover the rows");
    if (!grad_query && !grad_VT) return PA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {  // no products: the matrices' gradients are zero
        if (grad_VT)
            PA_CUDA_TRY(cudaMemsetAsync(grad_VT, 0, static_cast<size_t>(n_groups) * d_out * d *
                                                        (dtype == PA_F32 ? 4 : 2), s));
        return PA_OK;
    }
    PA_REQUIRE(grad && offsets && (!grad_query || VT) && (!grad_VT || query), "null pointer");
    if (dtype == PA_F32) {
        const float *dy = static_cast<const float *>(grad);
        if (grad_query)
            rc = grouped::rows_f32(static_cast<float *>(grad_query), dy,
                                   static_cast<const float *>(VT), offsets, rows, n_groups, d_out,
                                   d, ld_grad, ld_grad_query, true, s);
        if (rc == PA_OK && grad_VT)
            rc = grouped::matrices_f32(static_cast<float *>(grad_VT), dy,
                                       static_cast<const float *>(query), offsets, rows, n_groups,
                                       d, d_out, ld_grad, ld_query, s);
        return rc;
    }
    PA_REQUIRE(workspace || !pa_project_grouped_backward_workspace_bytes(
                                grad, query, VT, rows, n_groups, d, d_out, ld_grad, ld_query, dtype,
                                grad_query != nullptr, grad_VT != nullptr),
               "workspace missing (pa_project_grouped_backward_workspace_bytes)");
    PA_REQUIRE(aligned16(workspace), "workspace must be 16-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    rc = grouped::rows_make_ok(&grad, &ld_grad, rows, d_out, &ws, s);
    if (rc == PA_OK && grad_query) {
        int64_t ldw = d;
        rc = grouped::matrices_make_ok(&VT, &ldw, n_groups, d, d_out, offsets, rows, &ws, s);
        if (rc == PA_OK)
            rc = grouped::rows_16(grad_query, grad, ld_grad, VT, ldw, offsets, rows, n_groups,
                                  d_out, d, ld_grad_query, dtype, true, s);
    }
    if (rc == PA_OK && grad_VT) {
        rc = grouped::rows_make_ok(&query, &ld_query, rows, d, &ws, s);
        if (rc == PA_OK)
            rc = dtype == PA_BF16
                     ? grouped::matrices_mma<__nv_bfloat16>(grad_VT, grad, query, offsets, rows,
                                                            n_groups, d, d_out, ld_grad, ld_query, s)
                     : grouped::matrices_mma<__half>(grad_VT, grad, query, offsets, rows, n_groups,
                                                     d, d_out, ld_grad, ld_query, s);
    }
    return rc;
}
