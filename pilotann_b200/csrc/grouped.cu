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

// rows of 16-bit values that a bulk-tensor copy can start at
bool ldi_ok(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

template <typename T>
int rows_launch(void *out, const void *x, const void *w, const int64_t *offsets, int64_t rows,
                int n_groups, int d_sum, int d_out, int64_t ldx, int64_t ldo, bool transposed,
                cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        const int64_t ldw = transposed ? d_out : d_sum;
        if (ldi_ok(x, ldx) && ldi_ok(w, ldw))
            return rows_mma<T>(out, x, w, offsets, rows, n_groups, d_sum, d_out, ldx, ldo,
                               transposed, s);
    }
    dim3 grid(static_cast<unsigned>(rows / kT + n_groups + 2),
              static_cast<unsigned>((d_out + kT - 1) / kT));
    if (transposed)
        rows_kernel<T, false><<<grid, 256, 0, s>>>(static_cast<T *>(out), static_cast<const T *>(x),
                                                   static_cast<const T *>(w), offsets, rows,
                                                   n_groups, d_sum, d_out, ldx, ldo);
    else
        rows_kernel<T, true><<<grid, 256, 0, s>>>(static_cast<T *>(out), static_cast<const T *>(x),
                                                  static_cast<const T *>(w), offsets, rows,
                                                  n_groups, d_sum, d_out, ldx, ldo);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

template <typename T>
int matrices_launch(void *dw, const void *dy, const void *x, const int64_t *offsets, int64_t rows,
                    int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (rows > 0 && ldi_ok(dy, ldy) && ldi_ok(x, ldx))
            return matrices_mma<T>(dw, dy, x, offsets, rows, n_groups, d, d_out, ldy, ldx, s);
    }
    dim3 grid(static_cast<unsigned>((d + kT - 1) / kT), static_cast<unsigned>((d_out + kT - 1) / kT),
              static_cast<unsigned>(n_groups));
    matrices_kernel<T><<<grid, 256, 0, s>>>(static_cast<T *>(dw), static_cast<const T *>(dy),
                                            static_cast<const T *>(x), offsets, rows, n_groups, d,
                                            d_out, ldy, ldx);
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

int project_rows(void *out, const void *in, const void *w, const int64_t *offsets, int64_t rows,
                 int n_groups, int d_sum, int d_out, int64_t ldi, int64_t ldo, int dtype,
                 bool transposed, cudaStream_t s) {
    if (dtype == PA_F32)
        return rows_launch<float>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi, ldo,
                                  transposed, s);
    if (dtype == PA_BF16)
        return rows_launch<__nv_bfloat16>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi,
                                          ldo, transposed, s);
    return rows_launch<__half>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi, ldo,
                               transposed, s);
}

}  // namespace grouped
}  // namespace pa

extern "C" int pa_project_grouped(void *out, const void *query, const void *VT,
                                  const int64_t *offsets, int64_t rows, int n_groups, int d,
                                  int d_out, int64_t ld_query, int64_t ld_out, int dtype,
                                  void *stream) {
    using namespace pa;
    int rc = grouped::check(rows, n_groups, d, d_out, dtype);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(ld_query >= d && ld_out >= d_out, "row strides must cover the rows");
    if (rows == 0) return PA_OK;
    PA_REQUIRE(out && query && VT && offsets, "null pointer");
    return grouped::project_rows(out, query, VT, offsets, rows, n_groups, d, d_out, ld_query,
                                 ld_out, dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int pa_project_grouped_backward(void *grad_query, void *grad_VT, const void *grad,
                                           const void *query, const void *VT,
                                           const int64_t *offsets, int64_t rows, int n_groups,
                                           int d, int d_out, int64_t ld_grad, int64_t ld_query,
                                           int64_t ld_grad_query, int dtype, void *stream) {
    using namespace pa;
    int rc = grouped::check(rows, n_groups, d, d_out, dtype);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(ld_grad >= d_out, "row strides must cover the rows");
    PA_REQUIRE(!grad_query || ld_grad_query >= d, "row strides must cover the rows");
    PA_REQUIRE(!grad_VT || ld_query >= d, "row strides must cover the rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (grad_query && rows > 0) {
        PA_REQUIRE(grad && VT && offsets, "null pointer");
        rc = grouped::project_rows(grad_query, grad, VT, offsets, rows, n_groups, d_out, d, ld_grad,
                                   ld_grad_query, dtype, true, s);
        if (rc != PA_OK) return rc;
    }
    if (grad_VT) {
        PA_REQUIRE(offsets && (rows == 0 || (grad && query)), "null pointer");
        if (dtype == PA_F32)
            rc = grouped::matrices_launch<float>(grad_VT, grad, query, offsets, rows, n_groups, d,
                                                 d_out, ld_grad, ld_query, s);
        else if (dtype == PA_BF16)
            rc = grouped::matrices_launch<__nv_bfloat16>(grad_VT, grad, query, offsets, rows,
                                                         n_groups, d, d_out, ld_grad, ld_query, s);
        else
            rc = grouped::matrices_launch<__half>(grad_VT, grad, query, offsets, rows, n_groups, d,
                                                  d_out, ld_grad, ld_query, s);
    }
    return rc;
}
