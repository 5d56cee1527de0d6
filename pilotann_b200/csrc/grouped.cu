// Products of rows with the matrix of their group.  Rows of a group are contiguous:
// group g has rows [offsets[g], offsets[g + 1]).
//   forward   y[i, n]     = sum_k x[i, k]  w[g, n, k]
//   rows      dx[i, k]    = sum_n dy[i, n] w[g, n, k]
//   matrices  dw[g, n, k] = sum_{i in g} dy[i, n] x[i, k]
// Rows before offsets[0] and from offsets[n_groups] on belong to no group: y and dx are zero
// there.  Offsets are clamped to [0, rows], so that none of them makes an access leave the
// tensors, whatever they hold.
#include <cooperative_groups.h>

#include "grouped.cuh"
#include "tc05.cuh"

namespace pa {

namespace grouped {

namespace cg = cooperative_groups;

// ---- fp32 values: fma on the CUDA cores ---------------------------------------------
// Tiles of TR rows x TC columns by 256 threads, each TR / 16 x TC / 16 outputs:
//   C[r, c] = sum_t P(r, t) Q(c, t), P(r, t) = p[r * pr + t * pt], Q likewise,
// where the axis that is contiguous in memory is t (T_FAST) or r, c.  Slices of 16 t are copied to
// shared memory as they lie there, asynchronously and up to five slices ahead (a slice of a small
// tile is multiplied in 150 cycles, its data is 800 away), and read 16 bytes a thread.
// A sum is kept in two levels, 256 terms at a time, so that its error grows with the square root of
// 256 terms rather than of all (65536 rows in one sum: 5e-6 of the result in one level, below 1e-6 in
// two).  Where there are fewer tiles than the GPU can hold, a cluster of up to eight CTAs shares a tile
// and its sum, and adds the parts in order through distributed shared memory.
// 128 x 128 tiles keep the fma units 56 to 63 % busy, one CTA of eight warps an SM that waits for shared
// memory between them: 35, 37 and 39 TFLOP/s (forward, rows, matrices) for 8192 rows x 8 of 1024 x
// 1024, 40 to 45 for 16384 x 8 of 2048 x 2048.  Smaller tiles are bound by their loads: 30, 22 and 13
// TFLOP/s forward for 64, 32 and 16 rows a group, 64 groups of 1024 x 1024.
constexpr int kK = 16;
constexpr int kTerms = 256;
constexpr int kPitch = kK + 4;  // of a row of a T_FAST slice: 8 rows fall into different banks

template <int T, bool T_FAST> __host__ __device__ constexpr int slice_floats() {
    return T_FAST ? T * kPitch : kK * (T + 4);
}
template <int TR, int TC> __host__ __device__ constexpr int slices() {
    return TR * TC >= 128 * 128 ? 3 : TR * TC >= 64 * 64 ? 5 : 6;
}

__device__ __forceinline__ void copy_async(float *to, const float *from, int floats) {  // of 4
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc05::smem_u32(to)),
                 "l"(from), "r"(4 * floats)
                 : "memory");
}
__device__ __forceinline__ void copy_async1(float *to, const float *from, bool some) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc05::smem_u32(to)),
                 "l"(from), "r"(some ? 4 : 0)
                 : "memory");
}

// t0 .. t0 + 16 of the operand to `to`; zeros behind n_r, n_t.  vec: rows start on 16 bytes.
template <int T, bool T_FAST>
__device__ __forceinline__ void slice_load(float *to, const float *p, int64_t pr, int64_t pt, int n_r,
                                           int64_t t0, int64_t n_t, bool vec) {
    constexpr int kPieces = T * kK / 4;
    if (vec) {
#pragma unroll
        for (int j = threadIdx.x; j < kPieces; j += 256) {
            const int r = T_FAST ? j / 4 : 4 * (j % (T / 4)), t = T_FAST ? 4 * (j % 4) : j / (T / 4);
            const int64_t left = T_FAST ? (r < n_r ? n_t - t0 - t : 0) : (t0 + t < n_t ? n_r - r : 0);
            const int have = static_cast<int>(left < 0 ? 0 : left > 4 ? 4 : left);
            const float *from = T_FAST ? p + r * pr + t0 + t : p + (t0 + t) * pt + r;
            copy_async(to + (T_FAST ? r * kPitch + t : t * (T + 4) + r), have ? from : p, have);
        }
    } else {
#pragma unroll 4
        for (int j = threadIdx.x; j < 4 * kPieces; j += 256) {
            const int r = T_FAST ? j / kK : j % T, t = T_FAST ? j % kK : j / T;
            const bool some = r < n_r && t0 + t < n_t;
            copy_async1(to + (T_FAST ? r * kPitch + t : t * (T + 4) + r),
                        some ? p + r * pr + (t0 + t) * pt : p, some);
        }
    }
}

// the T / 16 rows of an operand that a thread has: every 16th of a T_FAST one, else four neighbours
// per 64 (or T / 16 neighbours)
template <int T, bool T_FAST> __device__ __forceinline__ int place(int thread, int i) {
    return T_FAST ? thread + 16 * i
           : T >= 64 ? 64 * (i / 4) + 4 * thread + i % 4 : (T / 16) * thread + i;
}
// v[k][i]: value t + k of row i of the thread
template <int T, bool T_FAST>
__device__ __forceinline__ void fetch4(float (&v)[4][T / 16], const float *s, int t, int thread) {
    if (T_FAST) {
#pragma unroll
        for (int i = 0; i < T / 16; ++i) {
            const float4 x = *reinterpret_cast<const float4 *>(s + (thread + 16 * i) * kPitch + t);
            v[0][i] = x.x; v[1][i] = x.y; v[2][i] = x.z; v[3][i] = x.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float *row = s + (t + k) * (T + 4);
            if constexpr (T >= 64) {
#pragma unroll
                for (int i = 0; i < T / 64; ++i) {
                    const float4 x = *reinterpret_cast<const float4 *>(row + 64 * i + 4 * thread);
                    v[k][4 * i] = x.x; v[k][4 * i + 1] = x.y;
                    v[k][4 * i + 2] = x.z; v[k][4 * i + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < T / 16; ++i) v[k][i] = row[(T / 16) * thread + i];
            }
        }
    }
}

template <int TR, int TC, bool PF, bool QF> __host__ __device__ constexpr int tile_bytes() {
    return 4 * slices<TR, TC>() * (slice_floats<TR, PF>() + slice_floats<TC, QF>());
}

struct Operand {
    const float *p;
    int64_t pr, pt;
    int n;
    bool vec;
};

template <int TR, int TC, bool PF, bool QF>
__device__ __forceinline__ void tile_product(float (&acc)[TR / 16][TC / 16], float *smem,
                                             const Operand &p, const Operand &q, int64_t n_t) {
    constexpr int S = slices<TR, TC>(), P = slice_floats<TR, PF>(), ALL = P + slice_floats<TC, QF>();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int n_slices = static_cast<int>((n_t + kK - 1) / kK);
    auto load = [&](int i) {
        if (i < n_slices) {
            float *to = smem + (i % S) * ALL;
            slice_load<TR, PF>(to, p.p, p.pr, p.pt, p.n, static_cast<int64_t>(i) * kK, n_t, p.vec);
            slice_load<TC, QF>(to + P, q.p, q.pr, q.pt, q.n, static_cast<int64_t>(i) * kK, n_t, q.vec);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float part[TR / 16][TC / 16] = {};
    for (int i = 0; i < S - 1; ++i) load(i);
    for (int i = 0; i < n_slices; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncthreads();  // slice i is here for all, slice i - 1 has been read by all
        load(i + S - 1);
        const float *ps = smem + (i % S) * ALL, *qs = ps + P;
#pragma unroll
        for (int t = 0; t < kK; t += 4) {
            float a[4][TR / 16], b[4][TC / 16];
            fetch4<TR, PF>(a, ps, t, ty);
            fetch4<TC, QF>(b, qs, t, tx);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int x = 0; x < TR / 16; ++x)
#pragma unroll
                    for (int y = 0; y < TC / 16; ++y)
                        part[x][y] = __fmaf_rn(a[k][x], b[k][y], part[x][y]);
        }
        if ((i + 1) % (kTerms / kK) == 0 || i + 1 == n_slices) {
#pragma unroll
            for (int x = 0; x < TR / 16; ++x)
#pragma unroll
                for (int y = 0; y < TC / 16; ++y) {
                    acc[x][y] += part[x][y];
                    part[x][y] = 0.0f;
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}

// The tile to memory.  In a cluster the CTAs have parts of the sum: each adds up, in the order of the
// CTAs, its share of the tile.
template <int TR, int TC, bool PF, bool QF>
__device__ __forceinline__ void tile_store(const float (&acc)[TR / 16][TC / 16], float *smem, float *out,
                                           int64_t ldo, int n_r, int n_c, bool vec) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks();
    if (parts == 1) {
#pragma unroll
        for (int i = 0; i < TR / 16; ++i) {
            const int r = place<TR, PF>(ty, i);
#pragma unroll
            for (int j = 0; j < TC / 16; j += QF ? 1 : 4) {
                const int c = place<TC, QF>(tx, j);
                if constexpr (!QF) {
                    if (r < n_r && c + 4 <= n_c && vec) {
                        *reinterpret_cast<float4 *>(out + r * ldo + c) =
                            make_float4(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (r < n_r && c + k < n_c) out[r * ldo + c + k] = acc[i][j + k];
                    }
                } else if (r < n_r && c < n_c) {
                    out[r * ldo + c] = acc[i][j];
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < TR / 16; ++i)
#pragma unroll
        for (int j = 0; j < TC / 16; ++j)
            smem[place<TR, PF>(ty, i) * TC + place<TC, QF>(tx, j)] = acc[i][j];
    cluster.sync();
    const int share = TR * TC / parts, first = share * cluster.block_rank();
    for (int e = first + threadIdx.x; e < first + share; e += 256) {
        float v = 0.0f;
        for (int k = 0; k < parts; ++k) v += cluster.map_shared_rank(smem, k)[e];
        const int r = e / TC, c = e % TC;
        if (r < n_r && c < n_c) out[r * ldo + c] = v;
    }
    cluster.sync();  // no CTA leaves while its part is read
}

// this CTA's share of a sum of n terms: whole slices
__device__ __forceinline__ void share_of(int64_t &lo, int64_t &hi) {
    const int parts = gridDim.z, k = blockIdx.z;  // a cluster spans z
    const int64_t n = hi - lo, each = (n + static_cast<int64_t>(parts) * kK - 1) / (parts * kK) * kK;
    const int64_t a = min(hi, lo + k * each);
    hi = min(hi, a + each);
    lo = a;
}

// The rows of slot `slot` of T rows: segment i owns the slots from floor(edge_i / T) + i on, which are
// enough for its tiles wherever it starts.  False: a slot without rows.  All threads of the CTA.
struct SlotRows { int seg; int64_t r0; int n_r; };
__device__ __forceinline__ bool slot_rows(SlotRows &s, const int64_t *offsets, int64_t rows,
                                          int n_groups, int64_t slot, int T) {
    int below = 0;  // segments that start at or before this slot
    for (int i0 = 0; i0 < n_groups + 2; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        below += __syncthreads_count(i < n_groups + 2 &&
                                     edge(offsets, n_groups, rows, i) / T + i <= slot);
    }
    s.seg = below - 1;
    const int64_t lo = edge(offsets, n_groups, rows, s.seg),
                  hi = edge(offsets, n_groups, rows, s.seg + 1);
    s.r0 = lo + (slot - (lo / T + s.seg)) * T;
    s.n_r = static_cast<int>(min(static_cast<int64_t>(T), hi - s.r0));
    return s.r0 >= lo && s.n_r > 0;
}

// Rows side: forward (W_T_FAST: w's last axis is summed) and the gradient of the rows.
template <int TR, int TC, bool W_T_FAST>
__global__ void __launch_bounds__(256)
rows_kernel(float *__restrict__ out, const float *__restrict__ x, const float *__restrict__ w,
            const int64_t *__restrict__ offsets, int64_t rows, int n_groups, int d_sum, int d_out,
            int64_t ldx, int64_t ldo, bool x_vec, bool w_vec, bool out_vec) {
    extern __shared__ __align__(16) float smem[];
    SlotRows slot;
    if (!slot_rows(slot, offsets, rows, n_groups, blockIdx.x, TR)) return;  // the whole cluster
    const int c0 = blockIdx.y * TC, n_c = min(TC, d_out - c0);
    float acc[TR / 16][TC / 16] = {};
    if (slot.seg >= 1 && slot.seg <= n_groups) {
        int64_t lo = 0, hi = d_sum;
        share_of(lo, hi);
        const float *wg = w + static_cast<int64_t>(slot.seg - 1) * d_sum * d_out;
        const Operand p{x + slot.r0 * ldx + lo, ldx, 1, slot.n_r, x_vec};
        const Operand q = W_T_FAST
                              ? Operand{wg + static_cast<int64_t>(c0) * d_sum + lo, d_sum, 1, n_c, w_vec}
                              : Operand{wg + lo * d_out + c0, 1, d_out, n_c, w_vec};
        tile_product<TR, TC, true, W_T_FAST>(acc, smem, p, q, hi - lo);
    }
    tile_store<TR, TC, true, W_T_FAST>(acc, smem, out + slot.r0 * ldo + c0, ldo, slot.n_r, n_c,
                                        out_vec);
}

// Gradient of the matrices: one tile of one group, summed over its rows.  blockIdx.x = tile along d
// and group.
template <int T>
__global__ void __launch_bounds__(256)
matrices_kernel(float *__restrict__ dw, const float *__restrict__ dy, const float *__restrict__ x,
                const int64_t *__restrict__ offsets, int64_t rows, int n_groups, int d, int d_out,
                int64_t ldy, int64_t ldx, bool y_vec, bool x_vec, bool out_vec) {
    extern __shared__ __align__(16) float smem[];
    const int d_tiles = (d + T - 1) / T, g = blockIdx.x / d_tiles;
    const int n0 = blockIdx.y * T, k0 = (blockIdx.x - g * d_tiles) * T;
    const int n_n = min(T, d_out - n0), n_k = min(T, d - k0);
    int64_t lo = edge(offsets, n_groups, rows, g + 1), hi = edge(offsets, n_groups, rows, g + 2);
    float acc[T / 16][T / 16] = {};
    if (hi > lo) {
        share_of(lo, hi);
        const Operand p{dy + lo * ldy + n0, 1, ldy, n_n, y_vec}, q{x + lo * ldx + k0, 1, ldx, n_k, x_vec};
        tile_product<T, T, false, false>(acc, smem, p, q, hi - lo);
    }
    tile_store<T, T, false, false>(acc, smem, dw + (static_cast<int64_t>(g) * d_out + n0) * d + k0, d,
                                   n_n, n_k, out_vec);
}

// Forward of groups of a few rows, which read their matrix and do little with it: a warp has two rows
// of w, its lanes run along them, four values (or one) each, and multiply them with up to eight
// rows of x from shared memory; butterfly over the lanes.  512 matrices of 1024 x 1024: 467 us for one
// row a group (4.6 TB/s, 70 % of the copy rate), 623 for four, 866 for eight, where its reads of x
// from shared memory bind; 16 x 64 tiles take 1243 for nine to sixteen.
constexpr int kFewRows = 8;
constexpr int kFewWarps = 8;
constexpr int kFewSlice = 1024;  // values of a row of x in shared memory

template <bool VEC>
__global__ void __launch_bounds__(32 * kFewWarps)
rows_few_kernel(float *__restrict__ out, const float *__restrict__ x, const float *__restrict__ w,
                const int64_t *__restrict__ offsets, int64_t rows, int n_groups, int d_sum,
                int d_out, int64_t ldx, int64_t ldo) {
    __shared__ __align__(16) float x_s[kFewRows][kFewSlice];
    const int lane = threadIdx.x & 31;
    SlotRows slot;
    if (!slot_rows(slot, offsets, rows, n_groups, blockIdx.x, kFewRows)) return;
    const int c0 = 2 * (blockIdx.y * kFewWarps + (threadIdx.x >> 5));
    const bool some = slot.seg >= 1 && slot.seg <= n_groups;
    const float *w0 = w + (static_cast<int64_t>(slot.seg - 1) * d_out + c0) * d_sum, *w1 = w0 + d_sum;
    float acc[kFewRows][2] = {};
    for (int t0 = 0; some && t0 < d_sum; t0 += kFewSlice) {
        const int len = min(kFewSlice, d_sum - t0);
        __syncthreads();
        for (int r = 0; r < slot.n_r; ++r)
            for (int t = threadIdx.x; t < len; t += 32 * kFewWarps)
                x_s[r][t] = __ldg(x + (slot.r0 + r) * ldx + t0 + t);
        __syncthreads();
        constexpr int N = VEC ? 4 : 1;
#pragma unroll 4
        for (int t = N * lane; t < len; t += 32 * N) {
            float a[N], b[N];
            if constexpr (VEC) {
                const float4 z = make_float4(0, 0, 0, 0);
                const float4 u = c0 < d_out ? __ldg(reinterpret_cast<const float4 *>(w0 + t0 + t)) : z;
                const float4 v = c0 + 1 < d_out ? __ldg(reinterpret_cast<const float4 *>(w1 + t0 + t)) : z;
                a[0] = u.x; a[1] = u.y; a[2] = u.z; a[3] = u.w;
                b[0] = v.x; b[1] = v.y; b[2] = v.z; b[3] = v.w;
            } else {
                a[0] = c0 < d_out ? __ldg(w0 + t0 + t) : 0.0f;
                b[0] = c0 + 1 < d_out ? __ldg(w1 + t0 + t) : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < kFewRows; ++r)
                if (r < slot.n_r) {  // uniform
                    float xv[N];
                    if constexpr (VEC) {
                        const float4 u = *reinterpret_cast<const float4 *>(&x_s[r][t]);
                        xv[0] = u.x; xv[1] = u.y; xv[2] = u.z; xv[3] = u.w;
                    } else {
                        xv[0] = x_s[r][t];
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        acc[r][0] = __fmaf_rn(xv[i], a[i], acc[r][0]);
                        acc[r][1] = __fmaf_rn(xv[i], b[i], acc[r][1]);
                    }
                }
        }
    }
#pragma unroll
    for (int r = 0; r < kFewRows; ++r)
        if (r < slot.n_r) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v = acc[r][c];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == c && c0 + c < d_out) out[(slot.r0 + r) * ldo + c0 + c] = v;
            }
        }
}

// ---- 16-bit operands that a bulk-tensor copy cannot read --------------------------
// Rows that do not start on 16 bytes (an odd width, a slice of a wider tensor) are copied into
// the workspace with a pitch of whole 16 bytes first; the products then run on that.  A copy
// reads and writes the operand once (of the matrices only those whose group has rows), which the
// tensor cores win back many times over plain loads: 4099 rows x 13 matrices of 333 x 200, all
// gradients, 178 us a step with 64 x 64 tiles of plain loads, 113 so (80 of it autograd's).
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

bool vec4(const void *p, int64_t ld) { return aligned16(p) && ld % 4 == 0; }

// CTAs that share a tile: until there are two for every SM, with 128 terms each at least
int parts_of(int64_t tiles, int64_t terms) {
    int parts = 1;
    while (parts < 8 && tiles * parts < 2 * 148 && terms >= 2 * 128 * parts) parts *= 2;
    return parts;
}

template <typename... P, typename... A>
int launch_tiles(void (*kernel)(P...), dim3 grid, int smem, cudaStream_t s, A... args) {
    if (smem > 48 * 1024)
        PA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(256);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = cluster.val.clusterDim.y = 1;
    cluster.val.clusterDim.z = grid.z;
    config.attrs = &cluster;
    config.numAttrs = 1;
    PA_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...));
    count_launch();
    return PA_OK;
}

template <int TR, int TC>
int rows_tiles(float *out, const float *x, const float *w, const int64_t *offsets, int64_t rows,
               int n_groups, int d_sum, int d_out, int64_t ldx, int64_t ldo, bool transposed,
               cudaStream_t s) {
    dim3 grid(static_cast<unsigned>(rows / TR + n_groups + 2),
              static_cast<unsigned>((d_out + TC - 1) / TC));
    // tiles that have rows: not more than the rows
    const int64_t tiles = (rows / TR + (rows < n_groups ? rows : n_groups)) * grid.y;
    grid.z = TR * TC > 64 * 64 ? 1 : parts_of(tiles, d_sum);
    const bool x_vec = vec4(x, ldx), w_vec = vec4(w, transposed ? d_out : d_sum);
    if (transposed)
        return launch_tiles(rows_kernel<TR, TC, false>, grid, tile_bytes<TR, TC, true, false>(), s, out,
                            x, w, offsets, rows, n_groups, d_sum, d_out, ldx, ldo, x_vec, w_vec,
                            vec4(out, ldo));
    return launch_tiles(rows_kernel<TR, TC, true>, grid, tile_bytes<TR, TC, true, true>(), s, out, x, w,
                        offsets, rows, n_groups, d_sum, d_out, ldx, ldo, x_vec, w_vec, vec4(out, ldo));
}

int rows_f32(float *out, const float *x, const float *w, const int64_t *offsets, int64_t rows,
             int n_groups, int d_sum, int d_out, int64_t ldx, int64_t ldo, bool transposed,
             cudaStream_t s) {
    const int64_t each = (rows + n_groups - 1) / n_groups;  // on average
    if (!transposed && each <= kFewRows) {
        dim3 grid(static_cast<unsigned>(rows / kFewRows + n_groups + 2),
                  static_cast<unsigned>((d_out + 2 * kFewWarps - 1) / (2 * kFewWarps)));
        if (vec4(w, d_sum))
            rows_few_kernel<true><<<grid, 32 * kFewWarps, 0, s>>>(out, x, w, offsets, rows, n_groups,
                                                                  d_sum, d_out, ldx, ldo);
        else
            rows_few_kernel<false><<<grid, 32 * kFewWarps, 0, s>>>(out, x, w, offsets, rows, n_groups,
                                                                   d_sum, d_out, ldx, ldo);
        count_launch();
        PA_CUDA_TRY(cudaGetLastError());
        return PA_OK;
    }
#define PA_GO(TR, TC) \
    return rows_tiles<TR, TC>(out, x, w, offsets, rows, n_groups, d_sum, d_out, ldx, ldo, transposed, s)
    if (each <= 16) PA_GO(16, 64);
    if (each <= 32) PA_GO(32, 64);
    // 128 x 128 needs a tile for every SM and groups that fill it
    if (each <= 192 || d_out <= 64 || (rows / 128) * ((d_out + 127) / 128) < 148) PA_GO(64, 64);
    PA_GO(128, 128);
#undef PA_GO
}

template <int T>
int matrices_tiles(float *dw, const float *dy, const float *x, const int64_t *offsets, int64_t rows,
                   int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s) {
    dim3 grid(static_cast<unsigned>((d + T - 1) / T) * n_groups,
              static_cast<unsigned>((d_out + T - 1) / T));
    grid.z = T > 64 ? 1 : parts_of(static_cast<int64_t>(grid.x) * grid.y, rows / n_groups);
    return launch_tiles(matrices_kernel<T>, grid, tile_bytes<T, T, false, false>(), s, dw, dy, x,
                        offsets, rows, n_groups, d, d_out, ldy, ldx, vec4(dy, ldy), vec4(x, ldx),
                        vec4(dw, d));
}

int matrices_f32(float *dw, const float *dy, const float *x, const int64_t *offsets, int64_t rows,
                 int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s) {
    const int64_t large = static_cast<int64_t>((d + 127) / 128) * ((d_out + 127) / 128) * n_groups;
    if (d > 64 && d_out > 64 && large >= 148)
        return matrices_tiles<128>(dw, dy, x, offsets, rows, n_groups, d, d_out, ldy, ldx, s);
    return matrices_tiles<64>(dw, dy, x, offsets, rows, n_groups, d, d_out, ldy, ldx, s);
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

bool aligned(int dtype, const int64_t *offsets, const void *a, const void *b, const void *c) {
    const size_t size = dtype == PA_F32 ? 4 : 2;
    return aligned_to(a, size) && aligned_to(b, size) && aligned_to(c, size) && aligned_to(offsets, 8);
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
    PA_REQUIRE(grouped::aligned(dtype, offsets, out, query, VT), "operands must be aligned to their values");
    if ((rc = product_check()) != PA_OK) return rc;
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
    PA_REQUIRE(grouped::aligned(dtype, offsets, grad_query, grad_VT, grad) &&
                   grouped::aligned(dtype, offsets, query, VT, nullptr),
               "operands must be aligned to their values");
    if ((rc = product_check()) != PA_OK) return rc;
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
