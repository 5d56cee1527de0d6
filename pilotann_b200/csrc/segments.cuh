// Tiles of the rows of each group, worked out by every CTA of a persistent kernel from the
// offsets on the device.
#pragma once

#include "grouped.cuh"

namespace pa {
namespace grouped {

struct Segments {
    int edge[PA_MAX_GROUPS + 3];   // first row of segment i, ascending
    int tiles[PA_MAX_GROUPS + 3];  // row tiles before segment i
    int part[32];                  // of the prefix sums
};

// inclusive prefix over the CTA's threads (all call it): maximum or sum; *all is over all of them
template <int THREADS, bool MAX>
__device__ __forceinline__ int cta_scan(int v, int *warp_part_s, int *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = MAX ? max(v, y) : v + y;
    }
    if (lane == 31) warp_part_s[warp] = v;
    __syncthreads();
    int before = 0, total = 0;  // the values are not negative
    for (int w = 0; w < THREADS / 32; ++w) {
        const int p = warp_part_s[w];
        if (w < warp) before = MAX ? max(before, p) : before + p;
        total = MAX ? max(total, p) : total + p;
    }
    __syncthreads();
    *all = total;
    return MAX ? max(before, v) : before + v;
}

// All threads of the CTA; a barrier is still needed behind it.  offsets == nullptr: one group that
// has all rows.
template <int THREADS>
__device__ __forceinline__ void segs_make(Segments &s, const int64_t *offsets, int n_groups,
                                          int rows, int tile_rows) {
    const int segs = n_groups + 2;
    int carry = 0;
    for (int i0 = 0; i0 <= segs; i0 += THREADS) {  // edges, made to ascend
        const int i = i0 + threadIdx.x;
        int e = 0;
        if (i <= segs)
            e = offsets ? static_cast<int>(edge(offsets, n_groups, rows, i)) : (i <= 1 ? 0 : rows);
        int all;
        const int v = cta_scan<THREADS, true>(e, s.part, &all);
        if (i <= segs) s.edge[i] = max(carry, v);
        carry = max(carry, all);
    }
    __syncthreads();
    carry = 0;
    for (int i0 = 0; i0 < segs; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        const int own =
            i < segs ? (static_cast<unsigned>(s.edge[i + 1] - s.edge[i]) + tile_rows - 1) / tile_rows
                     : 0;
        int all;
        const int v = cta_scan<THREADS, false>(own, s.part, &all);
        if (i < segs) s.tiles[i] = carry + v - own;
        carry += all;
    }
    if (threadIdx.x == 0) s.tiles[segs] = carry;
}

// The tiles of one CTA: every `step`-th of rows x n_col tiles, columns innermost, without a division
// a tile; the segment of the row is looked for from the last one on.  (Results fit the memory, so
// tile numbers fit 32 bits.)
struct Walk {
    int row, col, seg;
    int step_row, step_col, n_col, n_row;

    __device__ __forceinline__ Walk(int first, int step, int n_row_, int n_col_)
        : row(first / n_col_), col(first % n_col_), seg(0), step_row(step / n_col_),
          step_col(step % n_col_), n_col(n_col_), n_row(n_row_) {}
    __device__ __forceinline__ bool live() const { return row < n_row; }
    __device__ __forceinline__ void next() {
        row += step_row;
        col += step_col;
        if (col >= n_col) { col -= n_col; ++row; }
    }
    __device__ __forceinline__ int segment(const Segments &s) {
        while (s.tiles[seg + 1] <= row) ++seg;
        return seg;
    }
};

}  // namespace grouped
}  // namespace pa
