// Rows sorted by the router they were sent to: a stable counting sort of int64 ids.
//   offsets[g] = rows with an id in [0, g),  order = row numbers, ascending within a group;
// rows with an id outside [0, n_groups) come last, in order, behind offsets[n_groups].
//
// Rows are cut into blocks of kBlockRows; within a block every warp owns a run of
// consecutive rows and a counter per group in shared memory, so that the place of a row is
// (rows of earlier groups) + (earlier blocks) + (earlier warps) + (earlier rows of the warp):
// no counter is ever shared between rows whose order matters, and the result does not depend
// on timing.  One block: one launch.  More: a histogram per block, one CTA that turns the
// histograms into places, and the pass that writes.  Bound by launch latency up to some ten
// thousand rows; above that by the three passes over the ids (8 bytes a row each, from L2
// after the first).
#include "pa_common.cuh"

namespace pa {

namespace group {
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlockRows = 8192;
constexpr int kScanThreads = 1024;
}  // namespace group

__device__ __forceinline__ int group_of(int64_t id, int n_groups) {
    return id >= 0 && id < n_groups ? static_cast<int>(id) : n_groups;
}

__global__ void __launch_bounds__(group::kThreads)
group_count_kernel(int32_t *__restrict__ block_counts, const int64_t *__restrict__ ids,
                   int64_t rows, int n_groups) {
    extern __shared__ int32_t count_s[];  // [n_groups + 1]
    const int bins = n_groups + 1;
    for (int g = threadIdx.x; g < bins; g += group::kThreads) count_s[g] = 0;
    __syncthreads();
    const int64_t r0 = blockIdx.x * static_cast<int64_t>(group::kBlockRows);
    const int n = static_cast<int>(min(static_cast<int64_t>(group::kBlockRows), rows - r0));
    for (int i = threadIdx.x; i < n; i += group::kThreads)
        atomicAdd(&count_s[group_of(__ldg(ids + r0 + i), n_groups)], 1);
    __syncthreads();
    for (int g = threadIdx.x; g < bins; g += group::kThreads)
        block_counts[blockIdx.x * static_cast<int64_t>(bins) + g] = count_s[g];
}

// exclusive prefix of v over the CTA's threads (all call it); *total receives the sum
__device__ __forceinline__ int64_t cta_exclusive(int64_t v, int64_t *warp_sum_s, int64_t *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum_s[w] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < warps; ++i) {
        const int64_t s = warp_sum_s[i];
        if (i < w) before += s;
        all += s;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// histograms of the blocks -> places of the blocks within their group; offsets
__global__ void __launch_bounds__(group::kScanThreads)
group_scan_kernel(int64_t *__restrict__ offsets, int32_t *__restrict__ block_counts, int n_blocks,
                  int n_groups) {
    __shared__ int64_t warp_sum_s[32];
    const int bins = n_groups + 1;
    int64_t base = 0;
    for (int g0 = 0; g0 < bins; g0 += group::kScanThreads) {
        const int g = g0 + threadIdx.x;
        int32_t sum = 0;
        if (g < bins) {
            int32_t *p = block_counts + g;
            for (int b = 0; b < n_blocks; b += 8) {  // eight loads in flight
                int32_t c[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    c[j] = b + j < n_blocks ? p[static_cast<int64_t>(b + j) * bins] : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (b + j < n_blocks) p[static_cast<int64_t>(b + j) * bins] = sum;
                    sum += c[j];
                }
            }
        }
        int64_t total;
        const int64_t place = cta_exclusive(sum, warp_sum_s, &total) + base;
        if (g < bins) offsets[g] = place;  // offsets[n_groups]: where the ungrouped rows start
        base += total;
    }
}

// block_counts == nullptr: this CTA has all rows and makes the offsets itself
__global__ void __launch_bounds__(group::kThreads)
group_scatter_kernel(int64_t *__restrict__ order, int64_t *__restrict__ offsets,
                     const int32_t *__restrict__ block_counts, const int64_t *__restrict__ ids,
                     int64_t rows, int n_groups) {
    extern __shared__ int32_t count_s[];  // [kWarps][n_groups + 1]
    __shared__ int64_t warp_sum_s[32];
    const int bins = n_groups + 1, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < group::kWarps * bins; i += group::kThreads) count_s[i] = 0;
    __syncthreads();
    const int64_t r0 = blockIdx.x * static_cast<int64_t>(group::kBlockRows);
    const int n = static_cast<int>(min(static_cast<int64_t>(group::kBlockRows), rows - r0));
    // each warp a run of whole groups of 32 rows
    const int run = 32 * ((n + 32 * group::kWarps - 1) / (32 * group::kWarps));
    const int lo = min(n, w * run), hi = min(n, lo + run);
    int32_t *mine = count_s + w * bins;
    for (int i = lo + lane; i < hi; i += 32)
        atomicAdd(&mine[group_of(__ldg(ids + r0 + i), n_groups)], 1);
    __syncthreads();
    // places: rows of earlier groups and blocks, then of earlier warps (32 bits: rows < 2^31)
    int64_t base = 0;
    for (int g0 = 0; g0 < bins; g0 += group::kThreads) {
        const int g = g0 + threadIdx.x;
        int32_t sum = 0;
        if (g < bins)
            for (int i = 0; i < group::kWarps; ++i) sum += count_s[i * bins + g];
        int64_t place;
        if (block_counts == nullptr) {
            int64_t total;
            place = cta_exclusive(sum, warp_sum_s, &total) + base;
            base += total;
            if (g < bins) offsets[g] = place;
        } else {
            place = g < bins ? offsets[g] + block_counts[blockIdx.x * static_cast<int64_t>(bins) + g]
                             : 0;
        }
        if (g < bins) {
            int32_t at = static_cast<int32_t>(place);
            for (int i = 0; i < group::kWarps; ++i) {
                const int32_t c = count_s[i * bins + g];
                count_s[i * bins + g] = at;
                at += c;
            }
        }
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const bool live = i < hi;
        // lanes past the end share a key that no row has
        const int g = live ? group_of(__ldg(ids + r0 + i), n_groups) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, g);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        int32_t at = 0;
        if (live) at = mine[g];
        __syncwarp();
        if (live && rank == 0) mine[g] = at + __popc(peers);
        __syncwarp();
        if (live) order[at + rank] = r0 + i;
    }
}

}  // namespace pa

extern "C" int64_t pa_group_rows_workspace_bytes(int64_t rows, int n_groups) {
    if (rows <= pa::group::kBlockRows || n_groups < 1) return 0;
    const int64_t blocks = (rows + pa::group::kBlockRows - 1) / pa::group::kBlockRows;
    return blocks * (n_groups + 1) * static_cast<int64_t>(sizeof(int32_t));
}

extern "C" int pa_group_rows(int64_t *order, int64_t *offsets, const int64_t *router, int64_t rows,
                             int n_groups, void *workspace, void *stream) {
    using namespace pa;
    PA_REQUIRE(rows >= 0 && rows <= PA_MAX_ROWS, "rows out of range");
    PA_REQUIRE(n_groups >= 1 && n_groups <= PA_MAX_GROUPS, "n_groups must be in [1, %d]",
               PA_MAX_GROUPS);
    PA_REQUIRE(offsets && (rows == 0 || (order && router)), "null pointer");
    const int bins = n_groups + 1;
    const int blocks = static_cast<int>((rows + group::kBlockRows - 1) / group::kBlockRows);
    PA_REQUIRE(blocks <= 1 || workspace, "workspace missing (pa_group_rows_workspace_bytes)");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t scatter_smem = static_cast<size_t>(group::kWarps) * bins * sizeof(int32_t);
    if (scatter_smem > 48 * 1024)
        PA_CUDA_TRY(cudaFuncSetAttribute(group_scatter_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(scatter_smem)));
    int32_t *counts = blocks > 1 ? static_cast<int32_t *>(workspace) : nullptr;
    if (blocks > 1) {
        group_count_kernel<<<blocks, group::kThreads, bins * sizeof(int32_t), s>>>(counts, router,
                                                                                   rows, n_groups);
        group_scan_kernel<<<1, group::kScanThreads, 0, s>>>(offsets, counts, blocks, n_groups);
        count_launch(2);
    }
    group_scatter_kernel<<<blocks > 1 ? blocks : 1, group::kThreads, scatter_smem, s>>>(
        order, offsets, counts, router, rows, n_groups);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}
