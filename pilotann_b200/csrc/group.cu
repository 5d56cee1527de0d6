// Rows sorted by the router they were sent to: a stable counting sort of int64 ids.
//   offsets[g] = rows with an id in [0, g),  order = row numbers, ascending within a group;
// rows with an id outside [0, n_groups) come last, in order, behind offsets[n_groups].
//
// Rows are cut into blocks of kBlockRows; within a block every warp owns a run of
// consecutive rows and a counter per group in shared memory, so that the place of a row is
// (rows of earlier groups) + (earlier blocks) + (earlier warps) + (earlier rows of the warp):
// no counter is ever shared between rows whose order matters, and the result does not depend
// on timing.  Up to kSingleRows rows: one launch of one CTA, bound by its latency (1024 ids, 64
// groups: 5 us on the GPU, less than the call).  More: a histogram per block; the places of the
// blocks within each group, 32 groups a CTA, and the groups' sums; the pass that writes.
// The passes read 8 bytes a row twice, the second time from L2, and write 8.  1000000 ids, 1024 groups:
// 26.6 us, 5 + 8 + 13, bound by the chain of the three and by stores of 8 bytes to 1024 places.
#include "pa_common.cuh"

namespace pa {

namespace group {
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlockRows = 256 * kWarps;
constexpr int kSingleRows = 2 * kBlockRows;  // by a CTA of twice the warps
constexpr int kScanBlocks = 256;  // blocks of rows per step of the scan: 32 warps, 8 blocks each
}  // namespace group

__device__ __forceinline__ int group_of(int64_t id, int n_groups) {
    return id >= 0 && id < n_groups ? static_cast<int>(id) : n_groups;
}

__global__ void __launch_bounds__(group::kThreads)
group_count_kernel(int32_t *__restrict__ block_counts, unsigned *__restrict__ done,
                   const int64_t *__restrict__ ids, int64_t rows, int n_groups) {
    extern __shared__ int32_t count_s[];  // [n_groups + 1]
    const int bins = n_groups + 1;
    if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;
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

// exclusive prefix of v over the CTA's threads (all call it); *total receives the sum (32 bits: rows
// < 2^31)
__device__ __forceinline__ int32_t cta_exclusive(int32_t v, int32_t *warp_sum_s, int32_t *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum_s[w] = x;
    __syncthreads();
    int32_t sums = lane < warps ? warp_sum_s[lane] : 0;  // every warp adds them up for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t y = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += y;
    }
    *total = __shfl_sync(0xffffffffu, sums, 31);
    const int32_t before = __shfl_sync(0xffffffffu, sums, w == 0 ? 0 : w - 1);
    __syncthreads();
    return (w == 0 ? 0 : before) + x - v;
}

// Histograms of the blocks -> places of the blocks within their group; sums of the groups.  A lane
// has a group, a warp eight consecutive blocks, so that loads and stores are whole lines.  The CTA that
// is done last adds up the groups.
__global__ void __launch_bounds__(1024)
group_scan_kernel(int64_t *__restrict__ offsets, int32_t *__restrict__ totals, unsigned *done,
                  int32_t *__restrict__ block_counts, int n_blocks, int n_groups) {
    __shared__ int32_t part_s[32][33];
    const int bins = n_groups + 1, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int g = blockIdx.x * 32 + lane;
    int32_t carry = 0;
    for (int b0 = 0; b0 < n_blocks; b0 += group::kScanBlocks) {
        int32_t *p = block_counts + static_cast<int64_t>(b0 + 8 * w) * bins + g;
        int32_t c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            c[j] = g < bins && b0 + 8 * w + j < n_blocks ? p[static_cast<int64_t>(j) * bins] : 0;
        int32_t sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int32_t v = c[j];
            c[j] = sum;
            sum += v;
        }
        part_s[w][lane] = sum;
        __syncthreads();
        int32_t before = carry, all = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int32_t v = part_s[i][lane];
            if (i < w) before += v;
            all += v;
        }
        carry += all;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (g < bins && b0 + 8 * w + j < n_blocks)
                p[static_cast<int64_t>(j) * bins] = before + c[j];
        __syncthreads();
    }
    if (w == 0 && g < bins) totals[g] = carry;
    __shared__ bool last_s;
    __shared__ int32_t warp_sum_s[32];
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last_s = atomicAdd(done, 1u) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last_s) return;
    int32_t base = 0;
    for (int g0 = 0; g0 < bins; g0 += 1024) {
        const int i = g0 + threadIdx.x;
        int32_t total;
        const int32_t at = cta_exclusive(i < bins ? __ldcg(totals + i) : 0, warp_sum_s, &total) + base;
        if (i < bins) offsets[i] = at;  // [n_groups]: where the ungrouped rows start
        base += total;
    }
}

// A warp has 256 consecutive rows, eight a lane, kept in registers from the count to the end.
// block_counts == nullptr: this CTA has all rows and makes the offsets itself.
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
group_scatter_kernel(int64_t *__restrict__ order, int64_t *__restrict__ offsets,
                     const int32_t *__restrict__ block_counts, const int64_t *__restrict__ ids,
                     int64_t rows, int n_groups) {
    extern __shared__ int32_t count_s[];  // [WARPS][n_groups + 1]
    __shared__ int32_t warp_sum_s[32];
    constexpr int kThreads = 32 * WARPS, kEach = 8;
    const int bins = n_groups + 1, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t lo = (blockIdx.x * static_cast<int64_t>(WARPS) + w) * (32 * kEach) + lane;
    int g[kEach];  // -1: no row
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        g[j] = lo + 32 * j < rows ? group_of(__ldg(ids + lo + 32 * j), n_groups) : -1;
    for (int i = threadIdx.x; i < WARPS * bins; i += kThreads) count_s[i] = 0;
    __syncthreads();
    int32_t *mine = count_s + w * bins;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (g[j] >= 0) atomicAdd(&mine[g[j]], 1);
    __syncthreads();
    // places: rows of earlier groups and blocks, then of earlier warps
    int32_t base = 0;
    for (int g0 = 0; g0 < bins; g0 += kThreads) {
        const int i = g0 + threadIdx.x;
        int32_t place = 0;
        if (block_counts != nullptr) {
            if (i < bins)
                place = static_cast<int32_t>(__ldg(offsets + i)) +
                        __ldg(block_counts + blockIdx.x * static_cast<int64_t>(bins) + i);
        } else {
            int32_t sum = 0;
            if (i < bins)
                for (int k = 0; k < WARPS; ++k) sum += count_s[k * bins + i];
            int32_t total;
            place = cta_exclusive(sum, warp_sum_s, &total) + base;
            base += total;
            if (i < bins) offsets[i] = place;
        }
        if (i < bins) {
            int32_t at = place;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                const int32_t c = count_s[k * bins + i];
                count_s[k * bins + i] = at;
                at += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const unsigned peers = __match_any_sync(0xffffffffu, g[j]);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        int32_t at = 0;
        if (g[j] >= 0) at = mine[g[j]];
        __syncwarp();
        if (g[j] >= 0 && rank == 0) mine[g[j]] = at + __popc(peers);
        __syncwarp();
        if (g[j] >= 0) order[at + rank] = lo + 32 * j;
    }
}

template <int WARPS>
int scatter_launch(int64_t *order, int64_t *offsets, const int32_t *counts, const int64_t *ids,
                   int64_t rows, int n_groups, int blocks, cudaStream_t s) {
    const size_t smem = static_cast<size_t>(WARPS) * (n_groups + 1) * sizeof(int32_t);
    if (smem > 48 * 1024)
        PA_CUDA_TRY(cudaFuncSetAttribute(group_scatter_kernel<WARPS>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem)));
    group_scatter_kernel<WARPS><<<blocks, 32 * WARPS, smem, s>>>(order, offsets, counts, ids, rows,
                                                                 n_groups);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

}  // namespace pa

extern "C" int64_t pa_group_rows_workspace_bytes(int64_t rows, int n_groups) {
    if (rows <= pa::group::kSingleRows || n_groups < 1) return 0;
    const int64_t blocks = (rows + pa::group::kBlockRows - 1) / pa::group::kBlockRows;
    return ((blocks + 1) * (n_groups + 1) + 1) * static_cast<int64_t>(sizeof(int32_t));
}

extern "C" int pa_group_rows(int64_t *order, int64_t *offsets, const int64_t *router, int64_t rows,
                             int n_groups, void *workspace, void *stream) {
    using namespace pa;
    PA_REQUIRE(rows >= 0 && rows <= PA_MAX_ROWS, "rows out of range");
    PA_REQUIRE(n_groups >= 1 && n_groups <= PA_MAX_GROUPS, "n_groups must be in [1, %d]",
               PA_MAX_GROUPS);
    PA_REQUIRE(offsets && (rows == 0 || (order && router)), "null pointer");
    const bool single = rows <= group::kSingleRows;
    PA_REQUIRE(single || workspace, "workspace missing (pa_group_rows_workspace_bytes)");
    PA_REQUIRE(aligned_to(order, 8) && aligned_to(offsets, 8) && aligned_to(router, 8) &&
                   aligned_to(workspace, 4),
               "order, offsets and router must be aligned to 8 bytes, workspace to 4");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows <= group::kBlockRows)
        return scatter_launch<group::kWarps>(order, offsets, nullptr, router, rows, n_groups, 1, s);
    if (single)
        return scatter_launch<2 * group::kWarps>(order, offsets, nullptr, router, rows, n_groups, 1, s);
    const int bins = n_groups + 1;
    const int blocks = static_cast<int>((rows + group::kBlockRows - 1) / group::kBlockRows);
    int32_t *counts = static_cast<int32_t *>(workspace);
    int32_t *totals = counts + static_cast<int64_t>(blocks) * bins;
    unsigned *done = reinterpret_cast<unsigned *>(totals + bins);
    group_count_kernel<<<blocks, group::kThreads, bins * sizeof(int32_t), s>>>(counts, done, router,
                                                                               rows, n_groups);
    group_scan_kernel<<<(bins + 31) / 32, 1024, 0, s>>>(offsets, totals, done, counts, blocks,
                                                        n_groups);
    count_launch(2);
    PA_CUDA_TRY(cudaGetLastError());
    return scatter_launch<group::kWarps>(order, offsets, counts, router, rows, n_groups, blocks, s);
}
