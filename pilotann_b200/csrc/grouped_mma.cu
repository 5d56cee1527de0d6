// The grouped products of grouped.cu on the tensor cores, for 16-bit values whose rows start on
// 16 bytes.  All three have the form
//   D[m, c] = sum_t A(m, t) B(c, t)
// with m along the axis that is contiguous in the result (128 of them a tile: the lanes of
// TMEM) and c along its rows:
//   forward   m = n of y,   c = rows i of a group, t = k:  A = w[g] (t contiguous), B = x
//   rows      m = k of dx,  c = rows i of a group, t = n:  A = w[g] (m contiguous), B = dy
//   matrices  m = k of dw,  c = n of dw,           t = i:  A = x, B = dy (m and c contiguous)
// The rows of a group are on the narrow side of the tile (16 to 256 columns), so that groups
// of a few rows do not multiply 128; columns behind the group's last row are not stored, so a tile
// may hang over into the next group: those columns are dropped.  The last tile of a group loads
// and multiplies whole 64s and 16s of columns only.  In `matrices` t runs over rows: the tail of
// the last slice belongs to the next group and is cleared in shared memory, in both operands,
// so that a NaN there stays there.
//
// Persistent CTAs; warp 2 takes tiles (segments.cuh), warp 0 keeps bulk-tensor copies ahead, warp 1
// issues the MMAs, warps 4-7 store the tile before while the next is multiplied (two accumulators in
// TMEM).  Every wait is bounded.
//
// Measured: 128 rows x 64 matrices of 1024 x 2048 (bf16) 45 us, 5.2 TB/s, 79 % of the copy rate: the
// rest is the start (4 us to the first slice) and SMs that the memory serves later than others.
// Larger groups: grouped_pair.cu.
#include <atomic>

#include "epilogue.cuh"
#include "grouped.cuh"
#include "segments.cuh"
#include "tc05.cuh"
#include "tmap.cuh"

namespace pa {
namespace grouped {

namespace mma {
constexpr int BM = 128, BK = 64;
constexpr int THREADS = 256;
constexpr int A_BYTES = BM * BK * 2;
__host__ __device__ constexpr int b_bytes(int bn) { return bn * BK * 2; }
__host__ __device__ constexpr int stages(int bn) {
    return bn >= 256 ? 4 : bn >= 128 ? 6 : bn >= 64 ? 8 : bn >= 32 ? 9 : 10;
}
__host__ __device__ constexpr int smem_bytes(int bn) {
    return stages(bn) * (A_BYTES + b_bytes(bn)) + epilogue::bytes(bn) + 1024;
}
}  // namespace mma

template <typename T, int MODE, int BN>
__global__ void __launch_bounds__(mma::THREADS, 1)
mma_kernel(T *__restrict__ out, const __grid_constant__ CUtensorMap map_a,
           const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_tail,
           const int64_t *__restrict__ offsets, Shape sh, int *__restrict__ status) {
    using namespace mma;
    constexpr int STAGES = stages(BN), B_BYTES = b_bytes(BN), STAGE_BYTES = A_BYTES + B_BYTES;
    constexpr int BOX = BN < 64 ? BN : 64, BOX_BYTES = BOX * BK * 2;  // of B
    constexpr bool A_MN = MODE != kForward, B_MN = MODE == kMatrices;
    constexpr uint32_t COLS = 2 * BN < 32 ? 32 : 2 * BN;  // TMEM columns: a power of two
    static_assert(smem_bytes(BN) + sizeof(Segments) + sizeof(TileRing) + 512 <= 227 * 1024,
                  "shared memory of an SM");
    static_assert(BK == kSlice, "parts of a sum are whole slices");
    extern __shared__ uint8_t dyn_smem[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2],
        quit_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_s;
    __shared__ Segments segs;
    __shared__ TileRing tiles;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (tc05::smem_u32(dyn_smem) + 1023u) & ~1023u;

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc05::mbar_init(tc05::smem_u32(&full_bar[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&empty_bar[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc05::mbar_init(tc05::smem_u32(&acc_full[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&acc_empty[s]), 4);
        }
        tc05::mbar_init(tc05::smem_u32(&quit_bar), 1);
        ring_init(tiles, 6);
        abort_s = 0;
        tc05::fence_barrier_init();
        tc05::tma_prefetch_desc(&map_a);
        tc05::tma_prefetch_desc(&map_b);
    }
    if (warp == 0) tc05::tmem_alloc(tc05::smem_u32(&tmem_slot), COLS);
    segs_make<THREADS>(segs, offsets, sh.n_groups, sh.rows, BN);
    if (MODE == kMatrices) segs_order(segs, sh.n_groups);
    tc05::fence_before_sync();
    __syncthreads();
    tc05::fence_after_sync();
    const uint32_t tmem = tmem_slot;

    const int m_tiles = (sh.m_size + BM - 1) / BM;
    const int c_tiles = (sh.c_size + BN - 1) / BN;
    const int row_tiles = MODE == kMatrices ? sh.n_groups * c_tiles : segs.tiles[sh.n_groups + 2];
    auto make = [&](int index) {
        Tile r;
        const int row = index / m_tiles;
        r.g = kNoTile;
        if (row >= row_tiles) return r;
        r.m0 = (index - row * m_tiles) * BM;
        if (MODE == kMatrices) {
            const int nth = row / c_tiles;
            r.g = segs_group(segs, sh.n_groups, nth);
            r.c0 = (row - nth * c_tiles) * BN;
            r.c_end = sh.c_size;
            r.t0 = segs.edge[r.g + 1];
            r.t_end = segs.edge[r.g + 2];
        } else {
            const int seg = segs_find(segs, sh.n_groups, row);
            r.g = seg >= 1 && seg <= sh.n_groups ? seg - 1 : -1;
            r.c0 = segs.edge[seg] + (row - segs.tiles[seg]) * BN;
            r.c_end = segs.edge[seg + 1];
            r.t0 = 0;
            r.t_end = r.g >= 0 ? sh.t_size : 0;
        }
        return r;
    };

    uint32_t issued = 0;  // slices, by warp 0
    if (warp == 0) {
        const bool leader = tc05::elect_one();
        uint32_t it = 0;
        bool ok = true;
        Tile tile;
        for (uint32_t n = 0; ok && ring_take(tiles, abort_s, n, tile); ++n) {
            const int boxes = (min(BN, tile.c_end - tile.c0) + BOX - 1) / BOX;
            for (int t0 = tile.t0; t0 < tile.t_end; t0 += BK, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES)
                    ok = wait_warp(empty_bar[s], (it / STAGES - 1) & 1, abort_s);
                if (!ok) break;
                const uint32_t a = ring + s * STAGE_BYTES, b = a + A_BYTES;
                const uint32_t bar = tc05::smem_u32(&full_bar[s]);
                if (leader) {
                    tc05::mbar_expect_tx(bar, A_BYTES + boxes * BOX_BYTES);
                    if (MODE == kForward) {
                        tc05::tma_load_3d(a, &map_a, t0, tile.m0, tile.g, bar);
                    } else if (MODE == kRows) {
                        tc05::tma_load_3d(a, &map_a, tile.m0, t0, tile.g, bar);
                        tc05::tma_load_3d(a + A_BYTES / 2, &map_a, tile.m0 + 64, t0, tile.g, bar);
                    } else {
                        tc05::tma_load_2d(a, &map_a, tile.m0, t0, bar);
                        tc05::tma_load_2d(a + A_BYTES / 2, &map_a, tile.m0 + 64, t0, bar);
                    }
                    if (MODE != kMatrices && boxes * BOX == BN) {
                        tc05::tma_load_2d(b, &map_b, t0, tile.c0, bar);
                    } else {
                        for (int j = 0; j < boxes; ++j)
                            tc05::tma_load_2d(b + j * BOX_BYTES, &map_tail,
                                              MODE == kMatrices ? tile.c0 + BOX * j : t0,
                                              MODE == kMatrices ? t0 : tile.c0 + BOX * j, bar);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) abort_s = 1;
        issued = it;
    } else if (warp == 1) {
        const bool leader = tc05::elect_one();
        uint32_t it = 0, slot = 0, phases = 0;  // bit s: of accumulator s
        bool ok = true;
        // of the first stage; a descriptor counts 16 bytes, so others are sums
        const uint64_t desc_a = A_MN ? tc05::smem_desc_mn_sw128(ring, A_BYTES / 2)
                                     : tc05::smem_desc_sw128(ring);
        const uint64_t desc_b = B_MN ? tc05::smem_desc_mn_sw128(ring + A_BYTES, 8192)
                                     : tc05::smem_desc_sw128(ring + A_BYTES);
        Tile tile;
        for (uint32_t n = 0; ok && ring_take(tiles, abort_s, n, tile); ++n) {
            if (tile.t0 >= tile.t_end) continue;
            const int cols = min(BN, tile.c_end - tile.c0);
            const uint32_t idesc =
                tc05::idesc_f16(is_bf16<T>(), A_MN, B_MN, BM, (cols + 15) / 16 * 16);
            for (int p0 = tile.t0; ok && p0 < tile.t_end; p0 += kPart) {
                ok = wait_warp(acc_empty[slot], (phases >> slot & 1) ^ 1, abort_s);
                const uint32_t d = tmem + slot * BN;
                const int p_end = part_end(p0, tile.t_end);
                for (int t0 = p0; ok && t0 < p_end; t0 += BK, ++it) {
                    const int s = it % STAGES;
                    ok = wait_warp(full_bar[s], (it / STAGES) & 1, abort_s);
                    if (!ok) break;
                    const uint32_t a = ring + s * STAGE_BYTES, off = s * (STAGE_BYTES / 16);
                    const int live = MODE == kMatrices ? min(BK, p_end - t0) : BK;
                    if (MODE == kMatrices && live % 16 != 0) {
                        // rows of the next group up to the end of the last k step: 128 bytes each
                        const int dead = 16 - live % 16;
                        for (int i = lane; i < dead * 8 * (2 + (cols + 63) / 64); i += 32) {
                            const int chunk = i / (dead * 8), rest = i - chunk * dead * 8;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                             a + chunk * 8192 + live * 128 + rest * 16),
                                         "r"(0)
                                         : "memory");
                        }
                        tc05::fence_proxy_async_smem();
                    }
                    __syncwarp();
                    tc05::fence_after_sync();
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            if (16 * k < live) {
                                tc05::mma_f16(d, desc_a + off + k * (A_MN ? 2048 / 16 : 32 / 16),
                                              desc_b + off + k * (B_MN ? 2048 / 16 : 32 / 16), idesc,
                                              t0 > p0 || k > 0);
                            }
                        }
                        tc05::mma_commit(tc05::smem_u32(&empty_bar[s]));
                        if (t0 + BK >= p_end) tc05::mma_commit(tc05::smem_u32(&acc_full[slot]));
                    }
                    __syncwarp();
                }
                phases ^= 1u << slot;
                if (p0 == tile.t0) slot ^= 1;
            }
        }
        if (!ok) abort_s = 1;
    } else if (warp == 2) {
        if (lane == 0) {
            const int sum = MODE == kMatrices ? sh.rows / sh.n_groups : sh.t_size;  // on average
            ring_serve(tiles, abort_s, ring_depth((sum + BK - 1) / BK, STAGES), sh.unit,
                       ring_ahead((sum + BK - 1) / BK), make);
        }
    } else if (warp >= 4) {
        const int w = warp - 4;
        const uint32_t buf = ring + STAGES * STAGE_BYTES;
        constexpr int CHUNK = epilogue::cols(BN);
        uint32_t slot = 0, phases = 0, chunk = 0;
        for (uint32_t n = 0;; ++n) {
            // the four warps must agree on what they do: they meet at barriers below
            Tile tile;
            bool ok = ring_take(tiles, abort_s, n, tile);
            const bool some = ok && tile.t0 < tile.t_end;
            const uint32_t sum = slot;  // the accumulator that the sum is in, in the end
            if (some)
                ok = sum_parts<BN>(tile, acc_full, acc_empty, slot, phases, tmem, w, abort_s, tiles,
                                   sh.polls,
                                   [](uint64_t *bar) { tc05::mbar_arrive(tc05::smem_u32(bar)); });
            __syncwarp();
            if (!epilogue::all_agree(ok)) break;
            tc05::fence_after_sync();
            const int live = min(BN, tile.c_end - tile.c0);
            const int64_t first =
                (MODE == kMatrices ? static_cast<int64_t>(tile.g) * sh.c_size : 0) + tile.c0;
            T *dst = out + first * sh.ldo + tile.m0;
#pragma unroll 1
            for (int c0 = 0; c0 < live; c0 += CHUNK, ++chunk)
                epilogue::store_chunk<T, CHUNK, 0>(
                    dst + c0 * sh.ldo, sh.ldo, tmem + sum * BN + c0, some, live - c0,
                    sh.m_size - tile.m0, sh.piece, buf + (chunk & 1) * CHUNK * epilogue::kPitch, w,
                    lane, {}, {});
            if (some) {
                tc05::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc05::mbar_arrive(tc05::smem_u32(&acc_empty[sum]));
            }
        }
    }
    __syncwarp();
    tc05::fence_before_sync();
    __syncthreads();
    if (abort_s) {
        wind_down<STAGES>(tiles, full_bar, issued, &quit_bar);
        gave_up(out, MODE == kMatrices ? static_cast<int64_t>(sh.n_groups) * sh.c_size : sh.rows,
                sh.m_size, sh.ldo, status);
    }
    if (warp == 0) tc05::tmem_dealloc(tmem, COLS);
}

// ---- host -------------------------------------------------------------------------
static std::atomic<uint32_t> g_sum_polls{kTileWait};
uint32_t sum_polls() { return g_sum_polls.load(std::memory_order_relaxed); }

template <typename T, int MODE, int BN>
int launch(T *out, const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &tail,
           const int64_t *offsets, const Shape &sh, int64_t most_tiles, cudaStream_t s) {
    static bool configured[64] = {};
    int dev = 0;
    PA_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 64 && !configured[dev]) {
        PA_CUDA_TRY(cudaFuncSetAttribute(mma_kernel<T, MODE, BN>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         mma::smem_bytes(BN)));
        configured[dev] = true;
    }
    int *status = product_status_address();
    if (status == nullptr) return fail(PA_ERR_CUDA, "no host memory for the status of products");
    PA_REQUIRE(most_tiles <= 0x7fff0000, "too many rows for one call");
    const unsigned grid = static_cast<unsigned>((most_tiles + sh.unit - 1) / sh.unit);
    mma_kernel<T, MODE, BN><<<grid, mma::THREADS, mma::smem_bytes(BN), s>>>(out, a, b, tail, offsets, sh,
                                                                            status);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

template <typename T> constexpr CUtensorMapDataType map_type() {
    return is_bf16<T>() ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

template <typename T>
static int map_rows(CUtensorMap *map, const void *x, int64_t width, int64_t rows, int64_t ld,
                    int box_rows) {
    const uint64_t dims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
    const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows)};
    return tensor_map(map, map_type<T>(), x, 2, dims, strides, box);
}

template <typename T>
static int map_matrices(CUtensorMap *map, const void *w, int64_t d, int64_t d_out, int64_t n_groups,
                        int64_t ld, int box_rows) {
    const uint64_t dims[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(d_out),
                              static_cast<uint64_t>(n_groups)};
    const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(ld) * d_out * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(box_rows), 1};
    return tensor_map(map, map_type<T>(), w, 3, dims, strides, box);
}

template <typename T, int MODE, int BN>
static int rows_mma_bn(T *out, const T *in, const T *w, const int64_t *offsets, int64_t rows,
                       int n_groups, int d_sum, int d_out, int64_t ldi, int64_t ldw,
                       int64_t ldo, cudaStream_t s) {
    CUtensorMap a, b, tail;
    const bool fwd = MODE == kForward;
    int rc = map_matrices<T>(&a, w, fwd ? d_sum : d_out, fwd ? d_out : d_sum, n_groups,
                             ldw, fwd ? 128 : 64);
    if (rc != PA_OK) return rc;
    rc = map_rows<T>(&tail, in, d_sum, rows, ldi, BN < 64 ? BN : 64);
    if (rc != PA_OK) return rc;
    const int64_t most = (rows / BN + n_groups + 2) * ((d_out + 127) / 128);
    const Shape sh{static_cast<int>(rows), n_groups, d_out, 0, d_sum,
                   tiles_per_unit(most, (d_sum + mma::BK - 1) / mma::BK), ldo,
                   epilogue::piece_of(out, ldo, d_out), sum_polls()};
    if (BN == 256 && d_out > 128)  // pairs of CTAs have 256 neighbours of a result row
        return pair_launch<T, MODE>(out, a, tail, offsets, sh, s);
    b = tail;
    if (BN > 64 && (rc = map_rows<T>(&b, in, d_sum, rows, ldi, BN)) != PA_OK) return rc;
    return launch<T, MODE, BN>(out, a, b, tail, offsets, sh, most, s);
}

template <typename T, int MODE>
static int rows_mma_mode(T *out, const T *in, const T *w, const int64_t *offsets, int64_t rows,
                         int n_groups, int d_sum, int d_out, int64_t ldi, int64_t ldw,
                         int64_t ldo, cudaStream_t s) {
    // columns that a group fills on average, fewer where that leaves SMs without a tile
    const int64_t each = (rows + n_groups - 1) / n_groups;
    const int64_t m_tiles = (d_out + mma::BM - 1) / mma::BM, some = rows < n_groups ? rows : n_groups;
    int bn = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : each <= 128 ? 128 : 256;
    while (bn > 32 && (rows / bn + some) * m_tiles < 148) bn /= 2;
#define PA_GO(BN)                                                                             \
    if (bn == BN)                                                                             \
    return rows_mma_bn<T, MODE, BN>(out, in, w, offsets, rows, n_groups, d_sum, d_out, ldi, ldw, ldo, s)
    PA_GO(16);
    PA_GO(32);
    PA_GO(64);
    PA_GO(128);
    PA_GO(256);
    return fail(PA_ERR_ARG, "no tile of %d columns", bn);
#undef PA_GO
}

template <typename T>
int rows_mma(void *out, const void *in, const void *w, const int64_t *offsets, int64_t rows,
             int n_groups, int d_sum, int d_out, int64_t ldi, int64_t ldw, int64_t ldo,
             bool transposed,
             cudaStream_t s) {
    T *o = static_cast<T *>(out);
    const T *i = static_cast<const T *>(in), *m = static_cast<const T *>(w);
    if (transposed)
        return rows_mma_mode<T, kRows>(o, i, m, offsets, rows, n_groups, d_sum, d_out, ldi, ldw,
                                           ldo, s);
    return rows_mma_mode<T, kForward>(o, i, m, offsets, rows, n_groups, d_sum, d_out, ldi, ldw,
                                          ldo, s);
}

template <typename T, int BN>
static int matrices_mma_bn(T *dw, const T *dy, const T *x, const int64_t *offsets, int64_t rows,
                           int n_groups, int d, int d_out, int64_t ldy, int64_t ldx,
                           cudaStream_t s) {
    CUtensorMap a, b;
    int rc = map_rows<T>(&a, x, d, rows, ldx, 64);
    if (rc != PA_OK) return rc;
    rc = map_rows<T>(&b, dy, d_out, rows, ldy, 64);
    if (rc != PA_OK) return rc;
    const int64_t most =
        static_cast<int64_t>(n_groups) * ((d + 127) / 128) * ((d_out + BN - 1) / BN);
    const int64_t each = (rows + n_groups - 1) / n_groups;
    const Shape sh{static_cast<int>(rows), n_groups, d, d_out, 0,
                   tiles_per_unit(most, static_cast<int>((each + mma::BK - 1) / mma::BK)), d,
                   epilogue::piece_of(dw, d, d), sum_polls()};
    if (BN == 256 && d > 128) return pair_launch<T, kMatrices>(dw, a, b, offsets, sh, s);
    return launch<T, kMatrices, BN>(dw, a, b, b, offsets, sh, most, s);
}

template <typename T>
int matrices_mma(void *dw, const void *dy, const void *x, const int64_t *offsets, int64_t rows,
                 int n_groups, int d, int d_out, int64_t ldy, int64_t ldx, cudaStream_t s) {
    T *o = static_cast<T *>(dw);
    const T *y = static_cast<const T *>(dy), *i = static_cast<const T *>(x);
#define PA_GO(BN) return matrices_mma_bn<T, BN>(o, y, i, offsets, rows, n_groups, d, d_out, ldy, ldx, s)
    if (d_out <= 64) PA_GO(64);
    if (d_out <= 128) PA_GO(128);
    PA_GO(256);
#undef PA_GO
}

template int rows_mma<__half>(void *, const void *, const void *, const int64_t *, int64_t, int, int,
                              int, int64_t, int64_t, int64_t, bool, cudaStream_t);
template int rows_mma<__nv_bfloat16>(void *, const void *, const void *, const int64_t *, int64_t,
                                     int, int, int, int64_t, int64_t, int64_t, bool, cudaStream_t);
template int matrices_mma<__half>(void *, const void *, const void *, const int64_t *, int64_t, int,
                                  int, int, int64_t, int64_t, cudaStream_t);
template int matrices_mma<__nv_bfloat16>(void *, const void *, const void *, const int64_t *,
                                         int64_t, int, int, int, int64_t, int64_t, cudaStream_t);

}  // namespace grouped
}  // namespace pa

extern "C" int pa_selftest_sum_polls(int polls) {
    pa::grouped::g_sum_polls.store(polls < 0 ? pa::grouped::kTileWait : static_cast<uint32_t>(polls),
                                   std::memory_order_relaxed);
    return PA_OK;
}
