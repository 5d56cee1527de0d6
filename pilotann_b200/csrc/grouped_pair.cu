// The products of grouped_mma.cu for large groups, by pairs of CTAs: a tile of 256 x
// 256, 128 lanes of each CTA's TMEM.  Each CTA brings its 128 rows of A and half of B, and one MMA
// (cta_group::2) reads both halves: 32 KB a slice and CTA instead of 48 for the same products.  What
// bounds the single CTA is the traffic through shared memory (12 KB written and 12 KB read for
// products that take 128 cycles, at 128 bytes a cycle), and, in a long step, the power it takes.
//
// Measured: 65536 rows x 64 matrices of 1792 x 2048 (bf16): 320, 329 and 361 us alone (1500, 1460 and
// 1330 TFLOP/s), a fifth more in a row, where power bounds them; 369, 369 and 418 by single CTAs.
//
// CTA 0 issues the products and asks for tiles; it hands the answers to CTA 1.  Copies of both arrive
// on CTA 0's barriers, commits on both CTAs'.  In the gradient of the matrices the rows behind the end
// of a group are cleared by the CTA that holds them: in such a last slice, and only there (an
// arrival that publishes a CTA's stores to the other takes about 1 us), CTA 1's copies arrive on a
// barrier of its own, and it tells CTA 0 when it has cleared.  Otherwise as grouped_mma.cu.
#include "epilogue.cuh"
#include "grouped.cuh"
#include "segments.cuh"
#include "tc05.cuh"
#include "tmap.cuh"

namespace pa {
namespace grouped {

namespace pair {
constexpr int BM = 256, BN = 256, BK = 64;
constexpr int THREADS = 256, STAGES = 6;
constexpr int A_BYTES = 128 * BK * 2, B_BYTES = 128 * BK * 2;  // of one CTA
constexpr int BOX_BYTES = 64 * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int SMEM = STAGES * STAGE_BYTES + epilogue::bytes(BN) + 1024;
constexpr uint32_t COLS = 512;
}  // namespace pair

template <typename T, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::THREADS, 1)
pair_kernel(T *__restrict__ out, const __grid_constant__ CUtensorMap map_a,
            const __grid_constant__ CUtensorMap map_b, const int64_t *__restrict__ offsets, Shape sh,
            int *__restrict__ status) {
    using namespace pair;
    constexpr bool MATRICES = MODE == kMatrices, A_MN = MODE != kForward, B_MN = MATRICES;
    static_assert(SMEM + sizeof(Segments) + sizeof(TileRing) + 512 <= 227 * 1024,
                  "shared memory of an SM");
    static_assert(BK == kSlice, "parts of a sum are whole slices");
    extern __shared__ uint8_t dyn_smem[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2],
        ready_bar, told_bar, quit_bar, tail_bar[MATRICES ? STAGES : 1],
        other_bar[MATRICES ? STAGES : 1];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int told_s;  // CTA 1: the answer that CTA 0 got
    __shared__ volatile int abort_s;
    // what a pair that gives up has to wait for: slices, and bytes that each brought to CTA 0's barrier
    __shared__ uint32_t issued_s, bytes_s[STAGES];
    __shared__ uint32_t tails_s;  // bit s: phase that stage s's next last slice is copied in
    __shared__ Segments segs;
    __shared__ TileRing tiles;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = tc05::cluster_rank();
    const uint32_t ring = (tc05::smem_u32(dyn_smem) + 1023u) & ~1023u;

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc05::mbar_init(tc05::smem_u32(&full_bar[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&empty_bar[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc05::mbar_init(tc05::smem_u32(&acc_full[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&acc_empty[s]), 8);
        }
        for (int s = 0; MATRICES && s < STAGES; ++s) {
            tc05::mbar_init(tc05::smem_u32(&tail_bar[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&other_bar[s]), 1);
        }
        tc05::mbar_init(tc05::smem_u32(&ready_bar), 1);
        tc05::mbar_init(tc05::smem_u32(&told_bar), 1);
        tc05::mbar_init(tc05::smem_u32(&quit_bar), 1);
        ring_init(tiles, 6);
        abort_s = 0;
        tc05::fence_barrier_init();
        tc05::tma_prefetch_desc(&map_a);
        tc05::tma_prefetch_desc(&map_b);
    }
    if (warp == 0) tc05::tmem_alloc_pair(tc05::smem_u32(&tmem_slot), COLS);
    segs_make<THREADS>(segs, offsets, sh.n_groups, sh.rows, BN);
    if (MATRICES) segs_order(segs, sh.n_groups);
    tc05::fence_before_sync();
    __syncthreads();
    tc05::cluster_sync();  // the other CTA's barriers are there
    tc05::fence_after_sync();
    const uint32_t tmem = tmem_slot;

    const int m_tiles = (sh.m_size + BM - 1) / BM;
    const int c_tiles = (sh.c_size + BN - 1) / BN;
    const int row_tiles = MATRICES ? sh.n_groups * c_tiles : segs.tiles[sh.n_groups + 2];
    auto make = [&](int index) {
        Tile r;
        const int row = index / m_tiles;
        r.g = kNoTile;
        if (row >= row_tiles) return r;
        r.m0 = (index - row * m_tiles) * BM;
        if (MATRICES) {
            const int nth = row / c_tiles;
            r.g = segs_group(segs, sh.n_groups, nth);
            r.c0 = (row - nth * c_tiles) * BN;
            r.c_end = sh.c_size;
            r.t0 = segs.edge[r.g + 1];
            r.t_end = segs.edge[r.g + 2];
            return r;
        }
        const int seg = segs_find(segs, sh.n_groups, row);
        r.g = seg >= 1 && seg <= sh.n_groups ? seg - 1 : -1;
        r.c0 = segs.edge[seg] + (row - segs.tiles[seg]) * BN;
        r.c_end = segs.edge[seg + 1];
        r.t0 = 0;
        r.t_end = r.g >= 0 ? sh.t_size : 0;
        return r;
    };
    // columns that are multiplied: half of them from each CTA
    auto columns = [&](const Tile &tile) { return (min(BN, tile.c_end - tile.c0) + 31) / 32 * 32; };

    if (warp == 0) {
        const bool leader = tc05::elect_one();
        uint32_t it = 0, tails = 0;
        bool ok = true;
        Tile tile;
        for (uint32_t n = 0; ok && ring_take(tiles, abort_s, n, tile); ++n) {
            const int half = columns(tile) / 2, boxes = (half + 63) / 64;
            const int m = tile.m0 + 128 * static_cast<int>(rank);
            const int c = tile.c0 + half * static_cast<int>(rank);
            for (int t0 = tile.t0; t0 < tile.t_end; t0 += BK, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES)
                    ok = wait_warp(empty_bar[s], (it / STAGES - 1) & 1, abort_s);
                if (!ok) break;
                const uint32_t a = ring + s * STAGE_BYTES, b = a + A_BYTES;
                const uint32_t bar = tc05::map_rank(tc05::smem_u32(&full_bar[s]), 0);
                const int bytes = A_BYTES + boxes * BOX_BYTES;
                const bool tail = MATRICES && (tile.t_end - t0) % 16 != 0 && tile.t_end - t0 < BK;
                if (tail) tails ^= 1u << s;
                if (leader) bytes_s[s] = tail ? 0 : bytes;
                if (leader && tail) {
                    const uint32_t own = tc05::smem_u32(rank == 0 ? &full_bar[s] : &tail_bar[s]);
                    tc05::mbar_expect_tx(own, bytes);
                    tc05::tma_load_2d(a, &map_a, m, t0, own);
                    tc05::tma_load_2d(a + A_BYTES / 2, &map_a, m + 64, t0, own);
                    for (int j = 0; j < boxes; ++j)
                        tc05::tma_load_2d(b + j * BOX_BYTES, &map_b, c + 64 * j, t0, own);
                } else if (leader) {
                    if (rank == 0) tc05::mbar_expect_tx(tc05::smem_u32(&full_bar[s]), 2 * bytes);
                    if (MODE == kForward) {
                        tc05::tma_load_3d_pair(a, &map_a, t0, m, tile.g, bar);
                    } else if (MODE == kRows) {
                        tc05::tma_load_3d_pair(a, &map_a, m, t0, tile.g, bar);
                        tc05::tma_load_3d_pair(a + A_BYTES / 2, &map_a, m + 64, t0, tile.g, bar);
                    } else {
                        tc05::tma_load_2d_pair(a, &map_a, m, t0, bar);
                        tc05::tma_load_2d_pair(a + A_BYTES / 2, &map_a, m + 64, t0, bar);
                    }
                    for (int j = 0; j < boxes; ++j)
                        tc05::tma_load_2d_pair(b + j * BOX_BYTES, &map_b,
                                               MATRICES ? c + 64 * j : t0,
                                               MATRICES ? t0 : c + 64 * j, bar);
                }
                __syncwarp();
            }
        }
        if (!ok) abort_s = 1;
        if (lane == 0) {
            issued_s = it;
            tails_s = tails;
        }
    } else if (warp == 1) {
        const bool leader = tc05::elect_one();
        uint32_t it = 0, slot = 0, phases = 0;  // bit s: of accumulator s
        uint32_t tails = 0;  // bit s: phase of stage s's barriers for last slices
        bool ok = true;
        const uint64_t desc_a = A_MN ? tc05::smem_desc_mn_sw128(ring, A_BYTES / 2)
                                     : tc05::smem_desc_sw128(ring);
        const uint64_t desc_b = B_MN ? tc05::smem_desc_mn_sw128(ring + A_BYTES, BOX_BYTES)
                                     : tc05::smem_desc_sw128(ring + A_BYTES);
        Tile tile;
        for (uint32_t n = 0; ok && ring_take(tiles, abort_s, n, tile); ++n) {
            if (tile.g < 0 || tile.t0 >= tile.t_end) continue;
            const int boxes = (columns(tile) / 2 + 63) / 64;
            // clears the rows of the next group up to the end of the last k step: 128 bytes each
            auto clear = [&](int s, int live) {
                const int dead = 16 - live % 16;
                for (int i = lane; i < dead * 8 * (2 + boxes); i += 32) {
                    const int chunk = i / (dead * 8), rest = i - chunk * dead * 8;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                     ring + s * STAGE_BYTES + chunk * BOX_BYTES + live * 128 + rest * 16),
                                 "r"(0)
                                 : "memory");
                }
                tc05::fence_proxy_async_smem();
                __syncwarp();
            };
            if (rank != 0) {  // CTA 0 issues for both
                const int slices = (tile.t_end - tile.t0 + BK - 1) / BK;
                const int live = tile.t_end - tile.t0 - (slices - 1) * BK;
                it += slices;
                if (!MATRICES || live % 16 == 0) continue;
                const int s = (it - 1) % STAGES;
                ok = wait_warp(tail_bar[s], (tails >> s) & 1, abort_s);
                tails ^= 1u << s;
                if (!ok) break;
                clear(s, live);
                if (lane == 0)
                    tc05::mbar_arrive_cluster(tc05::map_rank(tc05::smem_u32(&other_bar[s]), 0));
                continue;
            }
            const uint32_t idesc = tc05::idesc_f16(is_bf16<T>(), A_MN, B_MN, BM, columns(tile));
            for (int p0 = tile.t0; ok && p0 < tile.t_end; p0 += kPart) {
                ok = wait_warp<true>(acc_empty[slot], (phases >> slot & 1) ^ 1, abort_s);
                const uint32_t d = tmem + slot * BN;
                const int p_end = part_end(p0, tile.t_end);
                for (int t0 = p0; ok && t0 < p_end; t0 += BK, ++it) {
                    const int s = it % STAGES;
                    ok = wait_warp<true>(full_bar[s], (it / STAGES) & 1, abort_s);
                    if (!ok) break;
                    const int live = MATRICES ? min(BK, p_end - t0) : BK;
                    if (MATRICES && live % 16 != 0) {
                        clear(s, live);
                        ok = wait_warp<true>(other_bar[s], (tails >> s) & 1, abort_s);
                        tails ^= 1u << s;
                        if (!ok) break;
                    }
                    tc05::fence_after_sync();
                    const uint32_t off = s * (STAGE_BYTES / 16);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            if (16 * k < live)
                                tc05::mma_f16_pair(d, desc_a + off + k * (A_MN ? 2048 / 16 : 32 / 16),
                                                   desc_b + off + k * (B_MN ? 2048 / 16 : 32 / 16),
                                                   idesc, t0 > p0 || k > 0);
                        tc05::mma_commit_pair(tc05::smem_u32(&empty_bar[s]));
                        if (t0 + BK >= p_end) tc05::mma_commit_pair(tc05::smem_u32(&acc_full[slot]));
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
            const uint32_t ready0 = tc05::map_rank(tc05::smem_u32(&ready_bar), 0),
                           told1 = tc05::map_rank(tc05::smem_u32(&told_bar), 1),
                           answer1 = tc05::map_rank(
                               tc05::smem_u32(const_cast<int *>(&told_s)), 1);
            auto ask = [&](uint32_t asked) -> int {
                if (rank == 0) {
                    int next = ring_ask(tiles);
                    if (next > 0) next /= 2;  // pairs
                    // CTA 1 has read the answer before
                    if (!wait_moving<true>(ready_bar, asked & 1, abort_s, tiles.moved)) next = -2;
                    tc05::store_cluster(answer1, static_cast<uint32_t>(next));
                    tc05::mbar_arrive_cluster(told1);
                    return next;
                }
                tc05::mbar_arrive_cluster(ready0);
                if (!wait_moving<true>(told_bar, asked & 1, abort_s, tiles.moved)) return -2;
                return told_s;
            };
            const int sum = MATRICES ? sh.rows / sh.n_groups : sh.t_size;  // on average
            ring_serve(tiles, abort_s, ring_depth((sum + BK - 1) / BK, STAGES), sh.unit,
                       ring_ahead((sum + BK - 1) / BK), static_cast<int>(blockIdx.x / 2), make,
                       ask);
        }
    } else if (warp >= 4) {
        const int w = warp - 4;
        const uint32_t buf = ring + STAGES * STAGE_BYTES;
        constexpr int CHUNK = epilogue::cols(BN);
        uint32_t slot = 0, phases = 0, chunk = 0;
        auto emptied = [](uint64_t *bar) {
            tc05::mbar_arrive_cluster(tc05::map_rank(tc05::smem_u32(bar), 0));
        };
        for (uint32_t n = 0;; ++n) {
            Tile tile;
            bool ok = ring_take(tiles, abort_s, n, tile);
            const bool some = ok && tile.t0 < tile.t_end;
            const uint32_t sum = slot;  // the accumulator that the sum is in, in the end
            if (some)
                ok = sum_parts<BN>(tile, acc_full, acc_empty, slot, phases, tmem, w, abort_s, tiles,
                                   sh.polls, emptied);
            __syncwarp();
            if (!epilogue::all_agree(ok)) break;
            tc05::fence_after_sync();
            const int live = min(BN, tile.c_end - tile.c0), m0 = tile.m0 + 128 * static_cast<int>(rank);
            const int64_t first =
                (MATRICES ? static_cast<int64_t>(tile.g) * sh.c_size : 0) + tile.c0;
            T *dst = out + first * sh.ldo + m0;
#pragma unroll 1
            for (int c0 = 0; c0 < live; c0 += CHUNK, ++chunk)
                epilogue::store_chunk<T, CHUNK, 0>(
                    dst + c0 * sh.ldo, sh.ldo, tmem + sum * BN + c0, some, live - c0,
                    sh.m_size - m0, sh.piece, buf + (chunk & 1) * CHUNK * epilogue::kPitch, w, lane,
                    {}, {});
            if (some) {
                tc05::fence_before_sync();
                __syncwarp();
                if (lane == 0) emptied(&acc_empty[sum]);
            }
        }
    }
    __syncwarp();
    tc05::fence_before_sync();
    __syncthreads();
    if (tid == 0 && abort_s)  // one that gives up takes the other along
        tc05::store_cluster(
            tc05::map_rank(tc05::smem_u32(const_cast<int *>(&abort_s)), rank ^ 1), 1);
    __syncwarp();
    tc05::cluster_sync();  // nothing of the other CTA reaches here any more, unless it gave up
    tc05::fence_after_sync();
    if (abort_s) {
        // what either has started lands before either ends
        if (warp == 0 && lane == 0) {
            const uint32_t mine = issued_s;
            if (rank == 0) {
                const uint32_t other = tc05::load_cluster(tc05::map_rank(tc05::smem_u32(&issued_s), 1));
                const uint32_t top = max(mine, other);
                for (uint32_t i = top > STAGES ? top - STAGES : 0; i < top; ++i) {
                    const int s = i % STAGES;
                    const uint32_t bar = tc05::smem_u32(&full_bar[s]);
                    if (i < mine) {
                        if (i >= other && bytes_s[s] != 0)  // CTA 1's half does not come
                            tc05::mbar_complete_tx(bar, bytes_s[s]);
                    } else {  // it comes alone
                        const uint32_t bytes =
                            tc05::load_cluster(tc05::map_rank(tc05::smem_u32(&bytes_s[s]), 1));
                        if (bytes == 0) continue;
                        tc05::mbar_expect_tx(bar, bytes);
                    }
                    tc05::mbar_wait_bounded(bar, (i / STAGES) & 1, kTileWait);
                }
            } else if (MATRICES) {
                for (uint32_t i = mine > STAGES ? mine - STAGES : 0; i < mine; ++i)
                    if (bytes_s[i % STAGES] == 0)
                        tc05::mbar_wait_bounded(tc05::smem_u32(&tail_bar[i % STAGES]),
                                                (tails_s >> (i % STAGES) & 1) ^ 1, kTileWait);
            }
        }
        __syncwarp();
        if (warp == 1 && tc05::elect_one()) {  // the lane that issues; both get an arrival
            if (rank == 0) tc05::mma_commit_pair(tc05::smem_u32(&quit_bar));
            tc05::mbar_wait_bounded(tc05::smem_u32(&quit_bar), 0, kTileWait);
        }
        if (tid == 64 && rank == 0) ring_close(tiles);
        gave_up(out, MATRICES ? static_cast<int64_t>(sh.n_groups) * sh.c_size : sh.rows, sh.m_size,
                sh.ldo, status);
        __syncthreads();
        tc05::cluster_sync();
    }
    if (warp == 0) tc05::tmem_dealloc_pair(tmem, COLS);
}

// maps: boxes of 64 values x 128 rows of the matrices (forward) or 64 rows (else), x 64 rows of the
// other operand
template <typename T, int MODE>
int pair_launch(T *out, const CUtensorMap &a, const CUtensorMap &b, const int64_t *offsets,
                const Shape &shape, cudaStream_t s) {
    static bool configured[64] = {};
    int dev = 0;
    PA_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 64 && !configured[dev]) {
        PA_CUDA_TRY(cudaFuncSetAttribute(pair_kernel<T, MODE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, pair::SMEM));
        configured[dev] = true;
    }
    int *status = product_status_address();
    if (status == nullptr) return fail(PA_ERR_CUDA, "no host memory for the status of products");
    const int64_t m_tiles = (shape.m_size + pair::BM - 1) / pair::BM;
    const int64_t most =
        m_tiles * (MODE == kMatrices
                       ? static_cast<int64_t>(shape.n_groups) * ((shape.c_size + pair::BN - 1) / pair::BN)
                       : static_cast<int64_t>(shape.rows) / pair::BN + shape.n_groups + 2);
    PA_REQUIRE(most <= 0x3fffffff, "too many rows for one call");
    Shape sh = shape;
    const int sum = MODE == kMatrices ? sh.rows / sh.n_groups : sh.t_size;
    sh.unit = tiles_per_unit(2 * most, (sum + pair::BK - 1) / pair::BK);
    const unsigned grid = 2 * static_cast<unsigned>((most + sh.unit - 1) / sh.unit);
    pair_kernel<T, MODE><<<grid, pair::THREADS, pair::SMEM, s>>>(out, a, b, offsets, sh, status);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

#define PA_PAIR(T, MODE)                                                                        \
    template int pair_launch<T, MODE>(T *, const CUtensorMap &, const CUtensorMap &,            \
                                      const int64_t *, const Shape &, cudaStream_t);
PA_PAIR(__half, kForward)
PA_PAIR(__half, kRows)
PA_PAIR(__half, kMatrices)
PA_PAIR(__nv_bfloat16, kForward)
PA_PAIR(__nv_bfloat16, kRows)
PA_PAIR(__nv_bfloat16, kMatrices)
#undef PA_PAIR

}  // namespace grouped
}  // namespace pa
