// Products of 4-bit rows with a 4-bit table, dense or with one table per group of rows:
//   out[i, n] = sum_k q(i, k) t(g, n, k)
// on the block-scaled tensor-core instructions (kind::mxf4: E8M0 per 32 values, kind::mxf4nvf4:
// E4M3 per 16), fp32 sums in TMEM.  The table is the wide side of the tile (128 rows, the
// lanes of TMEM), the queries the narrow one (16 to 192 columns), as in grouped_mma.cu: few
// queries do not multiply 128, and a result row is stored 32 neighbours at a time.
//
// Codes come by bulk-tensor copies, 256 values (128 bytes) of every row a stage.  Scales are
// row-major bytes in memory, while the instruction wants, for 128 rows and four bytes each,
// word (r % 32, r / 32) in TMEM, in each quarter of the lanes: a loader warp takes 16 bytes of rows
// l, l + 32, l + 64, l + 96 per lane (512 values of mxfp4, 256 of nvfp4), which is a 4 x 4 transpose
// in its registers, and stores four 16-byte rows without bank conflicts; four writer warps, one a
// quarter, take them to TMEM.  (tcgen05.cp from the issuing thread does the same, but each one, four
// columns, kept the thread and the products behind it for 160 cycles: 12 of them on 8 products, which
// take 96 each.  16384 x 4096 against 8192 rows took 458 us that way, 375 so.)  nvfp4's row scales
// multiply the finished sum.
//
// Measured: 16384 x 4096 against 8192 rows 300 us (3.7 PFLOP/s), bound by shared memory, which takes
// 10 KB in and gives 10 KB out for every product of 96 cycles; one query against 524288 rows of 768
// values 64 us (3.3 TB/s), bound by the issuing warp: twelve products and seven waits a tile.  nvfp4 the
// same: 427 to 460 us and 78 us; its kernels for 64 columns and more spill 40 bytes a thread.
#include <type_traits>

#include "epilogue.cuh"
#include "fp4.cuh"
#include "grouped.cuh"
#include "segments.cuh"
#include "tc05.cuh"
#include "tmap.cuh"

namespace pa {
namespace fp4 {

using grouped::kNoTile;
using grouped::Segments;
using grouped::Tile;
using grouped::TileRing;
using grouped::wait_warp;

namespace mma {
constexpr int BM = 128, BK = 256;        // values; 128 bytes of codes
constexpr int A_BYTES = BM * BK / 2;
constexpr int SCALE_SLOTS = 4;
__host__ __device__ constexpr int b_blocks(int bn) { return bn > 128 ? 2 : 1; }
// Loader warps of a block of 128 rows of scales: each has a piece of 16 bytes a row on its way,
// about 1 us from DRAM, while a tile of short rows needs a piece every 0.6 us.
__host__ __device__ constexpr int loaders(int bn) { return bn > 128 ? 2 : 3; }
// warps 0 codes, 1 products, 2 tiles, 4-7 results, 8-11 scales to TMEM, 12 on loaders of scales
__host__ __device__ constexpr int threads(int bn) {
    return 32 * (12 + (1 + b_blocks(bn)) * loaders(bn));
}
__host__ __device__ constexpr int scale_buffers(int bn) { return bn > 128 ? 2 : 4; }  // in TMEM
__host__ __device__ constexpr int stage_bytes(int bn) { return A_BYTES + bn * BK / 2; }
__host__ __device__ constexpr int scale_bytes(int bn) { return (1 + b_blocks(bn)) * 2048; }
__host__ __device__ constexpr int stages(int bn) {
    return bn >= 192 ? 4 : bn >= 128 ? 5 : bn >= 64 ? 7 : bn >= 32 ? 8 : 10;
}
__host__ __device__ constexpr int smem_bytes(int bn) {
    return stages(bn) * stage_bytes(bn) + SCALE_SLOTS * scale_bytes(bn) +
           epilogue::bytes(bn) + 1024;
}
}  // namespace mma

struct Args {
    void *out;
    const uint8_t *q_scales, *t_scales;
    const float *q_row_scale, *t_row_scale;
    const int64_t *offsets;
    int64_t d_out;
    int rows, n_groups, values;          // values of a row, padded to 32
    int q_pitch, t_pitch;                // bytes of scales from row to row
    int unit;                            // tiles a CTA takes at a time
    int out_dtype;
    int piece;                           // bytes that 16-bit result rows are stored in
    int *status;
    uint32_t polls;                      // limit of the wait for a sum
};

// Bytes [at, at + 16) of a row of `pitch` scale bytes, zero behind its end.  Only aligned 16-byte
// pieces that hold a byte of the row are read.
struct Piece { uint4 v0, v1; };
__device__ __forceinline__ Piece scales_fetch(const uint8_t *row, int at, int pitch, bool live) {
    Piece p = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    const int have = min(16, pitch - at);
    if (live && have > 0) {
        const uint8_t *src = row + at;
        const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15u);
        const uint4 *base = reinterpret_cast<const uint4 *>(src - shift);
        p.v0 = __ldg(base);
        if (shift + have > 16) p.v1 = __ldg(base + 1);
    }
    return p;
}
__device__ __forceinline__ uint4 scales_take(const Piece &p, const uint8_t *row, int at, int pitch) {
    const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + at) & 15u);
    uint32_t w[8] = {p.v0.x, p.v0.y, p.v0.z, p.v0.w, p.v1.x, p.v1.y, p.v1.z, p.v1.w};
    if (shift & 8u) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4u) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = 8u * (shift & 3u);
    uint32_t r[4];
    const int have = pitch - at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = __funnelshift_r(w[i], w[i + 1], bits);
        const int left = have - 4 * i;  // bytes of this word that are the row's
        if (left < 4) r[i] = left <= 0 ? 0u : r[i] & ((1u << (8 * left)) - 1u);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int METHOD, int BN>
__global__ void __launch_bounds__(mma::threads(BN), 1)
project_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_q,
               const __grid_constant__ CUtensorMap map_tail, const __grid_constant__ Args args) {
    using namespace mma;
    constexpr int THREADS = threads(BN), STAGES = stages(BN), STAGE_BYTES = stage_bytes(BN);
    constexpr int NB = b_blocks(BN), SLOT_BYTES = scale_bytes(BN);
    constexpr int GROUP = METHOD == PA_MXFP4 ? 2 : 1;   // stages that 16 scale bytes last
    constexpr int SCALE_COLS = 16 * (1 + NB);
    constexpr int BOX = BN < 64 ? BN : 64, BOX_BYTES = BOX * BK / 2;  // of the queries' codes
    constexpr int ACC_COLS = 2 * BN;
    constexpr int BUFS = scale_buffers(BN), ALL_COLS = ACC_COLS + BUFS * SCALE_COLS;
    constexpr uint32_t COLS = ALL_COLS <= 256 ? 256 : 512;
    static_assert(ALL_COLS <= 512, "TMEM has 512 columns");
    static_assert(smem_bytes(BN) + sizeof(Segments) + sizeof(TileRing) + 1024 +
                          (METHOD == PA_NVFP4 ? 8 * 4 * (BM + BN) : 4 * (BM + BN)) <= 227 * 1024,
                  "shared memory of an SM");
    extern __shared__ uint8_t dyn_smem[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], sc_full[SCALE_SLOTS],
        sc_empty[SCALE_SLOTS], tm_full[BUFS], tm_empty[BUFS], acc_full[2], acc_empty[2], quit_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_s;
    __shared__ Segments segs;
    __shared__ TileRing tiles;
    // nvfp4's row scales, of a tile each: the writers are at most five tiles ahead of the results
    constexpr int ROW_BUFS = METHOD == PA_NVFP4 ? 8 : 1;
    __shared__ float t_scale_s[ROW_BUFS][BM], q_scale_s[ROW_BUFS][BN];
    __shared__ __align__(8) uint64_t row_full[ROW_BUFS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = (tc05::smem_u32(dyn_smem) + 1023u) & ~1023u;
    const uint32_t scale_ring = ring + STAGES * STAGE_BYTES;

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc05::mbar_init(tc05::smem_u32(&full_bar[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&empty_bar[s]), 1);
        }
        for (int s = 0; s < SCALE_SLOTS; ++s) {
            tc05::mbar_init(tc05::smem_u32(&sc_full[s]), 1 + NB);
            tc05::mbar_init(tc05::smem_u32(&sc_empty[s]), 4);
        }
        for (int s = 0; s < ROW_BUFS; ++s) tc05::mbar_init(tc05::smem_u32(&row_full[s]), 4);
        for (int s = 0; s < BUFS; ++s) {
            tc05::mbar_init(tc05::smem_u32(&tm_full[s]), 4);
            tc05::mbar_init(tc05::smem_u32(&tm_empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc05::mbar_init(tc05::smem_u32(&acc_full[s]), 1);
            tc05::mbar_init(tc05::smem_u32(&acc_empty[s]), 4);
        }
        tc05::mbar_init(tc05::smem_u32(&quit_bar), 1);
        grouped::ring_init(tiles, 10 + (1 + NB) * loaders(BN));
        abort_s = 0;
        tc05::fence_barrier_init();
        tc05::tma_prefetch_desc(&map_t);
        tc05::tma_prefetch_desc(&map_q);
    }
    if (warp == 0) tc05::tmem_alloc(tc05::smem_u32(&tmem_slot), COLS);
    grouped::segs_make<THREADS>(segs, args.offsets, args.n_groups, args.rows, BN);
    tc05::fence_before_sync();
    __syncthreads();
    tc05::fence_after_sync();
    const uint32_t tmem = tmem_slot;

    const int m_tiles = static_cast<int>((args.d_out + BM - 1) / BM);
    const int n_stages = (args.values + BK - 1) / BK;
    const int row_tiles = segs.tiles[args.n_groups + 2];
    auto make = [&](int index) {
        Tile r;
        const int row = index / m_tiles;
        r.g = kNoTile;
        if (row >= row_tiles) return r;
        r.m0 = (index - row * m_tiles) * BM;
        const int seg = grouped::segs_find(segs, args.n_groups, row);
        r.g = seg >= 1 && seg <= args.n_groups ? seg - 1 : -1;
        r.c0 = segs.edge[seg] + (row - segs.tiles[seg]) * BN;
        r.c_end = segs.edge[seg + 1];
        r.t0 = r.t_end = 0;
        return r;
    };

    uint32_t issued = 0;  // slices of codes, by warp 0
    if (warp == 0) {
        // ---- codes ----
        const bool leader = tc05::elect_one();
        uint32_t it = 0;
        bool ok = true;
        Tile tile;
        for (uint32_t n = 0; ok && grouped::ring_take(tiles, abort_s, n, tile); ++n) {
            if (tile.g < 0) continue;
            const int boxes = (min(BN, tile.c_end - tile.c0) + BOX - 1) / BOX;
            for (int k = 0; k < n_stages; ++k, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES)
                    ok = wait_warp(empty_bar[s], (it / STAGES - 1) & 1, abort_s);
                if (!ok) break;
                const uint32_t a = ring + s * STAGE_BYTES;
                const uint32_t bar = tc05::smem_u32(&full_bar[s]);
                if (leader) {
                    tc05::mbar_expect_tx(bar, A_BYTES + boxes * BOX_BYTES);
                    tc05::tma_load_3d(a, &map_t, k * (BK / 2), tile.m0, tile.g, bar);
                    if (boxes * BOX == BN) {
                        tc05::tma_load_2d(a + A_BYTES, &map_q, k * (BK / 2), tile.c0, bar);
                    } else {
                        for (int j = 0; j < boxes; ++j)
                            tc05::tma_load_2d(a + A_BYTES + j * BOX_BYTES, &map_tail, k * (BK / 2),
                                              tile.c0 + BOX * j, bar);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) abort_s = 1;
        issued = it;
    } else if (warp == 1) {
        // ---- products: the warp runs together, one lane issues ----
        const bool leader = tc05::elect_one();
        uint32_t it = 0, sg = 0, acc_it = 0;
        bool ok = true;
        // of the first stage; a descriptor counts 16 bytes, so others are sums
        const uint64_t desc_a = tc05::smem_desc_sw128(ring);
        Tile tile;
        for (uint32_t n = 0; ok && grouped::ring_take(tiles, abort_s, n, tile); ++n) {
            if (tile.g < 0) continue;
            const int acc = acc_it & 1;
            if (acc_it >= 2)
                ok = wait_warp(acc_empty[acc], (acc_it / 2 - 1) & 1, abort_s);
            const uint32_t d = tmem + acc * BN;
            const int cols = min(BN, tile.c_end - tile.c0);
            const uint32_t idesc0 = tc05::idesc_mxf4(METHOD == PA_MXFP4, (cols + 15) / 16 * 16);
            uint32_t sa = 0, sb = 0;
            for (int k = 0; ok && k < n_stages; ++k, ++it) {
                const int s = it % STAGES, buf = sg % BUFS;
                if (k % GROUP == 0) {
                    ok = wait_warp(tm_full[buf], (sg / BUFS) & 1, abort_s);
                    sa = tmem + ACC_COLS + buf * SCALE_COLS;
                    sb = sa + 16;
                }
                ok = ok && wait_warp(full_bar[s], (it / STAGES) & 1, abort_s);
                if (!ok) break;
                tc05::fence_after_sync();
                const uint64_t a = desc_a + s * (STAGE_BYTES / 16), b = a + A_BYTES / 16;
                const int steps = min(4, (args.values - k * BK + 63) / 64);
                const bool last = k + 1 == n_stages;
                if (leader) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j < steps) {
                            // 64 values: two bytes of a scale word (mxfp4) or all four (nvfp4)
                            const int word = METHOD == PA_MXFP4 ? 2 * (k % GROUP) + j / 2 : j;
                            const uint32_t idesc =
                                idesc0 | tc05::idesc_scale_id(METHOD == PA_MXFP4 ? 2 * (j & 1) : 0);
                            tc05::mma_fp4<METHOD == PA_MXFP4>(
                                d, a + 2 * j, b + 2 * j, idesc, sa + 4 * word, sb + 4 * NB * word,
                                k > 0 || j > 0);
                        }
                    }
                    tc05::mma_commit(tc05::smem_u32(&empty_bar[s]));
                    if (k % GROUP == GROUP - 1 || last)
                        tc05::mma_commit(tc05::smem_u32(&tm_empty[buf]));
                    if (last) tc05::mma_commit(tc05::smem_u32(&acc_full[acc]));
                }
                __syncwarp();
                if (k % GROUP == GROUP - 1 || last) ++sg;
            }
            ++acc_it;
        }
        if (!ok) abort_s = 1;
    } else if (warp == 2) {
        if (lane == 0)
            grouped::ring_serve(tiles, abort_s, grouped::ring_depth(n_stages, STAGES), args.unit,
                                grouped::ring_ahead(n_stages), make);
    } else if (warp >= 8 && warp < 12) {
        // ---- scales to TMEM: lanes 32 (w % 4) on, for all the products of this CTA ----
        const uint32_t quarter = (32u * (warp & 3)) << 16;
        const int n_pieces = (n_stages + GROUP - 1) / GROUP;
        const int own = 32 * (warp & 3) + lane;
        Tile tile;
        uint32_t sg = 0, n_some = 0;
        bool ok = true;
        for (uint32_t n = 0; ok && grouped::ring_take(tiles, abort_s, n, tile); ++n) {
            if (tile.g < 0) continue;
            float t_row = 1.0f, q_row[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) q_row[j] = 1.0f;
            if (METHOD == PA_NVFP4) {  // on their way while the first scales are written
                if (tile.m0 + own < args.d_out)
                    t_row = __ldg(args.t_row_scale + tile.g * args.d_out + tile.m0 + own);
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    if (128 * j + own < BN && tile.c0 + 128 * j + own < tile.c_end)
                        q_row[j] = __ldg(args.q_row_scale + tile.c0 + 128 * j + own);
            }
            for (int piece = 0; piece < n_pieces; ++piece, ++sg) {
                const int slot = sg % SCALE_SLOTS, buf = sg % BUFS;
                ok = wait_warp(sc_full[slot], (sg / SCALE_SLOTS) & 1, abort_s);
                if (!ok) break;
                uint32_t r[1 + NB][16];
                const uint32_t from = scale_ring + slot * SLOT_BYTES + 16 * lane;
#pragma unroll
                for (int j = 0; j <= NB; ++j)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(r[j][4 * w]), "=r"(r[j][4 * w + 1]),
                                       "=r"(r[j][4 * w + 2]), "=r"(r[j][4 * w + 3])
                                     : "r"(from + 2048 * j + 512 * w)
                                     : "memory");
                if (sg >= BUFS)
                    ok = wait_warp(tm_empty[buf], (sg / BUFS - 1) & 1, abort_s);
                if (!ok) break;
                tc05::fence_after_sync();
                const uint32_t to = tmem + ACC_COLS + buf * SCALE_COLS + quarter;
                tc05::tmem_st_32x16(to, r[0]);
                if constexpr (NB == 1) {
                    tc05::tmem_st_32x16(to + 16, r[1]);
                } else {  // word w of both blocks side by side
                    uint32_t q[2][16];
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            q[w / 2][8 * (w % 2) + i] = r[1][4 * w + i];
                            q[w / 2][8 * (w % 2) + 4 + i] = r[NB][4 * w + i];
                        }
                    tc05::tmem_st_32x16(to + 16, q[0]);
                    tc05::tmem_st_32x16(to + 32, q[1]);
                }
                tc05::tmem_st_wait();
                tc05::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    tc05::mbar_arrive(tc05::smem_u32(&sc_empty[slot]));
                    tc05::mbar_arrive(tc05::smem_u32(&tm_full[buf]));
                }
                if (METHOD == PA_NVFP4 && piece == 0) {
                    const int at = n_some % ROW_BUFS;
                    t_scale_s[at][own] = t_row;
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        if (128 * j + own < BN) q_scale_s[at][128 * j + own] = q_row[j];
                    __syncwarp();
                    if (lane == 0) tc05::mbar_arrive(tc05::smem_u32(&row_full[at]));
                }
            }
            ++n_some;
        }
        if (!ok) abort_s = 1;
    } else if (warp >= 12) {
        // ---- scales: block 0 the table's 128 rows, 1 and 2 the queries' ----
        const int li = warp - 12;
        const int block = li % (1 + NB);
        const int pitch = block == 0 ? args.t_pitch : args.q_pitch;
        const int n_pieces = (n_stages + GROUP - 1) / GROUP;
        const int piece0 = li / (1 + NB);  // this warp has every loaders(BN)-th piece
        int piece = piece0;
        Tile tile = {};
        const uint8_t *row[4];
        bool live[4];
        uint32_t n = 0;
        auto rows_of_tile = [&]() {  // skips tiles without a group; false at the end
            do {
                if (!grouped::ring_take(tiles, abort_s, n++, tile)) return false;
            } while (tile.g < 0);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int r = 32 * b + lane;
                if (block == 0) {
                    live[b] = tile.m0 + r < args.d_out;
                    row[b] = args.t_scales +
                             (tile.g * args.d_out + tile.m0 + r) * static_cast<int64_t>(pitch);
                } else {
                    const int c = 128 * (block - 1) + r;
                    live[b] = c < BN && tile.c0 + c < tile.c_end;
                    row[b] = args.q_scales + (tile.c0 + c) * static_cast<int64_t>(pitch);
                }
            }
            return true;
        };
        // the piece of the current tile, or that far into the tiles behind it
        auto settle = [&]() {
            while (piece >= n_pieces) {
                piece -= n_pieces;
                if (!rows_of_tile()) return false;
            }
            return true;
        };
        bool more = rows_of_tile() && settle();
        Piece next[4];
        int at = 16 * piece;
        if (more) {
#pragma unroll
            for (int b = 0; b < 4; ++b) next[b] = scales_fetch(row[b], at, pitch, live[b]);
        }
        for (uint32_t sg = piece0; more; sg += loaders(BN)) {
            uint4 v[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) v[b] = scales_take(next[b], row[b], at, pitch);
            const int slot = sg % SCALE_SLOTS;
            if (sg >= SCALE_SLOTS && !wait_warp(sc_empty[slot], (sg / SCALE_SLOTS - 1) & 1, abort_s)) {
                abort_s = 1;
                break;
            }
            const uint32_t to = scale_ring + slot * SLOT_BYTES + 2048 * block + 16 * lane;
            const uint32_t w[4][4] = {{v[0].x, v[1].x, v[2].x, v[3].x},
                                      {v[0].y, v[1].y, v[2].y, v[3].y},
                                      {v[0].z, v[1].z, v[2].z, v[3].z},
                                      {v[0].w, v[1].w, v[2].w, v[3].w}};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 512 * i),
                             "r"(w[i][0]), "r"(w[i][1]), "r"(w[i][2]), "r"(w[i][3])
                             : "memory");
            __syncwarp();
            if (lane == 0) tc05::mbar_arrive(tc05::smem_u32(&sc_full[slot]));
            // only now: the tile of the next piece may have to wait for this one's product
            piece += loaders(BN);
            more = settle();
            at = 16 * piece;
            if (more) {
#pragma unroll
                for (int b = 0; b < 4; ++b) next[b] = scales_fetch(row[b], at, pitch, live[b]);
            }
        }
    } else if (warp >= 4) {
        // ---- results: warp w has lanes 32 (w - 4) .. of the accumulator ----
        const int w = warp - 4, own = 32 * w + lane;
        const uint32_t buf = scale_ring + SCALE_SLOTS * SLOT_BYTES;
        constexpr int CHUNK = epilogue::cols(BN);
        uint32_t acc_it = 0, n_tile = 0, chunk = 0;
        for (;; ++n_tile) {
            // the four warps must agree on what they do: they meet at barriers below
            Tile tile;
            bool ok = grouped::ring_take(tiles, abort_s, n_tile, tile);
            const bool some = ok && tile.g >= 0;
            const int acc = acc_it & 1, live = min(BN, tile.c_end - tile.c0);
            const float *ts = t_scale_s[acc_it % ROW_BUFS], *qs = q_scale_s[acc_it % ROW_BUFS];
            if (METHOD == PA_NVFP4 && some)
                ok = wait_warp(row_full[acc_it % ROW_BUFS], (acc_it / ROW_BUFS) & 1, abort_s);
            if (some && ok) ok = wait_warp(acc_full[acc], (acc_it / 2) & 1, abort_s, args.polls);
            if (some && !ok) abort_s = 1;
            __syncwarp();
            if (!epilogue::all_agree(ok)) break;
            tc05::fence_after_sync();
            const int m_left = static_cast<int>(min(args.d_out - tile.m0, static_cast<int64_t>(BM)));
            const int64_t first = tile.c0 * args.d_out + tile.m0;
            const uint32_t from = tmem + acc * BN;
            if (args.out_dtype == PA_F32) {
                // 32 lanes store 128 bytes of a row as they are
                float *dst = static_cast<float *>(args.out) + first + own;
                const float mine = METHOD == PA_NVFP4 && some ? ts[own] : 1.0f;
#pragma unroll 1
                for (int c0 = 0; c0 < live; c0 += CHUNK) {
                    uint32_t r[CHUNK];
                    if (some) {
                        const uint32_t col = from + ((32u * w) << 16) + c0;
                        if constexpr (CHUNK == 32) tc05::tmem_ld_32x32(col, r);
                        else tc05::tmem_ld_32x16(col, r);
                        tc05::tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int j = 0; j < CHUNK; ++j) r[j] = 0;
                    }
                    if (METHOD == PA_NVFP4 && some) {
#pragma unroll
                        for (int j = 0; j < CHUNK; ++j)
                            r[j] = __float_as_uint(epilogue::by_both(__uint_as_float(r[j]), mine,
                                                                     qs[c0 + j]));
                    }
                    if (own < m_left) {
                        if (c0 + CHUNK <= live) {
#pragma unroll
                            for (int j = 0; j < CHUNK; ++j, dst += args.d_out)
                                *dst = __uint_as_float(r[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < CHUNK; ++j, dst += args.d_out)
                                if (c0 + j < live) *dst = __uint_as_float(r[j]);
                        }
                    }
                }
            } else {
                float m_scale[4] = {}, c_scale[CHUNK / 4] = {};
                bool near = true;  // scales of this tile whose products need no second look
                if (METHOD == PA_NVFP4 && some) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) m_scale[i] = ts[32 * w + 8 * i + lane / 4];
                    near = epilogue::in_middle(ts[own]);
                    for (int c = own; c < BN; c += 128) near = near && epilogue::in_middle(qs[c]);
                    near = epilogue::all_agree(near);
                }
                auto store_scaled = [&](auto *out, auto scales) {
                    using O = typename std::remove_pointer<decltype(out)>::type;
                    constexpr int SCALES = decltype(scales)::value;
#pragma unroll 1
                    for (int c0 = 0; c0 < live; c0 += CHUNK, ++chunk) {
                        if (SCALES != 0 && some)
#pragma unroll
                            for (int j = 0; j < CHUNK / 4; ++j)
                                c_scale[j] = qs[c0 + 8 * (j / 2) + 2 * (lane % 4) + j % 2];
                        epilogue::store_chunk<O, CHUNK, SCALES>(
                            out + first + c0 * args.d_out, args.d_out, from + c0, some, live - c0,
                            m_left, args.piece, buf + (chunk & 1) * CHUNK * epilogue::kPitch, w, lane,
                            m_scale, c_scale);
                    }
                };
                auto store = [&](auto *out) {
                    if constexpr (METHOD == PA_MXFP4)
                        store_scaled(out, std::integral_constant<int, 0>());
                    else if (near)
                        store_scaled(out, std::integral_constant<int, 1>());
                    else
                        store_scaled(out, std::integral_constant<int, 2>());
                };
                if (args.out_dtype == PA_BF16) store(static_cast<__nv_bfloat16 *>(args.out));
                else store(static_cast<__half *>(args.out));
            }
            if (some) {
                tc05::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc05::mbar_arrive(tc05::smem_u32(&acc_empty[acc]));
                ++acc_it;
            }
        }
    }
    __syncwarp();
    tc05::fence_before_sync();
    __syncthreads();
    if (abort_s) {
        grouped::wind_down<STAGES>(tiles, full_bar, issued, &quit_bar);
        if (args.out_dtype == PA_F32)
            grouped::gave_up(static_cast<float *>(args.out), args.rows, args.d_out, args.d_out, args.status);
        else if (args.out_dtype == PA_BF16)
            grouped::gave_up(static_cast<__nv_bfloat16 *>(args.out), args.rows, args.d_out, args.d_out,
                             args.status);
        else
            grouped::gave_up(static_cast<__half *>(args.out), args.rows, args.d_out, args.d_out,
                             args.status);
    }
    if (warp == 0) tc05::tmem_dealloc(tmem, COLS);
}

// ---- host -------------------------------------------------------------------------
static int map_codes(CUtensorMap *map, const uint8_t *codes, int values, int64_t rows,
                     int64_t n_groups, int box_rows) {
    const uint64_t width = static_cast<uint64_t>(values) / 2;
    const uint64_t dims[3] = {width, static_cast<uint64_t>(rows), static_cast<uint64_t>(n_groups)};
    const uint64_t strides[2] = {width, width * rows};
    const uint32_t box[3] = {128, static_cast<uint32_t>(box_rows), 1};
    return tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, n_groups ? 3 : 2, dims, strides,
                      box);
}

template <int METHOD, int BN>
static int project_bn(Args args, const uint8_t *q_codes, const uint8_t *t_codes,
                      cudaStream_t s) {
    static bool configured[64] = {};
    int dev = 0;
    PA_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 64 && !configured[dev]) {
        PA_CUDA_TRY(cudaFuncSetAttribute(project_kernel<METHOD, BN>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         mma::smem_bytes(BN)));
        configured[dev] = true;
    }
    CUtensorMap map_t, map_q;
    int rc = map_codes(&map_t, t_codes, args.values, args.d_out, args.n_groups, mma::BM);
    if (rc != PA_OK) return rc;
    rc = map_codes(&map_q, q_codes, args.values, args.rows, 0, BN);
    if (rc != PA_OK) return rc;
    CUtensorMap tail = map_q;
    if (BN > 64 && (rc = map_codes(&tail, q_codes, args.values, args.rows, 0, 64)) != PA_OK)
        return rc;
    const int64_t most = (static_cast<int64_t>(args.rows) / BN + args.n_groups + 2) *
                         ((args.d_out + mma::BM - 1) / mma::BM);
    PA_REQUIRE(most <= 0x7fff0000, "too many rows for one call");
    args.unit = grouped::tiles_per_unit(most, (args.values + mma::BK - 1) / mma::BK);
    const unsigned grid = static_cast<unsigned>((most + args.unit - 1) / args.unit);
    project_kernel<METHOD, BN><<<grid, mma::threads(BN), mma::smem_bytes(BN), s>>>(map_t, map_q, tail,
                                                                                   args);
    count_launch();
    PA_CUDA_TRY(cudaGetLastError());
    return PA_OK;
}

template <int METHOD>
static int project_method(const Args &args, const uint8_t *q_codes, const uint8_t *t_codes,
                          cudaStream_t s) {
    const int each = (args.rows + args.n_groups - 1) / args.n_groups;  // on average
    if (each <= 16) return project_bn<METHOD, 16>(args, q_codes, t_codes, s);
    if (each <= 32) return project_bn<METHOD, 32>(args, q_codes, t_codes, s);
    if (each <= 64) return project_bn<METHOD, 64>(args, q_codes, t_codes, s);
    if (each <= 128) return project_bn<METHOD, 128>(args, q_codes, t_codes, s);
    return project_bn<METHOD, 192>(args, q_codes, t_codes, s);
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
    PA_REQUIRE(d_out >= 0 && d_out <= PA_MAX_ROWS / n_groups, "table rows out of range");
    if (rows == 0 || d_out == 0) return PA_OK;
    PA_REQUIRE(out && query_codes && query_scales && codes && scales, "null pointer");
    PA_REQUIRE(method == PA_MXFP4 || (query_row_scale && row_scale), "nvfp4 needs row scales");
    PA_REQUIRE(aligned16(query_codes) && aligned16(codes), "codes must be 16-byte aligned");
    PA_REQUIRE(aligned_to(out, out_dtype == PA_F32 ? 4 : 2) && aligned_to(query_row_scale, 4) &&
                   aligned_to(row_scale, 4) && aligned_to(offsets, 8),
               "out, row scales and offsets must be aligned to their values");
    const int rc = product_check();
    if (rc != PA_OK) return rc;
    int *status = product_status_address();
    if (status == nullptr) return fail(PA_ERR_CUDA, "no host memory for the status of products");
    const int values = static_cast<int>(fp4::padded(d));
    const int pitch = values / fp4::block_of(method);
    const fp4::Args args{out, query_scales, scales, query_row_scale, row_scale, offsets, d_out,
                         static_cast<int>(rows), n_groups, values, pitch, pitch, 1, out_dtype,
                         epilogue::piece_of(out, d_out, d_out), status,
                         grouped::sum_polls()};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return method == PA_MXFP4
               ? fp4::project_method<PA_MXFP4>(args, query_codes, codes, s)
               : fp4::project_method<PA_NVFP4>(args, query_codes, codes, s);
}
