// Tiles of the rows of each group, worked out by every CTA of a persistent kernel from the
// offsets on the device.
#pragma once

#include "grouped.cuh"
#include "tc05.cuh"
#include "tmap.cuh"

namespace pa {
namespace grouped {

// the tensor-core products: y, dx, dw
enum { kForward = 0, kRows = 1, kMatrices = 2 };
struct Shape {
    int rows, n_groups;
    int m_size;       // of D: contiguous axis
    int c_size;       // kMatrices: rows of one matrix
    int t_size;       // kForward, kRows: summed axis
    int unit;         // tiles a CTA takes at a time
    int64_t ldo;
    int piece;        // bytes that result rows are stored in
    uint32_t polls;   // limit of the wait for a sum
};

struct Segments {
    int edge[PA_MAX_GROUPS + 3];   // first row of segment i, ascending
    int tiles[PA_MAX_GROUPS + 3];  // row tiles before segment i
    int part[32];                  // of the prefix sums
    int order[128];                // groups, most rows first
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

// Groups by falling number of rows, for up to 128 of them (32 take 0.5 us): where a tile is summed
// over the rows of its group, the long ones start first and the short ones fill the end (16384 rows in
// 32 groups, the largest 1351: the SMs were done at 0.78 of the kernel's time on average).  All threads;
// a barrier is still needed behind it.
constexpr int kOrdered = 128;
__device__ __forceinline__ void segs_order(Segments &s, int n_groups) {
    const int g = threadIdx.x;
    if (n_groups <= kOrdered && g < n_groups) {
        const int mine = s.edge[g + 2] - s.edge[g + 1];
        int before = 0;
        for (int i = 0; i < n_groups; ++i) {
            const int other = s.edge[i + 2] - s.edge[i + 1];
            before += other > mine || (other == mine && i < g);
        }
        s.order[before] = g;
    }
}
__device__ __forceinline__ int segs_group(const Segments &s, int n_groups, int i) {
    return n_groups <= kOrdered ? s.order[i] : i;
}

// ---- tiles handed out while the kernel runs ----------------------------------------
// The grid has a CTA per tile that the offsets could make; one CTA fits an SM.  A CTA works on its own
// tile and then takes over the tile of a CTA that has not started (cluster launch control), until
// there is none: SMs finish 15 to 25 % apart where tiles differ or the memory serves some SMs
// sooner, and a fixed share of the tiles each waited for the slowest.  One warp asks, works the tile
// out and leaves it in a ring for the warps that load, multiply and store.  It asks as late as the loads
// allow: a tile taken early is one that an idle SM cannot have.
struct Tile {
    int g;            // group; -1: rows of no group, zeros; kNoTile: there are no more
    int m0;           // first of 128 along the contiguous axis of the result
    int c0, c_end;    // its rows: c0 .. min(c0 + BN, c_end)
    int t0, t_end;    // summed axis
};
constexpr int kNoTile = -2;

// ---- waits -----------------------------------------------------------------------------
// A wait polls an mbarrier, 4 us a poll while nothing happens, and gives up after kTileWait of them (2 s)
// or once another warp of the CTA has (quit).  No wait spans more than kPart terms of a sum, but the one
// for room in the ring of tiles: a tile sums up to 2^31 rows (9 s).  That one starts again whenever
// the warps that store have moved on.  A CTA that gives up waits for what it has started and
// keeps the rest of the grid from starting (wind_down), fills the result with NaN, sets the status word,
// frees its TMEM and returns.
constexpr uint32_t kTileWait = 1u << 19;

template <bool CLUSTER>
__device__ __forceinline__ bool over(uint32_t bar, uint32_t parity) {
    return CLUSTER ? tc05::mbar_try_wait_cluster(bar, parity) : tc05::mbar_try_wait(bar, parity);
}
// one thread
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_unless(uint64_t &bar, uint32_t parity, const volatile int &quit) {
    const uint32_t at = tc05::smem_u32(&bar);
    for (uint32_t i = 0; i < kTileWait; ++i) {
        if (over<CLUSTER>(at, parity)) return true;
        if (quit) return false;
    }
    return false;
}
// a converged warp, with the same answer in all lanes: they leave the loop together
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_warp(uint64_t &bar, uint32_t parity, const volatile int &quit,
                                          uint32_t limit = kTileWait) {
    const uint32_t at = tc05::smem_u32(&bar);
    for (uint32_t i = 0; i < limit; ++i) {
        if (__all_sync(0xffffffffu, over<CLUSTER>(at, parity))) return true;
        if (__any_sync(0xffffffffu, quit)) return false;
    }
    return false;
}
// starts again whenever `moved` changes
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_moving(uint64_t &bar, uint32_t parity, const volatile int &quit,
                                            const volatile uint32_t &moved) {
    const uint32_t at = tc05::smem_u32(&bar);
    uint32_t seen = moved;
    for (uint32_t i = 0; i < kTileWait; ++i) {
        if (over<CLUSTER>(at, parity)) return true;
        if (quit) return false;
        const uint32_t now = moved;
        if (now != seen) i = 0, seen = now;
    }
    return false;
}
// the limit of the wait for a sum that launches get (grouped_mma.cu)
uint32_t sum_polls();

struct TileRing {
    __align__(16) uint4 answer;
    __align__(16) int4 a[4];
    int2 b[4];
    __align__(8) uint64_t full[4], empty[4], answered;
    volatile uint32_t moved;  // counts what the first of the warps that store has done
    volatile uint32_t asked;  // how often launch control was asked
    volatile int due;         // the last answer was given up
    volatile int none;        // it said that there is nothing left
};

// Tiles known ahead of the slowest reader, for tiles of `slices` slices and a ring of `stages`: the
// loads run `stages` slices ahead, and an answer takes about 1 us.
__device__ __forceinline__ int ring_depth(int slices, int stages) {
    return min(4, 1 + 3 * stages / max(1, slices));
}

// one thread, before the barrier behind which the ring is used; readers: arrivals a tile gets
__device__ __forceinline__ void ring_init(TileRing &r, int readers) {
    for (int i = 0; i < 4; ++i) {
        tc05::mbar_init(tc05::smem_u32(&r.full[i]), 1);
        tc05::mbar_init(tc05::smem_u32(&r.empty[i]), readers);
    }
    tc05::mbar_init(tc05::smem_u32(&r.answered), 1);
    r.moved = r.asked = 0;
    r.due = r.none = 0;
}

// Whether tiles are so short that the next one is asked for before there is room for it: an answer
// takes 1 us, 3 in a cluster, a slice about a quarter.
__device__ __forceinline__ bool ring_ahead(int slices) { return slices <= 16; }

// Tiles that a CTA takes at a time: enough for 16 slices (an answer takes as long as a few), as
// long as every SM asks eight times.
inline int tiles_per_unit(int64_t tiles, int slices) {
    int unit = 1;
    while (unit < 8 && unit * slices < 16 && tiles / (2 * unit) >= 8 * 148) unit *= 2;
    return unit;
}

// The answer that has come: the number of the first CTA that was taken over, -1 if there was none.
__device__ __forceinline__ int ring_answer(TileRing &r) {
    uint32_t more, next;
    asm volatile(
        "{\n"
        ".reg .b128 h;\n"
        ".reg .pred p;\n"
        "ld.shared.b128 h, [%2];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "mov.u32 %1, 0;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n"
        "}\n"
        : "=r"(more), "=r"(next)
        : "r"(tc05::smem_u32(&r.answer))
        : "memory");
    tc05::fence_proxy_async_smem();  // the answer has been read before the next one is written
    if (!more) r.none = 1;
    return more ? static_cast<int>(next) : -1;
}

// Asks for the work of a CTA (or cluster) that has not started: the number of its first CTA, -1 if
// there is none, -2 if no answer came.
__device__ __forceinline__ int ring_ask(TileRing &r) {
    const uint32_t bar = tc05::smem_u32(&r.answered), phase = r.asked & 1;
    r.asked = r.asked + 1;
    tc05::mbar_expect_tx(bar, 16);
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 "
        "[%0], [%1];" ::"r"(tc05::smem_u32(&r.answer)), "r"(bar)
        : "memory");
    if (!tc05::mbar_wait_bounded(bar, phase, kTileWait)) {
        r.due = 1;
        return -2;
    }
    return ring_answer(r);
}

// One thread of a CTA that gives up: takes over what has not started, to leave it at that.  Nothing may
// be asked behind an answer that there is nothing left, nor before the last answer has come.
__device__ __forceinline__ void ring_close(TileRing &r) {
    if (r.due) {
        if (!tc05::mbar_wait_bounded(tc05::smem_u32(&r.answered), (r.asked - 1) & 1, kTileWait)) return;
        ring_answer(r);
    }
    while (!r.none)
        if (ring_ask(r) < 0) break;
}

// One thread hands out tiles: make(index) is the tile, or has g == kNoTile for an index that the
// offsets do not reach; ask(n) is the n-th answer.
template <typename Make, typename Ask>
__device__ __forceinline__ void ring_serve(TileRing &r, volatile int &abort_s, int depth, int unit,
                                           bool ahead, int index, Make make, Ask ask) {
    uint32_t n = 0;
    auto room = [&]() {  // for one more: tile n - depth has been taken by all
        const uint32_t old = n - depth;
        if (n >= static_cast<uint32_t>(depth) &&
            !wait_moving(r.empty[old & 3], (old / 4) & 1, abort_s, r.moved))
            abort_s = 1;
    };
    for (uint32_t asked = 0; !abort_s; ++asked) {
        for (int u = 0; u < unit && !abort_s; ++u) {
            const Tile tile = make(index * unit + u);
            if (tile.g == kNoTile) break;
            room();
            r.a[n & 3] = make_int4(tile.g, tile.m0, tile.c0, tile.c_end);
            r.b[n & 3] = make_int2(tile.t0, tile.t_end);
            tc05::mbar_arrive(tc05::smem_u32(&r.full[n & 3]));
            ++n;
        }
        if (!ahead) room();
        if (abort_s) break;
        index = ask(asked);
        if (index == -2) abort_s = 1;
        if (index < 0) break;
    }
    if (ahead && !abort_s) room();
    r.a[n & 3] = make_int4(kNoTile, 0, 0, 0);
    tc05::mbar_arrive(tc05::smem_u32(&r.full[n & 3]));
}

// the same for the tiles of CTAs without a cluster
template <typename Make>
__device__ __forceinline__ void ring_serve(TileRing &r, volatile int &abort_s, int depth, int unit,
                                           bool ahead, Make make) {
    ring_serve(r, abort_s, depth, unit, ahead, static_cast<int>(blockIdx.x), make,
               [&](uint32_t) { return ring_ask(r); });
}

// A reader's side: the n-th tile of this CTA, for a (converged) warp.  false: no more, or gave up.
__device__ __forceinline__ bool ring_take(TileRing &r, volatile int &abort_s, uint32_t n, Tile &tile) {
    const int slot = n & 3;
    // lanes that gave up must not leave others behind
    if (!__all_sync(0xffffffffu, wait_warp(r.full[slot], (n / 4) & 1, abort_s) && !abort_s)) {
        abort_s = 1;
        return false;
    }
    const int4 a = r.a[slot];
    const int2 b = r.b[slot];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc05::mbar_arrive(tc05::smem_u32(&r.empty[slot]));
    // one value for the warp
    tile.g = __shfl_sync(0xffffffffu, a.x, 0);
    tile.m0 = __shfl_sync(0xffffffffu, a.y, 0);
    tile.c0 = __shfl_sync(0xffffffffu, a.z, 0);
    tile.c_end = __shfl_sync(0xffffffffu, a.w, 0);
    tile.t0 = __shfl_sync(0xffffffffu, b.x, 0);
    tile.t_end = __shfl_sync(0xffffffffu, b.y, 0);
    return tile.g != kNoTile;
}

// ---- long sums ------------------------------------------------------------------------
// The tensor cores cut the sum in TMEM off at every step of 16 terms instead of rounding it: sums of
// positive terms came out 4.3e-4 too small after 65536 terms and 6.9e-3 after 2^20, where half a step
// of fp16 is 4.9e-4.  So a sum is multiplied in parts of 8192 terms (5e-5).  The first part stays
// where it is; the others go to the other accumulator, one after another, and the warps that store
// add each to the first, rounding to the nearest, while the products wait, about 2 us a part (one
// group of 65536 rows, 2048 x 2048: 377 us without parts, 390 with).  Sums of one part are as before:
// the accumulators take turns, and one is stored while the other is filled.
constexpr int kSlice = 64;  // terms
constexpr int kPart = 128 * kSlice;
__device__ __forceinline__ int part_end(int p0, int t_end) {
    return t_end - p0 <= kPart ? t_end : p0 + kPart;
}

// Warp w of the four that store: waits for the parts of the sum of `tile` and adds them up in the
// accumulator that `slot` names on entry.  phases: bit s, of full[s].  false: gave up.
template <int BN, typename Emptied>
__device__ __forceinline__ bool sum_parts(const Tile &tile, uint64_t *full, uint64_t *empty,
                                          uint32_t &slot, uint32_t &phases, uint32_t tmem, int w,
                                          volatile int &abort_s, TileRing &ring, uint32_t polls,
                                          Emptied emptied) {
    constexpr int N = BN < 32 ? 1 : 2;  // 16 columns each
    const uint32_t lanes = tmem + ((32u * w) << 16), sum = lanes + slot * BN;
    const int cols = min(BN, tile.c_end - tile.c0);
    for (int t = 0; t < tile.t_end - tile.t0; t += kPart) {
        if (!wait_warp(full[slot], phases >> slot & 1, abort_s, polls)) {
            abort_s = 1;
            return false;
        }
        if (w == 0 && (threadIdx.x & 31) == 0) ring.moved = ring.moved + 1;
        phases ^= 1u << slot;
        if (t == 0) {
            slot ^= 1;
            continue;
        }
        tc05::fence_after_sync();
        const uint32_t part = lanes + slot * BN;
#pragma unroll 1
        for (int c = 0; c < cols; c += 16 * N) {
            uint32_t a[N][16], b[N][16];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                tc05::tmem_ld_32x16(sum + c + 16 * i, a[i]);
                tc05::tmem_ld_32x16(part + c + 16 * i, b[i]);
            }
            tc05::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < N; ++i) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    a[i][j] = __float_as_uint(__uint_as_float(a[i][j]) + __uint_as_float(b[i][j]));
                tc05::tmem_st_32x16(sum + c + 16 * i, a[i]);
            }
        }
        tc05::tmem_st_wait();
        tc05::fence_before_sync();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) emptied(&empty[slot]);
    }
    return true;
}

// A CTA that gives up, behind a barrier behind which none of its warps starts anything: waits for the
// copies (`issued` by warp 0, in slices), the products (of warp 1) and the answer that are still on
// their way, so that none of them reaches memory that is no longer this CTA's, and keeps CTAs that have
// not started from it.  All threads.
template <int STAGES>
__device__ __forceinline__ void wind_down(TileRing &r, uint64_t *full, uint32_t issued, uint64_t *quit) {
    const int warp = threadIdx.x >> 5;
    if (warp == 0)
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
            tc05::mbar_wait_bounded(tc05::smem_u32(&full[i % STAGES]), (i / STAGES) & 1, kTileWait);
    if (warp == 1 && tc05::elect_one()) {  // the lane that issues
        tc05::mma_commit(tc05::smem_u32(quit));
        tc05::mbar_wait_bounded(tc05::smem_u32(quit), 0, kTileWait);
    }
    if (threadIdx.x == 64) ring_close(r);
    __syncthreads();
}

// A result of which tiles are missing becomes NaN, all of it: which tiles those are is not known of work
// that was taken over last.  (CTAs that do not give up may still store theirs.)  All threads.
template <typename T>
__device__ __forceinline__ void gave_up(T *out, int64_t rows, int64_t width, int64_t ld, int *status) {
    for (int64_t r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5)
        for (int64_t m = threadIdx.x & 31; m < width; m += 32)
            out[r * ld + m] = from_f32<T>(CUDART_NAN_F);
    if (threadIdx.x == 0) {
        *static_cast<volatile int *>(status) = 1;  // host memory
        __threadfence_system();
    }
}

// the segment that has row tile `tile`
__device__ __forceinline__ int segs_find(const Segments &s, int n_groups, int tile) {
    int lo = 0, hi = n_groups + 2;  // tiles[lo] <= tile < tiles[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.tiles[mid] <= tile) lo = mid; else hi = mid;
    }
    return lo;
}

// grouped_pair.cu
template <typename T, int MODE>
int pair_launch(T *out, const CUtensorMap &a, const CUtensorMap &b, const int64_t *offsets,
                const Shape &shape, cudaStream_t s);

}  // namespace grouped
}  // namespace pa
