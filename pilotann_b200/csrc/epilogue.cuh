// Accumulator tiles to 16-bit results.  A tile in TMEM has 128 neighbours of a result row in
// its lanes and rows in its columns: the transpose of what memory wants.  Four warps (32 lanes
// each) take `COLS` columns at a time in the fragment layout of 8 x 8 matrices, round, and store
// them transposed to shared memory (stmatrix), from where rows of 256 bytes go out 16 bytes a
// thread.  Storing straight from the lanes, 2 bytes a thread, cost 20 instructions a column and
// bound the products of short sums: 16384 rows x 32 matrices of 2048 x 768 took 115 us.
#pragma once

#include "grouped.cuh"
#include "tc05.cuh"

namespace pa {
namespace epilogue {

constexpr int kPitch = 272;  // bytes from row to row: 8 rows of 16 bytes fall into different banks
constexpr int kThreads = 128;
__host__ __device__ constexpr int cols(int bn) { return bn < 32 ? bn : 32; }
__host__ __device__ constexpr int bytes(int bn) { return 2 * cols(bn) * kPitch; }  // two buffers

__device__ __forceinline__ void sync() {
    asm volatile("barrier.cta.sync.aligned 1, 128;" ::: "memory");
}
// true if all four warps say so; they must agree before one leaves the others at a barrier
__device__ __forceinline__ bool all_agree(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 q, %1, 0;\n"
        "barrier.cta.red.and.aligned.pred p, 1, 128, q;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(ok))
        : "memory");
    return r != 0;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (grouped::is_bf16<T>())
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// v a b, without an overflow or underflow of a b that v would have undone
__device__ __forceinline__ float by_both(float v, float a, float b) {
    const float p = a * b;
    return p >= 1.1754944e-38f && p <= 3.4028235e38f ? v * p : (v * a) * b;
}

// two of these multiply to a normal number (looking at each product costs a quarter of the stores)
__device__ __forceinline__ bool in_middle(float a) {
    return a >= 1.0842022e-19f && a <= 9.223372e18f;  // 2^-63, 2^63
}

// Bytes that result rows of `width` 16-bit values can be stored in: all rows start on as many, and are
// whole pieces.
inline int piece_of(const void *out, int64_t ld, int64_t width) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(2 * ld) |
                           static_cast<uintptr_t>(2 * width);
    return bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
}

// rows of 256 bytes from shared memory, V a thread
template <typename V, typename T>
__device__ __forceinline__ void store_rows(T *dst, int64_t ld, uint32_t buf, int rows, int m_left,
                                           int tid) {
    constexpr int kEach = sizeof(V) / 2, kThreadsPerRow = 128 / kEach;
    const int m = kEach * (tid % kThreadsPerRow);
    if (m >= m_left) return;
    static_assert(kThreadsPerRow <= kThreads, "a row at a time at least");
#pragma unroll 4
    for (int c = tid / kThreadsPerRow; c < rows; c += kThreads / kThreadsPerRow) {
        V v;
        const uint32_t from = buf + c * kPitch + 2 * m;
        if constexpr (sizeof(V) == 16)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
        else if constexpr (sizeof(V) == 8)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                         : "=r"(v.x), "=r"(v.y) : "r"(from) : "memory");
        else if constexpr (sizeof(V) == 4)
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
        else
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
        *reinterpret_cast<V *>(dst + c * ld + m) = v;
    }
}

// One chunk: columns [c0, c0 + COLS) of the tile at `tmem` (`some` false: zeros instead), the
// first `live` of them wanted (all of them if it is more).  dst: element (lane 0, column c0).
// `m_left`: lanes that exist.
// With SCALES, element (m, c) is multiplied by m_scale[i] c_scale[j] before it is rounded (1: scales
// that are in_middle, 2: any): i counts
// the four lanes 32 w + 8 i + lane / 4 of this thread, j its columns 8 (j / 2) + 2 (lane % 4) + j % 2.
// All 128 threads.
template <typename T, int COLS, int SCALES>
__device__ __forceinline__ void store_chunk(T *dst, int64_t ld, uint32_t tmem, bool some, int live,
                                            int m_left, int piece, uint32_t buf, int w, int lane,
                                            const float (&m_scale)[4],
                                            const float (&c_scale)[COLS / 4]) {
    uint32_t r[2][COLS / 2], p[2][COLS / 8][2];
    if (some) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t at = tmem + ((32u * w + 16u * half) << 16);
            if constexpr (COLS == 32) tc05::tmem_ld_16x256_x4(at, r[half]);
            else tc05::tmem_ld_16x256_x2(at, r[half]);
        }
        tc05::tmem_ld_wait();
    } else {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) r[half][j] = 0;
    }
    auto round = [&](auto scaled) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < COLS / 8; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    p[half][i][h] = pack2<T>(
                        scaled(__uint_as_float(r[half][4 * i + 2 * h]), 2 * half + h, 2 * i),
                        scaled(__uint_as_float(r[half][4 * i + 2 * h + 1]), 2 * half + h, 2 * i + 1));
    };
    if constexpr (SCALES == 0)
        round([](float v, int, int) { return v; });
    else if constexpr (SCALES == 1)
        round([&](float v, int m, int c) { return v * (m_scale[m] * c_scale[c]); });
    else
        round([&](float v, int m, int c) { return by_both(v, m_scale[m], c_scale[c]); });
    // lane l names row l % 8 of matrix l / 8: column block l / 16, rows 8 (l / 8 % 2) on
    const uint32_t row = buf + (8 * (lane / 16) + lane % 8) * kPitch + (32 * w + 8 * (lane / 8 % 2)) * 2;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < COLS / 8; i += 2)
            asm volatile(
                "stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                    row + 8 * i * kPitch + 32 * half),
                "r"(p[half][i][0]), "r"(p[half][i][1]), "r"(p[half][i + 1][0]),
                "r"(p[half][i + 1][1])
                : "memory");
    sync();
    const int rows = live < COLS ? live : COLS;
    if (piece == 16) store_rows<uint4>(dst, ld, buf, rows, m_left, 32 * w + lane);
    else if (piece == 8) store_rows<uint2>(dst, ld, buf, rows, m_left, 32 * w + lane);
    else if (piece == 4) store_rows<uint32_t>(dst, ld, buf, rows, m_left, 32 * w + lane);
    else store_rows<uint16_t>(dst, ld, buf, rows, m_left, 32 * w + lane);
}

}  // namespace epilogue
}  // namespace pa
