// What the kernels on paged KV caches share: the batch's rows and the division of its sequences into tiles. The layout of
// the pools is stated with kt_hip_dec_page_bytes in include/kt_hip.h.
#pragma once

#include <stdint.h>

#include "kt_dpp.h"
#include "kt_kernels.h"

namespace kt {

// A sequence's rows t0 .. t0 + n - 1 of the batch, row t0 at position p0. kv_len is clamped to +-2^30 (tokens < 2^31, so p0
// stays within int32): a position that far off is outside every table as it stands.
struct PgRows {
    int t0, n, p0;
};

__device__ __forceinline__ int pg_start(const Paged& a, int b) {
    const int t = a.row_start[b];
    return t < 0 ? 0 : (t > a.tokens ? a.tokens : t);
}

__device__ __forceinline__ int pg_len(const Paged& a, int b) {
    const int L = a.kv_len[b];
    return L < -(1 << 30) ? -(1 << 30) : (L > (1 << 30) ? (1 << 30) : L);
}

__device__ __forceinline__ PgRows pg_rows(const Paged& a, int b) {
    const int t0 = pg_start(a, b), t1 = pg_start(a, b + 1), n = t1 > t0 ? t1 - t0 : 0;
    return {t0, n, pg_len(a, b) - n};
}

// Tiles of `step` units, sequence b with rows * mul units: its tiles begin at number floor(t0 mul / step) + per b, which
// leaves it at least floor(rows mul / step) + per of them, so the grid needs no lengths from the host:
// tokens mul / step + per seqs tiles in all. Returns the last sequence that begins at or before tile `t` and its first tile,
// -1 where none does. Each lane of a wave looks at every 64th sequence. row_start must not decrease; where it does, some
// sequence is returned all the same, and its tiles are bounded by its own rows.
__device__ __forceinline__ int pg_tile_seq(const Paged& a, int t, int mul, int step, int per, int* first) {
    const int lane = threadIdx.x & 63;
    auto begin = [&](int b) { return (int)((int64_t)pg_start(a, b) * mul / step) + per * b; };
    int c = 0;
    for (int b = lane; b < a.seqs; b += 64) c += begin(b) <= t;
    const int b = wave_sum_i32(c) - 1;
    if (b >= 0) *first = begin(b);
    return b;
}

// The page of position block `blk` (16 positions) of sequence b, or -1.
__device__ __forceinline__ int pg_page(const Paged& a, int b, int blk) {
    const int id = a.table[(size_t)b * a.max_pages + (blk >> (a.page_sh - 4))];
    return (unsigned)id < (unsigned)a.pages ? id : -1;
}

}  // namespace kt
