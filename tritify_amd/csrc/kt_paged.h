// What the kernels on paged KV caches share: the batch's rows and the division of its sequences into tiles. The layout of
// the pools is stated with kt_hip_dec_page_bytes in include/kt_hip.h.
#pragma once

#include <stdint.h>

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
// -1 where none does: the wave probes 64 sequences at even distances and goes on between two of them. Where row_start
// decreases the probes may end at a sequence that begins past `t`; that counts as none, so that a tile is never before its
// sequence's first.
__device__ __forceinline__ int pg_tile_seq(const Paged& a, int t, int mul, int step, int per, int* first) {
    const int lane = threadIdx.x & 63;
    auto begin = [&](int b) { return (int)((int64_t)pg_start(a, b) * mul / step) + per * b; };
    for (int lo = 0, n = a.seqs;;) {
        const int gap = (n + 63) / 64;
        const int c = __popcll(__ballot(lane * gap < n && begin(lo + lane * gap) <= t));
        if (c == 0) return -1;
        lo += (c - 1) * gap;
        if (gap == 1) {
            *first = begin(lo);
            return *first <= t ? lo : -1;
        }
        n = min(gap, n - (c - 1) * gap);
    }
}

// The page of position block `blk` (16 positions) of sequence b, or -1.
__device__ __forceinline__ int pg_page(const Paged& a, int b, int blk) {
    const int id = a.table[(size_t)b * a.max_pages + (blk >> (a.page_sh - 4))];
    return (unsigned)id < (unsigned)a.pages ? id : -1;
}

}  // namespace kt
