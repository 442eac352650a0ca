// Attention of a ragged batch's new rows over paged KV caches on gfx950 (kt_hip_dec_attention_paged, stated in
// include/kt_hip.h): chunks, whole prompts and single tokens by one kernel.
//
// A sequence's rows and the q heads of one kv head make columns (row i, head r: i rep + r). A CTA takes 16 of them, a wave
// 64 positions at a time, and both products run on 16x16x64 int8 MFMAs with the positions as rows of the first and as the
// summed index of the second. The integer softmax needs the largest score before any weight, exactly: pass 1 takes it over
// all positions (K alone), pass 2 forms the scores again or finds them in LDS, looks the weights up and multiplies V by
// their balanced base-256 digits, two of them (4-bit pages: three, of weight times multiplier); the digit sums are exact in
// int32 and meet as int64.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>
#include <type_traits>

#include "kt_paged.h"
#include "kt_w12_core.h"

namespace kt {

namespace {

typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef short ss2 __attribute__((ext_vector_type(2)));

struct PgAttend {
    const int8_t* q;
    int8_t* o;
    int64_t q_stride, o_stride;
    const int32_t* exp_tab;
    int rep, window, sinks, splits;
    int keep;                  // PG_KEEP: bytes of LDS for the scores kept between the passes
    int32_t* wlow;             // [unit][split][column]: the least negated scores
    unsigned long long* wsum;  // [unit][16 dimensions][register][lane], then the columns' sums of weights
    unsigned* wcnt;            // [unit]: the splits that have added theirs
    int32_t* stats;            // STATS: [row][head]: the largest score, the reciprocal of the weights' sum
};

// A CTA's part of the work. PG_WHOLE: both passes over all positions; PG_KEEP: the same with pass 1's scores kept in LDS as
// far as it goes. PG_MAX and PG_SUMS: the two passes as two launches, each over splits of the positions.
enum { PG_WHOLE = 0, PG_KEEP = 1, PG_MAX = 2, PG_SUMS = 3 };

constexpr int PG_COLS = 16;

// What a wave holds of a tile, 64 positions (four blocks of 16) of one kv head, in chunks (16 values: 16 bytes, or 8).
//
// Both K and V arrive as the caches hold them, lane l reading chunks l % 16 + 16 i of block l / 16. K goes through the
// wave's own LDS to its operand order: lane l has chunk l / 16 (+ 4 c) of position 16 (l / 4 % 4) + 4 t + l % 4 in k[t][c]. As
// the A operand of a product these rows give lane l the scores of positions 16 (l / 16) + 4 t + r in register r, so that a
// lane's 16 scores of the four products are one block's 16 positions in order: the layout of a B operand of the product
// with V, whose chunks (16 positions of a dimension) are its A operand as they stand.
template <int BITS>
struct PgChunk {
    typedef v4i T;
};
template <>
struct PgChunk<4> {
    typedef v2i T;
};
template <int HD, int BITS>
struct PgTile {
    typename PgChunk<BITS>::T x[HD / 16];
    v4i m;  // 4 bits: the multipliers of block l / 16
};

// -x of 16 int8 values, -128 taken as -127. A byte of sign h and low bits lo: 2^7 - lo takes no borrow from its neighbours and
// reaches 2^7 where lo is 0, that is for 0 and -128.
__device__ __forceinline__ v4i negate8(v4i x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = (uint32_t)x[i], h = u & 0x80808080u, t = 0x80808080u - (u & 0x7F7F7F7Fu);
        const uint32_t z = t & 0x80808080u, least = h & z;
        x[i] = (int)((t & 0x7F7F7F7Fu) | (~(h | z) & 0x80808080u) | (least - (least >> 7)));
    }
    return x;
}

// The swizzle of a row's chunks in the wave's LDS (row r of block n), by which the lanes that one LDS cycle serves (8 of 16
// bytes, 16 of 8: rows 4 t .. 4 t + 3 of two or four blocks) read different banks.
template <int HD, int BITS>
__device__ __forceinline__ int pg_swz(int n, int r) {
    if constexpr (BITS == 8) return HD == 64 ? ((r >> 1) & 1) | ((n & 1) << 1) : (r & 3) | ((n & 1) << 2);
    else return HD == 64 ? n : ((r >> 1) & 1) | (n << 1);
}

// Four neighbouring dimensions of an output row: clamp(round_half_away(a / b)), a = sum e v and b = sum e as the digits add up (both
// negated; 4 bits: v as 16 codes times 1/8 of a multiplier, so 128 sum e), zeros where nothing was seen. The quotient
// is a float estimate (relative error below 2^-20, so below 2^-12 for |a / b| < 256); where that is within 2^-12 of a half the
// exact remainder of 2 |a| + b by 2 b says which side.
template <int BITS>
__device__ __forceinline__ void pg_store(int8_t* to, const int64_t (&v)[4], int64_t dn, bool live) {
    const int64_t b = BITS == 8 ? -dn : -128 * dn;
    auto f = [](uint64_t x) { return __builtin_fmaf((float)(uint32_t)(x >> 32), 4294967296.0f, (float)(uint32_t)x); };
    uint32_t out = 0;
    if (live && b > 0) {
        const float rb = __builtin_amdgcn_rcpf(f((uint64_t)b));
        uint64_t m[4];
        int q[4];
        bool unsure = false;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            m[r] = v[r] < 0 ? 0 - (uint64_t)v[r] : (uint64_t)v[r];
            const float t = f(m[r]) * rb + 0.5f;
            unsure |= !(__builtin_fabsf(__builtin_amdgcn_fractf(t) - 0.5f) < 0.5f - 0x1p-12f);
            q[r] = (int)t;
        }
        if (unsure) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint64_t n = 2 * m[r] + (uint64_t)b, d = 2 * (uint64_t)b;
                const int64_t rem = (int64_t)(n - (uint64_t)(uint32_t)q[r] * d);
                q[r] += rem < 0 ? -1 : (rem >= (int64_t)d ? 1 : 0);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int x = min(q[r], 127);
            out |= (uint32_t)(uint8_t)(v[r] < 0 ? x : -x) << (8 * r);
        }
    }
    *reinterpret_cast<uint32_t*>(to) = out;
}

// STATS: the columns' statistics too (a kernel of its own: what it keeps of them costs 128 single tokens behind 6100 a fiftieth; us with /
// without: those 45.9 / 44.6, one behind 640 6.9 / 6.4, 3 x 1021 rows 26.4 / 25.4, 1024 rows behind 7777 85.2 / 84.5).
template <int HD, int BITS, int W, int MODE, bool STATS>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W == 8 || HD == 128 ? 2 : (BITS == 8 ? 4 : 3)))) void pg_attend_kernel(
    Paged a, PgAttend p) {
    constexpr int HH = HD / 2, KC = HD / 64, DT = HD / 16, ND = BITS == 8 ? 2 : 3;
    constexpr int NT = 64 * W, ET = 256 / NT > 1 ? 256 / NT : 1;  // fours of table entries a thread
    constexpr int ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;  // bytes of a K row of a slot, of a chunk
    constexpr bool MAXP = MODE != PG_SUMS, SUMP = MODE != PG_MAX;
    typedef PgTile<HD, BITS> Tile;
    typedef typename PgChunk<BITS>::T Chunk;
    __shared__ int64_t sSum[SUMP ? DT * 4 * 64 : 1], sDen[PG_COLS];
    __shared__ int sLow[MODE == PG_SUMS ? NT / PG_COLS : W][PG_COLS];
    __shared__ __attribute__((aligned(8))) uint16_t sE[1028];
    __shared__ __attribute__((aligned(16))) int8_t sK[W][64 * ROWB];
    extern __shared__ __attribute__((aligned(16))) int sS[];  // PG_KEEP: the scores of each wave's first tiles
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, gq = lane >> 4, kb = (lane >> 2) & 3, split = (int)blockIdx.y;
    typedef int tab4 __attribute__((ext_vector_type(4), aligned(4)));
    tab4 et[ET];
    if constexpr (SUMP) {  // the table is on its way while the batch is looked up
#pragma unroll
        for (int i = 0; i < ET; i++)
            if (NT <= 256 || tid < 256) et[i] = *reinterpret_cast<const tab4*>(p.exp_tab + 4 * (tid + i * NT));
    }

    // The kv head fastest: CTAs go to the XCDs in turn, so an XCD's L2 holds the heads congruent to it. Column tiles 0 .. seqs -
    // 1 are the sequences' first ones, the rest their further ones, from the last (of a prompt's, those see the most). Single
    // tokens may have first ones alone: CTAs that leave at once between those that stay would leave the XCDs different numbers
    // of them (numbered sequence by sequence, 256 on 256 CUs took two rounds: 68 us against 50).
    const int ntiles = (int)gridDim.x / a.nkv, g = (int)blockIdx.x % a.nkv, tile = ntiles - 1 - (int)blockIdx.x / a.nkv;
    int b = tile, nth = 0;
    if (tile >= a.seqs) {
        int first = 0;
        b = pg_tile_seq(a, tile - a.seqs, p.rep, PG_COLS, 0, &first);
        nth = tile - a.seqs - first + 1;
    }
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int m0 = nth * PG_COLS, mrows = s.n * p.rep;
    if (m0 >= mrows) return;
    const int cols = min(PG_COLS, mrows - m0), cap = a.max_pages << a.page_sh, nblk = cap >> 4;
    const int pmin = s.p0 + m0 / p.rep, pmax = min(s.p0 + (m0 + cols - 1) / p.rep, cap - 1);
    // the tiles of positions: those of the sinks, then those of the window
    const int ntile = pmax < 0 || a.pages == 0 ? 0 : pmax / 64 + 1;
    int nsink = 0, w0 = 0;
    if (p.window && ntile) {
        nsink = min((min(p.sinks, pmax + 1) + 63) / 64, ntile);
        w0 = max(nsink, (max(pmin, 0) - min(p.window - 1, max(pmin, 0))) / 64);
    }
    const int total = nsink + max(0, ntile - w0), step = p.splits * W, start = split * W + w;
    const int mine = start < total ? (total - 1 - start) / step + 1 : 0;  // this wave's tiles: every step-th from start
    auto at = [&](int n) {
        const int i = start + n * step;
        return i < nsink ? i : i - nsink + w0;
    };

    // the columns' rows and positions, and their negated q as B operands
    const int mcol = min(m0 + l16, mrows - 1), row = mcol / p.rep, head = g * p.rep + mcol - row * p.rep;
    const int pos = l16 < cols && s.p0 + row < cap ? s.p0 + row : -1;
    v4i q[KC];
#pragma unroll
    for (int c = 0; c < KC; c++)
        q[c] = negate8(*reinterpret_cast<const v4i*>(p.q + (size_t)(s.t0 + row) * p.q_stride + head * HD + 16 * gq + 64 * c));
    if constexpr (SUMP) {
#pragma unroll
        for (int i = 0; i < ET; i++) {
            uint32_t e[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                e[r] = (uint32_t)min(max(et[i][r], 0), 32768);
                // 8 bits: the two balanced base-256 digits of -e (2^15 itself has none, -2^15 does); 4 bits: -e
                e[r] = (BITS == 8 ? (0x8080u - e[r]) ^ 0x8080u : 0u - e[r]) & 0xFFFFu;
            }
            if (NT <= 256 || tid < 256)
                *reinterpret_cast<v2i*>(sE + 4 * (tid + i * NT)) = v2i{(int)(e[0] | e[1] << 16), (int)(e[2] | e[3] << 16)};
        }
        if (tid == 0) sE[1024] = 0;
        for (int i = tid; i < DT * 4 * 64; i += NT) sSum[i] = 0;
        if (tid < PG_COLS) sDen[tid] = 0;
    }

    // A lane's own block of a tile is block gq, for K and V alike: its page id, and its chunk l16's place in a pool
    const uint8_t *const kbase = a.k + (size_t)g * a.part, *const vbase = a.v + (size_t)g * a.part;
    const uint32_t stride = (uint32_t)a.nkv * (uint32_t)a.part;
    auto block_of = [&](int T) { return min(4 * T + gq, nblk - 1); };
    auto slot_of = [&](int T) { return (block_of(T) << 4) & ((1 << a.page_sh) - 1); };
    auto page_id = [&](int T) { return a.table[(size_t)b * a.max_pages + (block_of(T) >> (a.page_sh - 4))]; };
    auto page_ok = [&](int T, int id) { return ((unsigned)id < (unsigned)a.pages) & (4 * T + gq < nblk); };
    auto load = [&](const uint8_t* pool, int T, int id, Tile& x) {  // an id outside the pool reads page 0 and is masked
        const uint64_t part = (uint64_t)((unsigned)id < (unsigned)a.pages ? (uint32_t)id : 0u) * stride;
        const uint8_t* from = pool + (part + (uint32_t)(slot_of(T) * ROWB + l16 * CHB));
#pragma unroll
        for (int i = 0; i < DT; i++) x.x[i] = *reinterpret_cast<const Chunk*>(from + 16 * CHB * i);
        if constexpr (BITS == 4) x.m = *reinterpret_cast<const v4i*>(pool + (part + (uint32_t)((HH << a.page_sh) + slot_of(T))));
    };
    int8_t* const sk = sK[w];
    auto turn_k = [&](const Tile& x, Chunk (&k)[4][KC]) {
        __builtin_amdgcn_wave_barrier();  // the last tile's reads are issued; LDS takes a wave's accesses in order
#pragma unroll
        for (int i = 0; i < DT; i++) {
            const int r = (16 * i + l16) / DT, ch = l16 % DT;
            *reinterpret_cast<Chunk*>(sk + (16 * gq + r) * ROWB + (ch ^ pg_swz<HD, BITS>(gq, r)) * CHB) = x.x[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < KC; c++)
                k[t][c] = *reinterpret_cast<const Chunk*>(sk + (16 * kb + 4 * t + (lane & 3)) * ROWB +
                                                          ((4 * c + gq) ^ pg_swz<HD, BITS>(kb, lane & 3)) * CHB);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    // 4 bits: 16 times the 16 codes of a chunk, in order (byte 4 h + r: code 8 h + r low, code 8 h + 4 + r high)
    auto widen = [](Chunk x) {
        if constexpr (BITS == 8) {
            return x;
        } else {
            constexpr int M = (int)0xF0F0F0F0;
            return v4i{(x.x << 4) & M, x.x & M, (x.y << 4) & M, x.y & M};
        }
    };
    // the negated scores: register r of sc[t] is position 16 gq + 4 t + r of the tile, column l16
    auto scores = [&](const Chunk (&k)[4][KC], v4i m, v4i (&sc)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++) sc[t] = mfma16(widen(k[t][c]), q[c], sc[t]);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int r = 0; r < 4; r++)  // -((m (q . c) + 4) >> 3) of -16 (q . c)
                    sc[t][r] = (__mul24(sc[t][r], (m[t] >> (8 * r)) & 255) + 63) >> 7;
            }
        }
    };
    // what the column sees of a tile's block: its positions k <= hi and, with a window, k > lo or k < sink
    struct Mask {
        int hi, lo, sink;
    };
    auto mask_of = [&](int T, bool ok) {
        const int from = 64 * T + 16 * gq;
        return Mask{ok ? pos - from : -1, pos - p.window - from, p.sinks - from};
    };
    auto sees = [](auto how, const Mask& m, int k) {
        if constexpr (how == 0) return true;
        else if constexpr (how == 1) return k <= m.hi;
        else return (k <= m.hi) & ((k > m.lo) | (k < m.sink));
    };
    typedef std::integral_constant<int, 0> All;  // every position; those up to the column's own; and with a window
    typedef std::integral_constant<int, 1> Causal;
    typedef std::integral_constant<int, 2> Window;
    // whether every column sees every position of the tile (uniform)
    auto full = [&](int T, bool ok) {
        return __all(ok) && 64 * T + 63 <= pmin && (p.window == 0 || 64 * T > pmax - p.window || 64 * T + 63 < p.sinks);
    };

    // PG_KEEP: as many of the wave's tiles as the LDS holds keep their scores, a column's 16 bytes at a time (lanes side by
    // side); the others' are formed again from K, last tile first: its K is nearest. 128 single tokens behind about 6100
    // positions 50.3 -> 45.5 us.
    const int kept = MODE == PG_KEEP ? min(mine, p.keep / (256 * W * cols)) : 0;
    auto kept_place = [&](int n, int t) { return reinterpret_cast<v4i*>(sS) + (((n * W + w) * 4 + t) * 4 + gq) * cols + l16; };
    // V's ring over the kept tiles; at hd 64 there are registers to begin it before the maximum is known
    constexpr bool EARLY = MODE == PG_KEEP && HD == 64;
    constexpr int NV = EARLY ? 2 : 1;
    Tile xv[NV];
    int idv[NV], nidv[NV];
    auto begin_v = [&]() {
#pragma unroll
        for (int u = 0; u < NV; u++) {
            idv[u] = nidv[u] = 0;
            if (u < kept) idv[u] = page_id(at(u)), load(vbase, at(u), idv[u], xv[u]);
            if (u + NV < kept) nidv[u] = page_id(at(u + NV));
        }
    };

    // Tiles go through rings in registers, with 8 waves (one CTA a CU) two of K in pass 1 and two of V for kept scores, else one:
    // a tile's page ids are read a round of the ring before its loads are issued, and those a round before they are used, so a
    // wave waits for neither. No more, as every copy of a loop's body is fetched anew by each launch: with four of each and two
    // in pass 2, 128 single tokens took 48.2 us against 45.5 and one token behind 131000 positions of 4 bits 21.8 against 20.7; a
    // chunk of 1024 rows behind 7777 takes 83.7 traced.
    int low = INT_MAX;  // the least negated score of the column
    if constexpr (MAXP) {
        constexpr int NB = W == 8 ? 2 : 1;
        Tile x[NB];
        int id[NB], nid[NB];
#pragma unroll
        for (int u = 0; u < NB; u++) {
            id[u] = nid[u] = 0;
            if (u < mine) id[u] = page_id(at(u));
            if (u + NB < mine) nid[u] = page_id(at(u + NB));
        }
#pragma unroll
        for (int u = 0; u < NB; u++)
            if (u < mine) load(kbase, at(u), id[u], x[u]);
        if constexpr (EARLY) begin_v();
        for (int n0 = 0; n0 < mine; n0 += NB) {
#pragma unroll
            for (int u = 0; u < NB; u++) {
                const int n = n0 + u;
                if (n >= mine) break;
                const int T = at(n);
                const bool ok = page_ok(T, id[u]), all = full(T, ok);
                Chunk k[4][KC];
                turn_k(x[u], k);
                const v4i m = x[u].m;
                if (n + NB < mine) load(kbase, at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_id(at(n + 2 * NB));
                v4i sc[4];
                scores(k, m, sc);
                if (MODE == PG_KEEP && n < kept && l16 < cols) {
#pragma unroll
                    for (int t = 0; t < 4; t++) *kept_place(n, t) = sc[t];
                }
                auto least = [&](auto how) {
                    const Mask k = mask_of(T, ok);
#pragma unroll
                    for (int t = 0; t < 4; t++) {
#pragma unroll
                        for (int r = 0; r < 4; r++) sc[t][r] = sees(how, k, 4 * t + r) ? sc[t][r] : INT_MAX;
                        low = min(min(low, min(sc[t].x, sc[t].y)), min(sc[t].z, sc[t].w));
                    }
                };
                if (all) least(All());
                else if (p.window == 0) least(Causal());
                else least(Window());
            }
        }
        low = min(low, __shfl_xor(low, 16));
        low = min(low, __shfl_xor(low, 32));
        if (gq == 0) sLow[w][l16] = low;
    }
    const size_t unit = (size_t)tile * a.nkv + g;
    unsigned long long* const sum = p.wsum + unit * (size_t)(PG_COLS * (HD + 1));
    if constexpr (MODE == PG_SUMS) {  // the splits' least, each column's dealt to threads
        int m = INT_MAX;
        for (int i = tid / PG_COLS; i < p.splits; i += NT / PG_COLS) m = min(m, p.wlow[(unit * p.splits + i) * PG_COLS + tid % PG_COLS]);
        sLow[tid / PG_COLS][tid % PG_COLS] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (MODE == PG_SUMS ? NT / PG_COLS : W); i++) low = min(low, sLow[i][l16]);
    if constexpr (MODE == PG_MAX) {
        if (tid < PG_COLS) p.wlow[(unit * p.splits + split) * PG_COLS + tid] = low;
        // and what the sums are added to starts from zero, each split clearing its share
        for (int i = split * NT + tid; i < PG_COLS * (HD + 1); i += p.splits * NT) sum[i] = 0;
        if (split == 0 && tid == 0) p.wcnt[unit] = 0;
        return;
    }
    if constexpr (SUMP) {
        const int top = 128 - 2 * (low == INT_MAX ? 0 : low);  // 2 (max + 64); of a column that sees nothing every weight is masked
        v4i acc[DT][ND];
        int den[2] = {0, 0};
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int n = 0; n < ND; n++) acc[d][n] = v4i{0, 0, 0, 0};
        // y = 2 (max - s + 64); where the products are short, taken twice over on top of 2 (max + 64)
        auto lifted = [&](const Chunk (&k)[4][KC], v4i m, v4i (&y)[4]) {
            if constexpr (BITS == 8 && HD == 64) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    y[t] = v4i{top, top, top, top};
#pragma unroll
                    for (int c = 0; c < 2; c++) y[t] = mfma16(k[t][0], q[0], y[t]);
                }
            } else {
                scores(k, m, y);
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) y[t][r] = (int)((uint32_t)y[t][r] * 2 + (uint32_t)top);
            }
        };
        // The weights' digits as B operands: the table index is y >> 8, bytes 1 and 2 of y (|s| is at most 2^21, so y < 2^24
        // wherever the column sees the position; of other columns any index below 2^16 will do).
        auto weights = [&](auto how, int T, bool ok, v4i m, const v4i (&y)[4], v4i (&P)[ND]) {
            const Mask k = mask_of(T, ok);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                uint32_t u[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    u[r] = (uint32_t)y[t][r];
                    u[r] = sees(how, k, 4 * t + r) ? u[r] : 0x00FFFFFFu;
                }
                us2 e[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t ix = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(
                        __builtin_bit_cast(us2, __builtin_amdgcn_perm(u[2 * h + 1], u[2 * h], 0x06050201)), us2{1024, 1024}));
                    e[h] = us2{sE[ix & 0xFFFF], sE[ix >> 16]};
                }
                if constexpr (BITS == 8) {
                    const uint32_t e01 = __builtin_bit_cast(uint32_t, e[0]), e23 = __builtin_bit_cast(uint32_t, e[1]);
                    P[0][t] = (int)__builtin_amdgcn_perm(e23, e01, 0x06040200);
                    P[1][t] = (int)__builtin_amdgcn_perm(e23, e01, 0x07050301);
                    den[0] = __builtin_amdgcn_sdot4(P[0][t], 0x01010101, den[0], false);
                    den[1] = __builtin_amdgcn_sdot4(P[1][t], 0x01010101, den[1], false);
                } else {
                    uint32_t f[4];
#pragma unroll
                    for (int r = 0; r < 4; r++)  // the balanced digits of -e m: to -2^15 255 (m is any byte), which e m has not
                        f[r] = (uint32_t)(__mul24((int)(int16_t)e[r >> 1][r & 1], (int)(((uint32_t)m[t] >> (8 * r)) & 255)) + 0x808080) ^ 0x808080;
                    const uint32_t f01 = __builtin_amdgcn_perm(f[1], f[0], 0x05010400), f23 = __builtin_amdgcn_perm(f[3], f[2], 0x05010400);
                    P[0][t] = (int)__builtin_amdgcn_perm(f23, f01, 0x05040100);
                    P[1][t] = (int)__builtin_amdgcn_perm(f23, f01, 0x07060302);
                    P[ND - 1][t] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(f[3], f[2], 0x0c0c0602),
                                                              __builtin_amdgcn_perm(f[1], f[0], 0x0c0c0602), 0x05040100);
                    den[0] = __builtin_amdgcn_sdot2(__builtin_bit_cast(ss2, e[0]), ss2{1, 1}, den[0], false);
                    den[0] = __builtin_amdgcn_sdot2(__builtin_bit_cast(ss2, e[1]), ss2{1, 1}, den[0], false);
                }
            }
        };
        auto add_v = [&](int T, bool ok, const Tile& v, const v4i (&y)[4]) {
            v4i P[ND];
            if (full(T, ok)) weights(All(), T, ok, v.m, y, P);
            else if (p.window == 0) weights(Causal(), T, ok, v.m, y, P);
            else weights(Window(), T, ok, v.m, y, P);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < ND; e++) acc[d][e] = mfma16(widen(v.x[d]), P[e], acc[d][e]);
        };
        {
            constexpr int NB = 1;  // (as a loop without the ring's form the compiler's order of it is slower: the chunk above 86.6 us)
            Tile x[NB], v[NB];
            int id[NB], nid[NB];
            const int left = mine - kept;
            auto back = [&](int n) { return at(mine - 1 - n); };
#pragma unroll
            for (int u = 0; u < NB; u++) {
                id[u] = nid[u] = 0;
                if (u < left) id[u] = page_id(back(u));
                if (u + NB < left) nid[u] = page_id(back(u + NB));
            }
#pragma unroll
            for (int u = 0; u < NB; u++)
                if (u < left) load(kbase, back(u), id[u], x[u]), load(vbase, back(u), id[u], v[u]);
            for (int n0 = 0; n0 < left; n0 += NB) {
#pragma unroll
                for (int u = 0; u < NB; u++) {
                    const int n = n0 + u;
                    if (n >= left) break;
                    const int T = back(n);
                    Chunk k[4][KC];
                    turn_k(x[u], k);
                    const v4i m = x[u].m;
                    if (n + NB < left) load(kbase, back(n + NB), nid[u], x[u]);
                    v4i y[4];
                    lifted(k, m, y);
                    add_v(T, page_ok(T, id[u]), v[u], y);
                    if (n + NB < left) load(vbase, back(n + NB), nid[u], v[u]);
                    id[u] = nid[u];
                    if (n + 2 * NB < left) nid[u] = page_id(back(n + 2 * NB));
                }
            }
        }
        if constexpr (MODE == PG_KEEP) {
            if constexpr (!EARLY) begin_v();
            for (int n0 = 0; n0 < kept; n0 += NV) {
#pragma unroll
                for (int u = 0; u < NV; u++) {
                    const int n = n0 + u;
                    if (n >= kept) break;
                    const int T = at(n);
                    v4i y[4] = {};
                    if (l16 < cols) {
#pragma unroll
                        for (int t = 0; t < 4; t++) y[t] = *kept_place(n, t);
                    }
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) y[t][r] = (int)((uint32_t)y[t][r] * 2 + (uint32_t)top);
                    add_v(T, page_ok(T, idv[u]), xv[u], y);
                    if (n + NV < kept) load(vbase, at(n + NV), nidv[u], xv[u]);
                    idv[u] = nidv[u];
                    if (n + 2 * NV < kept) nidv[u] = page_id(at(n + 2 * NV));
                }
            }
        }

        // the waves' sums: register r of lane l is dimension 16 d + 4 (l / 16) + r of column l % 16
        if (mine > 0) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    int64_t v = (int64_t)acc[d][0][r] + ((int64_t)acc[d][1][r] << 8);
                    if constexpr (BITS == 4) v += (int64_t)acc[d][ND - 1][r] << 16;
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sSum[(d * 4 + r) * 64 + lane]), (unsigned long long)v);
                }
            const int64_t dn = BITS == 8 ? (int64_t)den[0] + ((int64_t)den[1] << 8) : (int64_t)den[0];
            atomicAdd(reinterpret_cast<unsigned long long*>(&sDen[l16]), (unsigned long long)dn);
        }
        __syncthreads();
        int8_t* const out = p.o + (size_t)(s.t0 + row) * p.o_stride + head * HD;  // (it % 16 is this thread's l16)
        auto put = [&](int it, const int64_t (&v)[4], int64_t dn) {  // dimensions 16 (it / 64) + 4 (it % 64 / 16) ..
            pg_store<BITS>(out + 16 * (it >> 6) + 4 * ((it & 63) >> 4), v, dn, pos >= 0);
        };
        [[maybe_unused]] auto leave = [&](int64_t dn) {  // by thread tid < cols, whose column is tid: `low` and the sum of its weights, negated
            const uint64_t R = dn < 0 && pos >= 0 ? (1ull << 40) / (uint64_t)-dn : 0;
            v2i* to = reinterpret_cast<v2i*>(p.stats + 2 * ((size_t)(s.t0 + row) * (p.rep * a.nkv) + head));
            *to = v2i{low == INT_MAX || pos < 0 ? 0 : -low, (int)(uint32_t)(R > 0xFFFFFFFFull ? 0xFFFFFFFFull : R)};
        };
        if constexpr (STATS && MODE != PG_SUMS) {
            if (tid < cols) leave(sDen[tid]);
        }
        for (int it = tid; it < DT * 64; it += NT) {
            if ((it & 15) >= cols) continue;
            int64_t v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = sSum[((it >> 6) * 4 + r) * 64 + (it & 63)];
            if constexpr (MODE == PG_SUMS) {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    (void)__hip_atomic_fetch_add(sum + ((it >> 6) * 4 + r) * 64 + (it & 63), (unsigned long long)v[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (it < PG_COLS)
                    (void)__hip_atomic_fetch_add(sum + PG_COLS * HD + it, (unsigned long long)sDen[it], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            } else {
                put(it, v, sDen[it & 15]);
            }
        }
        if constexpr (MODE == PG_SUMS) {  // the unit's last CTA has every split's sums (integers: in any order the same)
            if (!split_last(p.wcnt + unit)) return;
            if constexpr (STATS) {
                if (tid < cols) leave((int64_t)__hip_atomic_load(sum + PG_COLS * HD + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            }
            for (int it = tid; it < DT * 64; it += NT) {
                if ((it & 15) >= cols) continue;
                int64_t v[4];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    v[r] = (int64_t)__hip_atomic_load(sum + ((it >> 6) * 4 + r) * 64 + (it & 63), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                put(it, v, (int64_t)__hip_atomic_load(sum + PG_COLS * HD + (it & 15), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            }
        }
    }
}

struct Plan {
    int w, tiles, splits;  // waves of a CTA, column tiles (an upper bound), splits of the positions
};

// From the counts that the host knows. A unit is a column tile of one kv head. Waves: 8 a CTA, one CTA a CU, while the units
// fit the CUs; else 4, and 2 where that fills the chip by itself (a CTA's waves share its columns, so fewer of them join
// less). us with 2 / 4 / 8, 14 heads over 2, hd 64: 64 rows behind 4000 positions (56 units) 36.0 / 22.7 / 16.5; 512 behind
// 4000 (448) 45.9 / 30.9 / 35.3; 1024 alone (896) 15.1 / 12.4 / 23.6; 3 x 1021 alone (2682) 25.5 / 29.0 / 63.5. The same
// rows in 4 bits 53.3 / 29.6 / 21.9, 71.7 / 41.5 / 44.0, 19.1 / 18.0 / 25.6, 37.4 / 37.5 / 68.6. hd 128, 16 heads over 4: 64
// behind 4000 (68) 47.2 / 31.5 / 22.6, 320 behind 2000 (324) 34.3 / 24.3 / 27.3, 512 behind 4000 (516) 59.9 / 42.4 / 45.6,
// 1024 alone (1028) 19.1 / 21.0 / 28.2, 1600 alone (1604) 33.4 / 39.5 / 53.3; in 4 bits 64.5 / 38.3 / 28.5, 50.1 / 31.9 /
// 34.1, 91.9 / 54.5 / 58.2, 25.2 / 25.9 / 32.3, 43.4 / 47.6 / 61.5. So the first border holds for all of them, and at hd
// 128, with two waves a SIMD, two waves would already do from some 1000 units on, by a tenth. Single tokens differ less: 600
// behind 1000 (1200 units, hd 64) 36.8 / 41.3 / 54.0, 120 at hd 128 (480) 31.9 / 29.8 / 26.5. A wave never has more than
// 65536 positions: its digit sums stay within 2^14 2^16. Splits, where units leave CUs without one: to 128 CTAs, of at least
// 8 tiles; past that the extra launch, the second reading of K and the sums that meet in memory outweigh it. us with 1 / the
// rule's / twice its splits: one token behind 131000 (2 units) 353 / 17.8 / 20.2, 4 behind 32000 (8) 92.5 / 18.1 / 21.1, 16
// behind 8000 (32) 28.3 / 17.7 / 20.8, 64 (128) 37.1 / 37.1 / 53.8, one behind 5000 17.8 / 11.0 / 10.8; below 64 tiles it
// gains nothing (behind 2000 10.1 / 11.1 with two).
//
// Kernel times against the bytes and operations that cannot be left out (4 hd a column and visible position): 128 single
// tokens behind 6100 positions 45.5 us, 199 MB of K and V at 4.4 TB/s (the loads of ragged lengths end unevenly; a plain
// read of as much reaches 5.9); one token behind 131000 4-bit positions 6 + 14.5 us for 17 MB (two launches, four tiles a
// wave each, and a join; in the second, vector units are busy 45 % of the time and waves wait for half of theirs); 1024 rows
// behind 7777 74 us, 30.4 GOP at 0.41 POPS counted once (the scores are formed three times over, weights take two digits);
// there matrix units, vector units and LDS are busy 25, 50 and 58 % of the time and a wave waits for one of them in turn: 4
// waves on 64 columns sharing a tile's K and V in LDS (a third of the reads from the L2) took 87 us against 84 under the
// profiler. Two thirds of the LDS time are the turns of K (16 KB a tile over both passes), the rest the look-ups of weights.
// The same rows over 4-bit pages 123 us, vector units busy 83 %: a score's multiplier and rounding, and three digits of each
// weight, 465 instructions a tile against 161.
Plan plan(int64_t tokens, int64_t seqs, int64_t max_pos, int rep, int nkv) {
    const int64_t tiles = seqs + tokens * rep / PG_COLS, steps = max_pos / 64;
    const int64_t units = std::min(tiles, tokens * ((rep + PG_COLS - 1) / PG_COLS)) * nkv;
    int w = units <= 256 ? 8 : (units <= 1536 ? 4 : 2);
    while (w < 8 && max_pos > 65536 * w) w *= 2;
    const int64_t splits = w == 8 && steps >= 64 ? std::min(128 / std::max<int64_t>(units, 1), steps / 8) : 1;
    return {w, (int)tiles, (int)std::max<int64_t>(splits, 1)};
}

// The workspace's parts: the splits' least scores, the sums, the counts of arrived splits.
struct Parts {
    size_t sum, cnt, bytes;
};

Parts parts(const Plan& x, int nkv, int hd) {
    if (x.splits == 1) return {0, 0, 256};
    const size_t units = (size_t)x.tiles * nkv;
    const size_t sum = (units * x.splits * PG_COLS * 4 + 255) / 256 * 256, cnt = sum + units * PG_COLS * (hd + 1) * 8;
    return {sum, cnt, std::max<size_t>(256, cnt + (units * 4 + 255) / 256 * 256)};  // (0 says a shape refused)
}

template <int HD, int BITS, bool STATS>
hipError_t attend(const Paged& a, const PgAttend& p, const Plan& x, hipStream_t s) {
    const dim3 grid((unsigned)(x.tiles * a.nkv), (unsigned)x.splits), block(64 * x.w);
    if (x.w == 2) {
        pg_attend_kernel<HD, BITS, 2, PG_WHOLE, STATS><<<grid, block, 0, s>>>(a, p);
    } else if (x.w == 4) {
        pg_attend_kernel<HD, BITS, 4, PG_WHOLE, STATS><<<grid, block, 0, s>>>(a, p);
    } else if (x.splits == 1) {
        pg_attend_kernel<HD, BITS, 8, PG_KEEP, STATS><<<grid, block, (size_t)p.keep, s>>>(a, p);
    } else {
        pg_attend_kernel<HD, BITS, 8, PG_MAX, false><<<grid, block, 0, s>>>(a, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        pg_attend_kernel<HD, BITS, 8, PG_SUMS, STATS><<<grid, block, 0, s>>>(a, p);
    }
    return hipGetLastError();
}

}  // namespace

size_t pg_attend_workspace(int tokens, int seqs, int64_t max_pos, int nh, int nkv, int hd) {
    return parts(plan(tokens, seqs, max_pos, nh / nkv, nkv), nkv, hd).bytes;
}

hipError_t launch_pg_attend(const Paged& a, int hd, int bits, const int8_t* q, int64_t q_stride, int nh,
                            const int32_t* exp_tab, int window, int sinks, int8_t* o, int64_t o_stride, int32_t* stats,
                            void* ws, hipStream_t s) {
    const int64_t max_pos = (int64_t)a.max_pages << a.page_sh;
    const int rep = nh / a.nkv;
    // With a window a column tile's positions are fewer than window + sinks + 256 (15 of other rows, two tiles' ends each), whatever
    // the table's width: fewer splits than the workspace is made for, so no more of it.
    const int64_t reach = window ? std::min<int64_t>(max_pos, (int64_t)window + sinks + 256) : max_pos;
    const Plan x = plan(a.tokens, a.seqs, reach, rep, a.nkv);
    const Parts w = parts(x, a.nkv, hd);
    // kept scores: 256 bytes a column and tile, as far as a CTA's LDS (160 KB) goes beside the static arrays (K's 8 tiles, the
    // sums, 4 KB of others)
    const int64_t cols = a.tokens > a.seqs ? PG_COLS : std::min(rep, PG_COLS), most = (reach / 64 + 8) / 8 * 8 * cols * 256;
    const int64_t room = 163840 - 8 * 64 * (bits == 8 ? hd : hd / 2) - hd * 128 - 4096;
    const PgAttend p = {q, o, q_stride, o_stride, exp_tab, rep, window, sinks, x.splits, (int)std::min(most, room),
                        (int32_t*)ws, (unsigned long long*)((char*)ws + w.sum), (unsigned*)((char*)ws + w.cnt), stats};
    if (stats) {
        if (hd == 64) return bits == 8 ? attend<64, 8, true>(a, p, x, s) : attend<64, 4, true>(a, p, x, s);
        return bits == 8 ? attend<128, 8, true>(a, p, x, s) : attend<128, 4, true>(a, p, x, s);
    }
    if (hd == 64) return bits == 8 ? attend<64, 8, false>(a, p, x, s) : attend<64, 4, false>(a, p, x, s);
    return bits == 8 ? attend<128, 8, false>(a, p, x, s) : attend<128, 4, false>(a, p, x, s);
}

}  // namespace kt
