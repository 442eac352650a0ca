// Attention of a ragged batch's new rows over paged KV caches on gfx950 (kt_hip_dec_attention_paged, stated in
// include/kt_hip.h): chunks, whole prompts and single tokens by one kernel.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>
#include <stdlib.h>
#include <type_traits>

#include "kt_paged.h"
#include "kt_w12_core.h"

namespace kt {

namespace {

#ifndef PG_EU1
#define PG_EU1 3
#endif
#ifndef PG_NB1
#define PG_NB1 1
#endif
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

struct PgAttend {
    const int8_t* q;
    int8_t* o;
    int64_t q_stride, o_stride;
    const int32_t* exp_tab;
    int rep, window, sinks, splits;
    int keep;       // bytes of LDS for scores kept between the passes (PG_KEEP)
    int32_t* wlow;  // [tile][kv head][split][column]: the least negated scores
    unsigned long long* wsum;  // [tile][kv head][column group, 16 dimensions][register][lane], then the weights' sums
    unsigned* wcnt;            // [tile][kv head]
};

enum { PG_WHOLE = 0, PG_MAX = 1, PG_SUMS = 2, PG_KEEP = 3 };

// What a wave holds of a tile, 64 positions (four blocks of 16) of one kv head.
//
// Both arrive as the caches hold them, lane l reading chunks l % 16 + 16 i of block l / 16. K goes through the wave's own
// LDS to its operand order: lane l has chunk l / 16 (+ 4 c) of
// position 16 (l / 4 % 4) + 4 t + l % 4 in k[t][c]. As the A operand of a 16x16x64 product these rows give lane l the scores
// of positions 16 (l / 16) + 4 t + r in register r, so that a lane's 16 scores of the four products are one block's 16
// positions in order: the layout of a B operand of the product with V, whose chunks (16 positions of a dimension) are loaded
// as they stand.
template <int BITS>
struct PgChunk {
    typedef v4i T;
};
template <>
struct PgChunk<4> {
    typedef v2i T;
};

template <int HD, int BITS>
struct PgK {
    typename PgChunk<BITS>::T raw[HD / 16];
    v4i m;  // 4 bits: the multipliers of block l / 16
};
template <int HD, int BITS>
struct PgV {
    typename PgChunk<BITS>::T v[HD / 16];
    v4i m;
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

// Four neighbouring dimensions of an output row: clamp(round_half_away(sum e v / sum e)) of what the digits add up to (8
// bits: both negated; 4 bits: v as 16 codes times 1/8 of a multiplier), zeros where nothing was seen. The quotients
// floor((2 |a| + b) / (2 b)) are double estimates by one reciprocal (within one of the exact quotient, which is below 2^8 past
// the first test) and the exact remainders.
template <int BITS>
__device__ __forceinline__ void pg_store(int8_t* to, const int64_t (&v)[4], int64_t dn, bool live) {
    const uint64_t b = (uint64_t)(BITS == 8 ? -dn : 128 * dn), d = 2 * b;
    const double rd = 1.0 / (double)d;
    uint32_t out = 0;
    if (live && (int64_t)b > 0)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int64_t a = BITS == 8 ? -v[r] : v[r];
            const uint64_t m = a < 0 ? 0 - (uint64_t)a : (uint64_t)a, n = 2 * m + b;
            int q = (int)((double)n * rd);
            const int64_t rem = (int64_t)(n - (uint64_t)(uint32_t)q * d);
            q += rem < 0 ? -1 : (rem >= (int64_t)d ? 1 : 0);
            q = m >= 128 * b || q > 127 ? 127 : q;
            out |= (uint32_t)(uint8_t)(a < 0 ? -q : q) << (8 * r);
        }
    *reinterpret_cast<uint32_t*>(to) = out;
}

// Waves a SIMD is meant to hold: registers for 2, or lean ones for 4.
constexpr int pg_eu(int hd, int mt, int wp) { return wp == 8 ? 2 : (hd * mt == 64 ? PG_EU1 : 2); }

template <int HD, int BITS, int MT, int WM, int WP, int MODE>
__global__ __launch_bounds__(64 * WM * WP) __attribute__((amdgpu_waves_per_eu(pg_eu(HD, MT, WP)))) void pg_attend_kernel(Paged a, PgAttend p) {
    constexpr int HH = HD / 2, KC = HD / 64, DT = HD / 16, ND = BITS == 8 ? 2 : 3;
    constexpr int W = WM * WP, NT = 64 * W, CW = 16 * MT, COLS = CW * WM;  // threads; columns of a wave and of the CTA
    constexpr int NMAX = COLS * WP > NT ? WP : NT / COLS;
    constexpr int ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;  // bytes of a K row of a slot, of a chunk
    typedef PgK<HD, BITS> Tile;
    typedef PgV<HD, BITS> VTile;
    typedef typename PgChunk<BITS>::T Chunk;
    constexpr bool MAXP = MODE != PG_SUMS, SUMP = MODE != PG_MAX;
    __shared__ int64_t sSum[SUMP && WP > 1 ? WM * MT * DT * 4 * 64 : 1];
    __shared__ int64_t sDen[SUMP ? COLS : 1];
    __shared__ int sLow[NMAX][COLS];
    __shared__ uint16_t sE[1026];
    __shared__ __attribute__((aligned(16))) int8_t sK[W][64 * ROWB];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = w / WP, wp = w % WP, l16 = lane & 15, gq = lane >> 4, kb = (lane >> 2) & 3;
    extern __shared__ __attribute__((aligned(16))) int sS[];  // PG_KEEP: the scores of each wave's first tiles
    const int split = (int)blockIdx.y;
    int et[(1024 + NT - 1) / NT];
    if constexpr (SUMP) {  // the table is on its way while the batch is looked up
#pragma unroll
        for (int i = 0; i < (1024 + NT - 1) / NT; i++) et[i] = p.exp_tab[min(tid + i * NT, 1023)];
    }
    // The kv head fastest: CTAs go to the XCDs in turn, so an XCD's L2 holds the heads congruent to it. Numbers 0 .. seqs - 1
    // are the sequences' first tiles, the rest their further ones (from the last: of a prompt's, those see the most), and a
    // kind that may be empty comes last: single tokens have no further tiles, and CTAs that leave at once between others
    // would leave the XCDs different numbers of those that stay (256 of them on 256 CUs took two rounds).
    const int ntiles = (int)gridDim.x / a.nkv, g = (int)blockIdx.x % a.nkv, order = (int)blockIdx.x / a.nkv;
    const int tile = WP == 8 ? order : ntiles - 1 - order;
    int b = tile, nth = 0;
    if (tile >= a.seqs) {
        int first = 0;
        b = pg_tile_seq(a, tile - a.seqs, p.rep, COLS, 0, &first);
        nth = tile - a.seqs - first + 1;
    }
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int mc = nth * COLS, mrows = s.n * p.rep;  // m: row i, head r of the group as i rep + r
    if (mc >= mrows) return;
    const int m0 = mc + wm * CW, cols = max(0, min(CW, mrows - m0)), nmt = (cols + 15) / 16;  // this wave's columns
    const int cap = a.max_pages << a.page_sh, nblk = cap >> 4;
    const int pmin = s.p0 + m0 / p.rep, pmax = min(s.p0 + (m0 + cols - 1) / p.rep, cap - 1);
    // the tiles of 64 positions: those of the sinks, then those of the window
    const int ntile = cols == 0 || pmax < 0 || a.pages == 0 ? 0 : pmax / 64 + 1;
    int nsink = 0, w0 = 0;
    if (p.window && ntile) {
        nsink = min((min(p.sinks, pmax + 1) + 63) / 64, ntile);
        w0 = max(nsink, (max(pmin, 0) - min(p.window - 1, max(pmin, 0))) / 64);
    }
    const int total = nsink + max(0, ntile - w0);
    auto tile_at = [&](int i) { return i < nsink ? i : i - nsink + w0; };

    const uint8_t *const kbase = a.k + (size_t)g * a.part, *const vbase = a.v + (size_t)g * a.part;
    const uint8_t *const kmult = a.k + (size_t)g * a.part + (HH << a.page_sh), *const vmult = a.v + (size_t)g * a.part + (HH << a.page_sh);

    // the columns' rows and positions, and their negated q as B operands
    int pos[MT];
    v4i q[MT][KC];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int m = min(m0 + 16 * mt + l16, mrows - 1), i = m / p.rep, r = m - i * p.rep;
        pos[mt] = 16 * mt + l16 < cols && s.p0 + i < cap ? s.p0 + i : -1;
        const int8_t* qr = p.q + (size_t)(s.t0 + i) * p.q_stride + (g * p.rep + r) * HD + 16 * gq;
#pragma unroll
        for (int c = 0; c < KC; c++) q[mt][c] = negate8(*reinterpret_cast<const v4i*>(qr + 64 * c));
    }
    if constexpr (SUMP) {
#pragma unroll
        for (int i = 0; i < (1024 + NT - 1) / NT; i++) {
            const int e = min(max(et[i], 0), 32768);
            // 8 bits: the two balanced base-256 digits of -e (2^15 itself has none, -2^15 does); 4 bits: e
            if (tid + i * NT < 1024) sE[tid + i * NT] = BITS == 8 ? (uint16_t)((0x8080 - e) ^ 0x8080) : (uint16_t)e;
        }
        if (tid == 0) sE[1024] = 0;
        if constexpr (WP > 1) {
            for (int i = tid; i < WM * MT * DT * 4 * 64; i += NT) sSum[i] = 0;
            if (tid < COLS) sDen[tid] = 0;
        }
    }

    // A lane's own block of a tile is block gq, for K and V alike: its page id, and its chunk l16's place in a pool
    const int32_t* const table = a.table + (size_t)b * a.max_pages;
    const uint32_t stride = (uint32_t)a.nkv * (uint32_t)a.part;
    auto block_of = [&](int T) { return min(4 * T + gq, nblk - 1); };
    auto page_id = [&](int T) { return table[block_of(T) >> (a.page_sh - 4)]; };
    auto part_of = [&](int id) { return (uint64_t)((unsigned)id < (unsigned)a.pages ? (uint32_t)id : 0u) * stride; };
    auto slot_of = [&](int T) { return (block_of(T) << 4) & ((1 << a.page_sh) - 1); };
    auto load_k = [&](int T, int id, Tile& x) {
        const uint8_t* at = kbase + (part_of(id) + (uint32_t)(slot_of(T) * ROWB + l16 * CHB));
#pragma unroll
        for (int i = 0; i < DT; i++) x.raw[i] = *reinterpret_cast<const Chunk*>(at + 16 * CHB * i);
        if constexpr (BITS == 4) x.m = *reinterpret_cast<const v4i*>(kmult + part_of(id) + (uint32_t)slot_of(T));
    };
    auto load_v = [&](int T, int id, VTile& x) {
        const uint8_t* at = vbase + (part_of(id) + (uint32_t)(slot_of(T) * ROWB + l16 * CHB));
#pragma unroll
        for (int d = 0; d < DT; d++) x.v[d] = *reinterpret_cast<const Chunk*>(at + 16 * CHB * d);
        if constexpr (BITS == 4) x.m = *reinterpret_cast<const v4i*>(vmult + part_of(id) + (uint32_t)slot_of(T));
    };
    int8_t* const sk = sK[w];
    auto turn_k = [&](const Tile& x, Chunk (&k)[4][KC]) {
        __builtin_amdgcn_wave_barrier();  // the last tile's reads are issued; LDS takes a wave's accesses in order
#pragma unroll
        for (int i = 0; i < DT; i++) {
            const int r = (16 * i + l16) / DT, ch = l16 % DT;
            *reinterpret_cast<Chunk*>(sk + (16 * gq + r) * ROWB + (ch ^ pg_swz<HD, BITS>(gq, r)) * CHB) = x.raw[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < KC; c++)
                k[t][c] = *reinterpret_cast<const Chunk*>(sk + (16 * kb + 4 * t + (lane & 3)) * ROWB + ((4 * c + gq) ^ pg_swz<HD, BITS>(kb, lane & 3)) * CHB);
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
    // the negated scores of column group mt: register r of sc[t] is position 16 gq + 4 t + r of the tile
    auto scores = [&](const Chunk (&k)[4][KC], v4i km, int mt, v4i (&sc)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++) sc[t] = mfma16(widen(k[t][c]), q[mt][c], sc[t]);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int r = 0; r < 4; r++)  // -((m (q . c) + 4) >> 3) of -16 (q . c)
                    sc[t][r] = (__mul24(sc[t][r], (km[t] >> (8 * r)) & 255) + 63) >> 7;
            }
        }
    };
    auto sees = [&](int j, int pp) { return (j <= pp) & ((p.window == 0) | (j > pp - p.window) | (j < p.sinks)); };
    // whether every column sees every position of the tile (uniform)
    auto full = [&](int T, bool ok) {
        return __all(ok) && 64 * T + 63 <= pmin && (p.window == 0 || 64 * T > pmax - p.window || 64 * T + 63 < p.sinks);
    };
    auto page_ok = [&](int T, int id) { return (unsigned)id < (unsigned)a.pages && 4 * T + gq < nblk; };

    const int step = p.splits * WP, start = split * WP + wp;
    int low[MT];  // the least negated score of the columns
#pragma unroll
    for (int mt = 0; mt < MT; mt++) low[mt] = INT_MAX;
    // Tiles start, start + step, ... go through a ring of tiles in registers. A tile's page ids are read a round of the ring
    // before its loads are issued, and those a round before they are used: a wave waits for neither.
    const int mine = start < total ? (total - 1 - start) / step + 1 : 0;
    // PG_KEEP: as many of the wave's tiles as the LDS holds keep their scores, a column's 16 bytes at a time (lanes side by
    // side); the others' are formed again from K, last tile first: its K is nearest.
    const int kept = MODE == PG_KEEP ? min(mine, p.keep / (256 * WP * max(cols, 1))) : 0;
    auto kept_place = [&](int n, int t) { return reinterpret_cast<v4i*>(sS) + (((n * WP + wp) * 4 + t) * 4 + gq) * cols + l16; };
    auto keep_at = [&](int n, const v4i (&sc)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) *kept_place(n, t) = sc[t];
    };
    // V's ring over the kept tiles; at hd 64 there are registers to begin it before the maximum is known
    constexpr int NV = MODE == PG_KEEP && HD == 64 ? 4 : 1;
    constexpr bool EARLY = MODE == PG_KEEP && HD == 64;
    VTile xv[NV];
    int idv[NV], nidv[NV];
    auto at = [&](int n) { return tile_at(start + n * step); };
    auto begin_v = [&]() {
#pragma unroll
        for (int u = 0; u < NV; u++) {
            idv[u] = nidv[u] = 0;
            if (u < kept) idv[u] = page_id(at(u)), load_v(at(u), idv[u], xv[u]);
            if (u + NV < kept) nidv[u] = page_id(at(u + NV));
        }
    };
    if constexpr (MAXP) {
        constexpr int NB = WP == 8 ? (HD == 64 ? 4 : 2) : PG_NB1;
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
            if (u < mine) load_k(at(u), id[u], x[u]);
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
                const v4i km = x[u].m;
                if (n + NB < mine) load_k(at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_id(at(n + 2 * NB));
                if (all) {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        v4i sc[4];
                        scores(k, km, mt, sc);
                        if (MODE == PG_KEEP && n < kept && l16 < cols) keep_at(n, sc);
#pragma unroll
                        for (int t = 0; t < 4; t++) low[mt] = min(min(low[mt], min(sc[t].x, sc[t].y)), min(sc[t].z, sc[t].w));
                    }
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (mt >= nmt) break;
                        v4i sc[4];
                        scores(k, km, mt, sc);
                        if (MODE == PG_KEEP && n < kept && l16 < cols) keep_at(n, sc);
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                low[mt] = min(low[mt], ok & sees(64 * T + 16 * gq + 4 * t + r, pos[mt]) ? sc[t][r] : INT_MAX);
                    }
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            low[mt] = min(low[mt], __shfl_xor(low[mt], 16));
            low[mt] = min(low[mt], __shfl_xor(low[mt], 32));
            if (WP > 1 || MODE == PG_MAX)
                if (gq == 0) sLow[wp][wm * CW + 16 * mt + l16] = low[mt];
        }
    }
    const size_t unit = (size_t)tile * a.nkv + g;  // of the workspace's parts
    if constexpr (MODE == PG_SUMS) {  // the splits' least, each column's dealt to threads
        int m = INT_MAX;
        if (tid < NMAX * COLS)
            for (int i = tid / COLS; i < p.splits; i += NMAX) m = min(m, p.wlow[(unit * p.splits + i) * COLS + tid % COLS]);
        if (tid < NMAX * COLS) sLow[tid / COLS][tid % COLS] = m;
    }
    __syncthreads();
    if constexpr (MODE == PG_MAX) {
        for (int c = tid; c < COLS; c += NT) {
            int m = sLow[0][c];
#pragma unroll
            for (int i = 1; i < WP; i++) m = min(m, sLow[i][c]);
            p.wlow[(unit * p.splits + split) * COLS + c] = m;
        }
        // and what the sums are added to starts from zero, each split clearing its share
        for (int i = split * NT + tid; i < COLS * (HD + 1); i += p.splits * NT) p.wsum[unit * (size_t)(COLS * (HD + 1)) + i] = 0;
        if (split == 0 && tid == 0) p.wcnt[unit] = 0;
        return;
    }
    if constexpr (MODE == PG_SUMS || WP > 1) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < (MODE == PG_SUMS ? NMAX : WP); i++) low[mt] = min(low[mt], sLow[i][wm * CW + 16 * mt + l16]);
    }
    if constexpr (SUMP) {
        v4i acc[MT][DT][ND];
        int den[MT][2], top[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            // 2 (max + 64); of a column that sees nothing every weight is masked
            top[mt] = 128 - 2 * (low[mt] == INT_MAX ? 0 : low[mt]);
            den[mt][0] = den[mt][1] = 0;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int n = 0; n < ND; n++) acc[mt][d][n] = v4i{0, 0, 0, 0};
        }
        // The weights' digits as B operands, from y = 2 (max - s + 64): the table index is y >> 8, bytes 1 and 2 of y (|s| is
        // at most 2^21, so y < 2^24 wherever the column sees the position; of other columns any index below 2^16 will do).
        auto weights = [&](auto masked, int T, bool ok, v4i vm, int mt, const v4i (&y)[4], v4i (&P)[ND]) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                uint32_t u[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    u[r] = (uint32_t)y[t][r];
                    if constexpr (masked) u[r] = ok & sees(64 * T + 16 * gq + 4 * t + r, pos[mt]) ? u[r] : 0x00FFFFFFu;
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
                    den[mt][0] = __builtin_amdgcn_sdot4(P[0][t], 0x01010101, den[mt][0], false);
                    den[mt][1] = __builtin_amdgcn_sdot4(P[1][t], 0x01010101, den[mt][1], false);
                } else {
                    uint32_t f[4];
#pragma unroll
                    for (int r = 0; r < 4; r++)  // the balanced digits of e m
                        f[r] = (__umul24((uint32_t)e[r >> 1][r & 1], ((uint32_t)vm[t] >> (8 * r)) & 255) + 0x808080) ^ 0x808080;
                    const uint32_t f01 = __builtin_amdgcn_perm(f[1], f[0], 0x05010400), f23 = __builtin_amdgcn_perm(f[3], f[2], 0x05010400);
                    P[0][t] = (int)__builtin_amdgcn_perm(f23, f01, 0x05040100);
                    P[1][t] = (int)__builtin_amdgcn_perm(f23, f01, 0x07060302);
                    P[ND - 1][t] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(f[3], f[2], 0x0c0c0602), __builtin_amdgcn_perm(f[1], f[0], 0x0c0c0602), 0x05040100);
                    den[mt][0] = (int)__builtin_amdgcn_udot2(e[0], us2{1, 1}, (uint32_t)den[mt][0], false);
                    den[mt][0] = (int)__builtin_amdgcn_udot2(e[1], us2{1, 1}, (uint32_t)den[mt][0], false);
                }
            }
        };
        // y of the negated scores: 2 (-s) + 2 (max + 64); where the products are short, taken twice over on top of the latter.
        auto lift = [&](int mt, const v4i (&sc)[4], v4i (&y)[4]) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) y[t][r] = (int)((uint32_t)sc[t][r] * 2 + (uint32_t)top[mt]);
        };
        auto lifted = [&](const Chunk (&k)[4][KC], v4i km, int mt, v4i (&y)[4]) {
            if constexpr (BITS == 8 && HD == 64) {
                const v4i top4 = {top[mt], top[mt], top[mt], top[mt]};
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    y[t] = top4;
#pragma unroll
                    for (int c = 0; c < 2 * KC; c++) y[t] = mfma16(k[t][c >> 1], q[mt][c >> 1], y[t]);
                }
            } else {
                v4i sc[4];
                scores(k, km, mt, sc);
                lift(mt, sc, y);
            }
        };
        auto add_v = [&](const VTile& x, int mt, const v4i (&P)[ND]) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < ND; e++) acc[mt][d][e] = mfma16(widen(x.v[d]), P[e], acc[mt][d][e]);
        };
        {
            constexpr int NB = WP == 8 && HD == 64 && MODE != PG_KEEP ? 2 : 1;
            Tile x[NB];
            VTile y[NB];
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
                if (u < left) load_k(back(u), id[u], x[u]), load_v(back(u), id[u], y[u]);
            for (int n0 = 0; n0 < left; n0 += NB) {
#pragma unroll
                for (int u = 0; u < NB; u++) {
                    const int n = n0 + u;
                    if (n >= left) break;
                    const int T = back(n);
                    const bool ok = page_ok(T, id[u]), all = full(T, ok);
                    Chunk k[4][KC];
                    turn_k(x[u], k);
                    const v4i km = x[u].m;
                    if (n + NB < left) load_k(back(n + NB), nid[u], x[u]);
                    if (BITS == 8 && MT == 2 && all && nmt == MT) {  // one straight block: a group's lookups under the next one's products
                        v4i sc[MT][4], P[MT][ND];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) lifted(k, km, mt, sc[mt]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) weights(std::false_type(), T, ok, y[u].m, mt, sc[mt], P[mt]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) add_v(y[u], mt, P[mt]);
                    } else {
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            if (mt >= nmt) break;
                            v4i sc[4], P[ND];
                            lifted(k, km, mt, sc);
                            if ((BITS == 4 || MT == 1) && all) weights(std::false_type(), T, ok, y[u].m, mt, sc, P);
                            else weights(std::true_type(), T, ok, y[u].m, mt, sc, P);
                            add_v(y[u], mt, P);
                        }
                    }
                    if (n + NB < left) load_v(back(n + NB), nid[u], y[u]);
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
                    const bool ok = page_ok(T, idv[u]), all = full(T, ok);
                    v4i sc[4] = {}, y[4], P[ND];
                    if (l16 < cols) {
#pragma unroll
                        for (int t = 0; t < 4; t++) sc[t] = *kept_place(n, t);
                    }
                    lift(0, sc, y);
                    if (all) weights(std::false_type(), T, ok, xv[u].m, 0, y, P);
                    else weights(std::true_type(), T, ok, xv[u].m, 0, y, P);
                    add_v(xv[u], 0, P);
                    if (n + NV < kept) load_v(at(n + NV), nidv[u], xv[u]);
                    idv[u] = nidv[u];
                    if (n + 2 * NV < kept) nidv[u] = page_id(at(n + 2 * NV));
                }
            }
        }
        // register r of lane l is dimension 16 d + 4 (l / 16) + r of column l % 16
        auto total_of = [&](int mt, int d, int r) {
            int64_t v = (int64_t)acc[mt][d][0][r] + ((int64_t)acc[mt][d][1][r] << 8);
            if constexpr (BITS == 4) v += (int64_t)acc[mt][d][ND - 1][r] << 16;
            return v;
        };
        auto den_of = [&](int mt) { return BITS == 8 ? (int64_t)den[mt][0] + ((int64_t)den[mt][1] << 8) : (int64_t)den[mt][0]; };
        unsigned long long* const sum = p.wsum + unit * (size_t)(COLS * (HD + 1));
        auto place = [&](int cg, int d, int r, int ln) { return sum + ((cg * DT + d) * 4 + r) * 64 + ln; };
        auto put = [&](int cg, int d, int ln, const int64_t (&v)[4], int64_t dn) {
            const int m = mc + 16 * cg + (ln & 15), i = m / p.rep, r0 = m - i * p.rep, pp = s.p0 + i;
            if (m < mrows)
                pg_store<BITS>(p.o + (size_t)(s.t0 + i) * p.o_stride + (g * p.rep + r0) * HD + 16 * d + 4 * (ln >> 4), v, dn, pp >= 0 && pp < cap);
        };
        // four dimensions of a column (lane ln of 16 columns cg): to the output, or added to the other splits'
        auto give = [&](int cg, int d, int ln, const int64_t (&v)[4], int64_t dn) {
            if constexpr (MODE == PG_SUMS) {
                if (mc + 16 * cg + (ln & 15) < mrows) {
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        (void)__hip_atomic_fetch_add(place(cg, d, r, ln), (unsigned long long)v[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (d == 0 && ln < 16)
                        (void)__hip_atomic_fetch_add(sum + COLS * HD + 16 * cg + ln, (unsigned long long)dn, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            } else {
                put(cg, d, ln, v, dn);
            }
        };
        const int groups = min((mrows - mc + 15) / 16, COLS / 16);
        if constexpr (WP == 1) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if (mt >= nmt) break;
                int64_t dn = den_of(mt);
                dn += __shfl_xor(dn, 16);
                dn += __shfl_xor(dn, 32);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const int64_t v[4] = {total_of(mt, d, 0), total_of(mt, d, 1), total_of(mt, d, 2), total_of(mt, d, 3)};
                    give(wm * MT + mt, d, lane, v, dn);
                }
            }
        } else {
            if (mine > 0) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if (mt >= nmt) break;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            atomicAdd(reinterpret_cast<unsigned long long*>(&sSum[(((wm * MT + mt) * DT + d) * 4 + r) * 64 + lane]),
                                      (unsigned long long)total_of(mt, d, r));
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sDen[wm * CW + 16 * mt + l16]), (unsigned long long)den_of(mt));
                }
            }
            __syncthreads();
            for (int it = tid; it < groups * DT * 64; it += NT) {
                const int cg = it / (DT * 64), d = it / 64 % DT, ln = it & 63;
                int64_t v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = sSum[((cg * DT + d) * 4 + r) * 64 + ln];
                give(cg, d, ln, v, sDen[16 * cg + (ln & 15)]);
            }
        }
        if constexpr (MODE == PG_SUMS) {  // the tile's last CTA has every split's sums
            if (!split_last(p.wcnt + unit)) return;
            for (int it = tid; it < groups * DT * 64; it += NT) {
                const int cg = it / (DT * 64), d = it / 64 % DT, ln = it & 63;
                int64_t v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = (int64_t)__hip_atomic_load(place(cg, d, r, ln), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                put(cg, d, ln, v, (int64_t)__hip_atomic_load(sum + COLS * HD + 16 * cg + (ln & 15), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            }
        }
    }
}

struct Plan {
    int mt, wm, wp, tiles, splits;
};


static int tune(const char* n, int d) { const char* v = getenv(n); return v ? atoi(v) : d; }
Plan plan(int tokens, int seqs, int64_t max_pos, int nh, int nkv, int hd, int bits) {
    const int rep = nh / nkv;
    const int64_t each = ((int64_t)tokens * rep + seqs - 1) / std::max(seqs, 1);
    Plan x;
    if (each <= 16) x.mt = x.wm = 1, x.wp = 8;
    else x.mt = tune("PGT_MT", hd == 64 ? 2 : 1), x.wm = tune("PGT_WM", 4), x.wp = tune("PGT_WP", 2);
    const int64_t cols = 16 * x.mt * x.wm, tiles = (int64_t)tokens * rep / cols + seqs;
    x.tiles = (int)tiles;
    const int64_t ctas = std::min<int64_t>(tiles, tokens) * nkv, work = (max_pos + 63) / 64;
    x.splits = (int)std::max<int64_t>(1, std::min<int64_t>((tune("PGT_CTAS", 512) + ctas - 1) / ctas, work / (2 * x.wp)));
    if (ctas >= 256) x.splits = 1;
    x.splits = tune("PGT_S", x.splits);
    return x;
}

// The workspace's parts: the splits' maxima, the sums, the counts of arrived splits.
struct Parts {
    size_t sum, cnt, bytes;
};

Parts parts(const Plan& x, int nkv, int hd) {
    if (x.splits == 1) return {0, 0, 256};
    const size_t units = (size_t)x.tiles * nkv, cols = 16 * x.mt * x.wm;
    const size_t sum = (units * x.splits * cols * 4 + 255) / 256 * 256, cnt = sum + units * cols * (hd + 1) * 8;
    return {sum, cnt, cnt + (units * 4 + 255) / 256 * 256};
}

template <int HD, int BITS, int MT, int WM, int WP>
hipError_t attend(const Paged& a, PgAttend p, const Plan& x, hipStream_t s) {
    const dim3 grid((unsigned)(x.tiles * a.nkv), (unsigned)x.splits), block(64 * WM * WP);
    if (x.splits == 1) {
        if constexpr (WP == 8) {
            pg_attend_kernel<HD, BITS, MT, WM, WP, PG_KEEP><<<grid, block, (size_t)p.keep, s>>>(a, p);
        } else {
            pg_attend_kernel<HD, BITS, MT, WM, WP, PG_WHOLE><<<grid, block, 0, s>>>(a, p);
        }
        return hipGetLastError();
    }
    pg_attend_kernel<HD, BITS, MT, WM, WP, PG_MAX><<<grid, block, 0, s>>>(a, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    pg_attend_kernel<HD, BITS, MT, WM, WP, PG_SUMS><<<grid, block, 0, s>>>(a, p);
    return hipGetLastError();
}

template <int HD, int BITS>
hipError_t attend_by(const Paged& a, const PgAttend& p, const Plan& x, hipStream_t s) {
    constexpr int MT = HD == 64 ? 2 : 1;
    if (x.wp == 8) return attend<HD, BITS, 1, 1, 8>(a, p, x, s);
    if (x.mt == 1) {
    if (x.wm == 1 && x.wp == 4) return attend<HD, BITS, 1, 1, 4>(a, p, x, s);
    if (x.wm == 2 && x.wp == 2) return attend<HD, BITS, 1, 2, 2>(a, p, x, s);
    if (x.wm == 4 && x.wp == 2) return attend<HD, BITS, 1, 4, 2>(a, p, x, s);
    if (x.wm == 2 && x.wp == 4) return attend<HD, BITS, 1, 2, 4>(a, p, x, s);
    return attend<HD, BITS, 1, 4, 1>(a, p, x, s);
    }
    if (x.wm == 1 && x.wp == 4) return attend<HD, BITS, MT, 1, 4>(a, p, x, s);
    if (x.wm == 2 && x.wp == 2) return attend<HD, BITS, MT, 2, 2>(a, p, x, s);
    return attend<HD, BITS, MT, 4, 1>(a, p, x, s);
}

}  // namespace

// bits is not known here: the layout's larger need
size_t pg_attend_workspace(int tokens, int seqs, int64_t max_pos, int nh, int nkv, int hd) {
    return std::max(parts(plan(tokens, seqs, max_pos, nh, nkv, hd, 8), nkv, hd).bytes,
                    parts(plan(tokens, seqs, max_pos, nh, nkv, hd, 4), nkv, hd).bytes);
}

hipError_t launch_pg_attend(const Paged& a, int hd, int bits, const int8_t* q, int64_t q_stride, int nh,
                            const int32_t* exp_tab, int window, int sinks, int8_t* o, int64_t o_stride, void* ws,
                            hipStream_t s) {
    const int64_t max_pos = (int64_t)a.max_pages << a.page_sh;
    const Plan x = plan(a.tokens, a.seqs, max_pos, nh, a.nkv, hd, bits);
    const Parts w = parts(x, a.nkv, hd);
    const int rep = nh / a.nkv, cols = a.tokens > a.seqs ? 16 : std::min(rep, 16);
    // kept scores: 256 bytes a column and tile, as far as a CTA's LDS (160 KB) goes beside its static arrays
    const int64_t room = 163840 - 12288 - 8 * 64 * (bits == 8 ? hd : hd / 2) - hd * 128;
    const int64_t keep = std::min<int64_t>((max_pos / 64 + x.wp) / x.wp * x.wp * cols * 256, tune("PGT_KEEP", (int)room));
    const PgAttend p = {q, o, q_stride, o_stride, exp_tab, rep, window, sinks, x.splits, (int)keep, (int32_t*)ws,
                        (unsigned long long*)((char*)ws + w.sum), (unsigned*)((char*)ws + w.cnt)};
    if (hd == 64) return bits == 8 ? attend_by<64, 8>(a, p, x, s) : attend_by<64, 4>(a, p, x, s);
    return bits == 8 ? attend_by<128, 8>(a, p, x, s) : attend_by<128, 4>(a, p, x, s);
}

}  // namespace kt
