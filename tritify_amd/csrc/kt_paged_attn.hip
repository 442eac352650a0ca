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

struct PgAttend {
    const int8_t* q;
    int8_t* o;
    int64_t q_stride, o_stride;
    const int32_t* exp_tab;
    int rep, window, sinks, splits;
    int32_t* wmax;   // [tile][kv head][split][column]
    int64_t* wsum;   // [tile][kv head][split][column group, 16 dimensions][register][lane], then the weights' sums
};

enum { PG_WHOLE = 0, PG_MAX = 1, PG_SUMS = 2 };

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
struct PgTile {
    typedef typename PgChunk<BITS>::T Chunk;
    Chunk raw[HD / 16], v[HD / 16];
    v4i km, vm;  // 4 bits: the multipliers of block l / 16
};

// The swizzle of a row's chunks in the wave's LDS (row r of block n), by which the lanes that one LDS cycle serves (8 of 16
// bytes, 16 of 8: rows 4 t .. 4 t + 3 of two or four blocks) read different banks.
template <int HD, int BITS>
__device__ __forceinline__ int pg_swz(int n, int r) {
    if constexpr (BITS == 8) return HD == 64 ? ((r >> 1) & 1) | ((n & 1) << 1) : (r & 3) | ((n & 1) << 2);
    else return HD == 64 ? n : ((r >> 1) & 1) | (n << 1);
}

// Four neighbouring dimensions of an output row: clamp(round_half_away(sum e v / sum e)) of what the digits add up to (8
// bits: both negated; 4 bits: v as 16 codes times 1/8 of a multiplier), zeros where nothing was seen.
template <int BITS>
__device__ __forceinline__ void pg_store(int8_t* to, const int64_t (&v)[4], int64_t dn, bool live) {
    dn = BITS == 8 ? -dn : 128 * dn;
    uint32_t out = 0;
    if (live && dn > 0)
#pragma unroll
        for (int r = 0; r < 4; r++) out |= (uint32_t)(uint8_t)div_round_q8(BITS == 8 ? -v[r] : v[r], dn) << (8 * r);
    *reinterpret_cast<uint32_t*>(to) = out;
}

template <int HD, int BITS, int MT, int WM, int WP, int MODE>
__global__ __launch_bounds__(64 * WM * WP) void pg_attend_kernel(Paged a, PgAttend p) {
    constexpr int HH = HD / 2, KC = HD / 64, DT = HD / 16, ND = BITS == 8 ? 2 : 3;
    constexpr int W = WM * WP, NT = 64 * W, CW = 16 * MT, COLS = CW * WM;  // threads; columns of a wave and of the CTA
    constexpr int NMAX = COLS * WP > NT ? WP : NT / COLS;
    constexpr int ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;  // bytes of a K row of a slot, of a chunk
    typedef PgTile<HD, BITS> Tile;
    typedef typename Tile::Chunk Chunk;
    constexpr bool MAXP = MODE != PG_SUMS, SUMP = MODE != PG_MAX;
    __shared__ int64_t sSum[SUMP && WP > 1 ? WM * MT * DT * 4 * 64 : 1];
    __shared__ int64_t sDen[SUMP ? COLS : 1];
    __shared__ int sMax[NMAX][COLS];
    __shared__ uint16_t sE[1026];
    __shared__ __attribute__((aligned(16))) int8_t sK[W][64 * ROWB];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = w / WP, wp = w % WP, l16 = lane & 15, gq = lane >> 4, kb = (lane >> 2) & 3;
    const int split = (int)blockIdx.y;
    int et[(1024 + NT - 1) / NT];
    if constexpr (SUMP) {  // the table is on its way while the batch is looked up
#pragma unroll
        for (int i = 0; i < (1024 + NT - 1) / NT; i++) et[i] = p.exp_tab[min(tid + i * NT, 1023)];
    }
    // the kv head fastest: CTAs go to the XCDs in turn, so an XCD's L2 holds the heads congruent to it
    const int tile = (int)(gridDim.x / a.nkv) - 1 - (int)blockIdx.x / a.nkv, g = (int)blockIdx.x % a.nkv;
    int first = 0;
    const int b = pg_tile_seq(a, tile, p.rep, COLS, 1, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int mc = (tile - first) * COLS, mrows = s.n * p.rep;  // m: row i, head r of the group as i rep + r
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

    const uint8_t *const kbase = a.k + (size_t)g * a.part + l16 * CHB, *const vbase = a.v + (size_t)g * a.part + l16 * CHB;
    const uint8_t *const kmult = a.k + (size_t)g * a.part + (HH << a.page_sh), *const vmult = a.v + (size_t)g * a.part + (HH << a.page_sh);

    // the columns' rows and positions, and their q as B operands
    int pos[MT];
    v4i q[MT][KC];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int m = min(m0 + 16 * mt + l16, mrows - 1), i = m / p.rep, r = m - i * p.rep;
        pos[mt] = 16 * mt + l16 < cols && s.p0 + i < cap ? s.p0 + i : -1;
        const int8_t* qr = p.q + (size_t)(s.t0 + i) * p.q_stride + (g * p.rep + r) * HD + 16 * gq;
#pragma unroll
        for (int c = 0; c < KC; c++) q[mt][c] = *reinterpret_cast<const v4i*>(qr + 64 * c);
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
        const uint8_t* at = kbase + part_of(id) + (uint32_t)(slot_of(T) * ROWB);
#pragma unroll
        for (int i = 0; i < DT; i++) x.raw[i] = *reinterpret_cast<const Chunk*>(at + 16 * CHB * i);
        if constexpr (BITS == 4) x.km = *reinterpret_cast<const v4i*>(kmult + part_of(id) + (uint32_t)slot_of(T));
    };
    auto load_v = [&](int T, int id, Tile& x) {
        const uint8_t* at = vbase + part_of(id) + (uint32_t)(slot_of(T) * ROWB);
#pragma unroll
        for (int d = 0; d < DT; d++) x.v[d] = *reinterpret_cast<const Chunk*>(at + 16 * CHB * d);
        if constexpr (BITS == 4) x.vm = *reinterpret_cast<const v4i*>(vmult + part_of(id) + (uint32_t)slot_of(T));
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
    // the scores of column group mt: register r of s[t] is position 16 gq + 4 t + r of the tile
    auto scores = [&](const Chunk (&k)[4][KC], v4i km, int mt, v4i (&sc)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++) sc[t] = mfma16(widen(k[t][c]), q[mt][c], sc[t]);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int r = 0; r < 4; r++)  // (m (q . c) + 4) >> 3 of 16 (q . c)
                    sc[t][r] = (__mul24(sc[t][r], (km[t] >> (8 * r)) & 255) + 64) >> 7;
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
    int mx[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) mx[mt] = INT_MIN;
    // Tiles start, start + step, ... go through a ring of tiles in registers. A tile's page ids are read a round of the ring
    // before its loads are issued, and those a round before they are used: a wave waits for neither.
    const int mine = start < total ? (total - 1 - start) / step + 1 : 0;
    if constexpr (MAXP) {
        constexpr int NB = MT * HD <= 64 ? 4 : 2;
        Tile x[NB];
        int id[NB], nid[NB];
        auto at = [&](int n) { return tile_at(start + n * step); };
#pragma unroll
        for (int u = 0; u < NB; u++) {
            id[u] = nid[u] = 0;
            if (u < mine) id[u] = page_id(at(u));
            if (u + NB < mine) nid[u] = page_id(at(u + NB));
        }
#pragma unroll
        for (int u = 0; u < NB; u++)
            if (u < mine) load_k(at(u), id[u], x[u]);
        for (int n0 = 0; n0 < mine; n0 += NB) {
#pragma unroll
            for (int u = 0; u < NB; u++) {
                const int n = n0 + u;
                if (n >= mine) break;
                const int T = at(n);
                const bool ok = page_ok(T, id[u]), all = full(T, ok);
                Chunk k[4][KC];
                turn_k(x[u], k);
                const v4i km = x[u].km;
                if (n + NB < mine) load_k(at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_id(at(n + 2 * NB));
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if (mt >= nmt) break;
                    v4i sc[4];
                    scores(k, km, mt, sc);
                    if (all) {
#pragma unroll
                        for (int t = 0; t < 4; t++) mx[mt] = max(max(mx[mt], max(sc[t].x, sc[t].y)), max(sc[t].z, sc[t].w));
                    } else {
                        asm volatile("");  // keeps the masks out of the other tiles' path
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                mx[mt] = max(mx[mt], ok & sees(64 * T + 16 * gq + 4 * t + r, pos[mt]) ? sc[t][r] : INT_MIN);
                    }
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            mx[mt] = max(mx[mt], __shfl_xor(mx[mt], 16));
            mx[mt] = max(mx[mt], __shfl_xor(mx[mt], 32));
            if (WP > 1 || MODE == PG_MAX)
                if (gq == 0) sMax[wp][wm * CW + 16 * mt + l16] = mx[mt];
        }
    }
    const size_t unit = ((size_t)tile * a.nkv + g) * p.splits;  // of the workspace's parts
    if constexpr (MODE == PG_SUMS) {  // the splits' maxima, each column's dealt to threads
        int m = INT_MIN;
        if (tid < NMAX * COLS)
            for (int i = tid / COLS; i < p.splits; i += NMAX) m = max(m, p.wmax[(unit + i) * COLS + tid % COLS]);
        if (tid < NMAX * COLS) sMax[tid / COLS][tid % COLS] = m;
    }
    __syncthreads();
    if constexpr (MODE == PG_MAX) {
        for (int c = tid; c < COLS; c += NT) {
            int m = sMax[0][c];
#pragma unroll
            for (int i = 1; i < WP; i++) m = max(m, sMax[i][c]);
            p.wmax[(unit + split) * COLS + c] = m;
        }
        return;
    }
    if constexpr (MODE == PG_SUMS || WP > 1) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < (MODE == PG_SUMS ? NMAX : WP); i++) mx[mt] = max(mx[mt], sMax[i][wm * CW + 16 * mt + l16]);
    }
    if constexpr (SUMP) {
        v4i acc[MT][DT][ND];
        int den[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            mx[mt] = (mx[mt] == INT_MIN ? 0 : mx[mt]) + 64;  // of a column that sees nothing every weight is masked
            den[mt][0] = den[mt][1] = 0;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int n = 0; n < ND; n++) acc[mt][d][n] = v4i{0, 0, 0, 0};
        }
        constexpr int NB = MT * HD <= 64 ? 2 : 1;
        Tile x[NB];
        int id[NB], nid[NB];
        auto at = [&](int n) { return tile_at(start + (mine - 1 - n) * step); };  // from the end: its K is nearest
#pragma unroll
        for (int u = 0; u < NB; u++) {
            id[u] = nid[u] = 0;
            if (u < mine) id[u] = page_id(at(u));
            if (u + NB < mine) nid[u] = page_id(at(u + NB));
        }
#pragma unroll
        for (int u = 0; u < NB; u++)
            if (u < mine) load_k(at(u), id[u], x[u]), load_v(at(u), id[u], x[u]);
        for (int n0 = 0; n0 < mine; n0 += NB) {
#pragma unroll
            for (int u = 0; u < NB; u++) {
                const int n = n0 + u;
                if (n >= mine) break;
                const int T = at(n);
                const bool ok = page_ok(T, id[u]), all = full(T, ok);
                Chunk k[4][KC];
                turn_k(x[u], k);
                const v4i km = x[u].km, vm = x[u].vm;
                if (n + NB < mine) load_k(at(n + NB), nid[u], x[u]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if (mt >= nmt) break;
                    v4i sc[4], P[ND];
                    scores(k, km, mt, sc);
                    auto weights = [&](auto masked) {
                        if constexpr (masked) asm volatile("");  // keeps the masks out of the other tiles' path
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            uint32_t e[4];
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                uint32_t ix = min((uint32_t)(mx[mt] - sc[t][r]) >> 7, 1024u);
                                if constexpr (masked) ix = ok & sees(64 * T + 16 * gq + 4 * t + r, pos[mt]) ? ix : 1024u;
                                e[r] = sE[ix];
                                if constexpr (BITS == 4) {  // the digits of e m
                                    den[mt][0] += (int)e[r];
                                    e[r] = (__umul24(e[r], ((uint32_t)vm[t] >> (8 * r)) & 255) + 0x808080) ^ 0x808080;
                                }
                            }
                            const uint32_t e01 = __builtin_amdgcn_perm(e[1], e[0], 0x05010400), e23 = __builtin_amdgcn_perm(e[3], e[2], 0x05010400);
                            P[0][t] = (int)__builtin_amdgcn_perm(e23, e01, 0x05040100);
                            P[1][t] = (int)__builtin_amdgcn_perm(e23, e01, 0x07060302);
                            if constexpr (BITS == 4)
                                P[ND - 1][t] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(e[3], e[2], 0x0c0c0602), __builtin_amdgcn_perm(e[1], e[0], 0x0c0c0602), 0x05040100);
                            if constexpr (BITS == 8) {
                                den[mt][0] = __builtin_amdgcn_sdot4(P[0][t], 0x01010101, den[mt][0], false);
                                den[mt][1] = __builtin_amdgcn_sdot4(P[1][t], 0x01010101, den[mt][1], false);
                            }
                        }
                    };
                    if (all) weights(std::false_type());
                    else weights(std::true_type());
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < ND; e++)
                            acc[mt][d][e] = mfma16(widen(x[u].v[d]), P[e], acc[mt][d][e]);
                }
                if (n + NB < mine) load_v(at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_id(at(n + 2 * NB));
            }
        }
        // register r of lane l is dimension 16 d + 4 (l / 16) + r of column l % 16
        auto total_of = [&](int mt, int d, int r) {
            int64_t v = (int64_t)acc[mt][d][0][r] + ((int64_t)acc[mt][d][1][r] << 8);
            if constexpr (BITS == 4) v += (int64_t)acc[mt][d][ND - 1][r] << 16;
            return v;
        };
        auto den_of = [&](int mt) { return BITS == 8 ? (int64_t)den[mt][0] + ((int64_t)den[mt][1] << 8) : (int64_t)den[mt][0]; };
        int64_t* const to = p.wsum + ((unit + split) * WM) * (size_t)(CW * (HD + 1));
        // four dimensions of column c of wave group gm: to the output, or to this split's part of the workspace
        auto give = [&](int gm, int mt, int d, int ln, const int64_t (&v)[4], int64_t dn) {
            const int c = 16 * mt + (ln & 15), m = mc + gm * CW + c;
            if constexpr (MODE == PG_SUMS) {
                int64_t* x = to + (size_t)gm * (CW * (HD + 1));
#pragma unroll
                for (int r = 0; r < 4; r++) x[((mt * DT + d) * 4 + r) * 64 + ln] = v[r];
                if (d == 0 && ln < 16) x[CW * HD + c] = dn;
            } else if (m < mrows) {
                const int i = m / p.rep, r0 = m - i * p.rep, pp = s.p0 + i;
                pg_store<BITS>(p.o + (size_t)(s.t0 + i) * p.o_stride + (g * p.rep + r0) * HD + 16 * d + 4 * (ln >> 4), v, dn, pp >= 0 && pp < cap);
            }
        };
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
                    give(wm, mt, d, lane, v, dn);
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
            const int groups = min((mrows - mc + 15) / 16, COLS / 16);
            for (int it = tid; it < groups * DT * 64; it += NT) {
                const int cg = it / (DT * 64), d = it / 64 % DT, ln = it & 63;
                int64_t v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = sSum[((cg * DT + d) * 4 + r) * 64 + ln];
                give(cg / MT, cg % MT, d, ln, v, sDen[16 * cg + (ln & 15)]);
            }
        }
    }
}

// The splits' sums joined: one CTA per (tile, kv head, 16 columns, 16 dimensions), the splits dealt to its waves.
template <int HD, int BITS, int MT, int WM>
__global__ __launch_bounds__(512) void pg_join_kernel(Paged a, PgAttend p) {
    constexpr int CW = 16 * MT, COLS = CW * WM, DT = HD / 16;
    __shared__ int64_t sV[8][5][64];
    const int tile = (int)blockIdx.x / a.nkv, g = (int)blockIdx.x % a.nkv, cg = blockIdx.y, d = blockIdx.z;
    const int lane = threadIdx.x & 63, share = threadIdx.x >> 6, shares = blockDim.x >> 6;
    int first = 0;
    const int b = pg_tile_seq(a, tile, p.rep, COLS, 1, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int m = (tile - first) * COLS + 16 * cg + (lane & 15), mrows = s.n * p.rep;
    if (m - (lane & 15) >= mrows) return;
    const size_t part = CW * (HD + 1);
    const int64_t* from = p.wsum + (((size_t)tile * a.nkv + g) * p.splits * WM + cg / MT) * part;
    int64_t v[4] = {0, 0, 0, 0}, dn = 0;
    if (m < mrows) {
#pragma unroll 8
        for (int i = share; i < p.splits; i += shares) {
            const int64_t* x = from + (size_t)i * (WM * part);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] += x[(((cg % MT) * DT + d) * 4 + r) * 64 + lane];
            dn += x[CW * HD + 16 * (cg % MT) + (lane & 15)];
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sV[share][r][lane] = v[r];
    sV[share][4][lane] = dn;
    __syncthreads();
    if (share || m >= mrows) return;
    for (int k = 1; k < shares; k++) {
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] += sV[k][r][lane];
        dn += sV[k][4][lane];
    }
    const int i = m / p.rep, r0 = m - i * p.rep, pp = s.p0 + i;
    pg_store<BITS>(p.o + (size_t)(s.t0 + i) * p.o_stride + (g * p.rep + r0) * HD + 16 * d + 4 * (lane >> 4), v, dn,
                   pp >= 0 && pp < a.max_pages << a.page_sh);
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
    else x.mt = hd == 64 ? 2 : 1, x.wm = tune("PGT_WM", 4), x.wp = 8 / x.wm;
    const int64_t cols = 16 * x.mt * x.wm, tiles = (int64_t)tokens * rep / cols + seqs;
    x.tiles = (int)tiles;
    const int64_t ctas = std::min<int64_t>(tiles, tokens) * nkv, work = (max_pos + 63) / 64;
    x.splits = (int)std::max<int64_t>(1, std::min<int64_t>((tune("PGT_CTAS", 512) + ctas - 1) / ctas, work / (2 * x.wp)));
    if (ctas >= 256) x.splits = 1;
    x.splits = tune("PGT_S", x.splits);
    return x;
}

size_t ws_max_bytes(const Plan& x, int nkv) {
    return ((size_t)x.tiles * nkv * x.splits * 16 * x.mt * x.wm * 4 + 255) / 256 * 256;
}

size_t ws_bytes(const Plan& x, int nkv, int hd) {
    if (x.splits == 1) return 256;
    return ws_max_bytes(x, nkv) + (size_t)x.tiles * nkv * x.splits * 16 * x.mt * x.wm * (hd + 1) * 8;
}

template <int HD, int BITS, int MT, int WM, int WP>
hipError_t attend(const Paged& a, const PgAttend& p, const Plan& x, hipStream_t s) {
    const dim3 grid((unsigned)(x.tiles * a.nkv), (unsigned)x.splits), block(64 * WM * WP);
    if (x.splits == 1) {
        pg_attend_kernel<HD, BITS, MT, WM, WP, PG_WHOLE><<<grid, block, 0, s>>>(a, p);
        return hipGetLastError();
    }
    pg_attend_kernel<HD, BITS, MT, WM, WP, PG_MAX><<<grid, block, 0, s>>>(a, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    pg_attend_kernel<HD, BITS, MT, WM, WP, PG_SUMS><<<grid, block, 0, s>>>(a, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    int shares = 1;
    while (shares < 8 && 2 * shares <= x.splits) shares *= 2;
    pg_join_kernel<HD, BITS, MT, WM><<<dim3((unsigned)(x.tiles * a.nkv), MT * WM, HD / 16), dim3(64 * shares), 0, s>>>(a, p);
    return hipGetLastError();
}

template <int HD, int BITS>
hipError_t attend_by(const Paged& a, const PgAttend& p, const Plan& x, hipStream_t s) {
    constexpr int MT = HD == 64 ? 2 : 1;
    if (x.mt == 1 && x.wm == 1) return attend<HD, BITS, 1, 1, 8>(a, p, x, s);
    if (x.wm == 1) return attend<HD, BITS, MT, 1, 8>(a, p, x, s);
    if (x.wm == 2) return attend<HD, BITS, MT, 2, 4>(a, p, x, s);
    if (x.wm == 4) return attend<HD, BITS, MT, 4, 2>(a, p, x, s);
    return attend<HD, BITS, MT, 8, 1>(a, p, x, s);
}

}  // namespace

// bits is not known here: the layout's larger need
size_t pg_attend_workspace(int tokens, int seqs, int64_t max_pos, int nh, int nkv, int hd) {
    return std::max(ws_bytes(plan(tokens, seqs, max_pos, nh, nkv, hd, 8), nkv, hd),
                    ws_bytes(plan(tokens, seqs, max_pos, nh, nkv, hd, 4), nkv, hd));
}

hipError_t launch_pg_attend(const Paged& a, int hd, int bits, const int8_t* q, int64_t q_stride, int nh,
                            const int32_t* exp_tab, int window, int sinks, int8_t* o, int64_t o_stride, void* ws,
                            hipStream_t s) {
    const Plan x = plan(a.tokens, a.seqs, (int64_t)a.max_pages << a.page_sh, nh, a.nkv, hd, bits);
    const PgAttend p = {q, o, q_stride, o_stride, exp_tab, nh / a.nkv, window, sinks, x.splits, (int32_t*)ws,
                        (int64_t*)((char*)ws + ws_max_bytes(x, a.nkv))};
    if (hd == 64) return bits == 8 ? attend_by<64, 8>(a, p, x, s) : attend_by<64, 4>(a, p, x, s);
    return bits == 8 ? attend_by<128, 8>(a, p, x, s) : attend_by<128, 4>(a, p, x, s);
}

}  // namespace kt
