// Attention of a ragged batch's new rows over paged KV caches on gfx950 (kt_hip_dec_attention_paged, stated in
// include/kt_hip.h): chunks, whole prompts and single tokens by one kernel.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

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

constexpr int PG_W = 8;  // waves of a CTA
enum { PG_WHOLE = 0, PG_MAX = 1, PG_SUMS = 2 };

// What a wave holds of 64 positions (four blocks of 16) of one kv head. K: lane l has dimensions 16 (l / 16) .. of 64 from
// position 16 (l / 4 % 4) + 4 t + l % 4 in k[t][.]: as the A operand of a 16x16x64 product its 16 rows give lane l the
// scores of positions 16 (l / 16) + 4 t + r in register r. So a lane's 16 scores of the four products are one block's 16
// positions in order, which is the layout of a B operand of the product with V, whose chunks (16 positions of a dimension)
// are loaded as they stand.
template <int HD, int BITS>
struct PgTile {
    v4i k[4][HD / 64];
    v4i v[HD / 16];
    v4i km, vm;
};

template <int HD, int BITS, int MT, int W, int MODE>
__global__ __launch_bounds__(64 * W) void pg_attend_kernel(Paged a, PgAttend p) {
    constexpr int HH = HD / 2, KC = HD / 64, DT = HD / 16, ND = BITS == 8 ? 2 : 3, COLS = 16 * MT;
    constexpr int ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;
    constexpr bool MAXP = MODE != PG_SUMS, SUMP = MODE != PG_MAX;
    __shared__ int64_t sSum[SUMP ? MT * DT * 4 * 64 : 1];
    __shared__ int64_t sDen[COLS];
    __shared__ int sMax[W][COLS];
    __shared__ uint16_t sE[1026];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, gq = lane >> 4, kb = (lane >> 2) & 3;
    const int split = (int)blockIdx.y;
    // the kv head fastest: CTAs go to the XCDs in turn, so an XCD's L2 holds the heads congruent to it
    const int tile = (int)(gridDim.x / a.nkv) - 1 - (int)blockIdx.x / a.nkv, g = (int)blockIdx.x % a.nkv;
    int first = 0;
    const int b = pg_tile_seq(a, tile, p.rep, COLS, 1, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int m0 = (tile - first) * COLS, mrows = s.n * p.rep;  // m: row i, head r of the group as i rep + r
    if (m0 >= mrows) return;
    const int cols = min(COLS, mrows - m0), nmt = (cols + 15) / 16;
    const int cap = a.max_pages << a.page_sh, nblk = cap >> 4;
    const int pmin = s.p0 + m0 / p.rep, pmax = min(s.p0 + (m0 + cols - 1) / p.rep, cap - 1);
    // the tiles of 64 positions: those of the sinks, then those of the window
    const int ntile = pmax < 0 || a.pages == 0 ? 0 : pmax / 64 + 1;
    int nsink = 0, w0 = 0;
    if (p.window) {
        nsink = min((min(p.sinks, pmax + 1) + 63) / 64, ntile);
        w0 = max(nsink, (max(pmin, 0) - min(p.window - 1, max(pmin, 0))) / 64);
    }
    const int total = nsink + max(0, ntile - w0);
    auto tile_at = [&](int i) { return i < nsink ? i : i - nsink + w0; };

    if constexpr (SUMP) {
        for (int i = tid; i < 1025; i += 64 * W) {
            const int e = i < 1024 ? min(max(p.exp_tab[i], 0), 32768) : 0;
            // 8 bits: the two balanced base-256 digits of -e (2^15 itself has none, -2^15 does); 4 bits: e
            sE[i] = BITS == 8 ? (uint16_t)((0x8080 - e) ^ 0x8080) : (uint16_t)e;
        }
        for (int i = tid; i < MT * DT * 4 * 64; i += 64 * W) sSum[i] = 0;
        if (tid < COLS) sDen[tid] = 0;
    }

    // the columns' rows and positions, and their q as B operands
    int pos[MT];
    v4i q[MT][KC];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int m = m0 + min(16 * mt + l16, cols - 1), i = m / p.rep, r = m - i * p.rep;
        pos[mt] = 16 * mt + l16 < cols && s.p0 + i < cap ? s.p0 + i : -1;
        const int8_t* qr = p.q + (size_t)(s.t0 + i) * p.q_stride + (g * p.rep + r) * HD + 16 * gq;
#pragma unroll
        for (int c = 0; c < KC; c++) q[mt][c] = *reinterpret_cast<const v4i*>(qr + 64 * c);
    }

    // page ids of the tile's blocks kb (K) and gq (V and the multipliers)
    struct Ids {
        int k, v;
    };
    auto page_ids = [&](int T) {
        const int bk = min(4 * T + kb, nblk - 1), bv = min(4 * T + gq, nblk - 1);
        const int32_t* tab = a.table + (size_t)b * a.max_pages;
        return Ids{tab[bk >> (a.page_sh - 4)], tab[bv >> (a.page_sh - 4)]};
    };
    auto slot_of = [&](int blk) { return (blk << 4) & ((1 << a.page_sh) - 1); };
    auto part_of = [&](int id) { return ((size_t)((unsigned)id < (unsigned)a.pages ? id : 0) * a.nkv + g) * (size_t)a.part; };
    auto load_k = [&](int T, Ids id, PgTile<HD, BITS>& x) {
        const uint8_t* at = a.k + part_of(id.k) + (size_t)((slot_of(min(4 * T + kb, nblk - 1)) + (lane & 3)) * ROWB + gq * CHB);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < KC; c++) {
                if constexpr (BITS == 8) {
                    x.k[t][c] = *reinterpret_cast<const v4i*>(at + 4 * t * ROWB + 64 * c);
                } else {
                    const v2i y = *reinterpret_cast<const v2i*>(at + 4 * t * ROWB + 32 * c);
                    x.k[t][c].x = y.x, x.k[t][c].y = y.y;
                }
            }
        if constexpr (BITS == 4)
            x.km = *reinterpret_cast<const v4i*>(a.k + part_of(id.v) + (size_t)((HH << a.page_sh) + slot_of(min(4 * T + gq, nblk - 1))));
    };
    auto load_v = [&](int T, Ids id, PgTile<HD, BITS>& x) {
        const int slot = slot_of(min(4 * T + gq, nblk - 1));
        const uint8_t* at = a.v + part_of(id.v) + (size_t)(slot * ROWB + l16 * CHB);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if constexpr (BITS == 8) {
                x.v[d] = *reinterpret_cast<const v4i*>(at + 16 * CHB * d);
            } else {
                const v2i y = *reinterpret_cast<const v2i*>(at + 16 * CHB * d);
                x.v[d].x = y.x, x.v[d].y = y.y;
            }
        }
        if constexpr (BITS == 4)
            x.vm = *reinterpret_cast<const v4i*>(a.v + part_of(id.v) + (size_t)((HH << a.page_sh) + slot));
    };
    // 4 bits: 16 times the 16 codes of a chunk, in order (byte 4 h + r: code 8 h + r low, code 8 h + 4 + r high)
    auto widen = [](v4i x) {
        constexpr int M = (int)0xF0F0F0F0;
        return v4i{(x.x << 4) & M, x.x & M, (x.y << 4) & M, x.y & M};
    };
    // the scores of column group mt: register r of s[t] is position 16 gq + 4 t + r of the tile
    auto scores = [&](const PgTile<HD, BITS>& x, int mt, v4i (&sc)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++) sc[t] = mfma16(BITS == 8 ? x.k[t][c] : widen(x.k[t][c]), q[mt][c], sc[t]);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int r = 0; r < 4; r++)  // (m (q . c) + 4) >> 3 of 16 (q . c)
                    sc[t][r] = (__mul24(sc[t][r], (x.km[t] >> (8 * r)) & 255) + 64) >> 7;
            }
        }
    };
    auto sees = [&](int j, int pp) { return j <= pp && (p.window == 0 || j > pp - p.window || j < p.sinks); };
    // whether every column sees every position of the tile (uniform)
    auto full = [&](int T, bool ok) {
        return __all(ok) && 64 * T + 63 <= pmin && (p.window == 0 || 64 * T > pmax - p.window || 64 * T + 63 < p.sinks);
    };
    auto page_ok = [&](int T, Ids id) { return (unsigned)id.v < (unsigned)a.pages && 4 * T + gq < nblk; };

    const int step = p.splits * W, start = split * W + w;
    int mx[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) mx[mt] = INT_MIN;
    // Tiles start, start + step, ... go through a ring of tiles in registers. A tile's page ids are read a round of the ring
    // before its loads are issued, and those a round before they are used: a wave waits for neither.
    const int mine = start < total ? (total - 1 - start) / step + 1 : 0;
    if constexpr (MAXP) {
        constexpr int NB = MT == 1 ? 4 : 2;
        PgTile<HD, BITS> x[NB];
        Ids id[NB], nid[NB];
        auto at = [&](int n) { return tile_at(start + n * step); };
#pragma unroll
        for (int u = 0; u < NB; u++) {
            id[u] = nid[u] = Ids{0, 0};
            if (u < mine) id[u] = page_ids(at(u));
            if (u + NB < mine) nid[u] = page_ids(at(u + NB));
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
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if (mt >= nmt) break;
                    v4i sc[4];
                    scores(x[u], mt, sc);
                    if (all) {
#pragma unroll
                        for (int t = 0; t < 4; t++) mx[mt] = max(max(mx[mt], max(sc[t].x, sc[t].y)), max(sc[t].z, sc[t].w));
                    } else {
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (ok && sees(64 * T + 16 * gq + 4 * t + r, pos[mt])) mx[mt] = max(mx[mt], sc[t][r]);
                    }
                }
                if (n + NB < mine) load_k(at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_ids(at(n + 2 * NB));
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            mx[mt] = max(mx[mt], __shfl_xor(mx[mt], 16));
            mx[mt] = max(mx[mt], __shfl_xor(mx[mt], 32));
            if (gq == 0) sMax[w][16 * mt + l16] = mx[mt];
        }
    }
    __syncthreads();
    const size_t unit = ((size_t)tile * a.nkv + g) * p.splits;  // of the workspace's parts
    if constexpr (MODE == PG_MAX) {
        if (tid < COLS) {
            int m = sMax[0][tid];
#pragma unroll
            for (int i = 1; i < W; i++) m = max(m, sMax[i][tid]);
            p.wmax[(unit + split) * COLS + tid] = m;
        }
        return;
    }
    if constexpr (MODE == PG_WHOLE) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < W; i++) mx[mt] = max(mx[mt], sMax[i][16 * mt + l16]);
    }
    if constexpr (MODE == PG_SUMS) {
        for (int i = 0; i < p.splits; i++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) mx[mt] = max(mx[mt], p.wmax[(unit + i) * COLS + 16 * mt + l16]);
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
        constexpr int NB = MT == 1 ? 2 : 1;
        PgTile<HD, BITS> x[NB];
        Ids id[NB], nid[NB];
        auto at = [&](int n) { return tile_at(start + (mine - 1 - n) * step); };  // from the end: its K is nearest
#pragma unroll
        for (int u = 0; u < NB; u++) {
            id[u] = nid[u] = Ids{0, 0};
            if (u < mine) id[u] = page_ids(at(u));
            if (u + NB < mine) nid[u] = page_ids(at(u + NB));
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
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    if (mt >= nmt) break;
                    v4i sc[4], P[ND];
                    scores(x[u], mt, sc);
                    const v4i vm = x[u].vm;
                    if (mt == nmt - 1 && n + NB < mine) load_k(at(n + NB), nid[u], x[u]);
                    auto weights = [&](bool masked) {
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            uint32_t e[4];
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                uint32_t ix = min((uint32_t)(mx[mt] - sc[t][r]) >> 7, 1024u);
                                if (masked) ix = ok && sees(64 * T + 16 * gq + 4 * t + r, pos[mt]) ? ix : 1024u;
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
                    if (all) weights(false);
                    else weights(true);
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int k = 0; k < ND; k++)
                            acc[mt][d][k] = mfma16(BITS == 8 ? x[u].v[d] : widen(x[u].v[d]), P[k], acc[mt][d][k]);
                }
                if (n + NB < mine) load_v(at(n + NB), nid[u], x[u]);
                id[u] = nid[u];
                if (n + 2 * NB < mine) nid[u] = page_ids(at(n + 2 * NB));
            }
        }
        // the waves' sums: register r of lane l is dimension 16 d + 4 (l / 16) + r of column l % 16
        if (start < total) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if (mt >= nmt) break;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        int64_t v = (int64_t)acc[mt][d][0][r] + ((int64_t)acc[mt][d][1][r] << 8);
                        if constexpr (BITS == 4) v += (int64_t)acc[mt][d][ND - 1][r] << 16;
                        atomicAdd(reinterpret_cast<unsigned long long*>(&sSum[((mt * DT + d) * 4 + r) * 64 + lane]), (unsigned long long)v);
                    }
                const int64_t dn = BITS == 8 ? (int64_t)den[mt][0] + ((int64_t)den[mt][1] << 8) : (int64_t)den[mt][0];
                atomicAdd(reinterpret_cast<unsigned long long*>(&sDen[16 * mt + l16]), (unsigned long long)dn);
            }
        }
        __syncthreads();
        for (int it = tid; it < nmt * DT * 64; it += 64 * W) {
            const int mt = it / (DT * 64), d = it / 64 % DT, col = 16 * mt + (it & 15);
            int64_t v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = sSum[((mt * DT + d) * 4 + r) * 64 + (it & 63)];
            if constexpr (MODE == PG_SUMS) {
                int64_t* to = p.wsum + (unit + split) * (size_t)(COLS * (HD + 1));
#pragma unroll
                for (int r = 0; r < 4; r++) to[((mt * DT + d) * 4 + r) * 64 + (it & 63)] = v[r];
                if (d == 0 && (it & 63) < 16) to[COLS * HD + col] = sDen[col];
            } else if (col < cols) {
                const int i = (m0 + col) / p.rep, r0 = m0 + col - i * p.rep, pp = s.p0 + i;
                const int64_t dn = BITS == 8 ? -sDen[col] : 128 * sDen[col];
                uint32_t out = 0;
                if (pp >= 0 && pp < cap && dn > 0)
#pragma unroll
                    for (int r = 0; r < 4; r++) out |= (uint32_t)(uint8_t)div_round_q8(BITS == 8 ? -v[r] : v[r], dn) << (8 * r);
                *reinterpret_cast<uint32_t*>(p.o + (size_t)(s.t0 + i) * p.o_stride + (g * p.rep + r0) * HD + 16 * d + 4 * ((it & 63) >> 4)) = out;
            }
        }
    }
}

// The splits' sums joined: one CTA per (tile, kv head, 16 columns, 64 dimensions), four shares of the splits side by side.
template <int HD, int BITS, int MT>
__global__ __launch_bounds__(1024) void pg_join_kernel(Paged a, PgAttend p) {
    constexpr int DT = HD / 16, COLS = 16 * MT;
    __shared__ int64_t sV[4][4][256], sD[4][256];
    const int tile = (int)blockIdx.x / a.nkv, g = (int)blockIdx.x % a.nkv, mt = blockIdx.y;
    int first = 0;
    const int b = pg_tile_seq(a, tile, p.rep, COLS, 1, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int m0 = (tile - first) * COLS, cols = min(COLS, s.n * p.rep - m0), cap = a.max_pages << a.page_sh;
    if (16 * mt >= cols) return;
    const int64_t* from = p.wsum + ((size_t)tile * a.nkv + g) * p.splits * (size_t)(COLS * (HD + 1));
    const int it = threadIdx.x & 255, share = threadIdx.x >> 8;
    const int d = 4 * blockIdx.z + it / 64, lane = it & 63, col = 16 * mt + (lane & 15);
    int64_t v[4] = {0, 0, 0, 0}, dn = 0;
    if (col < cols) {
#pragma unroll 8
        for (int i = share; i < p.splits; i += 4) {
            const int64_t* x = from + (size_t)i * (COLS * (HD + 1));
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] += x[((mt * DT + d) * 4 + r) * 64 + lane];
            dn += x[COLS * HD + col];
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sV[share][r][it] = v[r];
    sD[share][it] = dn;
    __syncthreads();
    if (share || col >= cols) return;
    for (int k = 1; k < 4; k++) {
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] += sV[k][r][it];
        dn += sD[k][it];
    }
    const int i = (m0 + col) / p.rep, r0 = m0 + col - i * p.rep, pp = s.p0 + i;
    dn = BITS == 8 ? -dn : 128 * dn;
    uint32_t out = 0;
    if (pp >= 0 && pp < cap && dn > 0)
#pragma unroll
        for (int r = 0; r < 4; r++) out |= (uint32_t)(uint8_t)div_round_q8(BITS == 8 ? -v[r] : v[r], dn) << (8 * r);
    *reinterpret_cast<uint32_t*>(p.o + (size_t)(s.t0 + i) * p.o_stride + (g * p.rep + r0) * HD + 16 * d + 4 * (lane >> 4)) = out;
}

struct Plan {
    int mt, tiles, splits;
};

Plan plan(int tokens, int seqs, int64_t max_pos, int nh, int nkv, int hd, int bits) {
    const int rep = nh / nkv;
    const int64_t each = ((int64_t)tokens * rep + seqs - 1) / std::max(seqs, 1);
    Plan x;
    // as many columns as the registers hold beside a tile: a wave's loads serve them all
    x.mt = each <= 16 ? 1 : (hd == 64 ? 4 : 2) / (bits == 8 ? 1 : 2);
    const int64_t tiles = (int64_t)tokens * rep / (16 * x.mt) + seqs;
    x.tiles = (int)tiles;
    const int64_t ctas = std::min<int64_t>(tiles, tokens) * nkv, work = (max_pos + 63) / 64;
    x.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + ctas - 1) / ctas, work / (2 * PG_W)));
    if (ctas >= 256) x.splits = 1;
    return x;
}

size_t ws_max_bytes(const Plan& x, int nkv) {
    return ((size_t)x.tiles * nkv * x.splits * 16 * x.mt * 4 + 255) / 256 * 256;
}

size_t ws_bytes(const Plan& x, int nkv, int hd) {
    if (x.splits == 1) return 256;
    return ws_max_bytes(x, nkv) + (size_t)x.tiles * nkv * x.splits * 16 * x.mt * (hd + 1) * 8;
}

template <int HD, int BITS, int MT>
hipError_t attend(const Paged& a, const PgAttend& p, const Plan& x, hipStream_t s) {
    const dim3 grid((unsigned)(x.tiles * a.nkv), (unsigned)x.splits), block(64 * PG_W);
    if (x.splits == 1) {
        pg_attend_kernel<HD, BITS, MT, PG_W, PG_WHOLE><<<grid, block, 0, s>>>(a, p);
        return hipGetLastError();
    }
    pg_attend_kernel<HD, BITS, MT, PG_W, PG_MAX><<<grid, block, 0, s>>>(a, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    pg_attend_kernel<HD, BITS, MT, PG_W, PG_SUMS><<<grid, block, 0, s>>>(a, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    pg_join_kernel<HD, BITS, MT><<<dim3((unsigned)(x.tiles * a.nkv), MT, HD / 64), dim3(1024), 0, s>>>(a, p);
    return hipGetLastError();
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
    if (hd == 64) {
        if (x.mt == 1) return bits == 8 ? attend<64, 8, 1>(a, p, x, s) : attend<64, 4, 1>(a, p, x, s);
        return bits == 8 ? attend<64, 8, 4>(a, p, x, s) : attend<64, 4, 2>(a, p, x, s);
    }
    if (x.mt == 1) return bits == 8 ? attend<128, 8, 1>(a, p, x, s) : attend<128, 4, 1>(a, p, x, s);
    return attend<128, 8, 2>(a, p, x, s);
}

}  // namespace kt
