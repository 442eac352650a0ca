// The attention weights of a ragged batch's rows added up per held position and kv head, on gfx950 (kt_hip_dec_weigh_paged, stated
// in include/kt_hip.h): what an eviction from a paged cache goes by.
//
// With each row's largest score and the reciprocal R of its weights' sum in hand, one pass over K does: a wave holds 64 positions of K
// as B operands and goes through the columns (a row's q heads of one kv head, as in the attention), 64 of them a time. The scores are
// 16x16x64 int8 MFMAs with the columns as rows, so a lane has one position and 16 columns, whose weights' balanced base-256
// digits (of -e, two) are the A operand of a second product as they stand; its B operand is R's digits (five, each in a column of
// the result, and one further for e's high digit). Sums of e R are so exact in int32 and meet as int64.
//
// What it takes: 128 single tokens behind about 6100 (14 heads over 2 of 64) 28.7 us, K at 3.5 TB/s (vector units 0.42 busy, LDS 0.28,
// waves waiting for K 0.6 of their time), behind 6.0 us for the zeros of a fresh start, and 26.2 where the sums go on, as a decoder's do;
// 24.6 of that for equal lengths, as a sequence's tiles are dealt to a number of CTAs that the table's width gives and the longest decide;
// one token behind 131000 in 4 bits 7.5 us, behind 640 4.8; 1024 rows behind 7777 (15 GOP) 42.5 us: the table's look-ups have LDS busy 0.62
// of the time, over half of it with bank conflicts, vector units 0.60, a third of that for what each CTA begins and ends with, MFMAs 0.22.
// (Eight and sixteen copies of the table side by side, fewer conflicts: 49 to 51 us against 45.7, what the copies take to fill; 32, none,
// in a CTA of 16 waves a CU: 47 to 59 against 42.8.)

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

struct PgWeigh {
    const int8_t* q;
    int64_t q_stride;
    const int32_t* exp_tab;
    const int32_t* stats;
    int nh, rep, unit, window, sinks, splits;  // unit: columns of a CTA, at most WG_UNIT
    int64_t* w;
};

constexpr int WG_UNIT = 256;   // columns of a CTA: each digit sum stays within 2 2^14 256
constexpr int WG_WAVES = 4;
constexpr int WG_DIGITS = 5;   // of R, below 2^32
constexpr int WG_SUMS = 6;     // digits of e R before they carry: e's low one times R's d-th and its high one times the (d - 1)-th

// -x of 16 int8 values, -128 taken as -127.
__device__ __forceinline__ v4i negated(v4i x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = (uint32_t)x[i], h = u & 0x80808080u, t = 0x80808080u - (u & 0x7F7F7F7Fu);
        const uint32_t z = t & 0x80808080u, least = h & z;
        x[i] = (int)((t & 0x7F7F7F7Fu) | (~(h | z) & 0x80808080u) | (least - (least >> 7)));
    }
    return x;
}

// The sums of the batch's sequences begin from 0: two slots a thread, a page's (all its kv heads) side by side.
__global__ __launch_bounds__(256) void pg_weigh_zero_kernel(Paged a, int64_t* __restrict__ w) {
    typedef long long sums2 __attribute__((ext_vector_type(2)));
    const int b = blockIdx.y, end = min(pg_len(a, b), a.max_pages << a.page_sh);
    const int per = a.nkv << (a.page_sh - 1), pages = (max(end, 0) + (1 << a.page_sh) - 1) >> a.page_sh;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)pages * per; i += (int64_t)gridDim.x * 256) {
        const int pg = (int)((uint32_t)i / (uint32_t)per), at = 2 * ((int)i - pg * per);
        const int id = pg_page(a, b, pg << (a.page_sh - 4)), left = end - (pg << a.page_sh) - (at & ((1 << a.page_sh) - 1));
        if (id < 0 || left <= 0) continue;
        int64_t* to = w + ((size_t)id * a.nkv << a.page_sh) + at;
        if (left > 1 && ((uintptr_t)to & 15) == 0) *reinterpret_cast<sums2*>(to) = sums2{0, 0};
        else to[0] = 0, to[left > 1] = 0;
    }
}

// CT: 16 columns times CT a step. Waves a SIMD: with three instead of four the chunk of 1024 rows takes 45.5 us instead of 42.5, four spill some
// registers outside the loop over columns; in 4 bits, whose multipliers need more, four take 83 us and three 54.
template <int HD, int BITS, int CT>
__global__ __launch_bounds__(64 * WG_WAVES) __attribute__((amdgpu_waves_per_eu(HD == 64 ? (CT == 1 || BITS == 8 ? 4 : 3) : 2))) void
pg_weigh_kernel(Paged a, PgWeigh p) {
    constexpr int WG_GROUP = 16 * CT, QN = WG_GROUP * HD / 16 > 64 * WG_WAVES ? WG_GROUP * HD / 16 / (64 * WG_WAVES) : 1;
    constexpr int KC = HD / 64, CPR = HD / 16, NT = 64 * WG_WAVES, HH = HD / 2;
    constexpr int ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;
    typedef typename std::conditional<BITS == 8, v4i, v2i>::type Chunk;
    __shared__ __attribute__((aligned(16))) int8_t sQ[WG_GROUP * HD], sR[WG_DIGITS * WG_GROUP];
    __shared__ __attribute__((aligned(16))) int sTop[WG_GROUP], sPos[WG_GROUP];
    __shared__ __attribute__((aligned(8))) uint16_t sE[1028];
    __shared__ int sSum[WG_WAVES][64 * (WG_SUMS + 1)];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, gq = lane >> 4;
    typedef int tab4 __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int ET = 256 / NT > 1 ? 256 / NT : 1;
    tab4 et[ET];  // the table is on its way while the batch is looked up
#pragma unroll
    for (int i = 0; i < ET; i++)
        if (NT <= 256 || tid < 256) et[i] = *reinterpret_cast<const tab4*>(p.exp_tab + 4 * (tid + i * NT));

    // column units 0 .. seqs - 1 are the sequences' first ones, the rest their further ones
    const int ntiles = (int)gridDim.x / a.nkv, g = (int)blockIdx.x % a.nkv, unit = ntiles - 1 - (int)blockIdx.x / a.nkv;
    int b = unit, nth = 0;
    if (unit >= a.seqs) {
        int first = 0;
        b = pg_tile_seq(a, unit - a.seqs, p.rep, p.unit, 0, &first);
        nth = unit - a.seqs - first + 1;
    }
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int m0 = nth * p.unit, mrows = s.n * p.rep;
    if (m0 >= mrows) return;
    const int cols = min(p.unit, mrows - m0), groups = (cols + WG_GROUP - 1) / WG_GROUP;
    // column m0 + c is head (rem0 + c) % rep of row row0 + (rem0 + c) / rep; a float quotient of a whole number and a half below 2^13
    // is nearer to it than to a whole number, so its floor is exact
    const int row0 = nth ? m0 / p.rep : 0, rem0 = m0 - row0 * p.rep;
    const float inv = __builtin_amdgcn_rcpf((float)p.rep);
    auto over = [&](int c) { return (int)(((float)(rem0 + c) + 0.5f) * inv); };
    const int cap = a.max_pages << a.page_sh, nblk = cap >> 4, pos0 = s.p0 + row0;
    const int umin = pos0, umax = min(pos0 + __builtin_amdgcn_readfirstlane(over(cols - 1)), cap - 1);
    const int ntile = umax < 0 || a.pages == 0 ? 0 : umax / 64 + 1;
    int nsink = 0, w0 = 0;
    if (p.window && ntile) {
        nsink = min((min(p.sinks, umax + 1) + 63) / 64, ntile);
        w0 = max(nsink, (max(umin, 0) - min(p.window - 1, max(umin, 0))) / 64);
    }
    const int total = nsink + max(0, ntile - w0), step = p.splits * WG_WAVES, start = (int)blockIdx.y * WG_WAVES;
    const int rounds = start < total ? (total - 1 - start) / step + 1 : 0;  // of the CTA's first wave, which has the most
    if (rounds == 0) return;
    auto at = [&](int n) {  // this wave's n-th tile, or -1
        const int i = start + w + n * step;
        return i >= total ? -1 : (i < nsink ? i : i - nsink + w0);
    };

    // A tile's pages (a lane that of its block, lane / 16), read a round before its K is asked for.
    auto page_of = [&](int T) {
        const int blk = min(4 * max(T, 0) + gq, nblk - 1);
        return a.table[(size_t)b * a.max_pages + (blk >> (a.page_sh - 4))];
    };
    struct Keys {
        Chunk x[4][KC];
        int m[4];     // 4 bits: the multiplier of the lane's position
        int id;       // the page of the lane's block, or -1
        uint64_t ok;  // the lanes whose block has a page
    };
    const uint8_t* const kbase = a.k + (size_t)g * a.part;
    const uint32_t stride = (uint32_t)a.nkv * (uint32_t)a.part;
    const int from_lane = l16 * ROWB + gq * CHB;
    auto load = [&](int T, int id, Keys& k) {
        const bool ok = (unsigned)id < (unsigned)a.pages && 4 * T + gq < nblk;
        k.ok = __ballot(ok);
        k.id = ok ? id : -1;
        const int from_id = ok ? id : 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int slot = ((4 * T + t) << 4) & ((1 << a.page_sh) - 1);
            const uint8_t* from = kbase + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(from_id, 16 * t) * stride;
#pragma unroll
            for (int c = 0; c < KC; c++) k.x[t][c] = *reinterpret_cast<const Chunk*>(from + (slot * ROWB + 4 * c * CHB) + from_lane);
            if constexpr (BITS == 4) k.m[t] = from[((HH << a.page_sh) + slot) + l16];
        }
    };

    // a group's columns: negated q, 2 (top + 64), positions, R's digits; on their way while the group before is at work
    v4i qx[QN];
    v2i st = {0, 0};
    int at_row = 0;
    auto fetch = [&](int grp) {
        const int n = min(WG_GROUP, cols - grp * WG_GROUP);
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int it = tid + i * NT, c = grp * WG_GROUP + min(it / CPR, n - 1), up = over(c), row = row0 + up;
            if (QN > 1 || WG_GROUP * CPR >= NT || it < WG_GROUP * CPR)
                qx[i] = *reinterpret_cast<const v4i*>(p.q + (size_t)(s.t0 + row) * p.q_stride +
                                                      (g * p.rep + rem0 + c - up * p.rep) * HD + 16 * (it % CPR));
        }
        if (tid < WG_GROUP) {
            const int c = grp * WG_GROUP + min(tid, n - 1), up = over(c);
            at_row = row0 + up;
            st = *reinterpret_cast<const v2i*>(p.stats + 2 * ((size_t)(s.t0 + at_row) * p.nh + g * p.rep + rem0 + c - up * p.rep));
        }
    };
    auto put = [&](int grp) {
        const int n = min(WG_GROUP, cols - grp * WG_GROUP);
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int it = tid + i * NT, c = it / CPR, ch = it % CPR;
            if (QN > 1 || WG_GROUP * CPR >= NT || it < WG_GROUP * CPR)
                *reinterpret_cast<v4i*>(sQ + c * HD + 16 * (ch ^ swz<CPR>(c))) = negated(qx[i]);
        }
        if (tid < WG_GROUP) {
            const bool live = tid < n && s.p0 + at_row >= 0 && s.p0 + at_row < cap;
            sTop[tid] = (int)(128u + 2u * (uint32_t)st.x);
            sPos[tid] = live ? s.p0 + at_row : -1;
            const uint64_t r = (live ? (uint64_t)(uint32_t)st.y : 0) + 0x8080808080ull;
            // byte 4 t + r of the lanes of quarter q is column 16 t + 4 q + r
            const int to = ((tid >> 2) & 3) * 4 * CT + (tid >> 4) * 4 + (tid & 3);
#pragma unroll
            for (int d = 0; d < WG_DIGITS; d++) sR[d * WG_GROUP + to] = (int8_t)((r >> (8 * d)) ^ 0x80);
        }
    };

    Keys now, next;
    int id0 = page_of(at(0)), id1 = rounds > 1 ? page_of(at(1)) : 0;
    fetch(0);
#pragma unroll
    for (int i = 0; i < ET; i++) {
        uint32_t e[4];
#pragma unroll
        for (int r = 0; r < 4; r++) e[r] = ((0x8080u - (uint32_t)min(max(et[i][r], 0), 32768)) ^ 0x8080u) & 0xFFFFu;  // the two balanced digits of -e
        if (NT <= 256 || tid < 256) *reinterpret_cast<v2i*>(sE + 4 * (tid + i * NT)) = v2i{(int)(e[0] | e[1] << 16), (int)(e[2] | e[3] << 16)};
    }
    if (tid == 0) sE[1024] = 0;
    if (CT == 1 && at(0) >= 0) load(at(0), id0, now);

    auto widen = [](Chunk x) {  // 4 bits: 16 times the codes
        if constexpr (BITS == 8) {
            return x;
        } else {
            constexpr int M = (int)0xF0F0F0F0;
            return v4i{(x.x << 4) & M, x.x & M, (x.y << 4) & M, x.y & M};
        }
    };
    v4i acc[4];
    const int window = p.window ? p.window : 1 << 30;  // (positions lie within +-2^30, those that count below 2^20)
    // the weights of the tile's positions and a group's columns, times R; `all`: every column sees every position
    auto add = [&](auto all, int T, const Keys& k) {
        v4i rd[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        if constexpr (CT == 4) {
            if (l16 < WG_DIGITS) rd[0] = *reinterpret_cast<const v4i*>(sR + l16 * WG_GROUP + gq * 16);
            if (l16 >= 1 && l16 < WG_SUMS) rd[1] = *reinterpret_cast<const v4i*>(sR + (l16 - 1) * WG_GROUP + gq * 16);
        } else {  // e's two digits side by side in one product
            if (l16 < WG_DIGITS) rd[0].x = *reinterpret_cast<const int*>(sR + l16 * WG_GROUP + gq * 4);
            if (l16 >= 1 && l16 < WG_SUMS) rd[0].y = *reinterpret_cast<const int*>(sR + (l16 - 1) * WG_GROUP + gq * 4);
        }
        // all blocks of the tile for each 16 columns, whose q and top are read from LDS once (a block after the other, in fewer
        // registers and with a wave more: 1024 rows behind 7777 50 us against 44)
        v4i P[4][2] = {};
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const v4i top = *reinterpret_cast<const v4i*>(sTop + 16 * c + 4 * gq);
            v4i q[KC], pos = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KC; i++)
                q[i] = *reinterpret_cast<const v4i*>(sQ + (16 * c + l16) * HD + 16 * ((gq + 4 * i) ^ swz<CPR>(l16 + 16 * c)));
            if constexpr (!all) pos = *reinterpret_cast<const v4i*>(sPos + 16 * c + 4 * gq);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                v4i y = BITS == 8 && HD == 64 ? top : v4i{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KC; i++) {
                    y = mfma16(q[i], widen(k.x[t][i]), y);
                    if constexpr (BITS == 8 && HD == 64) y = mfma16(q[i], k.x[t][i], y);
                }
                uint32_t u[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {  // 2 (top - s + 64)
                    if constexpr (BITS == 4) y[r] = (__mul24(y[r], k.m[t]) + 63) >> 7;
                    u[r] = BITS == 8 && HD == 64 ? (uint32_t)y[r] : (uint32_t)y[r] * 2 + (uint32_t)top[r];
                }
                if constexpr (!all) {
                    const int j = (k.ok >> (16 * t)) & 1 ? 64 * T + 16 * t + l16 : INT_MAX;  // (of no page: past every row)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        u[r] = (j <= pos[r]) & ((j > pos[r] - window) | (j < p.sinks)) ? u[r] : 0x00FFFFFFu;
                }
                us2 e[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t ix = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(
                        __builtin_bit_cast(us2, __builtin_amdgcn_perm(u[2 * h + 1], u[2 * h], 0x06050201)), us2{1024, 1024}));
                    e[h] = us2{sE[ix & 0xFFFF], sE[ix >> 16]};
                }
                const uint32_t e01 = __builtin_bit_cast(uint32_t, e[0]), e23 = __builtin_bit_cast(uint32_t, e[1]);
                P[t][0][c] = (int)__builtin_amdgcn_perm(e23, e01, 0x06040200);
                P[t][CT == 4][CT == 4 ? c : 1] = (int)__builtin_amdgcn_perm(e23, e01, 0x07050301);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            acc[t] = mfma16(P[t][0], rd[0], acc[t]);
            if constexpr (CT == 4) acc[t] = mfma16(P[t][1], rd[1], acc[t]);
        }
    };

    for (int n = 0; n < rounds; n++) {
        const int T = at(n), T1 = n + 1 < rounds ? at(n + 1) : -1;
        if (CT == 1) {
            if (T1 >= 0) load(T1, id1, next);
        } else {
            if (T >= 0) load(T, id0, now);
            id0 = id1;
        }
        if (n + 2 < rounds) id1 = page_of(at(n + 2));
#pragma unroll
        for (int t = 0; t < 4; t++) acc[t] = v4i{0, 0, 0, 0};
        for (int grp = 0; grp < groups; grp++) {
            if (groups > 1 || n == 0) {
                if (groups > 1) __syncthreads();
                put(grp);
                __syncthreads();
                if (groups > 1 && (grp + 1 < groups || n + 1 < rounds)) fetch(grp + 1 < groups ? grp + 1 : 0);
            }
            const int gmin = pos0 + __builtin_amdgcn_readfirstlane(over(grp * WG_GROUP)),
                      gmax = pos0 + __builtin_amdgcn_readfirstlane(over(min(grp * WG_GROUP + WG_GROUP, cols) - 1));
            if (T < 0 || 64 * T > gmax) continue;
            if (now.ok == ~0ull && 64 * T + 63 <= gmin && gmax < cap &&
                (p.window == 0 || 64 * T > gmax - p.window || 64 * T + 63 < p.sinks))
                add(std::true_type(), T, now);
            else add(std::false_type(), T, now);
        }
        if (T >= 0) {
            // register r of acc[t], lane l: position 16 t + 4 (l / 16) + r, digit l % 16; turned to a position a lane
            int* const sum = sSum[w];
            __builtin_amdgcn_wave_barrier();
            if (l16 < WG_SUMS) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[(16 * t + 4 * gq + r) * (WG_SUMS + 1) + l16] = acc[t][r];
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            int64_t v = 0;  // of -e R
#pragma unroll
            for (int d = 0; d < WG_SUMS; d++) v += (int64_t)sum[lane * (WG_SUMS + 1) + d] * (1ll << (8 * d));
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (now.id >= 0 && v != 0)
                (void)__hip_atomic_fetch_sub(reinterpret_cast<unsigned long long*>(p.w) + ((((size_t)now.id * a.nkv + g)) << a.page_sh) +
                                                 ((64 * T + lane) & ((1 << a.page_sh) - 1)),
                                             (unsigned long long)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (CT == 1) now = next;
    }
}

}  // namespace

hipError_t launch_pg_weigh(const Paged& a, int hd, int bits, const int8_t* q, int64_t q_stride, int nh, const int32_t* exp_tab,
                           int window, int sinks, const int32_t* stats, bool fresh, int64_t* w, hipStream_t s) {
    const int64_t max_pos = (int64_t)a.max_pages << a.page_sh;
    if (fresh) {
        const int64_t blocks = std::min<int64_t>((max_pos * a.nkv + 511) / 512, std::max<int64_t>(1, 1024 / a.seqs));
        pg_weigh_zero_kernel<<<dim3((unsigned)blocks, (unsigned)a.seqs), dim3(256), 0, s>>>(a, w);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || a.tokens == 0) return e;
    }
    // A CTA's columns: 256, fewer where that leaves CUs without a CTA (us with 256 / fewer: 40 rows behind 2000 14.5 / 6.8, 150 rows 14.7 /
    // 7.9, 4 x 200 behind 500 15.1 / 9.0; of 1024 rows behind 7777 128 / 256 / 512 48 / 45 / 51). Its positions: all that leaves some 2048
    // CTAs (with 1024 / 2048 / 4096: 128 single tokens 28.9 / 28.5 / 31.5, the 1024 rows 48.8 / 45.2 / 45.6).
    const int rep = nh / a.nkv;
    const int64_t reach = window ? std::min<int64_t>(max_pos, (int64_t)window + sinks + WG_UNIT + 128) : max_pos;
    const int64_t rounds = (reach + 64 * WG_WAVES - 1) / (64 * WG_WAVES);
    auto units_of = [&](int unit) { return (a.seqs + (int64_t)a.tokens * rep / unit) * a.nkv; };
    int unit = WG_UNIT;
    while (unit > 64 && units_of(unit) * rounds < 1024) unit /= 2;
    const int64_t units = units_of(unit), splits = std::min(rounds, std::max<int64_t>(1, 2048 / units));
    const bool few = (int64_t)a.tokens * rep <= 24 * (int64_t)a.seqs;  // columns of a sequence, on average
    // 16 or 64 columns a step, us with 16 / 64 (7 heads a kv head): 64 sequences of 2 rows 6.3 / 8.5, of 3 7.9 / 8.6, of 5 9.4 /
    // 8.6; 64 of one row behind 4000 12.0 / 16.3, in heads of 128 17.1 / 26.1; one of 40 rows behind 2000 21.0 / 14.3. The average hides one
    // chunk beside many tokens: 64 single tokens and 150 rows take 16 columns, behind 1000 10.5 / 9.7, behind 4000 41.6 / 30.4.
    const PgWeigh p = {q, q_stride, exp_tab, stats, nh, rep, unit, window, sinks, (int)splits, w};
    auto go = [&](auto one, auto four) {
        if (few) one<<<dim3((unsigned)units, (unsigned)splits), dim3(64 * WG_WAVES), 0, s>>>(a, p);
        else four<<<dim3((unsigned)units, (unsigned)splits), dim3(64 * WG_WAVES), 0, s>>>(a, p);
        return hipGetLastError();
    };
    if (hd == 64)
        return bits == 8 ? go(pg_weigh_kernel<64, 8, 1>, pg_weigh_kernel<64, 8, 4>) : go(pg_weigh_kernel<64, 4, 1>, pg_weigh_kernel<64, 4, 4>);
    return bits == 8 ? go(pg_weigh_kernel<128, 8, 1>, pg_weigh_kernel<128, 8, 4>) : go(pg_weigh_kernel<128, 4, 1>, pg_weigh_kernel<128, 4, 4>);
}

}  // namespace kt
