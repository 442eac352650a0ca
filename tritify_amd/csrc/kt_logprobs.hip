// Log probabilities of rows of int32 logits on gfx950: of given tokens, the entropy, and the k likeliest alternatives
// (kt_hip_dec_logprobs_rows, stated in include/kt_hip.h). The softmax's sums are taken per block of 1024 logits against the block's own
// maximum, in integers, so one pass over the logits does and no order of waves or CTAs changes a bit; a block is what one wave
// holds in registers. A second launch joins a row's blocks (24 bytes each) and looks its alternatives up: the k largest logits lie in the
// k blocks with the largest maxima (of equal ones the first). 1021 rows of 151936 logits: 110 us in all, 5.65 TB/s, near what a read of this
// card's memory reaches (vector units 0.77 busy with 18 instructions a logit; the join 6.6 us of it); 64 rows 10.3 and 8.2 us, one row 3.4 and 6.9:
// the join's chain of blocks, ranks, candidates and ranks again.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>
#include <type_traits>

#include "kt_dpp.h"
#include "kt_kernels.h"

namespace kt {

namespace {

constexpr int LP_BLOCK = 1024, LP_MOST = 31 << 16, LP_FAR = 41 << 16;
constexpr int64_t LP_LN2 = 5814540;  // 2^23 ln 2

// 2^x and log2 x by their series, for tables that the compiler fills (entries are at least 2^-13 of a unit off a half, far more
// than the series' error).
constexpr double exp2_of(double x) {
    double t = 1, s = 1;
    for (int i = 1; i < 40; i++) t = t * (x * 0.69314718055994530942) / i, s += t;
    return s;
}
constexpr double log2_of(double x) {  // 1 <= x <= 2, by log x = 2 artanh((x - 1) / (x + 1))
    const double z = (x - 1) / (x + 1);
    double t = z, s = 0;
    for (int i = 1; i < 80; i += 2) s += t / i, t *= z * z;
    return 2 * s / 0.69314718055994530942;
}

struct LpTables {
    uint32_t e[512];  // round(2^31 2^(-i / 2^8)), round(2^31 2^(-i / 2^16))
    int32_t g[1025];  // round(2^24 log2(1 + i / 2^10))
    constexpr LpTables() : e(), g() {
        for (int i = 0; i < 256; i++) {
            e[i] = (uint32_t)(2147483648.0 * exp2_of(-i / 256.0) + 0.5);
            e[256 + i] = (uint32_t)(2147483648.0 * exp2_of(-i / 65536.0) + 0.5);
        }
        for (int i = 0; i <= 1024; i++) g[i] = (int32_t)(16777216.0 * log2_of(1 + i / 1024.0) + 0.5);
    }
};
__device__ constexpr LpTables lp_tables{};

// (mant, shift) as the blocks use them: t = (min(d, far) mant + round) >> shift, at most 31 2^16; from the difference `far` on t is there
// already, and it is less than 31 2^16 + mant there, so 32 bits of the product are enough: its high half from bit sh on (`high`, shift 32
// or more), or the 32 bits from bit sh.
struct LpScale {
    uint32_t mant, far, sh;
    bool high;
    uint64_t round;
};

struct LpRows {
    const int32_t* x;
    int64_t stride;
    int rows, n, nb, k;
    uint32_t mant;
    int shift;
    LpScale scale;
    int32_t* bm;                  // [row][block]: maximum
    unsigned long long *bs, *bw;  // sums
    const int32_t* token;
    int32_t *lp, *ent, *top, *top_lp;
};

typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));

// t(d), at most `most`.
__device__ __forceinline__ uint32_t lp_bits(uint32_t d, uint32_t mant, int shift, uint32_t most) {
    const uint64_t t = ((uint64_t)d * mant + ((1ull << shift) >> 1)) >> shift;
    return t > most ? most : (uint32_t)t;
}

// A wave a block: 16 logits a lane. HIGH: the shift is 32 or more, so t is of the product's high half.
template <bool HIGH>
__global__ __launch_bounds__(256) void lp_block_kernel(LpRows p) {
    __shared__ uint32_t sT[512];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t unit = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6), row = unit / (uint32_t)p.nb;
    const int blk = (int)(unit - row * (uint32_t)p.nb);
    const bool in = row < (uint32_t)p.rows;
    const int32_t* x = p.x + (size_t)row * p.stride + (size_t)blk * LP_BLOCK;
    const int left = in ? min(LP_BLOCK, p.n - blk * LP_BLOCK) : 0;
    int v[16];
    int top = INT_MIN;
    if (left == LP_BLOCK) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const i32x4 y = *reinterpret_cast<const i32x4*>(x + 4 * (lane + 64 * j));
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * j + e] = y[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int i = 4 * (lane + 64 * (j >> 2)) + (j & 3);
            v[j] = i < left ? x[i] : INT_MIN;
        }
    }
    sT[tid] = lp_tables.e[tid];
    sT[256 + tid] = lp_tables.e[256 + tid];
    __syncthreads();
    if (!in) return;
#pragma unroll
    for (int j = 0; j < 16; j++) top = max(top, v[j]);
    top = wave_max_i32(top);
    uint64_t S = 0, W = 0;
    const char* const table = reinterpret_cast<const char*>(sT);
    auto sums = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            uint32_t e[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t d = min((uint32_t)top - (uint32_t)v[j + h], p.scale.far);
                const uint64_t y = (uint64_t)d * p.scale.mant + p.scale.round;
                const uint32_t hi = (uint32_t)(y >> 32), lo = (uint32_t)y;
                const uint32_t t = min(HIGH ? hi >> p.scale.sh : __builtin_amdgcn_alignbit(hi, lo, p.scale.sh), (uint32_t)LP_MOST);
                e[h] = __umulhi(*reinterpret_cast<const uint32_t*>(table + ((t >> 6) & 0x3FC)),
                                *reinterpret_cast<const uint32_t*>(table + 1024 + ((t << 2) & 0x3FC))) >> (t >> 16);
                if (!whole && 4 * (lane + 64 * (j >> 2)) + (j & 3) + h >= left) e[h] = 0;
                W += (uint64_t)e[h] * t;
            }
            S += e[0] + e[1];  // (at most 2^31)
        }
    };
    if (left == LP_BLOCK) sums(std::true_type());
    else sums(std::false_type());
    S = wave_sum_u64(S);
    W = wave_sum_u64(W);
    if (lane == 0) {
        p.bm[unit] = top;
        p.bs[unit] = S;
        p.bw[unit] = W;
    }
}

constexpr int LP_CANDS = 1024;  // candidates for alternatives that a CTA keeps
constexpr int LP_BLOCKS = 1024;  // of a row at most

// A CTA a row: the blocks joined, then the alternatives. The k best blocks (of equal maxima the first) stay in registers, 8 fours of
// logits a thread at most; the least of their maxima is a lower bound of the k-th largest logit that hardly any other logit reaches, so
// those at or above it are collected and ranked against each other. A row of fewer than k blocks takes the k-th of its 64 lanes' maxima: of
// G lanes, all waves' logits dealt to them, some G ln(G / (G - k)) logits reach it, 24 for 20 alternatives.
// BEST: how many of the best blocks there is room for.
template <int NT, bool TOP, int BEST>
__global__ __launch_bounds__(NT) void lp_join_kernel(LpRows p) {
    constexpr int NW = NT / 64, PT = LP_BLOCKS / NT;
    __shared__ uint32_t sT[512];
    __shared__ int sMax[NW];
    __shared__ uint64_t sS[NW], sW[NW];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const int32_t* x = p.x + (size_t)row * p.stride;
    const size_t first = (size_t)row * p.nb;
    auto key = [](int v, uint32_t i) { return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (0xFFFFFFFFu - i); };  // (value, then the lower index)
    int bm[PT], M = INT_MIN;
    uint64_t bs[PT], bw[PT];
#pragma unroll
    for (int i = 0; i < PT; i++) {
        const int at = tid + i * NT;
        bm[i] = INT_MIN, bs[i] = bw[i] = 0;
        if (at < p.nb) bm[i] = p.bm[first + at], bs[i] = p.bs[first + at], bw[i] = p.bw[first + at];
    }
    int tok = -1, tok_x = 0;
    if (tid == 0) {
        tok = p.token[row];
        if ((unsigned)tok < (unsigned)p.n) tok_x = x[tok];
    }
    __shared__ int sG[TOP ? 1025 : 1];
    const int* const g = TOP ? sG : lp_tables.g;  // (with alternatives it is on its way early, for all that wait for L)
    for (int i = tid; i < 512; i += NT) sT[i] = lp_tables.e[i];
    if constexpr (TOP)
        for (int i = tid; i < 1025; i += NT) sG[i] = lp_tables.g[i];
#pragma unroll
    for (int i = 0; i < PT; i++) M = max(M, bm[i]);
    M = wave_max_i32(M);
    if (lane == 0) sMax[w] = M;
    __shared__ uint64_t sBm[TOP ? LP_BLOCKS : 1];
    __shared__ int sBlk[KT_LOGPROBS_MAX_K], sRank[64], sBound, sCount;
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < PT; i++)
            if (tid + i * NT < p.nb) sBm[tid + i * NT] = key(bm[i], (uint32_t)(tid + i * NT));
        if (tid == 0) sCount = 0;
        if (tid < 64) sRank[tid] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; i++) M = max(M, sMax[i]);
    uint64_t S = 0, W = 0;
#pragma unroll
    for (int i = 0; i < PT; i++) {
        const uint32_t u = lp_bits((uint32_t)M - (uint32_t)bm[i], p.mant, p.shift, LP_FAR), k = 22 + (u >> 16);
        const uint64_t m = __umulhi(sT[(u >> 8) & 255], sT[256 + (u & 255)]);
        S += ((bs[i] >> 8) * m) >> k;
        W += (((bw[i] + u * bs[i]) >> 21) * (m >> 8)) >> k;
    }
    S = wave_sum_u64(S);
    W = wave_sum_u64(W);
    if (lane == 0) sS[w] = S, sW[w] = W;
    const int kb = min(p.k, p.nb);
    if constexpr (TOP) {
        // each block's rank among the others: a few lanes a block, as many as there are threads for
        const int lg = p.nb >= NT ? 0 : min(6, 31 - __clz(NT / p.nb)), per = 1 << lg;
        for (int i = tid >> lg; i < p.nb; i += NT >> lg) {
            const uint64_t mine = sBm[i];
            int rank = 0;
#pragma unroll 8
            for (int j = tid & (per - 1); j < p.nb; j += per) rank += sBm[j] > mine;
            for (int o = 1; o < per; o <<= 1) rank += __shfl_xor(rank, o);
            if (rank < kb && (tid & (per - 1)) == 0) {
                sBlk[rank] = i;
                if (rank == p.k - 1) sBound = (int)((uint32_t)(mine >> 32) ^ 0x80000000u);
            }
        }
    }
    __syncthreads();
    S = W = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) S += sS[i], W += sW[i];
    const int a = 63 - __clzll((long long)S);
    const uint32_t y = (uint32_t)(a >= 31 ? S >> (a - 31) : S << (31 - a)) & 0x7FFFFFFFu;
    const int gi = (int)(y >> 21);
    const int64_t L = (int64_t)(a - 30) * (1 << 24) + g[gi] + (((int64_t)(g[gi + 1] - g[gi]) * (y & 0x1FFFFF)) >> 21);
    auto nats = [&](int64_t t) { return (int32_t)(((t * 256 + L) * LP_LN2 + (1 << 30)) >> 31); };
    auto lp_of = [&](int v) { return -nats(lp_bits((uint32_t)M - (uint32_t)v, p.mant, p.shift, INT_MAX)); };
    if constexpr (TOP) {
        __shared__ uint64_t sKey[LP_CANDS];
        __shared__ int sOut[NW], sLane[NT];
        constexpr int U = BEST * (LP_BLOCK / 4) / NT;
        i32x4 v[U];
        int at[U];  // the first of four logits; n where there are none
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int it = tid + u * NT;
            at[u] = p.n;
            if (it < kb * (LP_BLOCK / 4)) at[u] = min(p.n, sBlk[it / (LP_BLOCK / 4)] * LP_BLOCK + 4 * (it % (LP_BLOCK / 4)));
            if (at[u] + 4 <= p.n) {
                v[u] = *reinterpret_cast<const i32x4*>(x + at[u]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[u][e] = at[u] + e < p.n ? x[at[u] + e] : INT_MIN;
            }
        }
        if (tid == 0) {
            p.lp[row] = (unsigned)tok < (unsigned)p.n ? lp_of(tok_x) : INT_MIN;
            if (p.ent) p.ent[row] = nats((int64_t)((W << 18) / (S >> 3)));
        }
        auto each = [&](auto f) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (at[u] + e < p.n) f(v[u][e], at[u] + e);
        };
        auto count = [&](int c) {  // the sum over the CTA
            __syncthreads();
            c = wave_sum_i32(c);
            if (lane == 0) sOut[w] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (int i = 0; i < NW; i++) c += sOut[i];
            return c;
        };
        int T = sBound;
        if (p.nb < p.k) {  // the k-th of the lanes' maxima over all waves
            int big = INT_MIN, rank = 0;
            each([&](int v, int) { big = max(big, v); });
            sLane[tid] = big;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; i++) big = max(big, sLane[64 * i + lane]);
#pragma unroll
            for (int i = 0; i < 64 / NW; i++) {  // each wave counts against its share of the lanes
                const int j = 64 / NW * __builtin_amdgcn_readfirstlane(w) + i, o = __builtin_amdgcn_readlane(big, j);
                rank += (o > big) | ((o == big) & (j < lane));
            }
            atomicAdd(&sRank[lane], rank);
            __syncthreads();
            rank = sRank[lane];
            T = __builtin_amdgcn_readlane(big, __ffsll((unsigned long long)__ballot(rank == p.k - 1)) - 1);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (max(max(v[u].x, v[u].y), max(v[u].z, v[u].w)) < T) continue;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (v[u][e] >= T && at[u] + e < p.n) {
                    const int c = atomicAdd(&sCount, 1);
                    if (c < LP_CANDS) sKey[c] = key(v[u][e], (uint32_t)(at[u] + e));
                }
        }
        __syncthreads();
        int cands = sCount;
        if (cands > LP_CANDS && p.n > p.k) {
            // Too many at or above the bound, equal ones for the most part: the k-th largest value itself, bit by bit from the first
            // that the bound and the maximum differ in, then those above it and the first of those equal to it.
            uint32_t lo = (uint32_t)T ^ 0x80000000u;
            const uint32_t hi = (uint32_t)M ^ 0x80000000u;
            if (lo != hi) {
                const int top = 31 - __clz((int)(lo ^ hi));
                lo &= ~((2u << top) - 1);
                for (int b = top; b >= 0; b--) {
                    const uint32_t t = lo | (1u << b);
                    int c = 0;
                    each([&](int v, int) { c += ((uint32_t)v ^ 0x80000000u) >= t; });
                    if (count(c) >= p.k) lo = t;
                }
            }
            T = (int)(lo ^ 0x80000000u);
            __syncthreads();
            if (tid == 0) sCount = 0;
            __syncthreads();
            each([&](int v, int i) {
                if (v > T) sKey[atomicAdd(&sCount, 1)] = key(v, (uint32_t)i);  // fewer than k
            });
            __syncthreads();
            cands = sCount;
            __syncthreads();
            if (w == 0) {  // one wave looks for the first equal ones: the blocks in order of their number, then through each
                const int mine = lane < kb ? sBlk[lane] : INT_MAX;
                int rank = 0;
                for (int j = 0; j < kb; j++) rank += __shfl(mine, j) < mine;
                for (int q = 0; q < kb && cands < p.k; q++) {
                    const int blk = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)__ballot(lane < kb && rank == q)) - 1);
                    for (int j = 0; j < LP_BLOCK && cands < p.k; j += 64) {
                        const int i = blk * LP_BLOCK + j + lane;
                        const bool eq = i < p.n && x[i] == T;
                        const uint64_t all = __ballot(eq);
                        const int before = cands + __popcll(all & ((1ull << lane) - 1));
                        if (eq && before < p.k) sKey[before] = key(T, (uint32_t)i);
                        cands = min(p.k, cands + (int)__popcll(all));
                    }
                }
            }
            cands = p.k;
            __syncthreads();
        }
        for (int i = tid; i < cands; i += NT) {
            const uint64_t mine = sKey[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < cands; j++) rank += sKey[j] > mine;
            if (rank < p.k) {
                p.top[(size_t)row * p.k + rank] = (int32_t)(0xFFFFFFFFu - (uint32_t)mine);
                p.top_lp[(size_t)row * p.k + rank] = lp_of((int)((uint32_t)(mine >> 32) ^ 0x80000000u));
            }
        }
        if (p.n + tid < p.k) p.top[(size_t)row * p.k + p.n + tid] = -1, p.top_lp[(size_t)row * p.k + p.n + tid] = INT_MIN;
    } else if (tid == 0) {
        p.lp[row] = (unsigned)tok < (unsigned)p.n ? lp_of(tok_x) : INT_MIN;
        if (p.ent) p.ent[row] = nats((int64_t)((W << 18) / (S >> 3)));
    }
}

struct LpParts {
    size_t bs, bw, bytes;
};

LpParts lp_parts(int64_t rows, int64_t n) {
    const size_t blocks = (size_t)rows * (size_t)((n + LP_BLOCK - 1) / LP_BLOCK), bs = (4 * blocks + 255) / 256 * 256;
    return {bs, bs + 8 * blocks, std::max<size_t>(256, bs + 16 * blocks)};
}

}  // namespace

namespace {

LpScale lp_scale(uint32_t mant, int shift) {
    auto t = [&](uint64_t d) { return ((unsigned __int128)d * mant + ((1ull << shift) >> 1)) >> shift; };
    uint64_t lo = 0, hi = 0xFFFFFFFFu;  // the least difference whose t is past the bound, if there is one
    while (lo < hi) {
        const uint64_t mid = (lo + hi) / 2;
        if (t(mid) >= (unsigned)LP_MOST) hi = mid;
        else lo = mid + 1;
    }
    return {mant, (uint32_t)lo, (uint32_t)(shift >= 32 ? shift - 32 : shift), shift >= 32, (1ull << shift) >> 1};
}

}  // namespace

size_t lp_workspace(int64_t rows, int64_t n) { return lp_parts(rows, n).bytes; }

hipError_t launch_logprobs(const int32_t* logits, int rows, int n, int64_t stride, const int32_t* token, uint32_t mant,
                           int shift, int32_t* lp, int32_t* ent, int k, int32_t* top, int32_t* top_lp, void* ws,
                           hipStream_t s) {
    const LpParts w = lp_parts(rows, n);
    const int nb = (n + LP_BLOCK - 1) / LP_BLOCK;
    const LpScale sc = lp_scale(mant, shift);
    const LpRows p = {logits, stride, rows, n, nb, k, mant, shift, sc, (int32_t*)ws, (unsigned long long*)((char*)ws + w.bs),
                      (unsigned long long*)((char*)ws + w.bw), token, lp, ent, top, top_lp};
    const dim3 blocks((unsigned)(((int64_t)rows * nb + 3) / 4));  // (at most 2^24 - 256)
    if (sc.high) lp_block_kernel<true><<<blocks, dim3(256), 0, s>>>(p);
    else lp_block_kernel<false><<<blocks, dim3(256), 0, s>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Where eight blocks hold the alternatives 256 threads will do, in more CTAs at a time: us of the join with 256 / 1024 threads, 700 rows of
    // 300 logits 9.8 / 22, of 5000 11.7 / 23.4, of 151936 13.5 / 22.2; 300 of 50000 8.3 / 13.4; 128 of 30000 7.5 / 8.0; but few rows of many blocks
    // rank them faster with more: 64 of 151936 10.8 / 7.9, one 8.0 / 7.0.
    const bool small = std::min(k, nb) <= 8 && (rows > 256 || nb <= 32);
    if (k == 0) lp_join_kernel<256, false, 0><<<dim3((unsigned)rows), dim3(256), 0, s>>>(p);
    else if (small) lp_join_kernel<256, true, 8><<<dim3((unsigned)rows), dim3(256), 0, s>>>(p);
    else lp_join_kernel<1024, true, KT_LOGPROBS_MAX_K><<<dim3((unsigned)rows), dim3(1024), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace kt
