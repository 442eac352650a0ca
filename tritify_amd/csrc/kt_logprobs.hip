// Log probabilities of rows of int32 logits on gfx950: of given tokens, the entropy, and the k likeliest alternatives
// (kt_hip_dec_logprobs_rows, stated in include/kt_hip.h). The softmax's sums are taken per block of 1024 logits against the block's own
// maximum, in integers, so one pass over the logits does and no order of waves or CTAs changes a bit; a block is what one wave
// holds in registers. A second launch joins a row's blocks (24 bytes each) and looks its alternatives up: the k largest logits lie in the
// k blocks with the largest maxima (of equal ones the first).

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

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

struct LpRows {
    const int32_t* x;
    int64_t stride;
    int n, nb, k;
    uint32_t mant;
    int shift;
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

// A wave a block: 16 logits a lane.
__global__ __launch_bounds__(256) void lp_block_kernel(LpRows p) {
    __shared__ uint32_t sT[512];
    for (int i = threadIdx.x; i < 512; i += 256) sT[i] = lp_tables.e[i];
    __syncthreads();
    const int lane = threadIdx.x & 63, blk = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (blk >= p.nb) return;
    const int32_t* x = p.x + (size_t)blockIdx.y * p.stride + (size_t)blk * LP_BLOCK;
    const int left = min(LP_BLOCK, p.n - blk * LP_BLOCK);
    int v[16];
    int top = INT_MIN;
    if (left == LP_BLOCK) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const i32x4 y = *reinterpret_cast<const i32x4*>(x + 4 * (lane + 64 * j));
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * j + e] = y[e], top = max(top, y[e]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int i = 4 * (lane + 64 * (j >> 2)) + (j & 3);
            v[j] = i < left ? x[i] : INT_MIN;
            top = max(top, v[j]);
        }
    }
    top = wave_max_i32(top);
    uint64_t S = 0, W = 0;
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const uint32_t t = lp_bits((uint32_t)top - (uint32_t)v[j], p.mant, p.shift, LP_MOST);
        uint32_t e = __umulhi(sT[(t >> 8) & 255], sT[256 + (t & 255)]) >> (t >> 16);
        if (left < LP_BLOCK && 4 * (lane + 64 * (j >> 2)) + (j & 3) >= left) e = 0;
        S += e;
        W += (uint64_t)e * t;
    }
    S = wave_sum_u64(S);
    W = wave_sum_u64(W);
    if (lane == 0) {
        const size_t at = (size_t)blockIdx.y * p.nb + blk;
        p.bm[at] = top;
        p.bs[at] = S;
        p.bw[at] = W;
    }
}

constexpr int LP_CANDS = 1024;  // candidates for alternatives that a CTA keeps

// A CTA a row: the blocks joined, then the alternatives.
__global__ __launch_bounds__(256) void lp_join_kernel(LpRows p) {
    __shared__ uint64_t sKey[LP_CANDS];
    __shared__ uint32_t sT[512];
    __shared__ int sMax[4], sBlk[KT_LOGPROBS_MAX_K], sCount, sOut[4];
    __shared__ uint64_t sS[4], sW[4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const int32_t* x = p.x + (size_t)row * p.stride;
    const int32_t* bm = p.bm + (size_t)row * p.nb;
    for (int i = tid; i < 512; i += 256) sT[i] = lp_tables.e[i];
    int M = INT_MIN;
    for (int i = tid; i < p.nb; i += 256) M = max(M, bm[i]);
    M = wave_max_i32(M);
    if (lane == 0) sMax[w] = M;
    if (tid == 0) sCount = 0;
    __syncthreads();
    M = max(max(sMax[0], sMax[1]), max(sMax[2], sMax[3]));
    uint64_t S = 0, W = 0;
    for (int i = tid; i < p.nb; i += 256) {
        const size_t at = (size_t)row * p.nb + i;
        const uint32_t u = lp_bits((uint32_t)M - (uint32_t)bm[i], p.mant, p.shift, LP_FAR), k = 22 + (u >> 16);
        const uint64_t m = __umulhi(sT[(u >> 8) & 255], sT[256 + (u & 255)]), s = p.bs[at];
        S += ((s >> 8) * m) >> k;
        W += (((p.bw[at] + u * s) >> 21) * (m >> 8)) >> k;
    }
    S = wave_sum_u64(S);
    W = wave_sum_u64(W);
    if (lane == 0) sS[w] = S, sW[w] = W;
    __syncthreads();
    S = sS[0] + sS[1] + sS[2] + sS[3];
    W = sW[0] + sW[1] + sW[2] + sW[3];
    const int a = 63 - __clzll((long long)S);
    const uint32_t y = (uint32_t)(a >= 31 ? S >> (a - 31) : S << (31 - a)) & 0x7FFFFFFFu;
    const int gi = (int)(y >> 21);
    const int64_t L = (int64_t)(a - 30) * (1 << 24) + lp_tables.g[gi] +
                      (((int64_t)(lp_tables.g[gi + 1] - lp_tables.g[gi]) * (y & 0x1FFFFF)) >> 21);
    auto nats = [&](int64_t t) { return (int32_t)(((t * 256 + L) * LP_LN2 + (1 << 30)) >> 31); };
    auto lp_of = [&](int v) { return -nats(lp_bits((uint32_t)M - (uint32_t)v, p.mant, p.shift, INT_MAX)); };
    if (tid == 0) {
        const int t = p.token[row];
        p.lp[row] = (unsigned)t < (unsigned)p.n ? lp_of(x[t]) : INT_MIN;
        if (p.ent) p.ent[row] = nats((int64_t)((W << 18) / (S >> 3)));
    }
    if (p.k == 0) return;

    // the blocks that hold the alternatives, in order of their number
    const int kb = min(p.k, p.nb);
    auto key = [](int v, uint32_t i) { return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (0xFFFFFFFFu - i); };
    for (int i = tid; i < p.nb; i += 256) {
        const uint64_t mine = key(bm[i], (uint32_t)i);
        int rank = 0;
        for (int j = 0; j < p.nb && rank < kb; j++) rank += key(bm[j], (uint32_t)j) > mine;
        if (rank < kb) sBlk[rank] = i;
    }
    __syncthreads();
    if (w == 0) {
        const int mine = lane < kb ? sBlk[lane] : INT_MAX;
        int rank = 0;
        for (int j = 0; j < kb; j++) rank += __shfl(mine, j) < mine;
        if (lane < kb) sBlk[rank] = mine;  // (a wave's reads come before its writes)
    }
    __syncthreads();
    // A lower bound of the k-th largest: of each wave's lanes' maxima the k-th.
    const int items = kb * 256;  // fours of logits
    auto each = [&](auto f) {
        for (int it = tid; it < items; it += 256) {
            const int i = sBlk[it >> 8] * LP_BLOCK + 4 * (it & 255);
            if (i + 4 <= p.n) {
                const i32x4 v = *reinterpret_cast<const i32x4*>(x + i);
#pragma unroll
                for (int e = 0; e < 4; e++) f(v[e], i + e);
            } else {
                for (int e = 0; i + e < p.n; e++) f(x[i + e], i + e);
            }
        }
    };
    int big = INT_MIN, rank = 0;
    each([&](int v, int) { big = max(big, v); });
    for (int j = 0; j < 64; j++) {
        const int o = __builtin_amdgcn_readlane(big, j);
        rank += o > big || (o == big && j < lane);
    }
    const int kth = __builtin_amdgcn_readlane(big, __ffsll((unsigned long long)__ballot(rank == p.k - 1)) - 1);
    if (lane == 0) sOut[w] = kth;
    __syncthreads();
    int T = max(max(sOut[0], sOut[1]), max(sOut[2], sOut[3]));
    each([&](int v, int i) {
        if (v >= T) {
            const int c = atomicAdd(&sCount, 1);
            if (c < LP_CANDS) sKey[c] = key(v, (uint32_t)i);
        }
    });
    __syncthreads();
    int cands = sCount;
    auto count_block = [&](int c) {  // the sum over the CTA
        __syncthreads();
        c = wave_sum_i32(c);
        if (lane == 0) sOut[w] = c;
        __syncthreads();
        return sOut[0] + sOut[1] + sOut[2] + sOut[3];
    };
    if (cands > LP_CANDS && p.n > p.k) {
        // Too many at or above the bound, equal ones for the most part: the k-th largest value itself, bit by bit from the first that
        // the bound and the maximum differ in, then those above it and the first of those equal to it.
        uint32_t lo = (uint32_t)T ^ 0x80000000u;
        const uint32_t hi = (uint32_t)M ^ 0x80000000u;
        if (lo != hi) {
            const int top = 31 - __clz((int)(lo ^ hi));
            lo &= ~((2u << top) - 1);
            for (int b = top; b >= 0; b--) {
                const uint32_t t = lo | (1u << b);
                int c = 0;
                each([&](int v, int) { c += ((uint32_t)v ^ 0x80000000u) >= t; });
                if (count_block(c) >= p.k) lo = t;
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
        if (w == 0) {  // one wave looks for the first equal ones, in order
            for (int it = 0; it < kb * LP_BLOCK && cands < p.k; it += 64) {
                const int i = sBlk[it >> 10] * LP_BLOCK + (it & (LP_BLOCK - 1)) + lane;
                const bool eq = i < p.n && x[i] == T;
                const uint64_t all = __ballot(eq);
                const int before = cands + __popcll(all & ((1ull << lane) - 1));
                if (eq && before < p.k) sKey[before] = key(T, (uint32_t)i);
                cands = min(p.k, cands + (int)__popcll(all));
            }
        }
        cands = p.k;
        __syncthreads();
    }
    for (int i = tid; i < cands; i += 256) {
        const uint64_t mine = sKey[i];
        int rank = 0;
        for (int j = 0; j < cands; j++) rank += sKey[j] > mine;
        if (rank < p.k) {
            p.top[(size_t)row * p.k + rank] = (int32_t)(0xFFFFFFFFu - (uint32_t)mine);
            p.top_lp[(size_t)row * p.k + rank] = lp_of((int)((uint32_t)(mine >> 32) ^ 0x80000000u));
        }
    }
    for (int i = p.n + tid; i < p.k; i += 256) p.top[(size_t)row * p.k + i] = -1, p.top_lp[(size_t)row * p.k + i] = INT_MIN;
}

struct LpParts {
    size_t bs, bw, bytes;
};

LpParts lp_parts(int64_t rows, int64_t n) {
    const size_t blocks = (size_t)rows * (size_t)((n + LP_BLOCK - 1) / LP_BLOCK), bs = (4 * blocks + 255) / 256 * 256;
    return {bs, bs + 8 * blocks, std::max<size_t>(256, bs + 16 * blocks)};
}

}  // namespace

size_t lp_workspace(int64_t rows, int64_t n) { return lp_parts(rows, n).bytes; }

hipError_t launch_logprobs(const int32_t* logits, int rows, int n, int64_t stride, const int32_t* token, uint32_t mant,
                           int shift, int32_t* lp, int32_t* ent, int k, int32_t* top, int32_t* top_lp, void* ws,
                           hipStream_t s) {
    const LpParts w = lp_parts(rows, n);
    const int nb = (n + LP_BLOCK - 1) / LP_BLOCK;
    const LpRows p = {logits, stride, n, nb, k, mant, shift, (int32_t*)ws, (unsigned long long*)((char*)ws + w.bs),
                      (unsigned long long*)((char*)ws + w.bw), token, lp, ent, top, top_lp};
    lp_block_kernel<<<dim3((unsigned)((nb + 3) / 4), (unsigned)rows), dim3(256), 0, s>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    lp_join_kernel<<<dim3((unsigned)rows), dim3(256), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace kt
