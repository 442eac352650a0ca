// Eviction from paged KV caches by accumulated attention weight on gfx950 (kt_hip_dec_evict_paged, stated in include/kt_hip.h): for
// each sequence and kv head the heaviest positions are chosen, then their k, v, multipliers and sums go to other pages.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "kt_dpp.h"
#include "kt_paged.h"
#include "kt_w12_core.h"

namespace kt {

namespace {

struct PgEvict {
    const int32_t* to;
    int to_pages, budget, recent, sinks;
    int32_t* kept;
    int64_t* w;
};

constexpr int EV_NT = 1024, EV_WAVES = EV_NT / 64;

// The order of sums as unsigned numbers, 0 for a position without a page.
__device__ __forceinline__ uint64_t weight_key(const Paged& a, const PgEvict& p, int b, int g, int j) {
    const int id = pg_page(a, b, j >> 4);
    if (id < 0) return 0;
    const int64_t w = p.w[(((size_t)id * a.nkv + g) << a.page_sh) + (j & ((1 << a.page_sh) - 1))];
    const uint64_t k = (uint64_t)w ^ (1ull << 63);
    return k ? k : 1;
}

// A CTA a sequence and kv head. The heaviest `most` of the positions lo .. hi - 1: digit by digit from the first that they differ in, the
// bits of the least that stays; then, wave by wave over neighbouring positions, those above it and the first of those equal to it.
__global__ __launch_bounds__(EV_NT) void pg_select_kernel(Paged a, PgEvict p) {
    __shared__ uint64_t sAnd[EV_WAVES], sOr[EV_WAVES];
    __shared__ int sHist[256], sDigit, sNeed, sGt[EV_WAVES], sEq[EV_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, g = blockIdx.x, b = blockIdx.y;
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh));
    int32_t* kept = p.kept + ((size_t)b * a.nkv + g) * p.budget;
    if (L <= p.budget) {
        for (int i = tid; i < p.budget; i += EV_NT) kept[i] = i < L ? i : -1;
        return;
    }
    const int lo = p.sinks, hi = L - p.recent, most = p.budget - p.sinks - p.recent;
    for (int i = tid; i < p.sinks; i += EV_NT) kept[i] = i;
    for (int i = tid; i < p.recent; i += EV_NT) kept[p.budget - p.recent + i] = hi + i;
    if (most == 0) return;
    uint64_t all = ~0ull, any = 0;
    for (int j = lo + tid; j < hi; j += EV_NT) {
        const uint64_t k = weight_key(a, p, b, g, j);
        all &= k, any |= k;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) all &= __shfl_xor(all, o), any |= __shfl_xor(any, o);
    if (lane == 0) sAnd[wv] = all, sOr[wv] = any;
    __syncthreads();
    for (int i = 0; i < EV_WAVES; i++) all &= sAnd[i], any |= sOr[i];
    uint64_t least = all, mask = ~0ull;  // the bits of the least key that are known
    int need = most;
    if (all != any) {
        int sh = (63 - __clzll((long long)(all ^ any))) & ~7;
        mask = sh == 56 ? 0 : ~0ull << (sh + 8);
        least = all & mask;
        for (; sh >= 0; sh -= 8) {
            if (tid < 256) sHist[tid] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += EV_NT) {
                const uint64_t k = weight_key(a, p, b, g, j);
                if ((k & mask) == least) atomicAdd(&sHist[(k >> sh) & 255], 1);
            }
            __syncthreads();
            if (wv == 0) {  // lane l: digits 252 - 4 l .. 255 - 4 l
                int c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) c[i] = sHist[255 - 4 * lane - i], sum += c[i];
                int above = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int v = __shfl_up(above, o);
                    above += lane >= o ? v : 0;
                }
                above -= sum;  // of all lanes before
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (above < need && above + c[i] >= need) sDigit = 255 - 4 * lane - i, sNeed = need - above;
                    above += c[i];
                }
            }
            __syncthreads();
            least |= (uint64_t)sDigit << sh;
            mask |= 255ull << sh;
            need = sNeed;
            __syncthreads();
        }
    }
    const int seg = ((hi - lo + EV_WAVES - 1) / EV_WAVES + 63) & ~63, j0 = min(lo + wv * seg, hi), j1 = min(j0 + seg, hi);
    int gt = 0, eq = 0;
    for (int j = j0 + lane; j < j1; j += 64) {
        const uint64_t k = weight_key(a, p, b, g, j);
        gt += k > least, eq += k == least;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) gt += __shfl_xor(gt, o), eq += __shfl_xor(eq, o);
    if (lane == 0) sGt[wv] = gt, sEq[wv] = eq;
    __syncthreads();
    gt = eq = 0;
    for (int i = 0; i < wv; i++) gt += sGt[i], eq += sEq[i];
    const uint64_t before = (1ull << lane) - 1;
    for (int j = j0; j < j1; j += 64) {
        const uint64_t k = j + lane < j1 ? weight_key(a, p, b, g, j + lane) : 0;
        const bool in = j + lane < j1;
        const uint64_t bg = __ballot(in && k > least), be = __ballot(in && k == least);
        const int g0 = gt + __popcll(bg & before), e0 = eq + __popcll(be & before);
        if (in && (k > least || (k == least && e0 < need))) kept[p.sinks + g0 + min(e0, need)] = j + lane;
        gt += __popcll(bg), eq += __popcll(be);
    }
}

// A CTA (2 HD threads) a block of 16 slots, sequence and kv head: the first half of the threads moves K's chunks, the other gathers V's
// (16 positions of a dimension, from as many chunks).
template <int HD, int BITS>
__global__ __launch_bounds__(2 * HD) void pg_move_kernel(Paged a, PgEvict p, int nblk) {
    constexpr int HH = HD / 2, CH = HD / 16, ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;
    typedef typename std::conditional<BITS == 8, v4i, v2i>::type Chunk;
    __shared__ int sId[16], sSlot[16];
    const int b = (int)blockIdx.x / nblk, blk = (int)blockIdx.x - b * nblk, g = blockIdx.y, tid = threadIdx.x;
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh)), n = min(16, min(L, p.budget) - 16 * blk);
    if (n <= 0) return;
    const int id = p.to[(size_t)b * p.to_pages + (blk >> (a.page_sh - 4))], slot = (16 * blk) & ((1 << a.page_sh) - 1);
    if ((unsigned)id >= (unsigned)a.pages) return;
    const size_t to = ((size_t)id * a.nkv + g) * (size_t)a.part, mult = (size_t)(HH << a.page_sh);
    if (tid < 16) {
        const int j = tid < n ? p.kept[((size_t)b * a.nkv + g) * p.budget + 16 * blk + tid] : -1;
        const int from = j < 0 ? -1 : pg_page(a, b, j >> 4), sl = j & ((1 << a.page_sh) - 1);
        sId[tid] = from;
        sSlot[tid] = sl;
        if (tid < n) {
            p.w[(((size_t)id * a.nkv + g) << a.page_sh) + slot + tid] = from < 0 ? 0 : p.w[(((size_t)from * a.nkv + g) << a.page_sh) + sl];
            if constexpr (BITS == 4) {
                const size_t part = ((size_t)max(from, 0) * a.nkv + g) * (size_t)a.part + mult + sl;
                a.k[to + mult + slot + tid] = from < 0 ? 0 : a.k[part];
                a.v[to + mult + slot + tid] = from < 0 ? 0 : a.v[part];
            }
        }
    }
    __syncthreads();
    auto part_of = [&](int r) { return ((size_t)sId[r] * a.nkv + g) * (size_t)a.part; };
    if (tid < HD) {
        const int r = tid / CH, c = tid % CH;
        if (r >= n) return;
        Chunk x = {};
        if (sId[r] >= 0) x = *reinterpret_cast<const Chunk*>(a.k + part_of(r) + sSlot[r] * ROWB + c * CHB);
        *reinterpret_cast<Chunk*>(a.k + to + (slot + r) * ROWB + c * CHB) = x;
        return;
    }
    const int d = tid - HD;
    if constexpr (BITS == 8) {
        uint8_t* out = a.v + to + slot * HD + 16 * d;
        v4i x = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (sId[r] >= 0) x[r >> 2] |= (int)((uint32_t)a.v[part_of(r) + (sSlot[r] >> 4) * 16 * HD + 16 * d + (sSlot[r] & 15)] << (8 * (r & 3)));
        if (n == 16) {
            *reinterpret_cast<v4i*>(out) = x;
        } else {
            for (int r = 0; r < n; r++) out[r] = (uint8_t)((uint32_t)x[r >> 2] >> (8 * (r & 3)));
        }
    } else {
        uint32_t* out = reinterpret_cast<uint32_t*>(a.v + to + slot * HH + 8 * d);
        uint32_t x[2] = {0, 0}, keep[2] = {0, 0};
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int sh = 8 * (r & 3) + 4 * ((r >> 2) & 1);
            if (r >= n) keep[r >> 3] |= 15u << sh;
            if (sId[r] < 0) continue;
            const int sl = sSlot[r], e = sl & 15;
            const uint32_t c = a.v[part_of(r) + (sl >> 4) * 16 * HH + 8 * d + 4 * (e >> 3) + (e & 3)] >> (4 * ((e >> 2) & 1)) & 15;
            x[r >> 3] |= c << sh;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) out[h] = n == 16 ? x[h] : (x[h] | (out[h] & keep[h]));
    }
}

}  // namespace

hipError_t launch_pg_evict(const Paged& a, int hd, int bits, const int32_t* to, int budget, int recent, int sinks, int32_t* kept,
                           int64_t* w, hipStream_t s) {
    const int page = 1 << a.page_sh, nblk = (budget + 15) / 16;
    const PgEvict p = {to, (budget + page - 1) / page, budget, recent, sinks, kept, w};
    pg_select_kernel<<<dim3((unsigned)a.nkv, (unsigned)a.seqs), dim3(EV_NT), 0, s>>>(a, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    auto go = [&](auto kern) {
        kern<<<dim3((unsigned)(a.seqs * nblk), (unsigned)a.nkv), dim3(2 * hd), 0, s>>>(a, p, nblk);
        return hipGetLastError();
    };
    if (hd == 64) return bits == 8 ? go(pg_move_kernel<64, 8>) : go(pg_move_kernel<64, 4>);
    return bits == 8 ? go(pg_move_kernel<128, 8>) : go(pg_move_kernel<128, 4>);
}

}  // namespace kt
