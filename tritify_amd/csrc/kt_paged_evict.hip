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
constexpr int EV_BINS = 4096;   // of sums
constexpr int EV_CANDS = 1024;  // positions of one bin that are ranked against each other
constexpr int EV_U = 8;         // positions of a lane in flight

// The bin of a sum: the values below 64 one each, from there on 32 to a power of two, mirrored for negative ones; bin 0 for a position
// without a page (no sum has it).
__device__ __forceinline__ int weight_bin(int64_t w) {
    const uint64_t m = (uint64_t)(w < 0 ? ~w : w);
    const int sh = max(0, 58 - __clzll((long long)(m | 1)));
    const int b = 32 * sh + (int)(m >> sh);
    return w < 0 ? 2047 - b : 2048 + b;
}
// The order of sums as unsigned numbers, 0 for a position without a page.
__device__ __forceinline__ uint64_t weight_key(int64_t w, bool page) {
    const uint64_t k = (uint64_t)w ^ (1ull << 63);
    return page ? (k ? k : 1) : 0;
}

// A CTA a sequence and kv head. Which positions stay: the sums' histogram says in which bin the least that stays lies and how many of the
// bin do; a second sweep notes a bit for each position above that bin, and its members are ranked against each other (their sums, then
// their positions). The bits give the order. Each wave sweeps neighbouring positions, 64 a step.
//
// Two sweeps of the sums, whatever the length: 131001 positions (2 kv heads, two CTAs at work) XX us; 64 sequences of up to 2200, 2 kv
// heads, YY us.
__global__ __launch_bounds__(EV_NT) void pg_select_kernel(Paged a, PgEvict p) {
    extern __shared__ uint64_t sBits[];  // a word for 64 positions
    __shared__ int sHist[EV_BINS];
    __shared__ uint64_t sKey[EV_CANDS], sAnd[EV_WAVES], sOr[EV_WAVES];
    __shared__ int sAt[EV_CANDS], sWave[EV_WAVES], sBin, sNeed, sCount;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.x, b = blockIdx.y;
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
    for (int i = tid; i < EV_BINS; i += EV_NT) sHist[i] = 0;
    if (tid == 0) sCount = 0;

    // the wave's words, and f(word, position or -1, sum, whether it has a page) for each of them, all lanes at work
    const int words = (hi - lo + 63) / 64, seg = (words + EV_WAVES - 1) / EV_WAVES, w0 = min(wv * seg, words), w1 = min(w0 + seg, words);
    auto sweep = [&](auto f) {
        for (int wd = w0; wd < w1; wd += EV_U) {
            int id[EV_U];
            int64_t x[EV_U];
#pragma unroll
            for (int u = 0; u < EV_U; u++) {
                const int j = lo + 64 * (wd + u) + lane;
                id[u] = wd + u < w1 && j < hi ? pg_page(a, b, j >> 4) : -1;
            }
#pragma unroll
            for (int u = 0; u < EV_U; u++) {
                const int j = lo + 64 * (wd + u) + lane;
                x[u] = 0;
                if (id[u] >= 0) x[u] = p.w[(((size_t)id[u] * a.nkv + g) << a.page_sh) + (j & ((1 << a.page_sh) - 1))];
            }
#pragma unroll
            for (int u = 0; u < EV_U; u++) {
                const int j = lo + 64 * (wd + u) + lane;
                if (wd + u < w1) f(wd + u, j < hi ? j : -1, x[u], id[u] >= 0);
            }
        }
    };
    __syncthreads();
    sweep([&](int, int j, int64_t x, bool page) {
        // lanes with the first lane's bin are counted together: one bin may have most positions (zeros)
        const int bin = j < 0 ? -1 : (page ? weight_bin(x) : 0), one = __builtin_amdgcn_readfirstlane(bin);
        const int same = (int)__popcll(__ballot(bin == one));
        if (lane == 0 && one >= 0) atomicAdd(&sHist[one], same);
        if (bin != one && bin >= 0) atomicAdd(&sHist[bin], 1);
    });
    __syncthreads();
    {  // from the largest bin: thread t has bins 4095 - 4 t and the three below
        int c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = sHist[EV_BINS - 1 - 4 * tid - i], sum += c[i];
        int above = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(above, o);
            above += lane >= o ? v : 0;
        }
        if (lane == 63) sWave[wv] = above;
        above -= sum;
        __syncthreads();
        for (int i = 0; i < wv; i++) above += sWave[i];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (above < most && above + c[i] >= most) sBin = EV_BINS - 1 - 4 * tid - i, sNeed = most - above;
            above += c[i];
        }
    }
    __syncthreads();
    const int bin = sBin, members = sHist[bin];
    int need = sNeed;  // of the bin's members
    const bool all = need == members, few = members <= EV_CANDS;
    sweep([&](int word, int j, int64_t x, bool page) {
        const int mine = j < 0 ? -1 : (page ? weight_bin(x) : 0);
        const uint64_t stay = __ballot(mine > bin || (all && mine == bin));
        if (lane == 0) sBits[word] = stay;
        if (mine == bin && few && !all) {
            const int c = atomicAdd(&sCount, 1);
            sKey[c] = weight_key(x, page);
            sAt[c] = j;
        }
    });
    __syncthreads();
    if (!all && few) {
        if (tid < members) {
            const uint64_t mine = sKey[tid];
            const int at = sAt[tid];
            int rank = 0;
            for (int i = 0; i < members; i++) rank += (sKey[i] > mine) | ((sKey[i] == mine) & (sAt[i] < at));
            if (rank < need) atomicOr(reinterpret_cast<unsigned long long*>(&sBits[(at - lo) >> 6]), 1ull << ((at - lo) & 63));
        }
        __syncthreads();
    } else if (!all) {
        // More members than that, equal ones for the most part: the least sum that stays, eight bits at a time from the first that the
        // members differ in; then those above it and the first of those equal to it.
        uint64_t both = ~0ull, any = 0;
        auto members_of = [&](auto f) {
            sweep([&](int word, int j, int64_t x, bool page) {
                const bool in = j >= 0 && (page ? weight_bin(x) : 0) == bin;
                f(word, in, weight_key(x, page));
            });
        };
        members_of([&](int, bool in, uint64_t k) {
            if (in) both &= k, any |= k;
        });
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) both &= __shfl_xor(both, o), any |= __shfl_xor(any, o);
        if (lane == 0) sAnd[wv] = both, sOr[wv] = any;
        __syncthreads();
        for (int i = 0; i < EV_WAVES; i++) both &= sAnd[i], any |= sOr[i];
        uint64_t least = both, mask = ~0ull;
        if (both != any) {
            int sh = (63 - __clzll((long long)(both ^ any))) & ~7;
            mask = sh == 56 ? 0 : ~0ull << (sh + 8);
            least = both & mask;
            for (; sh >= 0; sh -= 8) {
                if (tid < 256) sHist[tid] = 0;
                __syncthreads();
                members_of([&](int, bool in, uint64_t k) {
                    if (in && (k & mask) == least) atomicAdd(&sHist[(k >> sh) & 255], 1);
                });
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
                    above -= sum;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (above < need && above + c[i] >= need) sBin = 255 - 4 * lane - i, sNeed = need - above;
                        above += c[i];
                    }
                }
                __syncthreads();
                least |= (uint64_t)sBin << sh;
                mask |= 255ull << sh;
                need = sNeed;
                __syncthreads();
            }
        }
        int before = 0;
        members_of([&](int, bool in, uint64_t k) { before += (int)__popcll(__ballot(in && k == least)); });
        if (lane == 0) sWave[wv] = before;
        __syncthreads();
        before = 0;
        for (int i = 0; i < wv; i++) before += sWave[i];
        members_of([&](int word, bool in, uint64_t k) {
            const uint64_t eq = __ballot(in && k == least);
            const bool first = before + (int)__popcll(eq & ((1ull << lane) - 1)) < need;
            const uint64_t stay = __ballot(in && (k > least || (k == least && first)));
            if (lane == 0) sBits[word] |= stay;
            before += (int)__popcll(eq);
        });
        __syncthreads();
    }
    // each wave its words, after the bits of the waves before
    int mine = 0;
    for (int wd = w0 + lane; wd < w1; wd += 64) mine += (int)__popcll(sBits[wd]);
    mine = wave_sum_i32(mine);
    __syncthreads();  // (the counts of the ties are read)
    if (lane == 0) sWave[wv] = mine;
    __syncthreads();
    int at = p.sinks;
    for (int i = 0; i < wv; i++) at += sWave[i];
#pragma unroll 4
    for (int wd = w0; wd < w1; wd++) {
        const uint64_t bits = sBits[wd];
        if ((bits >> lane) & 1) kept[at + (int)__popcll(bits & ((1ull << lane) - 1))] = lo + 64 * wd + lane;
        at += (int)__popcll(bits);
    }
}

constexpr int EV_MOVE = 64;  // slots of a CTA

// A CTA 64 slots of a sequence's and kv head's new pages: where each comes from, then all at once K's chunks, a thread each, and V's, whose
// 16 positions of a dimension come from as many chunks (their bytes, or halves of them, one by one: neighbours lie in the same few lines).
template <int HD, int BITS>
__global__ __launch_bounds__(256) void pg_move_kernel(Paged a, PgEvict p, int nblk) {
    constexpr int HH = HD / 2, CH = HD / 16, ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8;
    typedef typename std::conditional<BITS == 8, v4i, v2i>::type Chunk;
    __shared__ const uint8_t *sK[EV_MOVE], *sV[EV_MOVE];  // the slot's row in K, its first byte in V; null without a page
    __shared__ int sOdd[EV_MOVE], sTo[EV_MOVE / 16];
    const int b = (int)blockIdx.x / nblk, first = ((int)blockIdx.x - b * nblk) * EV_MOVE, g = blockIdx.y, tid = threadIdx.x;
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh)), n = min(EV_MOVE, min(L, p.budget) - first);
    if (n <= 0) return;
    const int mask = (1 << a.page_sh) - 1;
    const size_t mult = (size_t)(HH << a.page_sh);
    if (tid < EV_MOVE) {
        const int j = tid < n ? p.kept[((size_t)b * a.nkv + g) * p.budget + first + tid] : -1;
        const int id = tid < n ? p.to[(size_t)b * p.to_pages + ((first + tid) >> a.page_sh)] : -1;
        const int from = j < 0 ? -1 : pg_page(a, b, j >> 4), sl = j & mask, to_sl = (first + tid) & mask;
        const bool there = (unsigned)id < (unsigned)a.pages;
        const size_t part = ((size_t)max(from, 0) * a.nkv + g) * (size_t)a.part;
        sK[tid] = from < 0 ? nullptr : a.k + part + sl * ROWB;
        const int e = sl & 15;
        sV[tid] = from < 0 ? nullptr : a.v + part + (size_t)(sl >> 4) * 16 * ROWB + (BITS == 8 ? e : 4 * (e >> 3) + (e & 3));
        sOdd[tid] = BITS == 8 ? 0 : 4 * ((e >> 2) & 1);
        if ((tid & 15) == 0) sTo[tid >> 4] = there ? id : -1;
        if (there) {
            p.w[(((size_t)id * a.nkv + g) << a.page_sh) + to_sl] = from < 0 ? 0 : p.w[(((size_t)from * a.nkv + g) << a.page_sh) + sl];
            if constexpr (BITS == 4) {
                const size_t to = ((size_t)id * a.nkv + g) * (size_t)a.part + mult + to_sl;
                a.k[to] = from < 0 ? 0 : a.k[part + mult + sl];
                a.v[to] = from < 0 ? 0 : a.v[part + mult + sl];
            }
        }
    }
    __syncthreads();
    auto to_of = [&](int r) { return ((size_t)sTo[r >> 4] * a.nkv + g) * (size_t)a.part; };
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        const int it = tid + 256 * i, r = it / CH, c = it % CH;
        if (r >= n || sTo[r >> 4] < 0) continue;
        Chunk x = {};
        if (sK[r]) x = *reinterpret_cast<const Chunk*>(sK[r] + c * CHB);
        *reinterpret_cast<Chunk*>(a.k + to_of(r) + ((first + r) & mask) * ROWB + c * CHB) = x;
    }
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        const int it = tid + 256 * i, d = it % HD, r0 = 16 * (it / HD), left = n - r0;
        if (left <= 0 || sTo[r0 >> 4] < 0) continue;
        uint32_t v[16];
#pragma unroll
        for (int r = 0; r < 16; r++) v[r] = sV[r0 + r] ? sV[r0 + r][d * CHB] : 0;
        uint8_t* const out = a.v + to_of(r0) + (size_t)(((first + r0) & mask) >> 4) * 16 * ROWB + d * CHB;
        if constexpr (BITS == 8) {
            v4i x = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 16; r++) x[r >> 2] |= (int)(v[r] << (8 * (r & 3)));
            if (left >= 16) {
                *reinterpret_cast<v4i*>(out) = x;
            } else {
                for (int r = 0; r < left; r++) out[r] = (uint8_t)((uint32_t)x[r >> 2] >> (8 * (r & 3)));
            }
        } else {
            uint32_t x[2] = {0, 0}, keep[2] = {0, 0};
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int sh = 8 * (r & 3) + 4 * ((r >> 2) & 1);
                x[r >> 3] |= ((v[r] >> sOdd[r0 + r]) & 15) << sh;
                if (r >= left) keep[r >> 3] |= 15u << sh;
            }
            uint32_t* const to = reinterpret_cast<uint32_t*>(out);
#pragma unroll
            for (int h = 0; h < 2; h++) to[h] = left >= 16 ? x[h] : ((x[h] & ~keep[h]) | (to[h] & keep[h]));
        }
    }
}

}  // namespace

hipError_t launch_pg_evict(const Paged& a, int hd, int bits, const int32_t* to, int budget, int recent, int sinks, int32_t* kept,
                           int64_t* w, hipStream_t s) {
    const int page = 1 << a.page_sh, nblk = (budget + EV_MOVE - 1) / EV_MOVE;
    const PgEvict p = {to, (budget + page - 1) / page, budget, recent, sinks, kept, w};
    const size_t words = ((size_t)a.max_pages * page + 63) / 64 * 8;  // at most 64 KB
    pg_select_kernel<<<dim3((unsigned)a.nkv, (unsigned)a.seqs), dim3(EV_NT), words, s>>>(a, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    auto go = [&](auto kern) {
        kern<<<dim3((unsigned)(a.seqs * nblk), (unsigned)a.nkv), dim3(256), 0, s>>>(a, p, nblk);
        return hipGetLastError();
    };
    if (hd == 64) return bits == 8 ? go(pg_move_kernel<64, 8>) : go(pg_move_kernel<64, 4>);
    return bits == 8 ? go(pg_move_kernel<128, 8>) : go(pg_move_kernel<128, 4>);
}

}  // namespace kt
