// Eviction from paged KV caches by accumulated attention weight on gfx950 (kt_hip_dec_evict_paged, stated in include/kt_hip.h): for
// each sequence and kv head the heaviest positions are chosen, then their k, v, multipliers and sums go to other pages. 64 sequences of about
// 2200 cut to 1024 (2 kv heads of 64): 10 to 11 us to choose, a chain of two passes over the sums (in registers), a histogram and a ranking with
// a CTA to two CUs; 9.7 us to move 34 MB; 64 of 8000 cut to 4096 41.8 us for 142 MB, with the rest of the lines that kept bytes lie in some
// 210 at 5 TB/s (128 or 256 slots a CTA: no change). One of 131000 to 16384 in 4 bits: 21 us to choose, 5.6 to move.
//
// These are sums spread as attention leaves them. Many positions in the bin of the least sum that stays cost more: up to EV_CANDS of
// them are compared with each other, by one lane each where they are over 512 (64 x 2200 to 1024, seven in ten sums 0 and the cut among them: 63 us to choose
// against 11), past that the sums are read again for each step (64 x 8000 to 4096 of the same kind 22.6 us against 13.1), and by each of
// several CTAs (one of 131000 to 16384, 95 in 100 sums 0: 136 us in the last of the four launches against 7.9; all sums within one power
// of two: 312).

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
constexpr int EV_U = 8;         // words of a wave in flight: 64 positions each

// The bin of a sum: the values below 128 one each, from there on 64 to a power of two; bin 1 for negative ones, which only a caller's own
// sums hold, and bin 0 for positions without a page, below them all. (With 32 to a power of two a bin of 131000 positions has twice the
// members to rank: to 16384 16.9 us for the last two steps against 13.9; of 64 x 2200, in one CTA each, no change. Where few members are to be
// ranked the wider histogram only costs: the figures in brackets above ev_shared.)
__device__ __forceinline__ int weight_bin(int64_t w, bool page) {
    const uint64_t m = (uint64_t)w;
    const int sh = max(0, 57 - __clzll((long long)(m | 1)));
    return page ? (w >= 0 ? 2 + 64 * sh + (int)(m >> sh) : 1) : 0;
}
// The order of a bin's sums as unsigned numbers (those of positions without a page, which are read as 0, are equal).
__device__ __forceinline__ uint64_t weight_key(int64_t w) { return (uint64_t)w ^ (1ull << 63); }

// What several CTAs of a sequence and kv head share where its positions are too many for one: in the workspace, for each.
struct EvShared {
    int* hist;       // [EV_BINS], then the count of candidates
    uint64_t* key;   // [EV_CANDS]
    int* at;         // [EV_CANDS]
    uint64_t* bits;  // a word for 64 positions
};
struct EvSpace {
    char* base;
    size_t stride, key, at, bits;
    __host__ __device__ EvShared of(size_t i) const {
        char* const x = base + i * stride;
        return {(int*)x, (uint64_t*)(x + key), (int*)(x + at), (uint64_t*)(x + bits)};
    }
};

// The positions that a sequence and kv head choose from, and the words of 64 that a wave of a CTA reads, eight at a time.
struct EvSweep {
    const Paged& a;
    const int32_t* table;
    const int64_t* sums;
    uint32_t stride;
    int lo, hi, lane;
    int64_t x[EV_U];
    uint32_t page;  // bit u: the position of word u has a page
    __device__ EvSweep(const Paged& a, const PgEvict& p, int b, int g, int lo, int hi)
        : a(a), table(a.table + (size_t)b * a.max_pages), sums(p.w + ((size_t)g << a.page_sh)),
          stride((uint32_t)a.nkv << a.page_sh), lo(lo), hi(hi), lane(threadIdx.x & 63), page(0) {}
    __device__ void load(int word, int end) {
        int id[EV_U];
        page = 0;
#pragma unroll
        for (int u = 0; u < EV_U; u++) {
            const int j = lo + 64 * (word + u) + lane;
            id[u] = -1;
            if (word + u < end && j < hi) id[u] = table[j >> a.page_sh];
        }
#pragma unroll
        for (int u = 0; u < EV_U; u++) {
            const int j = lo + 64 * (word + u) + lane;
            const bool ok = (unsigned)id[u] < (unsigned)a.pages;
            page |= (uint32_t)ok << u;
            x[u] = 0;
            if (ok) x[u] = sums[(uint64_t)(uint32_t)id[u] * stride + (uint32_t)(j & ((1 << a.page_sh) - 1))];
        }
    }
    // f(word, position or -1, sum, whether it has a page) for the loaded words below `end`, all lanes at work
    template <class F>
    __device__ void each(int word, int end, F f) {
#pragma unroll
        for (int u = 0; u < EV_U; u++) {
            const int j = lo + 64 * (word + u) + lane;
            if (word + u < end) f(word + u, j < hi ? j : -1, x[u], (bool)((page >> u) & 1));
        }
    }
    template <class F>
    __device__ void all(int w0, int w1, F f) {
        for (int w = w0; w < w1; w += EV_U) load(w, w1), each(w, w1, f);
    }
};

// A position's bin counted. Lanes with the first lane's bin are counted together: one bin may have most positions (zeros).
__device__ __forceinline__ void count_bin(int* hist, int bin) {
    const int one = __builtin_amdgcn_readfirstlane(bin), same = (int)__popcll(__ballot(bin == one));
    if ((threadIdx.x & 63) == 0 && one >= 0) atomicAdd(&hist[one], same);
    if (bin != one && bin >= 0) atomicAdd(&hist[bin], 1);
}

// Of a histogram, from the largest bin: the bin that the most-th position is in, and how many of the bin those are. By the whole CTA.
struct EvBin {
    int bin, need, members;
};
__device__ __forceinline__ EvBin find_bin(const int* hist, int most) {
    __shared__ int sWave[EV_WAVES];
    __shared__ EvBin sOut;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    constexpr int N = EV_BINS / EV_NT;
    int c[N], sum = 0;
#pragma unroll
    for (int i = 0; i < N; i++) c[i] = hist[EV_BINS - 1 - N * tid - i], sum += c[i];
    int above = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(above, o);
        above += lane >= o ? v : 0;
    }
    if (lane == 63) sWave[wv] = above;
    above -= sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EV_WAVES; i++) above += i < wv ? sWave[i] : 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (above < most && above + c[i] >= most) sOut = {EV_BINS - 1 - N * tid - i, most - above, c[i]};
        above += c[i];
    }
    __syncthreads();
    return sOut;
}

// Several CTAs a sequence and kv head: the histogram cleared, its parts added, and the positions above its bin noted, the bin's own listed.
__global__ __launch_bounds__(256) void pg_select_clear_kernel(EvSpace sp) {
    int* const hist = sp.of(blockIdx.x).hist;
    for (int i = threadIdx.x; i <= EV_BINS; i += 256) hist[i] = 0;
}

// Words of a wave here, four: us of the two kernels with two / four / eight for one sequence of 131000 (2 kv heads) 10.8 / 12.0 / 14.3, 16 of
// them 33.4 / 25.0 / 24.5, 64 of 32000 32.0 / 24.4 / 23.9.
constexpr int EV_PU = 4, EV_PART = EV_WAVES * EV_PU;

template <bool MARK>
__global__ __launch_bounds__(EV_NT) void pg_select_part_kernel(Paged a, PgEvict p, EvSpace sp) {
    __shared__ int sHist[MARK ? 1 : EV_BINS];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.y, b = blockIdx.z;
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh));
    const int lo = p.sinks, hi = L - p.recent, most = p.budget - p.sinks - p.recent;
    const int words = (hi - lo + 63) / 64, w0 = (int)blockIdx.x * EV_PART + wv * EV_PU, w1 = min(w0 + EV_PU, words);
    if (L <= p.budget || most == 0 || (int)blockIdx.x * EV_PART >= words) return;
    EvSweep s(a, p, b, g, lo, hi);
    s.load(w0, w1);
    const EvShared sh = sp.of((size_t)b * a.nkv + g);
    if constexpr (!MARK) {
        for (int i = tid; i < EV_BINS; i += EV_NT) sHist[i] = 0;
        __syncthreads();
        s.each(w0, w1, [&](int, int j, int64_t x, bool page) { count_bin(sHist, j < 0 ? -1 : weight_bin(x, page)); });
        __syncthreads();
        for (int i = tid; i < EV_BINS; i += EV_NT)
            if (sHist[i]) atomicAdd(&sh.hist[i], sHist[i]);
    } else {
        const EvBin e = find_bin(sh.hist, most);
        s.each(w0, w1, [&](int word, int j, int64_t x, bool page) {
            const int bin = j < 0 ? -1 : weight_bin(x, page);
            const uint64_t stay = __ballot(bin > e.bin || (e.need == e.members && bin == e.bin));
            if (lane == 0) sh.bits[word] = stay;
            if (bin == e.bin && e.need < e.members && e.members <= EV_CANDS) {
                const int c = atomicAdd(&sh.hist[EV_BINS], 1);
                if (c < EV_CANDS) sh.key[c] = weight_key(x), sh.at[c] = j;  // (more only if the sums change under the call)
            }
        });
    }
}

// Which positions stay, a CTA a sequence and kv head: the sums' histogram says in which bin the least that stays lies and how many of
// the bin do; a bit is noted for each position above that bin, and its members are ranked against each other (their sums, then their
// positions). The bits give the order. SHARED: histogram, bits and members are in the workspace, and each of the CTAs (grid x) writes its
// share of the positions.
template <bool SHARED>
__global__ __launch_bounds__(EV_NT) void pg_select_kernel(Paged a, PgEvict p, EvSpace sp) {
    extern __shared__ uint64_t sBits[];  // a word for 64 positions
    __shared__ int sHist[EV_BINS];
    __shared__ uint64_t sKey[EV_CANDS], sAnd[EV_WAVES], sOr[EV_WAVES];
    __shared__ int sAt[EV_CANDS], sWave[EV_WAVES], sBin, sNeed, sCount;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.y, b = blockIdx.z;
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh)), part = (int)blockIdx.x, parts = (int)gridDim.x;
    int32_t* const kept = p.kept + ((size_t)b * a.nkv + g) * p.budget;
    if (L <= p.budget) {
        for (int i = part * EV_NT + tid; i < p.budget; i += parts * EV_NT) kept[i] = i < L ? i : -1;
        return;
    }
    const int lo = p.sinks, hi = L - p.recent, most = p.budget - p.sinks - p.recent;
    for (int i = part * EV_NT + tid; i < p.sinks; i += parts * EV_NT) kept[i] = i;
    for (int i = part * EV_NT + tid; i < p.recent; i += parts * EV_NT) kept[p.budget - p.recent + i] = hi + i;
    if (most == 0) return;
    // each wave's neighbouring words
    const int words = (hi - lo + 63) / 64, seg = (words + EV_WAVES - 1) / EV_WAVES, w0 = min(wv * seg, words), w1 = min(w0 + seg, words);
    EvSweep s(a, p, b, g, lo, hi);
    EvBin e;
    if constexpr (SHARED) {
        const EvShared sh = sp.of((size_t)b * a.nkv + g);
        e = find_bin(sh.hist, most);
        for (int i = tid; i < words; i += EV_NT) sBits[i] = sh.bits[i];
        if (e.need < e.members && tid < min(e.members, EV_CANDS)) sKey[tid] = sh.key[tid], sAt[tid] = sh.at[tid];
    } else {
        s.load(w0, w1);
        for (int i = tid; i < EV_BINS; i += EV_NT) sHist[i] = 0;
        if (tid == 0) sCount = 0;
        __syncthreads();
        auto count = [&](int, int j, int64_t x, bool page) { count_bin(sHist, j < 0 ? -1 : weight_bin(x, page)); };
        s.each(w0, w1, count);
        if (seg > EV_U) s.all(w0 + EV_U, w1, count);
        __syncthreads();
        e = find_bin(sHist, most);
        auto mark = [&](int word, int j, int64_t x, bool page) {
            const int bin = j < 0 ? -1 : weight_bin(x, page);
            const uint64_t stay = __ballot(bin > e.bin || (e.need == e.members && bin == e.bin));
            if (lane == 0) sBits[word] = stay;
            if (bin == e.bin && e.need < e.members && e.members <= EV_CANDS) {
                const int c = atomicAdd(&sCount, 1);
                if (c < EV_CANDS) sKey[c] = weight_key(x), sAt[c] = j;  // (more only if the sums change under the call)
            }
        };
        if (seg > EV_U) s.all(w0, w1, mark);
        else s.each(w0, w1, mark);  // (still in registers)
    }
    __syncthreads();
    int need = e.need;
    if (need < e.members && e.members <= EV_CANDS) {
        // a few lanes a member, as many as there are threads for
        const int lg = min(6, 31 - __clz(EV_NT / e.members)), per = 1 << lg, m = tid >> lg;
        const uint64_t mine = sKey[m];
        const int at = sAt[m];
        int rank = 0;
#pragma unroll 8
        for (int i = tid & (per - 1); i < e.members; i += per) rank += (sKey[i] > mine) | ((sKey[i] == mine) & (sAt[i] < at));
        for (int o = 1; o < per; o <<= 1) rank += __shfl_xor(rank, o);
        if (m < e.members && rank < need && (tid & (per - 1)) == 0 && (unsigned)(at - lo) < (unsigned)(hi - lo))  // (fewer if they change)
            atomicOr(reinterpret_cast<unsigned long long*>(&sBits[(at - lo) >> 6]), 1ull << ((at - lo) & 63));
        __syncthreads();
    } else if (need < e.members) {
        // More members than that, equal ones for the most part: the least sum that stays, eight bits at a time from the first that the
        // members differ in; then those above it and the first of those equal to it.
        uint64_t both = ~0ull, any = 0;
        auto members_of = [&](auto f) {
            s.all(w0, w1, [&](int word, int j, int64_t x, bool page) { f(word, j >= 0 && weight_bin(x, page) == e.bin, weight_key(x)); });
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
    // each wave its words (of the CTA's share), after the bits of all words before
    const int share = (words + parts - 1) / parts, s0 = min(part * share, words), s1 = min(s0 + share, words);
    const int sseg = (s1 - s0 + EV_WAVES - 1) / EV_WAVES, v0 = min(s0 + wv * sseg, s1), v1 = min(v0 + sseg, s1);
    int bits_before = 0, mine = 0;
    if constexpr (SHARED)
        for (int i = tid; i < s0; i += EV_NT) bits_before += (int)__popcll(sBits[i]);
    for (int i = v0 + lane; i < v1; i += 64) mine += (int)__popcll(sBits[i]);
    mine = wave_sum_i32(mine);
    __syncthreads();  // (the counts of the ties are read)
    if (lane == 0) sWave[wv] = mine;
    if constexpr (SHARED) {
        bits_before = wave_sum_i32(bits_before);
        if (lane == 0) sAnd[wv] = (uint64_t)bits_before;
    }
    __syncthreads();
    int at = p.sinks;
#pragma unroll
    for (int i = 0; i < EV_WAVES; i++) {
        at += i < wv ? sWave[i] : 0;
        if constexpr (SHARED) at += (int)sAnd[i];
    }
#pragma unroll 4
    for (int i = v0; i < v1; i++) {
        const uint64_t bits = sBits[i];
        const int to = at + (int)__popcll(bits & ((1ull << lane) - 1));
        if (((bits >> lane) & 1) && to < p.budget - p.recent) kept[to] = lo + 64 * i + lane;
        at += (int)__popcll(bits);
    }
}

constexpr int EV_MOVE = 64;   // slots of a CTA
constexpr int EV_CHUNKS = 4;  // chunks' rows of V that a wave holds in LDS

// A CTA 64 slots of a sequence's and kv head's new pages: where each comes from, then K's chunks, a thread each, and V's, by a wave the 16
// slots of 64 dimensions. What these come from are chunks of 16 positions: of a few, where most positions stay, the rows go to LDS whole
// and a lane picks its dimension's bytes (or halves of them) there; of more, each slot's bytes are loaded, neighbours in the same lines. us
// with up to 4 chunks in LDS / bytes alone (up to 6: within a tenth, or more): 64 sequences of 8000 to their last 4096 34.6 / 48.8, to the
// heaviest 4096 41.8 / 48.7 (4 bits 35.6 / 43.7), to 2000 30.1 / 30.4, to 1000 19.1 / 18.8; of 2200 to 1024 9.8 / 13.6.
template <int HD, int BITS>
__global__ __launch_bounds__(256) void pg_move_kernel(Paged a, PgEvict p, int nblk) {
    constexpr int HH = HD / 2, CH = HD / 16, ROWB = BITS == 8 ? HD : HH, CHB = BITS == 8 ? 16 : 8, U = HD / 64;
    typedef typename std::conditional<BITS == 8, v4i, v2i>::type Chunk;
    __shared__ const uint8_t *sK[EV_MOVE], *sV[EV_MOVE];  // the slot's row in K, its chunks' row in V; null without a page
    __shared__ int sE[EV_MOVE], sTo[EV_MOVE / 16];        // its byte of a chunk, with 4 bits and 4 more where it is the high half
    __shared__ __attribute__((aligned(16))) int8_t sChunk[4][EV_CHUNKS * 64 * CHB];
    const int b = (int)blockIdx.x / nblk, first = ((int)blockIdx.x - b * nblk) * EV_MOVE, g = blockIdx.y, tid = threadIdx.x;
    const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int L = max(0, min(pg_len(a, b), a.max_pages << a.page_sh)), n = min(EV_MOVE, min(L, p.budget) - first);
    if (n <= 0 || a.pages == 0) return;
    const int mask = (1 << a.page_sh) - 1;
    const size_t mult = (size_t)(HH << a.page_sh);
    if (tid < EV_MOVE) {
        const int j = tid < n ? p.kept[((size_t)b * a.nkv + g) * p.budget + first + tid] : -1;
        const int id = tid < n ? p.to[(size_t)b * p.to_pages + ((first + tid) >> a.page_sh)] : -1;
        const int from = (unsigned)j < (unsigned)L ? pg_page(a, b, j >> 4) : -1, sl = j & mask, to_sl = (first + tid) & mask;
        const bool there = (unsigned)id < (unsigned)a.pages;
        const size_t part = ((size_t)max(from, 0) * a.nkv + g) * (size_t)a.part;
        sK[tid] = from < 0 ? nullptr : a.k + part + sl * ROWB;
        const int e = sl & 15;
        sV[tid] = from < 0 ? nullptr : a.v + part + (size_t)(sl >> 4) * 16 * ROWB;
        sE[tid] = BITS == 8 ? e : (4 * (e >> 3) + (e & 3)) | ((e & 4) << 4);
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
    Chunk k[U];
#pragma unroll
    for (int i = 0; i < U; i++) {  // (what is not there is read from the pool's start)
        const int it = tid + 256 * i;
        const uint8_t* const from = sK[it / CH];
        k[i] = *reinterpret_cast<const Chunk*>(from ? from + it % CH * CHB : a.k);
    }
    int8_t* const lds = sChunk[w];
#pragma unroll 1
    for (int i = 0; i < U; i++) {
        const int r0 = 16 * ((w + 4 * i) / U), d0 = 64 * ((w + 4 * i) % U), left = n - r0;
        // the 16 slots' chunks and bytes, a lane each; the slots whose chunk is not that of the slot before
        const uint64_t from = (uint64_t)sV[r0 + (lane & 15)], before = __shfl_up(from, 1);
        const int e = sE[r0 + (lane & 15)];
        const uint32_t news = ((uint32_t)__ballot(from != before) & 0xFFFF) | 1, there = (uint32_t)__ballot(from != 0) & 0xFFFF;
        auto base = [&](int r) {
            return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)from, r) |
                                                    (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(from >> 32), r) << 32);
        };
        uint32_t v[16];
        if (__builtin_popcount(news) <= EV_CHUNKS) {
            uint32_t more = news;
#pragma unroll
            for (int c = 0; c < EV_CHUNKS; c++) {
                if (more == 0) break;
                const int r = __builtin_ctz(more);
                more &= more - 1;
                if (((there >> r) & 1) && (BITS == 8 || lane < 32)) dma16(make_rsrc(base(r) + d0 * CHB, 64 * CHB), lds + c * 64 * CHB, 16 * lane, 0);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int r = 0; r < 16; r++)
                v[r] = (uint8_t)lds[(__builtin_popcount(news & ((2u << r) - 1)) - 1) * 64 * CHB + (__builtin_amdgcn_readlane(e, r) & 15) + CHB * lane];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before a wave's next chunks take their place
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) v[r] = ((there >> r) & 1 ? base(r) : a.v)[(d0 + lane) * CHB + (__builtin_amdgcn_readlane(e, r) & 15)];
        }
#pragma unroll
        for (int r = 0; r < 16; r++) v[r] = (there >> r) & 1 ? v[r] : 0;
        if (i == 0) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int it = tid + 256 * u, r = it / CH, c = it % CH;
                if (r < n && sTo[r >> 4] >= 0)
                    *reinterpret_cast<Chunk*>(a.k + to_of(r) + ((first + r) & mask) * ROWB + c * CHB) = sK[r] ? k[u] : Chunk{};
            }
        }
        if (left <= 0 || sTo[r0 >> 4] < 0) continue;
        uint8_t* const out = a.v + to_of(r0) + (size_t)(((first + r0) & mask) >> 4) * 16 * ROWB + (d0 + lane) * CHB;
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
                x[r >> 3] |= ((v[r] >> (__builtin_amdgcn_readlane(e, r) >> 4)) & 15) << sh;
                if (r >= left) keep[r >> 3] |= 15u << sh;
            }
            uint32_t* const to = reinterpret_cast<uint32_t*>(out);
#pragma unroll
            for (int h = 0; h < 2; h++) to[h] = left >= 16 ? x[h] : ((x[h] & ~keep[h]) | (to[h] & keep[h]));
        }
    }
}

EvSpace ev_space(int64_t max_pos) {
    const size_t key = (EV_BINS + 2) * 4, at = key + EV_CANDS * 8, bits = at + EV_CANDS * 4;
    return {nullptr, (bits + (size_t)(max_pos + 63) / 64 * 8 + 255) / 256 * 256, key, at, bits};
}

// One CTA a sequence and kv head takes one launch, and a long one's sums alone: us for one sequence of 4000 positions (2 kv heads) 8.4, of 8000
// 11.3, 16000 19.2, 24000 25, 32000 31, 131000 114, for 64 of 4000 9.2, of 16000 21.1. Several take four launches (and of the caller 10 us
// more): one of 25000 17.9, 32000 17.8, 131000 18.2 (19.0 with the bins as they are now), 64 of 32000 36.6 (39.2). The rule goes by the
// table's width, which is all that the host knows: 63 sequences of 1000 beside one of 17000 take the four launches too, 21 us against 7.9
// for 64 of 1000.
bool ev_shared(int64_t max_pos) { return max_pos > 16384; }

}  // namespace

size_t pg_evict_workspace(int64_t seqs, int64_t nkv, int64_t max_pos) {
    return ev_shared(max_pos) ? std::max<size_t>(256, (size_t)seqs * nkv * ev_space(max_pos).stride) : 256;  // (0 says a shape refused)
}

hipError_t launch_pg_evict(const Paged& a, int hd, int bits, const int32_t* to, int budget, int recent, int sinks, int32_t* kept,
                           int64_t* w, void* ws, hipStream_t s) {
    const int page = 1 << a.page_sh, nblk = (budget + EV_MOVE - 1) / EV_MOVE;
    const int64_t max_pos = (int64_t)a.max_pages * page;
    const PgEvict p = {to, (budget + page - 1) / page, budget, recent, sinks, kept, w};
    const size_t lds = (size_t)(max_pos + 63) / 64 * 8;  // the bits: at most 64 KB
    EvSpace sp = ev_space(max_pos);
    sp.base = (char*)ws;
    if (ev_shared(max_pos)) {
        const dim3 grid((unsigned)((max_pos + 64 * EV_PART - 1) / (64 * EV_PART)), (unsigned)a.nkv, (unsigned)a.seqs);
        pg_select_clear_kernel<<<dim3((unsigned)(a.seqs * a.nkv)), dim3(256), 0, s>>>(sp);
        pg_select_part_kernel<false><<<grid, dim3(EV_NT), 0, s>>>(a, p, sp);
        pg_select_part_kernel<true><<<grid, dim3(EV_NT), 0, s>>>(a, p, sp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        // a CTA a CU: each repeats the choice among the bin's members (16 sequences of 131000 with 8 / 16 / 32 CTAs each 9.3 / 14.5 / 25 us, 64
        // of 32000 with 1 / 2 / 4 / 8 9.8 / 8.4 / 13 / 22.4)
        const unsigned parts = (unsigned)std::min<int64_t>(64, std::max<int64_t>(1, 256 / ((int64_t)a.seqs * a.nkv)));
        pg_select_kernel<true><<<dim3(parts, grid.y, grid.z), dim3(EV_NT), lds, s>>>(a, p, sp);
    } else {
        pg_select_kernel<false><<<dim3(1, (unsigned)a.nkv, (unsigned)a.seqs), dim3(EV_NT), lds, s>>>(a, p, sp);
    }
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
