// The int8 decoder's paged KV caches on gfx950: the new rows' RoPE with the write of k and v to their pages (8 bits, or
// quantised to 4), the read back, and the greedy choice of a batch's rows. The attention is kt_paged_attn.hip. The rules
// and the layout of the pools are stated with kt_hip_dec_*_paged in include/kt_hip.h; the decoder these serve is the one of
// kt_decoder.hip (DecoderModel, crates/01-engine/kt-core/src/model.rs:168-188, 290-353), for many sequences at once.

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "kt_dpp.h"
#include "kt_paged.h"
#include "kt_w12_core.h"

namespace kt {

namespace {

// The low bytes of four ints.
__device__ __forceinline__ int pack4(const int (&v)[4]) {
    return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm((uint32_t)v[3], (uint32_t)v[2], 0x0C0C0400),
                                      __builtin_amdgcn_perm((uint32_t)v[1], (uint32_t)v[0], 0x0C0C0400), 0x05040100);
}

template <int SH = 14>
__device__ __forceinline__ int rope_round(int v) {  // clamp(round_half_away(v / 2^SH)), |v| <= 2^30
    return max(-127, min((v + (1 << (SH - 1)) + (v >> 31)) >> SH, 127));
}

__device__ __forceinline__ int byte_of(int w, int i) { return (int)(int8_t)(w >> (8 * i)); }

// The multiplier of a row whose largest magnitude is `top` (0 .. 128): ceil(8 top / 7), at most 147.
__device__ __forceinline__ int mult4(int top) { return (8 * top + 6) / 7; }

// 2^20 / (2 m) rounded up: n / (2 m) = (n inv) >> 20 for 0 <= n <= 2195 (n inv / 2^20 exceeds n / (2 m) by less than
// n / 2^20 < 1 / 294 <= 1 / (2 m), and n inv < 2^31 from m = 2 on, the least multiplier of a row that is not zeros).
__device__ __forceinline__ int mult4_inv(int m) { return m ? ((1 << 20) + 2 * m - 1) / (2 * m) : 0; }

// clamp(round_half_away(8 x / m), +-7): floor((16 |x| + m) / (2 m)); 0 where m is 0 (x is then too).
__device__ __forceinline__ int code4(int x, int m, int inv) {
    const int a = x < 0 ? -x : x;
    int c = ((16 * a + m) * inv) >> 20;
    c = c > 7 ? 7 : c;
    return x < 0 ? -c : c;
}

// clamp(round_half_away(c m / 8)).
__device__ __forceinline__ int value4(int c, int m) {
    const int t = c * m;
    int q = ((t < 0 ? -t : t) + 4) >> 3;
    q = q > 127 ? 127 : q;
    return t < 0 ? -q : q;
}

// What the append with the heads' norms has beside the plain one.
struct PgNorm {
    const int16_t *q, *k;  // weights, or null
    const int32_t* shift;  // or null
    int64_t* w;            // the sums of weights of a slot, or null
};

// floor(sqrt(v)), v <= 2^30: the float root is off by less than one.
__device__ __forceinline__ int isqrt30(int v) {
    int r = (int)__builtin_amdgcn_sqrtf((float)v);
    r -= r * r > v;
    r += (r + 1) * (r + 1) <= v;
    return r;
}

// clamp(round_half_away(128 y / R), +-16383), |y| <= 2^22, 1 <= R <= 2^15, in floats: c is 128 / R short of it by 2^-21 to 2^-20 of itself,
// more than what the product's rounding adds, so the floor (below 2^14) is the whole one or one less, which the remainder, exact in an
// fma, says. r = R / 128.
__device__ __forceinline__ int norm_code(int y, float r, float c) {
    const float a = __builtin_fabsf((float)y);
    float q = __builtin_floorf(__builtin_fmaf(a, c, 0.5f));
    q += __builtin_fmaf(-q, r, a) >= 0.5f * r ? 1.0f : 0.0f;
    return (int)__builtin_copysignf(__builtin_fminf(q, 16383.0f), (float)y);
}

// One CTA per (block of 16 positions that a sequence's rows reach, kv head): it rotates the q heads of the group and the k
// head of the rows in the block, four pairs a thread, stages k and v in LDS and writes the block's bytes. The block is the
// unit because V's chunk is 16 positions of a dimension, in 4 bits with two positions to a byte: what rows fill goes out in
// dwords, what only some of them belong to byte by byte (4 bits: read, merged and written back by its only owner).
//
// Bound by the chain of one block (batch, rows, RoPE, LDS, pages) while few are at work: 64 single tokens 4.0 us for 0.15 MB,
// 4 x 512 rows (14 heads over 2, hd 64) 5.9 us for 4.8 MB, where waves wait 60 % of their time and vector instructions take 0.36
// of the busy time; by vector instructions where CTAs fill the CUs: 3 x 4000 rows (hd 64) 11.3 us for 31 MB, 0.69 busy with 16 a
// value of qkv, and 2048 rows in 4 bits (16 heads over 4, hd 128; two CTAs a CU, one round) 9.8 us for 12 MB, 0.66 with 30.
// LDS is busy less than a tenth of the time in each.
//
// NORM: a head's values are in the HH / 4 neighbouring lanes that hold its pairs, so its sum of squares is a few DPP steps. Its quotients and
// the wider products make it vector instructions again: 4 x 512 rows (16 heads over 4, hd 128) 11.5 us for 13 MB, 0.69 busy with 31 a value of
// qkv; a chunk of 2048 in 4 bits 12.0 us, 0.72 with 43; 64 single tokens 4.4 us.
template <int HD, int BITS, int NT, bool NORM>
__global__ __launch_bounds__(NT) void pg_append_kernel(Paged a, const int8_t* __restrict__ qkv, int64_t stride, int nh,
                                                        const int16_t* __restrict__ cosT,
                                                        const int16_t* __restrict__ sinT, int max_pos,
                                                        int8_t* __restrict__ q, int64_t q_stride, PgNorm nm) {
    constexpr int HH = HD / 2, CH = HD / 16;
    __shared__ __attribute__((aligned(16))) int8_t sKV[2][16][HD];
    __shared__ int sM[2][16], sInv[2][16];
    const int tid = threadIdx.x, g = blockIdx.y, rep = nh / a.nkv;
    int first = 0;
    const int b = pg_tile_seq(a, (int)blockIdx.x, 1, 16, 2, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    const int blk = (s.p0 >> 4) + ((int)blockIdx.x - first);
    const int lo = max(16 * blk, s.p0), hi = min(16 * blk + 16, s.p0 + s.n);
    if (lo >= hi) return;
    // the rows whose position the tables and the caches have
    int cap = min(max_pos, a.max_pages << a.page_sh), vlo = max(lo, 0), shift = 0;
    if constexpr (NORM) {
        if (nm.shift) shift = max(-(1 << 30), min(nm.shift[b], 1 << 30));
        const int64_t left = (int64_t)max_pos - shift;
        cap = left < (a.max_pages << a.page_sh) ? (int)left : a.max_pages << a.page_sh;
        vlo = max(vlo, -shift);
    }
    vlo = min(vlo, hi);  // (0 <= vhi - vlo <= 16 wherever the block is)
    const int vhi = max(min(hi, cap), vlo);
    for (int i = tid; i < (vhi - vlo) * CH; i += NT) {
        const int p = vlo + i / CH, c = i % CH;
        const int8_t* src = qkv + (size_t)(s.t0 + (p - s.p0)) * stride + (nh + a.nkv + g) * HD + 16 * c;
        *reinterpret_cast<v4i*>(&sKV[1][p & 15][16 * c]) = *reinterpret_cast<const v4i*>(src);
    }
    // a thread's dimensions are the same ones in all of its turns, and so are their norms' weights
    [[maybe_unused]] v2i wq[2], wk[2];
    if constexpr (NORM) {
        const int d = 4 * (tid % (HH / 4));
        if (nm.q) wq[0] = *reinterpret_cast<const v2i*>(nm.q + d), wq[1] = *reinterpret_cast<const v2i*>(nm.q + d + HH);
        if (nm.k) wk[0] = *reinterpret_cast<const v2i*>(nm.k + d), wk[1] = *reinterpret_cast<const v2i*>(nm.k + d + HH);
    }
    const int items = (hi - lo) * (rep + 1) * (HH / 4);
    const uint32_t inv = 0xFFFFFFFFu / (uint32_t)(rep + 1) + 1;  // x / (rep + 1) = x inv >> 32 while x (rep + 1) < 2^32
    for (int i = tid; i < items; i += NT) {
        const int c = i % (HH / 4), x4 = i / (HH / 4), r = (int)__umulhi((uint32_t)x4, inv);
        const int hv = x4 - r * (rep + 1), p = lo + r;
        const size_t t = (size_t)(s.t0 + (p - s.p0));
        const bool live = p >= vlo && p < vhi;
        int xs[4] = {}, ys[4] = {};
        if (live) {
            const int8_t* src = qkv + t * stride + (hv < rep ? g * rep + hv : nh + g) * HD + 4 * c;
            const int xa = *reinterpret_cast<const int*>(src), xb = *reinterpret_cast<const int*>(src + HH);
            const v2i C = *reinterpret_cast<const v2i*>(cosT + (size_t)(p + shift) * HH + 4 * c);
            const v2i S = *reinterpret_cast<const v2i*>(sinT + (size_t)(p + shift) * HH + 4 * c);
            if (NORM && (hv < rep ? nm.q : nm.k)) {
                const v2i A = hv < rep ? wq[0] : wk[0], B = hv < rep ? wq[1] : wk[1];
                uint32_t V = (uint32_t)__builtin_amdgcn_sdot4(xa, xa, __builtin_amdgcn_sdot4(xb, xb, 0, false), false);
                V += dpp32<DPP_XOR1>(V);  // (a head's lanes are all here, and all live or none)
                V += dpp32<DPP_XOR2>(V);
                V += dpp32<DPP_HALF_MIRROR>(V);
                if constexpr (HD == 128) V += dpp32<DPP_MIRROR>(V);
                const int R = max(1, isqrt30((int)(V << (HD == 64 ? 10 : 9))));
                const float r = (float)R * 0x1p-7f, inv = __builtin_amdgcn_rcpf(r) * (1 - 0x1.8p-21f);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int cc = (int)(int16_t)(C[e >> 1] >> (16 * (e & 1))), ss = (int)(int16_t)(S[e >> 1] >> (16 * (e & 1)));
                    const int u = norm_code(byte_of(xa, e) * (int)(int16_t)(A[e >> 1] >> (16 * (e & 1))), r, inv);
                    const int w = norm_code(byte_of(xb, e) * (int)(int16_t)(B[e >> 1] >> (16 * (e & 1))), r, inv);
                    xs[e] = rope_round<20>(__mul24(u, cc) - __mul24(w, ss));
                    ys[e] = rope_round<20>(__mul24(w, cc) + __mul24(u, ss));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int cc = (int)(int16_t)(C[e >> 1] >> (16 * (e & 1))), ss = (int)(int16_t)(S[e >> 1] >> (16 * (e & 1)));
                    const int u = byte_of(xa, e), w = byte_of(xb, e);
                    xs[e] = rope_round(u * cc - w * ss);
                    ys[e] = rope_round(w * cc + u * ss);
                }
            }
        }
        const int x = pack4(xs), y = pack4(ys);
        if (hv < rep) {
            int8_t* to = q + t * q_stride + (g * rep + hv) * HD + 4 * c;
            *reinterpret_cast<int*>(to) = x;
            *reinterpret_cast<int*>(to + HH) = y;
        } else if (live) {
            *reinterpret_cast<int*>(&sKV[0][p & 15][4 * c]) = x;
            *reinterpret_cast<int*>(&sKV[0][p & 15][4 * c + HH]) = y;
        }
    }
    if (vlo >= vhi) return;
    const int id = pg_page(a, b, blk);
    if (id < 0) return;
    __syncthreads();
    const int r0 = vlo & 15, r1 = vhi - 16 * blk;  // the block's rows r0 .. r1 - 1
    const size_t part = ((size_t)id * a.nkv + g) * (size_t)a.part;
    const int slot = (16 * blk) & ((1 << a.page_sh) - 1);
    if constexpr (NORM) {
        if (nm.w && tid >= r0 && tid < r1) nm.w[(((size_t)id * a.nkv + g) << a.page_sh) + slot + tid] = 0;
    }
    if constexpr (BITS == 8) {
        uint8_t* kd = a.k + part + slot * HD;
        uint8_t* vd = a.v + part + slot * HD;
        for (int i = tid; i < 16 * CH + 4 * HD; i += NT) {
            if (i < 16 * CH) {  // a chunk of K
                const int r = i / CH, c = i % CH;
                if (r >= r0 && r < r1) *reinterpret_cast<v4i*>(kd + r * HD + 16 * c) = *reinterpret_cast<const v4i*>(&sKV[0][r][16 * c]);
            } else {  // four positions of a dimension of V
                const int d = (i - 16 * CH) >> 2, r = 4 * ((i - 16 * CH) & 3);
                if (r >= r0 && r + 4 <= r1) {
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) w |= (uint32_t)(uint8_t)sKV[1][r + e][d] << (8 * e);
                    *reinterpret_cast<uint32_t*>(vd + 16 * d + r) = w;
                } else {
                    for (int e = max(r, r0); e < min(r + 4, r1); e++) vd[16 * d + e] = (uint8_t)sKV[1][e][d];
                }
            }
        }
    } else {
        constexpr int RT = HD / 4;  // threads of a row: its largest magnitude, four values each
        for (int i = tid; i < 32 * RT; i += NT) {
            const int w = i / (16 * RT), r = i / RT % 16, x = *reinterpret_cast<const int*>(&sKV[w][r][4 * (i % RT)]);
            int top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, max(byte_of(x, e), -byte_of(x, e)));
#pragma unroll
            for (int o = RT / 2; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o));
            if (i % RT == 0 && r >= r0 && r < r1) {
                const int m = mult4(top);
                sM[w][r] = m;
                sInv[w][r] = mult4_inv(m);
                (w ? a.v : a.k)[part + (size_t)(HH << a.page_sh) + slot + r] = (uint8_t)m;
            }
        }
        __syncthreads();
        uint8_t* kd = a.k + part + slot * HH;
        uint8_t* vd = a.v + part + slot * HH;
        for (int i = tid; i < 32 * CH + 2 * HD; i += NT) {  // half a chunk, 8 codes, each
            uint32_t w = 0;
            if (i < 32 * CH) {
                const int r = i / (2 * CH), x = i % (2 * CH);
                if (r < r0 || r >= r1) continue;
                const int m = sM[0][r], inv = sInv[0][r];
#pragma unroll
                for (int e = 0; e < 8; e++) w |= (uint32_t)(code4(sKV[0][r][8 * x + e], m, inv) & 15) << (8 * (e & 3) + 4 * (e >> 2));
                *reinterpret_cast<uint32_t*>(kd + r * HH + 4 * x) = w;
            } else {
                const int d = (i - 32 * CH) >> 1, r = 8 * ((i - 32 * CH) & 1);
                if (r >= r1 || r + 8 <= r0) continue;
                uint32_t* to = reinterpret_cast<uint32_t*>(vd + 8 * d + (r >> 1));
                if (r < r0 || r + 8 > r1) w = *to;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (r + e < r0 || r + e >= r1) continue;
                    const int sh = 8 * (e & 3) + 4 * (e >> 2);
                    w = (w & ~(15u << sh)) | ((uint32_t)(code4(sKV[1][r + e][d], sM[1][r + e], sInv[1][r + e]) & 15) << sh);
                }
                *to = w;
            }
        }
    }
}

// One CTA per (block of 16 positions of a sequence, kv head), 2 HD threads: the first HD move K's chunks, the others take four
// dimensions by four positions of V each (the chunks hold positions side by side, the rows dimensions). One load and one store
// of a thread after the other's latency: 24 x 200 positions of 4 bits (2 kv heads, hd 64) 3.5 us, 2048 (4, hd 128) 3.9 us for 3.2 MB.
template <int HD, int BITS>
__global__ __launch_bounds__(2 * HD) void pg_read_kernel(Paged a, int8_t* __restrict__ k, int8_t* __restrict__ v,
                                                         int64_t max_pos, int nblk) {
    constexpr int HH = HD / 2, CH = HD / 16;
    const int b = (int)blockIdx.x / nblk, blk = (int)blockIdx.x - b * nblk, g = blockIdx.y;
    int end = min(pg_len(a, b), a.max_pages << a.page_sh);
    end = (int64_t)end < max_pos ? end : (int)max_pos;
    const int n = min(16, end - 16 * blk);
    if (n <= 0) return;
    const int id = pg_page(a, b, blk), slot = (16 * blk) & ((1 << a.page_sh) - 1);
    const size_t part = ((size_t)(id < 0 ? 0 : id) * a.nkv + g) * (size_t)a.part, mult = part + (size_t)(HH << a.page_sh) + slot;
    const size_t out = (((size_t)b * max_pos + 16 * blk) * a.nkv + g) * HD, row = (size_t)a.nkv * HD;
    if (threadIdx.x < HD) {
        const int c = threadIdx.x % CH, r = threadIdx.x / CH;
        if (r >= n) return;
        v4i w = {0, 0, 0, 0};
        if (id >= 0) {
            if constexpr (BITS == 8) {
                w = *reinterpret_cast<const v4i*>(a.k + part + (slot + r) * HD + 16 * c);
            } else {
                const v2i x = *reinterpret_cast<const v2i*>(a.k + part + (slot + r) * HH + 8 * c);
                const int m = a.k[mult + r];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int code = (x[e >> 3] << (28 - 8 * (e & 3) - 4 * ((e >> 2) & 1))) >> 28;
                    w[e >> 2] |= (value4(code, m) & 255) << (8 * (e & 3));
                }
            }
        }
        *reinterpret_cast<v4i*>(k + out + r * row + 16 * c) = w;
        return;
    }
    const int d = 4 * ((threadIdx.x - HD) % (HD / 4)), t = (threadIdx.x - HD) / (HD / 4);  // positions 4 t .. 4 t + 3
    if (4 * t >= n) return;
    int w[4] = {0, 0, 0, 0};
    if (id >= 0) {
        int m = 0;
        if constexpr (BITS == 4) m = *reinterpret_cast<const int*>(a.v + mult + 4 * t);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (BITS == 8) {
                const int x = *reinterpret_cast<const int*>(a.v + part + slot * HD + 16 * (d + e) + 4 * t);
#pragma unroll
                for (int r = 0; r < 4; r++) w[r] |= (byte_of(x, r) & 255) << (8 * e);
            } else {
                const int x = *reinterpret_cast<const int*>(a.v + part + slot * HH + 8 * (d + e) + 4 * (t >> 1)) << (4 - 4 * (t & 1));
#pragma unroll
                for (int r = 0; r < 4; r++) w[r] |= (value4((x << (24 - 8 * r)) >> 28, (m >> (8 * r)) & 255) & 255) << (8 * e);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (4 * t + r < n) *reinterpret_cast<int*>(v + out + (4 * t + r) * row + d) = w[r];
}

// The greedy choice. A key is (value, then the lower index) in 64 bits, the largest key the first maximum:
// ((v ^ 2^31) << 32) | (2^32 - 1 - i).
template <int NT>
__device__ __forceinline__ uint64_t block_max_key(uint64_t best, uint64_t* s_key) {
    best = (uint64_t)wave_max_i64((int64_t)(best ^ (1ull << 63))) ^ (1ull << 63);
    if ((threadIdx.x & 63) == 0) s_key[threadIdx.x >> 6] = best;
    __syncthreads();
    best = s_key[0];
#pragma unroll
    for (int q = 1; q < NT / 64; q++) best = s_key[q] > best ? s_key[q] : best;
    return best;
}

typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));

// Grid (parts, rows): the best key of a part of a row; with one part a row, its index is the answer. One pass over the logits:
// 256 rows of 151936 in 28.8 us, 156 MB at 5.4 TB/s; 64 rows in 10.9 us with the second launch, 39 MB at 3.6 TB/s.
template <int NT>
__global__ __launch_bounds__(NT) void pg_argmax_kernel(const int32_t* __restrict__ logits, int n, int64_t stride,
                                                        int per, uint64_t* __restrict__ part,
                                                        int32_t* __restrict__ token) {
    __shared__ uint64_t s_key[NT / 64];
    const int32_t* x = logits + (size_t)blockIdx.y * stride;
    const uint32_t i0 = min(blockIdx.x * (uint32_t)per, (uint32_t)n), i1 = min(i0 + (uint32_t)per, (uint32_t)n);
    // fours of logits (on any boundary of four bytes), then the up to three that are left
    const uint32_t first = i0 + 4 * threadIdx.x, end = i0 + ((i1 - i0) & ~3u);
    auto four = [&](uint32_t i) { return *reinterpret_cast<const i32x4*>(x + i); };
    auto key = [](int v, uint32_t i) { return ((uint64_t)((uint32_t)v ^ 0x80000000u) << 32) | (0xFFFFFFFFu - i); };
    int top = INT_MIN;
    uint32_t at = first;  // the first four with the largest value yet
    constexpr int U = NT == 1024 ? 8 : 4;  // loads in flight; past the end the last four again
    for (uint32_t i = first; i < end; i += U * 4 * NT) {
        i32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = four(min(i + u * 4 * NT, end - 4));
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int m = max(max(v[u].x, v[u].y), max(v[u].z, v[u].w));
            at = m > top ? min(i + u * 4 * NT, end - 4) : at;
            top = max(top, m);
        }
    }
    uint64_t best = 0;
    if (first < end) {
        const i32x4 v = four(at);
        best = key(top, at + (v.x == top ? 0 : (v.y == top ? 1 : (v.z == top ? 2 : 3))));
    }
    if (end + threadIdx.x < i1) {
        const uint64_t last = key(x[end + threadIdx.x], end + threadIdx.x);
        best = last > best ? last : best;
    }
    best = block_max_key<NT>(best, s_key);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) token[blockIdx.y] = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
        else part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = best;
    }
}

__global__ __launch_bounds__(256) void pg_argmax_join_kernel(const uint64_t* __restrict__ part, int parts,
                                                             int32_t* __restrict__ token) {
    __shared__ uint64_t s_key[4];
    uint64_t best = 0;
    for (int i = threadIdx.x; i < parts; i += 256) {
        const uint64_t key = part[(size_t)blockIdx.x * parts + i];
        best = key > best ? key : best;
    }
    best = block_max_key<256>(best, s_key);
    if (threadIdx.x == 0) token[blockIdx.x] = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
}

}  // namespace

hipError_t launch_pg_append(const Paged& a, int hd, int bits, const int8_t* qkv, int64_t stride, int nh,
                            const int16_t* cosT, const int16_t* sinT, int max_pos, const int16_t* q_norm,
                            const int16_t* k_norm, const int32_t* shift, int64_t* w, int8_t* q, int64_t q_stride,
                            hipStream_t s) {
    const dim3 grid((unsigned)(a.tokens / 16 + 2 * a.seqs), (unsigned)a.nkv);
    const PgNorm nm = {q_norm, k_norm, shift, w};
    // Few CTAs get more threads each, as long as the chip holds them side by side (two of 1024 a CU, some of them empty). us
    // with 256 / 1024: 132 single tokens' CTAs 4-bit 5.0 / 4.6, a chunk of 100 rows 5.0 / 4.2, 512 rows 4-bit 6.7 / 5.6, 498 CTAs
    // 7.2 / 6.8, 520 (hd 128, 4-bit) 13.2 / 10.6; 948 9.8 / 11.1, 1008 (hd 128, 4-bit) 16.0 / 17.1, 1056 of single tokens 4.9 / 7.4. With norms:
    // 132 single tokens 4.3 / 4.4, 544 (hd 128) 12.0 / 11.5, 520 (hd 128, 4-bit) 15.8 / 12.0.
    const bool wide = (int64_t)grid.x * grid.y <= 768;
    auto go = [&](auto few, auto lots) {
        if (wide) lots<<<grid, dim3(1024), 0, s>>>(a, qkv, stride, nh, cosT, sinT, max_pos, q, q_stride, nm);
        else few<<<grid, dim3(256), 0, s>>>(a, qkv, stride, nh, cosT, sinT, max_pos, q, q_stride, nm);
        return hipGetLastError();
    };
    if (q_norm || k_norm || shift || w) {
        if (hd == 64)
            return bits == 8 ? go(pg_append_kernel<64, 8, 256, true>, pg_append_kernel<64, 8, 1024, true>)
                             : go(pg_append_kernel<64, 4, 256, true>, pg_append_kernel<64, 4, 1024, true>);
        return bits == 8 ? go(pg_append_kernel<128, 8, 256, true>, pg_append_kernel<128, 8, 1024, true>)
                         : go(pg_append_kernel<128, 4, 256, true>, pg_append_kernel<128, 4, 1024, true>);
    }
    if (hd == 64)
        return bits == 8 ? go(pg_append_kernel<64, 8, 256, false>, pg_append_kernel<64, 8, 1024, false>)
                         : go(pg_append_kernel<64, 4, 256, false>, pg_append_kernel<64, 4, 1024, false>);
    return bits == 8 ? go(pg_append_kernel<128, 8, 256, false>, pg_append_kernel<128, 8, 1024, false>)
                     : go(pg_append_kernel<128, 4, 256, false>, pg_append_kernel<128, 4, 1024, false>);
}

hipError_t launch_pg_read(const Paged& a, int hd, int bits, int8_t* k, int8_t* v, int64_t max_pos, hipStream_t s) {
    const int nblk = (int)((std::min<int64_t>(max_pos, (int64_t)a.max_pages << a.page_sh) + 15) / 16);
    auto go = [&](auto kern) {
        kern<<<dim3((unsigned)(a.seqs * nblk), (unsigned)a.nkv), dim3(2 * hd), 0, s>>>(a, k, v, max_pos, nblk);
        return hipGetLastError();
    };
    if (hd == 64) return bits == 8 ? go(pg_read_kernel<64, 8>) : go(pg_read_kernel<64, 4>);
    return bits == 8 ? go(pg_read_kernel<128, 8>) : go(pg_read_kernel<128, 4>);
}

// One CTA a row saves the second launch, and reads what is left of a long row alone. us a call, one / parts: 1 row of 8192 to 65536
// 4.3 / 7.5, of 100000 5.1 / 7.6, of 151936 8.2 / 7.6, of 300000 13.7 / 7.4; 64 rows of 65536 5.9 / 7.3, of 100000 7.5 / 8.2, of 151936
// 14.8 / 10.9; 256 rows fill the chip: of 32768 6.9 / 9.4, of 151936 28.8 / 32.5, of 300000 53.7 / 58.8. Parts are of 4096 logits,
// the rows' parts together some 2048 CTAs.
int pg_argmax_parts(int64_t rows, int64_t n) {
    if (n <= 100000 || rows >= 256) return 1;
    return (int)std::max<int64_t>(1, std::min((n + 4095) / 4096, (2048 + rows - 1) / std::max<int64_t>(rows, 1)));
}

hipError_t launch_pg_argmax(const int32_t* logits, int rows, int n, int64_t stride, int32_t* token, uint64_t* part,
                            hipStream_t s) {
    const int parts = pg_argmax_parts(rows, n), per = (int)(((int64_t)n + parts - 1) / parts);
    const dim3 grid((unsigned)parts, (unsigned)rows);
    if (parts == 1) pg_argmax_kernel<1024><<<grid, dim3(1024), 0, s>>>(logits, n, stride, per, part, token);
    else pg_argmax_kernel<256><<<grid, dim3(256), 0, s>>>(logits, n, stride, per, part, token);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || parts == 1) return e;
    pg_argmax_join_kernel<<<dim3((unsigned)rows), dim3(256), 0, s>>>(part, parts, token);
    return hipGetLastError();
}

}  // namespace kt
