// Attention of a ragged batch's new rows over paged KV caches on gfx950 (kt_hip_dec_attention_paged).

#include <algorithm>
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "kt_paged.h"
#include "kt_w12_core.h"

namespace kt {

namespace {

// clamp(round_half_away(a / b)), b > 0.
__device__ __forceinline__ int div_round_q8(int64_t a, int64_t b) {
    const uint64_t m = a < 0 ? 0 - (uint64_t)a : (uint64_t)a;
    uint64_t q = (2 * m + (uint64_t)b) / (2 * (uint64_t)b);
    q = q > 127 ? 127 : q;
    return a < 0 ? -(int)q : (int)q;
}

// One CTA per (row, q head): the scores of 256 positions at a time, one a thread, their maximum; then the scores again,
// the weights to LDS and the weighted sum of v, a thread per (dimension, share of the positions).
template <int HD, int BITS>
__global__ __launch_bounds__(256) void pg_attend_row_kernel(Paged a, const int8_t* __restrict__ q, int64_t q_stride,
                                                            int nh, const int32_t* __restrict__ exp_tab, int window,
                                                            int sinks, int8_t* __restrict__ o, int64_t o_stride) {
    constexpr int HH = HD / 2, SH = 256 / HD;
    __shared__ __attribute__((aligned(16))) int8_t sQ[HD];
    __shared__ int sE[256], sMul[256], sRed[8];
    __shared__ const int8_t* sV[256];
    __shared__ int64_t sDen[4], sSum[SH][HD];
    const int t = (int)blockIdx.x / nh, h = (int)blockIdx.x - t * nh, g = h / (nh / a.nkv), tid = threadIdx.x;
    int first = 0;
    const int b = pg_tile_seq(a, t, 1, 1, 0, &first);
    if (b < 0) return;
    const PgRows s = pg_rows(a, b);
    if (t < s.t0 || t >= s.t0 + s.n) return;
    const int p = s.p0 + (t - s.t0);
    int8_t* to = o + (size_t)t * o_stride + h * HD;
    if (p < 0 || p >= a.max_pages << a.page_sh) {
        if (tid < HD) to[tid] = 0;
        return;
    }
    if (tid < HD) sQ[tid] = q[(size_t)t * q_stride + h * HD + tid];
    __syncthreads();
    auto score = [&](int j, int& sc) {
        if (j > p || (window && j <= p - window && j >= sinks)) return false;
        const int id = pg_page(a, b, j >> 4);
        if (id < 0) return false;
        const size_t part = ((size_t)id * a.nkv + g) * (size_t)a.part;
        const int slot = j & ((1 << a.page_sh) - 1);
        const int8_t* k = reinterpret_cast<const int8_t*>(a.k) + part;
        sc = 0;
        if constexpr (BITS == 8) {
            for (int d = 0; d < HD; d++) sc += sQ[d] * k[slot * HD + d];
        } else {
            for (int d = 0; d < HD; d++) {
                const int x = (uint8_t)k[slot * HH + d / 16 * 8 + d % 16 / 8 * 4 + d % 4];
                sc += sQ[d] * ((d % 8 >= 4 ? x << 24 : x << 28) >> 28);
            }
            sc = (sc * (uint8_t)k[(HH << a.page_sh) + slot] + 4) >> 3;
        }
        sV[tid] = reinterpret_cast<const int8_t*>(a.v) + part;
        return true;
    };
    int mx = INT_MIN;
    for (int j = tid; j <= p; j += 256) {
        int sc;
        if (score(j, sc)) mx = max(mx, sc);
    }
    mx = wave_max_i32(mx);
    if ((tid & 63) == 0) sRed[tid >> 6] = mx;
    __syncthreads();
    mx = max(max(sRed[0], sRed[1]), max(sRed[2], sRed[3]));
    int64_t den = 0, sum = 0;
    const int d = tid % HD, sh = tid / HD;
    for (int j0 = 0; j0 <= p; j0 += 256) {
        __syncthreads();
        int sc, e = 0;
        if (score(j0 + tid, sc)) {
            const int i = (mx - sc + 64) >> 7;
            e = i < 1024 ? min(max(exp_tab[i], 0), 32768) : 0;
        }
        sE[tid] = e;
        den += e;
        __syncthreads();
        for (int i = sh; i < 256; i += SH) {
            if (sE[i] == 0) continue;
            const int slot = (j0 + i) & ((1 << a.page_sh) - 1);
            if constexpr (BITS == 8) {
                sum += sE[i] * sV[i][(slot >> 4) * 16 * HD + 16 * d + (slot & 15)];
            } else {
                const int r = slot & 15, x = (uint8_t)sV[i][(slot >> 4) * 8 * HD + 8 * d + (r >> 3) * 4 + (r & 3)];
                sum += (int64_t)(sE[i] * (uint8_t)sV[i][(HH << a.page_sh) + slot]) * ((r & 4 ? x << 24 : x << 28) >> 28);
            }
        }
    }
    den = (int64_t)wave_sum_u64((uint64_t)den);
    if ((tid & 63) == 0) sDen[tid >> 6] = den;
    sSum[sh][d] = sum;
    __syncthreads();
    if (tid < HD) {
        int64_t top = 0;
        for (int i = 0; i < SH; i++) top += sSum[i][tid];
        den = (sDen[0] + sDen[1] + sDen[2] + sDen[3]) * (BITS == 8 ? 1 : 8);
        to[tid] = den ? (int8_t)div_round_q8(top, den) : 0;
    }
}

}  // namespace

size_t pg_attend_workspace(int, int, int64_t, int, int, int) { return 256; }

hipError_t launch_pg_attend(const Paged& a, int hd, int bits, const int8_t* q, int64_t q_stride, int nh,
                            const int32_t* exp_tab, int window, int sinks, int8_t* o, int64_t o_stride, void*,
                            hipStream_t s) {
    auto go = [&](auto kern) {
        kern<<<dim3((unsigned)(a.tokens * nh)), dim3(256), 0, s>>>(a, q, q_stride, nh, exp_tab, window, sinks, o, o_stride);
        return hipGetLastError();
    };
    if (hd == 64) return bits == 8 ? go(pg_attend_row_kernel<64, 8>) : go(pg_attend_row_kernel<64, 4>);
    return bits == 8 ? go(pg_attend_row_kernel<128, 8>) : go(pg_attend_row_kernel<128, 4>);
}

}  // namespace kt
