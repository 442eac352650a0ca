/*
 * kt_oracle_paged.c -- TEST INFRASTRUCTURE ONLY. The W12 decoder's attention over paged KV caches, restated value by
 * value in 64 bits: RoPE with the append to pages (8 bits, or quantised to 4), the read back, the attention of a ragged
 * batch's rows, the batch's greedy choice, the append with head norms, the attention's weights added up, the eviction by them, and
 * log probabilities. The rules are this build's (include/kt_hip.h, kt_hip_dec_*_paged); with 8
 * bits they are those of kt_dec_rope_row and kt_dec_attend on contiguous caches, which tests/test_paged.py checks.
 * Integer arithmetic only.
 */
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include "kt_oracle.h"

typedef struct {
    int64_t tokens, seqs, max_pages, pages, page, nkv, hd, bits;
    const int32_t *row_start, *kv_len, *table;
    uint8_t *k, *v;
} kt_pg;

static int64_t clampv(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
static int64_t round_div(int64_t a, int64_t b) { /* b > 0, half away from zero */
    int64_t q = (2 * (a < 0 ? -a : a) + b) / (2 * b);
    return a < 0 ? -q : q;
}

static int64_t page_bytes(const kt_pg* P) { return P->bits == 8 ? P->page * P->hd : P->page * (P->hd / 2 + 1); }

/* The page of (sequence b, position j) and kv head g in a pool, or NULL where the table names none. */
static uint8_t* page_of(const kt_pg* P, uint8_t* pool, int64_t b, int64_t j, int64_t g) {
    if (j < 0 || j >= P->max_pages * P->page) return NULL;
    int64_t id = P->table[b * P->max_pages + j / P->page];
    if (id < 0 || id >= P->pages) return NULL;
    return pool + (id * P->nkv + g) * page_bytes(P);
}

/* Where value d of slot s stands in a page: the index of its chunk of 16 values and its place in the chunk. */
static void place(const kt_pg* P, int is_v, int64_t s, int64_t d, int64_t* chunk, int64_t* at) {
    if (is_v) {
        *chunk = (s / 16) * P->hd + d;
        *at = s % 16;
    } else {
        *chunk = s * (P->hd / 16) + d / 16;
        *at = d % 16;
    }
}

static int64_t get_code(const kt_pg* P, const uint8_t* pg, int is_v, int64_t s, int64_t d) {
    int64_t chunk, at;
    place(P, is_v, s, d, &chunk, &at);
    if (P->bits == 8) return (int8_t)pg[chunk * 16 + at];
    int64_t x = pg[chunk * 8 + (at / 8) * 4 + at % 4];
    x = at % 8 >= 4 ? x >> 4 : x & 15;
    return x > 7 ? x - 16 : x;
}

static void put_code(const kt_pg* P, uint8_t* pg, int is_v, int64_t s, int64_t d, int64_t c) {
    int64_t chunk, at;
    place(P, is_v, s, d, &chunk, &at);
    if (P->bits == 8) {
        pg[chunk * 16 + at] = (uint8_t)c;
        return;
    }
    uint8_t* x = pg + chunk * 8 + (at / 8) * 4 + at % 4;
    *x = at % 8 >= 4 ? (uint8_t)((*x & 0x0F) | ((c & 15) << 4)) : (uint8_t)((*x & 0xF0) | (c & 15));
}

static int64_t get_mult(const kt_pg* P, const uint8_t* pg, int64_t s) {
    return P->bits == 8 ? 8 : pg[P->page * P->hd / 2 + s];
}

static void put_row(const kt_pg* P, uint8_t* pg, int is_v, int64_t s, const int8_t* x) {
    int64_t m = 8, top = 0;
    if (P->bits == 4) {
        for (int64_t d = 0; d < P->hd; d++) {
            int64_t a = x[d] < 0 ? -(int64_t)x[d] : x[d];
            top = a > top ? a : top;
        }
        m = (8 * top + 6) / 7;
        pg[P->page * P->hd / 2 + s] = (uint8_t)m;
    }
    for (int64_t d = 0; d < P->hd; d++)
        put_code(P, pg, is_v, s, d, P->bits == 8 ? x[d] : (m ? clampv(round_div(8 * (int64_t)x[d], m), -7, 7) : 0));
}

/* Rows first .. last - 1 of sequence b, and the position of its first row. */
static void rows_of(const kt_pg* P, int64_t b, int64_t* first, int64_t* last, int64_t* pos) {
    *first = clampv(P->row_start[b], 0, P->tokens);
    *last = clampv(P->row_start[b + 1], *first, P->tokens);
    *pos = (int64_t)P->kv_len[b] - (*last - *first);
}

void kt_pg_rope_append(const kt_pg* P, const int8_t* qkv, int64_t stride, int64_t nh, const int16_t* cos_t,
                       const int16_t* sin_t, int64_t max_pos, int8_t* q, int64_t q_stride) {
    const int64_t hd = P->hd, nkv = P->nkv;
    int8_t* row = (int8_t*)malloc((size_t)((nh + 2 * nkv) * hd));
    for (int64_t b = 0; b < P->seqs; b++) {
        int64_t t0, t1, p0;
        rows_of(P, b, &t0, &t1, &p0);
        for (int64_t t = t0; t < t1; t++) {
            const int64_t p = p0 + t - t0;
            if (p < 0 || p >= max_pos || p >= P->max_pages * P->page) {
                memset(q + t * q_stride, 0, (size_t)(nh * hd));
                continue;
            }
            memcpy(row, qkv + t * stride, (size_t)((nh + 2 * nkv) * hd));
            for (int64_t h = 0; h < nh + nkv; h++)
                for (int64_t i = 0; i < hd / 2; i++) {
                    int8_t *x = row + h * hd + i, *y = x + hd / 2;
                    const int64_t a = *x, c = *y, C = cos_t[p * (hd / 2) + i], S = sin_t[p * (hd / 2) + i];
                    *x = (int8_t)clampv(round_div(a * C - c * S, 16384), -127, 127);
                    *y = (int8_t)clampv(round_div(c * C + a * S, 16384), -127, 127);
                }
            memcpy(q + t * q_stride, row, (size_t)(nh * hd));
            for (int64_t g = 0; g < nkv; g++) {
                uint8_t* pk = page_of(P, P->k, b, p, g);
                if (!pk) continue;
                put_row(P, pk, 0, p % P->page, row + (nh + g) * hd);
                put_row(P, page_of(P, P->v, b, p, g), 1, p % P->page, row + (nh + nkv + g) * hd);
            }
        }
    }
    free(row);
}

void kt_pg_read(const kt_pg* P, int8_t* k, int8_t* v, int64_t max_pos) {
    for (int64_t b = 0; b < P->seqs; b++)
        for (int64_t j = 0; j < P->kv_len[b] && j < max_pos && j < P->max_pages * P->page; j++)
            for (int64_t g = 0; g < P->nkv; g++)
                for (int w = 0; w < 2; w++) {
                    int8_t* to = (w ? v : k) + ((b * max_pos + j) * P->nkv + g) * P->hd;
                    const uint8_t* pg = page_of(P, w ? P->v : P->k, b, j, g);
                    for (int64_t d = 0; d < P->hd; d++)
                        to[d] = !pg ? 0
                                    : (int8_t)(P->bits == 8
                                                   ? get_code(P, pg, w, j % P->page, d)
                                                   : clampv(round_div(get_code(P, pg, w, j % P->page, d) *
                                                                          get_mult(P, pg, j % P->page), 8), -127, 127));
                }
}

void kt_pg_attend(const kt_pg* P, const int8_t* q, int64_t q_stride, int64_t nh, const int32_t* exp_tab, int64_t window,
                  int64_t sinks, int8_t* o, int64_t o_stride) {
    const int64_t hd = P->hd, rep = nh / P->nkv, cap = P->max_pages * P->page;
    int64_t* e = (int64_t*)malloc((size_t)(cap ? cap : 1) * sizeof(int64_t));
    for (int64_t b = 0; b < P->seqs; b++) {
        int64_t t0, t1, p0;
        rows_of(P, b, &t0, &t1, &p0);
        for (int64_t t = t0; t < t1; t++)
            for (int64_t h = 0; h < nh; h++) {
                const int64_t p = p0 + t - t0, g = h / rep;
                const int8_t* qr = q + t * q_stride + h * hd;
                int8_t* to = o + t * o_stride + h * hd;
                int64_t top = INT64_MIN, den = 0;
                if (p < 0 || p >= cap) {
                    memset(to, 0, (size_t)hd);
                    continue;
                }
                for (int64_t j = 0; j <= p; j++) {
                    const uint8_t* pk = page_of(P, P->k, b, j, g);
                    e[j] = INT64_MIN;
                    if (!pk || (window && j <= p - window && j >= sinks)) continue;
                    int64_t s = 0;
                    for (int64_t d = 0; d < hd; d++) s += clampv(qr[d], -127, 127) * get_code(P, pk, 0, j % P->page, d);
                    if (P->bits == 4) {
                        s = s * get_mult(P, pk, j % P->page) + 4;
                        s = s >= 0 ? s / 8 : -((-s + 7) / 8); /* floor */
                    }
                    e[j] = s;
                    top = s > top ? s : top;
                }
                for (int64_t j = 0; j <= p; j++) {
                    if (e[j] == INT64_MIN) {
                        e[j] = 0;
                        continue;
                    }
                    const int64_t i = (top - e[j] + 64) / 128;
                    e[j] = i < 1024 ? clampv(exp_tab[i], 0, 32768) : 0;
                    den += e[j];
                }
                for (int64_t d = 0; d < hd; d++) {
                    int64_t sum = 0;
                    for (int64_t j = 0; j <= p; j++)
                        if (e[j]) {
                            const uint8_t* pv = page_of(P, P->v, b, j, g);
                            sum += e[j] * get_code(P, pv, 1, j % P->page, d) * get_mult(P, pv, j % P->page);
                        }
                    to[d] = den ? (int8_t)clampv(round_div(sum, 8 * den), -127, 127) : 0;
                }
            }
    }
    free(e);
}

void kt_pg_argmax(const int32_t* logits, int64_t rows, int64_t n, int64_t stride, int32_t* token) {
    for (int64_t r = 0; r < rows; r++) {
        int64_t best = 0;
        for (int64_t i = 1; i < n; i++)
            if (logits[r * stride + i] > logits[r * stride + best]) best = i;
        token[r] = (int32_t)best;
    }
}

static int64_t isqrt(int64_t n) {
    int64_t r = 0;
    for (int64_t b = (int64_t)1 << 30; b; b >>= 1)
        if ((r + b) * (r + b) <= n) r += b;
    return r;
}

static int64_t clamp30(int64_t v) { return clampv(v, -((int64_t)1 << 30), (int64_t)1 << 30); }

void kt_pg_norm_rope_append(const kt_pg* P, const int8_t* qkv, int64_t stride, int64_t nh, const int16_t* cos_t,
                            const int16_t* sin_t, int64_t max_pos, const int16_t* q_norm, const int16_t* k_norm,
                            const int32_t* shift, int8_t* q, int64_t q_stride, int64_t* w) {
    const int64_t hd = P->hd, nkv = P->nkv;
    int64_t* n = (int64_t*)malloc((size_t)hd * sizeof(int64_t));
    int8_t* row = (int8_t*)malloc((size_t)((nh + 2 * nkv) * hd));
    for (int64_t b = 0; b < P->seqs; b++) {
        int64_t t0, t1, p0;
        rows_of(P, b, &t0, &t1, &p0);
        for (int64_t t = t0; t < t1; t++) {
            const int64_t p = clamp30(P->kv_len[b]) - (t1 - t0) + t - t0, at = p + (shift ? clamp30(shift[b]) : 0);
            if (p < 0 || p >= P->max_pages * P->page || at < 0 || at >= max_pos) {
                memset(q + t * q_stride, 0, (size_t)(nh * hd));
                continue;
            }
            memcpy(row, qkv + t * stride, (size_t)((nh + 2 * nkv) * hd));
            for (int64_t h = 0; h < nh + nkv; h++) {
                const int16_t* norm = h < nh ? q_norm : k_norm;
                int8_t* x = row + h * hd;
                int64_t V = 0, one = 16384;
                for (int64_t d = 0; d < hd; d++) V += (int64_t)x[d] * x[d];
                const int64_t R = isqrt(V * 65536 / hd);
                for (int64_t d = 0; d < hd; d++)
                    n[d] = !norm ? x[d] : (R ? clampv(round_div(128 * (int64_t)x[d] * norm[d], R), -16383, 16383) : 0);
                if (norm) one = 1048576;
                for (int64_t i = 0; i < hd / 2; i++) {
                    const int64_t C = cos_t[at * (hd / 2) + i], S = sin_t[at * (hd / 2) + i], a = n[i], c = n[i + hd / 2];
                    x[i] = (int8_t)clampv(round_div(a * C - c * S, one), -127, 127);
                    x[i + hd / 2] = (int8_t)clampv(round_div(c * C + a * S, one), -127, 127);
                }
            }
            memcpy(q + t * q_stride, row, (size_t)(nh * hd));
            for (int64_t g = 0; g < nkv; g++) {
                uint8_t* pk = page_of(P, P->k, b, p, g);
                if (!pk) continue;
                put_row(P, pk, 0, p % P->page, row + (nh + g) * hd);
                put_row(P, page_of(P, P->v, b, p, g), 1, p % P->page, row + (nh + nkv + g) * hd);
                if (w) w[(P->table[b * P->max_pages + p / P->page] * nkv + g) * P->page + p % P->page] = 0;
            }
        }
    }
    free(n);
    free(row);
}

/* The score of row q for (sequence b, position j, kv head g), or INT64_MIN where the row at p does not see it. */
static int64_t score(const kt_pg* P, const int8_t* q, int64_t b, int64_t j, int64_t g, int64_t p, int64_t window, int64_t sinks) {
    const uint8_t* pk = page_of(P, P->k, b, j, g);
    if (!pk || j > p || (window && j <= p - window && j >= sinks)) return INT64_MIN;
    int64_t s = 0;
    for (int64_t d = 0; d < P->hd; d++) s += clampv(q[d], -127, 127) * get_code(P, pk, 0, j % P->page, d);
    if (P->bits == 4) {
        s = s * get_mult(P, pk, j % P->page) + 4;
        s = s >= 0 ? s / 8 : -((-s + 7) / 8); /* floor */
    }
    return s;
}

static int64_t weight(const int32_t* exp_tab, int64_t top, int64_t s) {
    const int64_t i = (top - s + 64) / 128;
    return i < 1024 ? clampv(exp_tab[i], 0, 32768) : 0;
}

void kt_pg_stats(const kt_pg* P, const int8_t* q, int64_t q_stride, int64_t nh, const int32_t* exp_tab, int64_t window,
                 int64_t sinks, int32_t* stats) {
    const int64_t cap = P->max_pages * P->page, rep = nh / P->nkv;
    for (int64_t b = 0; b < P->seqs; b++) {
        int64_t t0, t1, p0;
        rows_of(P, b, &t0, &t1, &p0);
        for (int64_t t = t0; t < t1; t++)
            for (int64_t h = 0; h < nh; h++) {
                const int64_t p = p0 + t - t0;
                int64_t top = INT64_MIN, den = 0;
                for (int64_t j = 0; p >= 0 && p < cap && j <= p; j++) {
                    const int64_t s = score(P, q + t * q_stride + h * P->hd, b, j, h / rep, p, window, sinks);
                    top = s > top ? s : top;
                }
                for (int64_t j = 0; p >= 0 && p < cap && j <= p; j++) {
                    const int64_t s = score(P, q + t * q_stride + h * P->hd, b, j, h / rep, p, window, sinks);
                    if (s != INT64_MIN) den += weight(exp_tab, top, s);
                }
                const int64_t R = den ? ((int64_t)1 << 40) / den : 0;
                stats[(t * nh + h) * 2] = top == INT64_MIN ? 0 : (int32_t)top;
                stats[(t * nh + h) * 2 + 1] = (int32_t)(uint32_t)(R > 0xFFFFFFFFLL ? 0xFFFFFFFFLL : R);
            }
    }
}

static int64_t* w_of(const kt_pg* P, int64_t* w, int64_t b, int64_t j, int64_t g) {
    if (!page_of(P, P->k, b, j, g)) return NULL;
    return w + (P->table[b * P->max_pages + j / P->page] * P->nkv + g) * P->page + j % P->page;
}

void kt_pg_weigh(const kt_pg* P, const int8_t* q, int64_t q_stride, int64_t nh, const int32_t* exp_tab, int64_t window,
                 int64_t sinks, const int32_t* stats, int64_t fresh, int64_t* w) {
    const int64_t cap = P->max_pages * P->page, rep = nh / P->nkv;
    for (int64_t b = 0; fresh && b < P->seqs; b++)
        for (int64_t j = 0; j < P->kv_len[b] && j < cap; j++)
            for (int64_t g = 0; g < P->nkv; g++)
                if (w_of(P, w, b, j, g)) *w_of(P, w, b, j, g) = 0;
    for (int64_t b = 0; b < P->seqs; b++) {
        int64_t t0, t1, p0;
        rows_of(P, b, &t0, &t1, &p0);
        for (int64_t t = t0; t < t1; t++)
            for (int64_t h = 0; h < nh; h++) {
                const int64_t p = p0 + t - t0, top = stats[(t * nh + h) * 2];
                const int64_t R = (uint32_t)stats[(t * nh + h) * 2 + 1];
                for (int64_t j = 0; p >= 0 && p < cap && j <= p; j++) {
                    const int64_t s = score(P, q + t * q_stride + h * P->hd, b, j, h / rep, p, window, sinks);
                    if (s != INT64_MIN) *w_of(P, w, b, j, h / rep) += weight(exp_tab, top, s) * R;
                }
            }
    }
}

typedef struct {
    int64_t w, j, page;
} kt_held;

static int heavier(const void* a, const void* b) {
    const kt_held *x = (const kt_held*)a, *y = (const kt_held*)b;
    if (x->page != y->page) return x->page > y->page ? -1 : 1;
    if (x->w != y->w) return x->w > y->w ? -1 : 1;
    return x->j < y->j ? -1 : 1;
}

static int earlier(const void* a, const void* b) { return ((const kt_held*)a)->j < ((const kt_held*)b)->j ? -1 : 1; }

/* `T`: P with the pages that the positions move to as its table. */
void kt_pg_evict(const kt_pg* P, const kt_pg* T, int64_t budget, int64_t recent, int64_t sinks, int64_t* w, int32_t* kept) {
    const int64_t cap = P->max_pages * P->page, hd = P->hd;
    kt_held* x = (kt_held*)malloc((size_t)cap * sizeof(kt_held));
    for (int64_t b = 0; b < P->seqs; b++)
        for (int64_t g = 0; g < P->nkv; g++) {
            const int64_t L = clampv(P->kv_len[b], 0, cap), n = L < budget ? L : budget;
            for (int64_t j = 0; j < L; j++) {
                const int64_t* at = w_of(P, w, b, j, g);
                x[j].j = j, x[j].w = at ? *at : 0, x[j].page = at != NULL;
            }
            if (L > budget) {
                const int64_t most = budget - sinks - recent;
                qsort(x + sinks, (size_t)(L - recent - sinks), sizeof *x, heavier);
                qsort(x + sinks, (size_t)most, sizeof *x, earlier);
                memmove(x + sinks + most, x + L - recent, (size_t)recent * sizeof *x);
            }
            for (int64_t i = 0; i < budget; i++) kept[(b * P->nkv + g) * budget + i] = i < n ? (int32_t)x[i].j : -1;
            for (int64_t i = 0; i < n; i++) {
                const int64_t j = x[i].j, s = j % P->page, d = i % P->page;
                const uint8_t *fk = page_of(P, P->k, b, j, g), *fv = page_of(P, P->v, b, j, g);
                uint8_t *tk = page_of(T, T->k, b, i, g), *tv = page_of(T, T->v, b, i, g);
                if (!tk) continue;
                for (int64_t e = 0; e < hd; e++) {
                    put_code(T, tk, 0, d, e, fk ? get_code(P, fk, 0, s, e) : 0);
                    put_code(T, tv, 1, d, e, fv ? get_code(P, fv, 1, s, e) : 0);
                }
                if (P->bits == 4) {
                    tk[P->page * hd / 2 + d] = fk ? (uint8_t)get_mult(P, fk, s) : 0;
                    tv[P->page * hd / 2 + d] = fv ? (uint8_t)get_mult(P, fv, s) : 0;
                }
                *w_of(T, w, b, i, g) = fk ? *w_of(P, w, b, j, g) : 0;
            }
        }
    free(x);
}

typedef unsigned __int128 u128;
static int64_t bits_of(int64_t d, int64_t mant, int shift, int64_t most) {
    const u128 t = ((u128)d * (u128)mant + (shift ? (u128)1 << (shift - 1) : 0)) >> shift;
    return t > (u128)most ? most : (int64_t)t;
}

/* a, f (256) and g (1025): the tables. */
void kt_pg_logprobs(const int32_t* logits, int64_t rows, int64_t n, int64_t stride, const int32_t* token, int64_t mant, int shift,
                    const int64_t* a, const int64_t* f, const int64_t* g, int32_t* lp, int32_t* entropy, int64_t k,
                    int32_t* top, int32_t* top_lp) {
    const int64_t most = (int64_t)31 << 16;
    for (int64_t r = 0; r < rows; r++) {
        const int32_t* x = logits + r * stride;
        int64_t M = x[0], S = 0, W = 0;
        for (int64_t i = 0; i < n; i++) M = x[i] > M ? x[i] : M;
        for (int64_t i0 = 0; i0 < n; i0 += 1024) {
            const int64_t i1 = i0 + 1024 < n ? i0 + 1024 : n;
            int64_t mb = x[i0], s = 0, w = 0;
            for (int64_t i = i0; i < i1; i++) mb = x[i] > mb ? x[i] : mb;
            for (int64_t i = i0; i < i1; i++) {
                const int64_t t = bits_of(mb - x[i], mant, shift, most), e = ((a[(t >> 8) & 255] * f[t & 255]) >> 32) >> (t >> 16);
                s += e, w += e * t;
            }
            const int64_t u = bits_of(M - mb, mant, shift, (int64_t)41 << 16), m = (a[(u >> 8) & 255] * f[u & 255]) >> 32;
            S += ((s >> 8) * m) >> (22 + (u >> 16));
            W += (((w + u * s) >> 21) * (m >> 8)) >> (22 + (u >> 16));
        }
        int64_t e = 0;
        while (S >> (e + 1)) e++;
        const int64_t y = (int64_t)(((u128)S << 31) >> e) - ((int64_t)1 << 31), i = y >> 21;
        const int64_t L = (e - 30) * ((int64_t)1 << 24) + g[i] + (((g[i + 1] - g[i]) * (y & ((1 << 21) - 1))) >> 21);
#define NATS(t) ((((t) * 256 + L) * 5814540 + ((int64_t)1 << 30)) >> 31)
#define LP(v) ((int32_t)-NATS(bits_of(M - (v), mant, shift, 0x7FFFFFFF)))
        lp[r] = token[r] < 0 || token[r] >= n ? INT32_MIN : LP(x[token[r]]);
        if (entropy) entropy[r] = (int32_t)NATS((W << 18) / (S >> 3));
        int64_t last = INT64_MAX, at = -1; /* the alternative before */
        for (int64_t q = 0; q < k; q++) {
            int64_t best = -1;
            for (int64_t j = 0; q < n && j < n; j++)
                if ((x[j] < last || (x[j] == last && j > at)) && (best < 0 || x[j] > x[best])) best = j;
            top[r * k + q] = (int32_t)best;
            top_lp[r * k + q] = best < 0 ? INT32_MIN : LP(x[best]);
            if (best >= 0) last = x[best], at = best;
        }
#undef NATS
#undef LP
    }
}
