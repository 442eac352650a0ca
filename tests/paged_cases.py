"""Batches on paged caches for tests/test_paged.py and tests/test_gpu_paged.py: random pools, tables and lengths, and what
the oracle (oracle/kt_oracle_paged.c, value by value in 64 bits) makes of them. Everything is integers, so every comparison
is exact."""
import numpy as np

from oracle import oracle as O


def part_bytes(page, hd, bits):
    return page * hd if bits == 8 else page * (hd // 2 + 1)


def exp_table(hd=64):
    """round(2^15 exp(-i / w)), w table entries to a unit of logit."""
    return np.round(32768.0 * np.exp(-np.arange(1024) / (8.0 * hd ** 0.5))).astype(np.int32)


def rope_tables(n, hd):
    a = np.arange(n)[:, None] * 1.0e6 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.round(16384 * np.cos(a)).astype(np.int16), np.round(16384 * np.sin(a)).astype(np.int16)


class Case:
    """lens: (rows, positions with them) of each sequence. Random pools (every byte a value that a write can leave), a
    table of distinct pages in random order, -1 past each sequence's pages; `behind` rows after the last sequence's."""

    def __init__(self, seed, lens, nh, nkv, hd, page, bits, spare=2, behind=0, pad=0, sigma=32):
        g = self.g = np.random.default_rng(seed)
        self.lens, self.nh, self.nkv, self.hd, self.page, self.bits = lens, nh, nkv, hd, page, bits
        self.kv_len = np.array([L for _, L in lens], dtype=np.int32)
        self.row_start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.tokens = int(self.row_start[-1]) + behind
        need = [max(0, -(-L // page)) for _, L in lens]
        self.max_pages, self.pages = max([1] + need), sum(need) + spare
        order = g.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lens), self.max_pages), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = self.pool(sigma), self.pool(sigma)
        self.width = nh * hd + pad
        self.q = self.rows8(self.tokens, self.width, sigma=sigma)
        self.qkv = self.rows8(self.tokens, (nh + 2 * nkv) * hd + pad, sigma=sigma)
        self.exp = exp_table(hd)

    def rows8(self, *shape, sigma=32):
        return np.clip(np.round(self.g.normal(0, sigma, shape)), -128, 127).astype(np.int8)

    def pool(self, sigma):
        n = self.pages * self.nkv
        if self.bits == 8:
            return self.rows8(n, self.page * self.hd, sigma=sigma).view(np.uint8)
        codes = self.g.integers(-7, 8, size=(n, self.page * self.hd // 2, 2))
        mult = self.g.integers(0, 148, size=(n, self.page))
        return np.concatenate([(codes[..., 0] & 15) | ((codes[..., 1] & 15) << 4), mult], axis=1).astype(np.uint8)

    def oracle(self, k=None, v=None):
        return O.paged(self.tokens, self.row_start, self.kv_len, self.table, self.k if k is None else k,
                       self.v if v is None else v, self.page, self.nkv, self.hd, self.bits)

    def attend(self, window=0, sinks=0, fill=77):
        """The oracle's output rows, those of no sequence left at `fill`."""
        o = np.full((self.tokens, self.width), fill, dtype=np.int8)
        O.paged_attend(self.oracle(), self.q, self.nh, self.exp, o, window, sinks)
        return o

    def append(self, cos, sin, fill=77):
        """The oracle's q rows and pools after the write."""
        q = np.full((self.tokens, self.width), fill, dtype=np.int8)
        k, v = self.k.copy(), self.v.copy()
        O.paged_append(self.oracle(k, v), self.qkv, self.nh, cos, sin, q)
        return q, k, v
