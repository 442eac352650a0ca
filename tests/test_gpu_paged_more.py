"""Head norms in the append, softmax statistics, accumulated attention weights, eviction by them and log probabilities
(kt_hip_dec_norm_rope_kv_paged, _attention_paged_stats, _weigh_paged, _evict_paged, kt_hip_dec_logprobs_rows) on the GPU against the
oracle's value-by-value restatement, byte for byte: whole pools, whole sums, and rows and slots that a call leaves alone."""
import numpy as np
import pytest

from oracle import oracle as O
from paged_cases import Case, rope_tables
from test_gpu_paged import FILL, Dev, same, say

pytestmark = pytest.mark.gpu
HD_BITS = [(8, 64), (4, 64), (8, 128), (4, 128)]


def put(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class More(Dev):
    """A Case on the GPU with accumulated weights, which start from random sums."""

    def __init__(self, torch, c):
        from tritify_amd.paged import PagedKV

        super().__init__(torch, c)
        self.w0 = c.g.integers(0, 1 << 50, size=(c.pages, c.nkv, c.page))
        self.kv = PagedKV(c.pages, c.page, c.nkv, c.hd, c.bits, k=self.kv.k, v=self.kv.v, w=put(torch, self.w0))
        self.stats = torch.full((c.tokens, c.nh, 2), FILL, dtype=torch.int32, device="cuda")

    def attend(self, window=0, sinks=0, stream=None):
        self.kv.attend(self.q, self.b, self.c.nh, self.exp, self.o, self.ws, window, sinks, stream, stats=self.stats)
        return self.o

    def weigh(self, window=0, sinks=0, fresh=False, stream=None):
        self.kv.weigh(self.q, self.b, self.c.nh, self.exp, self.stats, window, sinks, fresh, stream)
        return self.kv.w


# -- the append with norms -------------------------------------------------------------------------------------------


def check_norm(torch, c, max_pos, q_norm, k_norm, shift, w=True):
    cos, sin = rope_tables(max_pos, c.hd)
    d = More(torch, c)
    if not w:
        d.kv.w = None
    q = np.full((c.tokens, c.width), FILL, dtype=np.int8)
    k, v, sums = c.k.copy(), c.v.copy(), d.w0.copy()
    O.paged_norm_append(c.oracle(k, v), c.qkv, c.nh, cos, sin, q, q_norm, k_norm, shift, sums if w else None)
    opt = lambda a, t: None if a is None else put(torch, a.astype(t))  # noqa: E731
    for _ in range(2):
        d.kv.append(d.qkv, d.b, c.nh, put(torch, cos), put(torch, sin), d.o, q_norm=opt(q_norm, np.int16), k_norm=opt(k_norm, np.int16),
                    shift=opt(shift, np.int32))
        same(d.o, q, "q")
        same(d.kv.k, k.view(np.int8), "k pool")
        same(d.kv.v, v.view(np.int8), "v pool")
        if w:
            same(d.kv.w, sums, "sums")


LENS = [(1, 1), (1, 16), (1, 17), (0, 20), (16, 16), (16, 40), (15, 15), (47, 63), (1, 200), (33, 300), (0, 0)]


@pytest.mark.parametrize("nh,nkv,hd,page", [(14, 2, 64, 16), (8, 8, 64, 64), (16, 4, 128, 32), (3, 1, 128, 256)])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("which", ["both", "q", "k", "shift", "w", "norms"])
def test_norm_append(torch_dev, nh, nkv, hd, page, bits, which):
    c = Case(nh + bits, LENS, nh, nkv, hd, page, bits, behind=2, pad=32)
    say(f"case: norm append heads={nh}/{nkv} hd={hd} page={page} bits={bits} {which}")
    wt = lambda: np.round(4096 * (1 + 0.4 * c.g.normal(size=hd))).astype(np.int16)  # noqa: E731
    shift = c.g.integers(-20, 60, size=len(LENS))
    q_norm, k_norm = (wt() if which in ("both", "q", "norms") else None), (wt() if which in ("both", "k", "norms") else None)
    check_norm(torch_dev, c, 320, q_norm, k_norm, shift if which in ("both", "shift") else None, w=which != "norms")


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("sigma", [0, 1, 3, 32, 1000])
def test_norm_append_values(torch_dev, bits, sigma):
    """Rows of zeros, of one small value, of ends of the range; weights at the ends of theirs."""
    c = Case(5, [(90, 120), (40, 40)], 4, 2, 64, 16, bits, sigma=sigma)
    c.qkv[7, 64:128] = 0
    c.qkv[8, :] = 0
    c.qkv[8, 3] = c.qkv[8, 64 * 4 + 5] = 1
    c.qkv[9] = -128
    say(f"case: norm values sigma={sigma} bits={bits}")
    for weights in (np.full(64, 4096), c.g.integers(-32768, 32768, size=64), np.where(np.arange(64) % 2, 32767, -32768), np.zeros(64)):
        check_norm(torch_dev, c, 130, weights, weights[::-1].copy(), None)


@pytest.mark.parametrize("bits", [8, 4])
def test_norm_append_tables_and_shifts_at_their_ends(torch_dev, bits):
    torch = torch_dev
    c = Case(6, [(20, 7), (40, 60), (5, 5), (3, 50), (2, 18), (4, 30), (4, 30), (9, 40)], 4, 2, 64, 16, bits, behind=3)
    c.table[1, 1], c.table[3, 3] = -1, c.pages
    c.kv_len[4] = 16 * c.max_pages + 1
    shift = np.array([0, 10, -1, 2 ** 31 - 1, 0, -(2 ** 31), 40, -34])
    say(f"case: norm append outside bits={bits}")
    check_norm(torch, c, 64, np.full(64, 5000), np.full(64, -3000), shift)
    check_norm(torch, c, 0, np.full(64, 5000), None, shift)
    d = More(torch, c)
    cos = c.g.choice([-32768, 32767, 16384, 0], size=(64, 32)).astype(np.int16)
    q, k, v, sums = np.full((c.tokens, c.width), FILL, dtype=np.int8), c.k.copy(), c.v.copy(), d.w0.copy()
    norm = np.full(64, 32767, dtype=np.int16)
    O.paged_norm_append(c.oracle(k, v), c.qkv, 4, cos, cos[::-1].copy(), q, norm, norm, None, sums)
    d.kv.append(d.qkv, d.b, 4, put(torch, cos), put(torch, cos[::-1]), d.o, q_norm=put(torch, norm), k_norm=put(torch, norm))
    same(d.o, q, "q")
    same(d.kv.k, k.view(np.int8), "k pool")


@pytest.mark.parametrize("bits,hd", HD_BITS)
def test_append_far_outside_reaches_no_other_memory(torch_dev, bits, hd):
    """Lengths at the ends of 32 bits, with norms and without: blocks whose distance to the tables' positions, times a row's chunks, is
    past 32 bits. The rows lie between others of their tensors."""
    torch = torch_dev
    c = Case(24, [(20, 30), (40, 60), (3, 50), (33, 40), (1, 9), (17, 40)], 4, 2, hd, 16, bits)
    c.kv_len = np.array([2 ** 31 - 1, -(2 ** 31), 2 ** 30, 2 ** 30 + 7, -(2 ** 30), 2 ** 30 - 60], dtype=np.int32)
    cos, sin = rope_tables(64, hd)
    for norm in (None, np.full(hd, 4096, dtype=np.int16)):
        for shift in (None, np.array([-(2 ** 31), 2 ** 31 - 1, -(2 ** 30), -(2 ** 30) + 20, 2 ** 30, -(2 ** 30) + 70], dtype=np.int32)):
            say(f"case: append far outside bits={bits} hd={hd} norm={norm is not None} shift={shift is not None}")
            d = More(torch, c)
            if norm is None and shift is None:
                d.kv.w = None  # the plain append
            q, k, v, w = np.full((c.tokens, c.width), FILL, dtype=np.int8), c.k.copy(), c.v.copy(), d.w0.copy()
            O.paged_norm_append(c.oracle(k, v), c.qkv, 4, cos, sin, q, norm, norm, shift, w)
            opt = lambda a: None if a is None else put(torch, a)  # noqa: E731
            d.kv.append(d.qkv, d.b, 4, put(torch, cos), put(torch, sin), d.o, q_norm=opt(norm), k_norm=opt(norm), shift=opt(shift))
            same(d.o, q, "q")
            same(d.kv.k, k.view(np.int8), "k pool")
            same(d.kv.v, v.view(np.int8), "v pool")


def test_norm_append_many_blocks(torch_dev):
    """More blocks than the chip takes at once, where a CTA has 256 threads."""
    lens = [(50, 70 + i) if i % 40 == 3 else (int(i % 7 > 0), 1 + (i * 29) % 90) for i in range(430)]
    for bits, hd in HD_BITS:
        c = Case(22, lens, 4, 4, hd, 32, bits, behind=2, pad=16)
        say(f"case: norm append many bits={bits} hd={hd}")
        check_norm(torch_dev, c, 600, c.g.integers(-8000, 8000, size=hd), c.g.integers(-8000, 8000, size=hd), c.g.integers(0, 90, size=430))


# -- statistics and weights ------------------------------------------------------------------------------------------


def check_weigh(torch, c, window=0, sinks=0, seen_only=False):
    """Attention with statistics, then the weights: added to what is there, then from zero."""
    say(f"case: weigh lens={c.lens[:6]} heads={c.nh}/{c.nkv} hd={c.hd} page={c.page} bits={c.bits} window={window}/{sinks}")
    d = More(torch, c)
    same(d.attend(window, sinks), c.attend(window, sinks, FILL), "attend")
    stats = O.paged_stats(c.oracle(), c.q, c.nh, c.exp, window, sinks)
    got = d.stats.cpu().numpy()
    rows = np.zeros(c.tokens, dtype=bool)
    for b in range(len(c.kv_len)):
        rows[max(0, c.row_start[b]):max(0, c.row_start[b + 1])] = True
    assert (got[~rows] == FILL).all()
    assert np.array_equal(got[rows], stats[rows])
    for fresh in (False, True):
        w = d.kv.w.cpu().numpy()
        O.paged_weigh(c.oracle(), c.q, c.nh, c.exp, stats, w, window, sinks, fresh)
        same(d.weigh(window, sinks, fresh), w, f"sums fresh={fresh}")
    return d


HEADS = [(1, 1, 64), (14, 2, 64), (4, 4, 64), (20, 1, 64), (16, 4, 128), (9, 3, 128), (33, 1, 128), (70, 1, 64)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("bits", [8, 4])
def test_weigh_heads(torch_dev, nh, nkv, hd, bits):
    page = {1: 16, 14: 32, 4: 64, 20: 128, 16: 256, 9: 16, 33: 64, 70: 16}[nh]
    check_weigh(torch_dev, Case(nh, [(1, 1), (1, 77), (0, 50), (13, 90), (35, 35), (1, 300)], nh, nkv, hd, page, bits, behind=3, pad=16))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 255, 257, 511, 513, 1025, 2500])
def test_weigh_one_row_lengths(torch_dev, L, bits):
    check_weigh(torch_dev, Case(L, [(1, L)], 14, 2, 64, 16, bits))


@pytest.mark.parametrize("bits,hd", HD_BITS)
@pytest.mark.parametrize("n,L", [(2, 2), (9, 700), (10, 64), (73, 73), (74, 333), (130, 600)])
def test_weigh_chunks(torch_dev, n, L, bits, hd):
    """Columns of one group, several, and past a CTA's (7 heads a kv head: 512 columns are 73 rows)."""
    check_weigh(torch_dev, Case(n, [(n, L), (max(1, n - 3), L + 40)], 7, 1, hd, 32, bits))


@pytest.mark.parametrize("bits,hd", HD_BITS)
def test_weigh_long(torch_dev, bits, hd):
    check_weigh(torch_dev, Case(5, [(1, 20011), (2, 9000)], 7, 1, hd, 64, bits))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (65, 4), (100, 20), (300, 64), (128, 1000), (5000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_weigh_window(torch_dev, window, sinks, bits):
    check_weigh(torch_dev, Case(8, [(1, 1), (1, 900), (30, 700), (70, 70), (150, 600)], 7, 1, 64, 16, bits), window, sinks)


@pytest.mark.parametrize("window,sinks", [(300, 5), (9000, 700)])
def test_weigh_window_in_a_wide_table(torch_dev, window, sinks):
    check_weigh(torch_dev, Case(12, [(1, 20011), (2, 9000), (1, 100)], 7, 1, 64, 64, 8), window, sinks)


@pytest.mark.parametrize("bits", [8, 4])
def test_weigh_many_sequences(torch_dev, bits):
    lens = [((i * 7) % 5, (i * 7) % 5 + (i * 53) % 200) for i in range(150)]
    check_weigh(torch_dev, Case(6, lens, 4, 2, 64, 16, bits, behind=2))
    check_weigh(torch_dev, Case(7, [(int(i % 9 > 0), 1 + (i * 53) % 140) for i in range(1100)], 4, 4, 64, 16, bits))


@pytest.mark.parametrize("bits", [8, 4])
def test_weigh_pages_left_out_and_positions_outside(torch_dev, bits):
    c = Case(9, [(1, 400), (40, 200), (1, 64), (3, 33), (1, 2000)], 4, 2, 64, 16, bits)
    c.table[0, [0, 3, 4, 20]] = [-1, c.pages, 2 ** 31 - 1, -(2 ** 31)]
    c.table[1, [1, 11, 12]] = [-7, c.pages + 5, -1]
    c.table[2] = -1
    c.table[3, 2] = c.pages
    c.table[4, :100] = -1
    check_weigh(torch_dev, c)
    c = Case(10, [(5, 3), (4, 70), (2, 8), (3, 9)], 4, 2, 64, 16, bits, behind=6)
    c.kv_len = np.array([3, 2 ** 31 - 1, -(2 ** 31), 16 * c.max_pages + 1], dtype=np.int32)
    check_weigh(torch_dev, c)
    c.row_start = (c.row_start + 4).astype(np.int32)
    c.kv_len = np.array([5, 70, 3, 16 * c.max_pages + 1], dtype=np.int32)
    check_weigh(torch_dev, c)


@pytest.mark.parametrize("bits,hd", HD_BITS)
def test_weigh_of_a_chunk_is_that_of_its_parts(torch_dev, bits, hd):
    """Chunks large enough that a CTA takes 256 columns, against calls of a few rows each, whose CTAs take 64: the same sums."""
    from tritify_amd.paged import PagedBatch

    torch = torch_dev
    c = Case(15, [(900, 4000), (1, 3000)], 16, 4, hd, 64, bits)
    say(f"case: weigh in parts bits={bits} hd={hd}")
    d = More(torch, c)
    for window, sinks in ((0, 0), (1500, 70)):
        d.attend(window, sinks)
        whole = d.weigh(window, sinks, fresh=True).clone()
        d.kv.w[:] = torch.where(whole == put(torch, d.w0), d.kv.w, 0)  # the slots that no position has keep what they had
        d.kv.weigh(d.q, d.b, 16, d.exp, d.stats, window, sinks, fresh=True)
        assert torch.equal(d.kv.w, whole)
        d.kv.weigh(d.q[:0], PagedBatch(d.b.row_start * 0, d.b.kv_len, d.b.table, 0), 16, d.exp, d.stats[:0], window, sinks, fresh=True)
        for at in list(range(0, 900, 61)) + [900]:
            n = 1 if at == 900 else min(61, 900 - at)
            one = 1 if at == 900 else 0
            lens = torch.tensor([3000 if one else 3100 + at + n], dtype=torch.int32, device="cuda")
            b = PagedBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"), lens, d.b.table[one:one + 1], n)
            d.kv.weigh(d.q[at:at + n], b, 16, d.exp, d.stats[at:at + n], window, sinks)
        assert torch.equal(d.kv.w, whole)


def test_weigh_shared_pages(torch_dev):
    """A common prompt's pages in several tables: each slot has the sum over the sequences."""
    c = Case(14, [(1, 100), (3, 90), (1, 100)], 6, 2, 64, 16, 8)
    c.table[1, :4] = c.table[2, :4] = c.table[0, :4]
    check_weigh(torch_dev, c)


@pytest.mark.parametrize("bits,hd", HD_BITS)
@pytest.mark.parametrize("what", ["peaks", "flat", "zeros", "beyond", "step", "low"])
def test_weigh_tables_and_extremes(torch_dev, what, bits, hd):
    c = Case(11, [(1, 700), (33, 250), (1, 5), (1, 6000)], 7, 1, hd, 16, bits, sigma=200 if what == "peaks" else 32)
    if what == "flat":
        c.exp[:] = 32768
    if what == "zeros":
        c.exp[:] = 0
    if what == "beyond":
        c.exp[::3], c.exp[1::3] = 2 ** 31 - 1, -5
    if what == "step":
        c.exp[1:] = 0
    if what == "low":  # sums of weights below 2^8: the reciprocal's bound
        c.exp[:] = 0
        c.exp[0] = 1
    if what == "peaks":
        for a in (c.q, c.k.view(np.int8) if bits == 8 else c.q):
            a[:] = np.where(a < 0, -128, 127)
        if bits == 4:
            c.k[:, : c.page * hd // 2] = c.g.choice([0x77, 0x99], size=(c.pages, c.page * hd // 2))
            c.k[:, c.page * hd // 2:] = 147
    check_weigh(torch_dev, c)


def test_weigh_any_statistics_reach_no_other_memory(torch_dev):
    from tritify_amd.paged import PagedBatch

    torch = torch_dev
    for row_start in ([0, 90, 40, 60], [90, 0, 90, 30, 90], [-5, 200, -7, 50], [70, 10]):
        c = Case(70, [(1, 200)] * (len(row_start) - 1), 14, 2, 64, 16, 8, spare=6)
        d = More(torch, c)
        b = PagedBatch(torch.tensor(row_start, dtype=torch.int32, device="cuda"), d.b.kv_len, d.b.table, 90)
        q = put(torch, c.rows8(90, 14 * 64))
        stats = put(torch, c.g.integers(-(2 ** 31), 2 ** 31, size=(90, 14, 2)).astype(np.int32))
        say(f"case: weigh row_start={row_start}")
        d.kv.weigh(q, b, 14, d.exp, stats)
        unused = [p for p in range(c.pages) if p not in c.table]
        same(d.kv.w[unused], d.w0[unused])


def test_weigh_offsets_past_32_bits(torch_dev):
    """A K pool of more than 4 GiB and sums of more than 2^32 bytes, the pages in use at their end."""
    from tritify_amd.paged import PagedBatch, PagedKV

    torch = torch_dev
    c = Case(21, [(1, 700), (20, 300)], 8, 4, 128, 256, 8)
    d = More(torch, c)
    pages = (5 << 30) // (4 * 256 * 8)
    part = c.k.shape[1]
    say(f"case: {pages} pages of {4 * part} bytes, sums of {pages * 4 * 256 * 8}")
    k, w = torch.empty(pages, 4, part, dtype=torch.int8, device="cuda"), torch.zeros(pages, 4, 256, dtype=torch.int64, device="cuda")
    v = torch.empty(pages, 4, part, dtype=torch.int8, device="cuda")
    k[-c.pages:], v[-c.pages:] = d.kv.k, d.kv.v
    kv = PagedKV(pages, 256, 4, 128, 8, k=k, v=v, w=w)
    table = np.where(c.table >= 0, c.table + pages - c.pages, -1).astype(np.int32)
    b = PagedBatch(d.b.row_start, d.b.kv_len, put(torch, table), c.tokens)
    kv.attend(d.q, b, 8, d.exp, d.o, d.ws, stats=d.stats)
    kv.weigh(d.q, b, 8, d.exp, d.stats)
    want = np.zeros((c.pages, 4, 256), dtype=np.int64)
    O.paged_weigh(c.oracle(), c.q, 8, c.exp, O.paged_stats(c.oracle(), c.q, 8, c.exp), want)
    same(w[-c.pages:], want, "sums")
    # cut down within the same pools
    free = torch.tensor([[5], [pages // 2]], dtype=torch.int32, device="cuda")
    kept = torch.zeros(2, 4, 100, dtype=torch.int32, device="cuda")
    kv.evict(b, free, 100, kept, recent=30, sinks=2)
    k1, v1, w1 = c.k.copy(), c.v.copy(), want.copy()
    ot = np.array([[c.pages], [c.pages + 1]], dtype=np.int32)
    grow = lambda a: np.concatenate([a, np.zeros((2,) + a.shape[1:], dtype=a.dtype)])  # noqa: E731
    k1, v1, w1 = grow(c.k.reshape(c.pages, -1)), grow(c.v.reshape(c.pages, -1)), grow(want)
    P = O.paged(c.tokens, c.row_start, c.kv_len, c.table, k1, v1, 256, 4, 128, 8)
    same(kept, O.paged_evict(P, ot, 100, 30, 2, w1), "kept")
    for i, page in enumerate((5, pages // 2)):
        same(k[page].reshape(4, 256, 128)[:, :100], k1[c.pages + i].view(np.int8).reshape(4, 256, 128)[:, :100], "k")
        same(w[page][:, :100], w1[c.pages + i][:, :100], "w")
        rows = lambda a: a.reshape(4, 16, 128, 16).swapaxes(2, 3).reshape(4, 256, 128)[:, :100]  # noqa: E731
        same(rows(v[page]), rows(v1[c.pages + i].view(np.int8)), "v")


# -- eviction --------------------------------------------------------------------------------------------------------


def check_evict(torch, c, budget, recent=0, sinks=0, w=None, to=None):
    """The pages that the positions go to are the pool's last ones."""
    say(f"case: evict lens={[L for _, L in c.lens][:8]} heads={c.nkv} hd={c.hd} page={c.page} bits={c.bits} budget={budget} {recent}/{sinks}")
    need = -(-budget // c.page)
    free = np.setdiff1d(np.arange(c.pages), c.table)
    if to is None:
        to = c.g.permutation(free)[: len(c.kv_len) * need].reshape(len(c.kv_len), need)
    d = More(torch, c)
    if w is not None:
        d.w0 = w
        d.kv.w.copy_(put(torch, w))
    k, v, sums = c.k.copy(), c.v.copy(), d.w0.copy()
    want = O.paged_evict(c.oracle(k, v), to, budget, recent, sinks, sums)
    kept = torch.full((len(c.kv_len), c.nkv, budget), FILL, dtype=torch.int32, device="cuda")
    for again in range(2):
        d.kv.evict(d.b, put(torch, to.astype(np.int32)), budget, kept, recent, sinks)
        same(kept, want, "kept")
        same(d.kv.k, k.view(np.int8), "k pool")
        same(d.kv.v, v.view(np.int8), "v pool")
        same(d.kv.w, sums, "sums")
    return want


def spare_case(seed, lens, nkv, hd, page, bits, budget):
    return Case(seed, [(0, L) for L in lens], nkv, nkv, hd, page, bits, spare=len(lens) * -(-budget // page) + 2)


@pytest.mark.parametrize("bits,hd", HD_BITS)
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (17, 5, 3), (64, 0, 0), (64, 64, 0), (64, 30, 34), (100, 7, 0), (300, 1, 200)])
def test_evict(torch_dev, bits, hd, page, budget, recent, sinks):
    c = spare_case(budget + page, [0, 1, 15, 16, 17, 63, 64, 65, 100, 101, 299, 300, 301, 700], 3, hd, page, bits, budget)
    check_evict(torch_dev, c, budget, recent, sinks)


@pytest.mark.parametrize("what", ["zeros", "few", "equal top", "negative", "ends", "small", "low bits"])
@pytest.mark.parametrize("L", [300, 5000])
def test_evict_sums(torch_dev, what, L):
    """Ties (the lower position stays), sums of either sign and at the ends of 64 bits, sums that differ in low or high bits alone."""
    c = spare_case(3, [L, L // 2, L - 1], 2, 64, 16, 8, 128)
    shape = (c.pages, 2, 16)
    w = {"zeros": lambda: np.zeros(shape, dtype=np.int64), "few": lambda: c.g.integers(0, 3, size=shape),
         "equal top": lambda: np.where(c.g.random(shape) < 0.4, 1 << 45, c.g.integers(0, 1 << 45, size=shape)),
         "negative": lambda: c.g.integers(-(2 ** 62), 2 ** 62, size=shape), "small": lambda: c.g.integers(-40, 40, size=shape),
         "ends": lambda: c.g.choice(np.array([-(2 ** 63) + 1, 2 ** 63 - 1, 0, -1, 1]), size=shape),
         "low bits": lambda: (np.int64(5) << 50) + c.g.integers(0, 200, size=shape)}[what]()
    check_evict(torch_dev, c, 128, 10, 4, w)
    check_evict(torch_dev, c, 100, 0, 0, w)


@pytest.mark.parametrize("L,budget", [(16384 + 20, 1000), (16384 + 21, 16384), (40011, 12345), (131000, 300)])
def test_evict_long(torch_dev, L, budget):
    c = spare_case(4, [L, 700], 2, 64, 64, 4, budget)
    check_evict(torch_dev, c, budget, min(100, budget // 3), 4)
    check_evict(torch_dev, c, budget, 0, 0, c.g.integers(0, 50, size=(c.pages, 2, 64)))


def test_evict_from_the_widest_table(torch_dev):
    """524288 positions in pages that are named many times over: sums of 64 to a page, so 8192 positions have each."""
    c = spare_case(8, [64 * 256], 1, 64, 256, 8, 1000)
    table = np.resize(c.table[0, :64], 2048)
    c.table, c.max_pages = table[None].astype(np.int32), 2048
    c.kv_len = np.array([524288], dtype=np.int32)
    check_evict(torch_dev, c, 1000, 100, 7)
    c.kv_len = np.array([524288 - 1000], dtype=np.int32)
    check_evict(torch_dev, c, 1000, 0, 0, c.g.integers(0, 1 << 45, size=(c.pages, 1, 256)))


@pytest.mark.parametrize("bits", [8, 4])
def test_evict_many_sequences(torch_dev, bits):
    c = spare_case(5, [(i * 37) % 200 for i in range(300)], 2, 64, 16, bits, 60)
    check_evict(torch_dev, c, 60, 20, 2)


@pytest.mark.parametrize("bits", [8, 4])
def test_evict_pages_left_out(torch_dev, bits):
    """A position without a page is below all others, and leaves zeros where it stays all the same; entries of `to` outside the pool
    drop what goes there; lengths past the table and below zero."""
    c = spare_case(6, [100, 90, 200, 50, 64, 70], 2, 64, 16, bits, 48)
    c.table[0, [1, 3]] = [-1, c.pages]
    c.table[1, 1:] = -5  # fewer positions with a page than the budget
    c.table[2] = -1
    c.kv_len[3], c.kv_len[4], c.kv_len[5] = -9, 2 ** 31 - 1, -(2 ** 31)
    need = 3
    to = c.g.permutation(np.setdiff1d(np.arange(c.pages), c.table))[: 6 * need].reshape(6, need).astype(np.int32)
    to[4, 1], to[0, 2] = -1, c.pages
    w = c.g.integers(-100, 100, size=(c.pages, 2, 16))
    check_evict(torch_dev, c, 48, 3, 2, w, to)
    check_evict(torch_dev, c, 48, 0, 0, w, to)


@pytest.mark.parametrize("L,many", [(300, True), (5000, True), (20000, True), (5000, False), (20000, False)])
def test_evict_the_least_sums(torch_dev, L, many):
    """The least of 64 bits is below the next one, whichever has the lower position, and above a position without a page: with cuts among
    the negative sums and, where most are negative, among the positions without a page (more than a bin's candidates, or fewer)."""
    c = spare_case(12, [L, L - 7], 2, 64, 16, 8, L - L // 5 if many else L - 100)
    gone = L // 50 if many else 1
    for b in range(2):
        c.table[b, c.g.permutation(L // 16)[:gone]] = -1
    least = -(2 ** 63) + c.g.integers(0, 3, size=(c.pages, 2, 16))
    w = least if many else np.where(c.g.random(least.shape) < 300 / L, least, c.g.integers(0, 1 << 45, size=least.shape))
    for budget in (L // 2, L - L // 5) if many else (L - 100,):
        check_evict(torch_dev, c, budget, 10, 4, w)


@pytest.mark.parametrize("width", [4, 2048])
def test_evict_of_no_sequences(torch_dev, width):
    from tritify_amd.paged import PagedBatch, PagedKV

    torch = torch_dev
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    kv, b = PagedKV(5, 16, 2, 64, weights=True), PagedBatch(z(1), z(0), z(0, width), 0)
    assert kv.evict_workspace_bytes(b) > 0
    kv.evict(b, z(0, 3), 40, z(0, 2, 40), recent=3)
    torch.cuda.synchronize()
    assert not kv.k.any() and not kv.v.any() and not kv.w.any()


# -- log probabilities -----------------------------------------------------------------------------------------------


def run_logprobs(torch, x, n, tokens, scale, k, stream=None):
    import tritify_amd as TA

    rows = x.shape[0]
    i32 = lambda *s: torch.full(s, FILL, dtype=torch.int32, device="cuda")  # noqa: E731
    lp, ent, top, top_lp = i32(rows + 1), i32(rows + 1), i32(rows + 1, max(k, 1)), i32(rows + 1, max(k, 1))
    ws = torch.full((TA.dec_logprobs_rows_workspace(rows, n, k),), 0x6D, dtype=torch.int8, device="cuda")
    for _ in range(2):
        TA.dec_logprobs_rows(put(torch, x), rows, n, put(torch, tokens), scale, lp, ws, ent, top if k else None, top_lp if k else None, k,
                             stride=x.shape[1])
    for t in (lp, ent, top, top_lp):
        assert (t[rows:] == FILL).all()
    return [t[:rows].cpu().numpy() for t in (lp, ent)] + ([t[:rows].cpu().numpy() for t in (top, top_lp)] if k else [])


def check_logprobs(torch, x, n, tokens, unit, k):
    from tritify_amd import backend as B

    scale = unit if isinstance(unit, tuple) else B.logit_scale(unit)
    say(f"case: logprobs rows={x.shape[0]} n={n} k={k} scale={scale}")
    got = run_logprobs(torch, x, n, tokens.astype(np.int32), scale, k)
    want = O.logprobs_rows(x, n, tokens, *scale, k)
    for g, w, what in zip(got, want, ("lp", "entropy", "top", "top lp")):
        assert np.array_equal(g, w), (what, np.argwhere(g != w)[:3], g[g != w][:3], w[g != w][:3])
    return got


SIZES = [1, 2, 3, 5, 63, 97, 1000, 1023, 1024, 1025, 2048, 4095, 4097, 5000, 20000, 32769, 100001, 151936]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("k", [0, 1, 5, 20, 32])
def test_logprobs_sizes(torch_dev, n, k):
    g = np.random.default_rng(n + k)
    rows = 3 if n > 50000 else 5
    x = np.round(g.normal(0, 1 << 18, size=(rows, n + 3))).astype(np.int32)
    x[1, n // 2] += 1 << 21
    x[:, n:] = 2 ** 31 - 1  # past the rows
    check_logprobs(torch_dev, x, n, g.integers(0, n, size=rows), 87381, k)


@pytest.mark.parametrize("n", [40, 1024, 6000, 70000, 1 << 20])
@pytest.mark.parametrize("k", [1, 20, 32])
@pytest.mark.parametrize("what", ["equal", "two", "few", "sorted", "falling", "ends", "blocks", "tail"])
def test_logprobs_ties_and_orders(torch_dev, n, k, what):
    g = np.random.default_rng(n)
    x = {"equal": lambda: np.full((2, n), -7), "two": lambda: g.integers(0, 2, size=(2, n)), "few": lambda: g.integers(-40, 40, size=(2, n)),
         "sorted": lambda: np.tile(np.arange(n), (2, 1)) - n, "falling": lambda: -np.tile(np.arange(n), (2, 1)),
         "ends": lambda: g.choice(np.array([-(2 ** 31), 2 ** 31 - 1]), size=(2, n)),
         "blocks": lambda: np.where(np.arange(n) // 1024 % 3 == 1, 500, g.integers(0, 500, size=(2, n))),
         "tail": lambda: np.where(np.arange(n) >= n - 40, 10 ** 6 + np.arange(n) // 2, g.integers(0, 10 ** 6, size=(2, n)))}[what]()
    check_logprobs(torch_dev, x.astype(np.int32), n, np.array([0, n - 1]), 8.0 if what in ("few", "two") else 5000, k)


@pytest.mark.parametrize("scale", [(1, 0), (1, 62), ((1 << 31) - 1, 0), ((1 << 31) - 1, 62), ((1 << 31) - 1, 31), (1 << 30, 30), (12345, 1),
                                   (1161815935, 33), (1161815935, 32), (1161815935, 40)])
def test_logprobs_scales(torch_dev, scale):
    g = np.random.default_rng(scale[1])
    x = np.concatenate([np.round(g.normal(0, 10.0 ** e, size=(1, 3000))).clip(-(2 ** 31), 2 ** 31 - 1) for e in (0, 1, 3, 5, 7, 9)]).astype(np.int32)
    check_logprobs(torch_dev, x, 3000, g.integers(0, 3000, size=6), scale, 7)


def test_logprobs_many_rows_and_tokens_outside(torch_dev):
    g = np.random.default_rng(1)
    x = np.round(g.normal(0, 1 << 17, size=(700, 300))).astype(np.int32)
    tokens = g.integers(-3, 303, size=700)
    tokens[:4] = [-(2 ** 31), 2 ** 31 - 1, 300, -1]
    lp = check_logprobs(torch_dev, x, 300, tokens, 30000, 4)[0]
    assert ((lp == -(2 ** 31)) == ((tokens < 0) | (tokens >= 300))).all()


@pytest.mark.parametrize("k", [1, 8, 9])
def test_logprobs_many_rows_of_many_blocks(torch_dev, k):
    g = np.random.default_rng(7)
    x = np.round(g.normal(0, 1 << 18, size=(260, 40001))).astype(np.int32)
    x[3], x[4] = -5, g.integers(0, 3, size=40001)
    x[5, ::1024] += 1 << 22  # every block's maximum far above its others
    x[6] = np.sort(x[6])
    check_logprobs(torch_dev, x, 40000, g.integers(0, 40000, size=260), 87381, k)


def test_logprobs_of_a_batch_are_those_of_each_row(torch_dev):
    g = np.random.default_rng(2)
    x = np.round(g.normal(0, 1 << 18, size=(9, 50000))).astype(np.int32)
    t = g.integers(0, 50000, size=9)
    all_rows = check_logprobs(torch_dev, x, 50000, t, 87381, 20)
    for r in range(9):
        for a, b in zip(all_rows, check_logprobs(torch_dev, x[r:r + 1], 50000, t[r:r + 1], 87381, 20)):
            assert np.array_equal(a[r:r + 1], b)


# -- together --------------------------------------------------------------------------------------------------------


class Chain:
    """Sequences through append (norms, shifts), attention, weights and a cut, by the GPU and by the oracle side by side."""

    def __init__(self, torch, bits, hd=64, seed=90):
        self.torch, self.hd = torch, hd
        c = self.c = Case(seed, [(30, 30), (1, 50), (9, 70)], 8, 2, hd, 16, bits, spare=12)
        self.d = More(torch, c)
        self.cos, self.sin = rope_tables(300, hd)
        self.qn, self.kn = (c.g.integers(2000, 7000, size=hd).astype(np.int16) for _ in range(2))
        self.k, self.v, self.w = c.k.copy(), c.v.copy(), self.d.w0.copy()
        self.shift = np.zeros(3, dtype=np.int32)
        self.dev = [put(torch, a) for a in (self.cos, self.sin, self.qn, self.kn)]
        self.shift_dev = put(torch, self.shift)
        self.kept = torch.zeros(3, 2, 40, dtype=torch.int32, device="cuda")
        free = np.setdiff1d(np.arange(c.pages), c.table)
        self.to = free[:9].reshape(3, 3).astype(np.int32)
        self.to_dev = put(torch, self.to)
        self.qrot = torch.zeros_like(self.d.q)

    def gpu(self, s=None):
        d, (cos, sin, qn, kn) = self.d, self.dev
        d.kv.append(d.qkv, d.b, 8, cos, sin, self.qrot, s, qn, kn, self.shift_dev)
        d.kv.attend(self.qrot, d.b, 8, d.exp, d.o, d.ws, 0, 0, s, stats=d.stats)
        d.kv.weigh(self.qrot, d.b, 8, d.exp, d.stats, 0, 0, False, s)

    def cut(self, s=None):
        self.d.kv.evict(self.d.b, self.to_dev, 40, self.kept, 10, 2, s)

    def oracle(self):
        c = self.c
        P = c.oracle(self.k, self.v)
        q = np.zeros((c.tokens, c.width), dtype=np.int8)
        O.paged_norm_append(P, c.qkv, 8, self.cos, self.sin, q, self.qn, self.kn, self.shift, self.w)
        o = np.full((c.tokens, c.width), FILL, dtype=np.int8)
        O.paged_attend(P, q, 8, c.exp, o)
        O.paged_weigh(P, q, 8, c.exp, O.paged_stats(P, q, 8, c.exp), self.w)
        return o

    def oracle_cut(self):
        return O.paged_evict(self.c.oracle(self.k, self.v), self.to, 40, 10, 2, self.w)

    def check(self, o, kept, what):
        same(self.d.o, o, f"o {what}")
        same(self.kept, kept, f"kept {what}")
        same(self.d.kv.k, self.k.view(np.int8), f"k {what}")
        same(self.d.kv.v, self.v.view(np.int8), f"v {what}")
        same(self.d.kv.w, self.w, f"w {what}")


@pytest.mark.parametrize("bits,hd", HD_BITS)
def test_together(torch_dev, bits, hd):
    """Append, attend, weigh and cut; then single tokens on the cut sequences, whose rotations go on from their shifts."""
    torch = torch_dev
    t = Chain(torch, bits, hd)
    say(f"case: together bits={bits} hd={hd}")
    t.gpu()
    t.cut()
    o, kept = t.oracle(), t.oracle_cut()
    t.check(o, kept, "first")
    # the cut sequences as they go on: two of them (the first was shorter than the budget), one new token each
    c, d = t.c, t.d
    c.lens = [(1, min(L, 40) + 1) for _, L in c.lens]
    t.shift = np.array([max(0, int(L) - 40) for L in c.kv_len], dtype=np.int32)
    c.kv_len = np.array([L for _, L in c.lens], dtype=np.int32)
    c.row_start, c.tokens = np.arange(4, dtype=np.int32), 3
    c.table, c.max_pages = t.to, 3
    c.q, c.qkv = c.q[:3], c.rows8(3, c.qkv.shape[1])
    from tritify_amd.paged import PagedBatch

    d.b = PagedBatch(put(torch, c.row_start), put(torch, c.kv_len), t.to_dev, 3)
    d.ws, d.stats, d.o, d.qkv, t.qrot = d.kv.workspace(d.b, 8), d.stats[:3], d.o[:3], put(torch, c.qkv), t.qrot[:3]
    t.shift_dev = put(torch, t.shift)
    t.gpu()
    t.check(t.oracle(), kept, "then")


def test_together_captured(torch_dev):
    """The four calls and the logits' log probabilities captured once: each replay follows what its arrays then hold, with eager
    calls of other shapes between the replays."""
    import tritify_amd as TA

    torch = torch_dev
    t, other = Chain(torch, 8), Chain(torch, 4, 128, seed=91)
    x = torch.zeros(3, 9000, dtype=torch.int32, device="cuda")
    tok, lp, ent = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    top, top_lp = (torch.zeros(3, 6, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = torch.empty(TA.dec_logprobs_rows_workspace(3, 9000, 6), dtype=torch.int8, device="cuda")
    scale = TA.logit_scale(90000)

    def step(s):
        t.gpu(s)
        t.cut(s)
        TA.dec_logprobs_rows(x, 3, 9000, tok, scale, lp, ws, ent, top, top_lp, 6, stream=s)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        step(s)
        g.capture_end()
    torch.cuda.synchronize()
    for i in range(4):
        say(f"case: replay {i}")
        c = t.c
        c.kv_len = np.array([30 - i, 50 - 9 * i, 70 + i], dtype=np.int32)
        c.qkv = c.rows8(*c.qkv.shape)
        t.shift = np.array([i, 5 * i, 0], dtype=np.int32)
        logits = np.round(c.g.normal(0, 1 << 18, size=(3, 9000))).astype(np.int32)
        tokens = c.g.integers(0, 9000, size=3).astype(np.int32)
        for to, a in ((t.d.b.kv_len, c.kv_len), (t.d.qkv, c.qkv), (t.shift_dev, t.shift), (x, logits), (tok, tokens)):
            to.copy_(torch.from_numpy(a))
        other.gpu()
        other.cut()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        o = t.oracle()
        t.check(o, t.oracle_cut(), f"replay {i}")
        for got, want in zip((lp, ent, top, top_lp), O.logprobs_rows(logits, 9000, tokens, *scale, 6)):
            assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("own", [True, False])
def test_a_long_table_captured(torch_dev, own):
    """Attention in splits with its statistics, the weights from 0 and a cut by several CTAs captured once, with the cut's scratch
    given or of its own; between the replays eager calls of the same pools."""
    torch = torch_dev
    c = Case(95, [(1, 30000), (3, 260)], 4, 2, 64, 64, 4, spare=14)
    d = More(torch, c)
    kept = torch.zeros(2, 2, 400, dtype=torch.int32, device="cuda")
    to = np.setdiff1d(np.arange(c.pages), c.table)[:14].reshape(2, 7).astype(np.int32)
    to_dev = put(torch, to)
    ws = None if own else torch.empty(d.kv.evict_workspace_bytes(d.b), dtype=torch.int8, device="cuda")
    assert d.kv.evict_workspace_bytes(d.b) > 256

    def step(s):
        d.kv.attend(d.q, d.b, 4, d.exp, d.o, d.ws, 0, 0, s, stats=d.stats)
        d.kv.weigh(d.q, d.b, 4, d.exp, d.stats, 0, 0, True, s)
        d.kv.evict(d.b, to_dev, 400, kept, 50, 4, s, ws)

    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.capture_begin()
        step(s)
        g.capture_end()
    torch.cuda.synchronize()
    k, v, w = c.k.copy(), c.v.copy(), d.w0.copy()

    def want():
        stats = O.paged_stats(c.oracle(k, v), c.q, 4, c.exp)
        for b in range(2):  # fresh
            for j in range(int(c.kv_len[b])):
                w[c.table[b, j // 64], :, j % 64] = 0
        O.paged_weigh(c.oracle(k, v), c.q, 4, c.exp, stats, w)
        return O.paged_evict(c.oracle(k, v), to, 400, 50, 4, w)

    for i in range(3):
        say(f"case: replay {i}")
        c.kv_len = np.array([30000 - 777 * i, 260 - 60 * i], dtype=np.int32)
        c.q = c.rows8(*c.q.shape)
        d.b.kv_len.copy_(torch.from_numpy(c.kv_len))
        d.q.copy_(torch.from_numpy(c.q))
        torch.cuda.synchronize()
        for by in (g.replay, lambda: step(None)):
            kept.fill_(FILL)
            torch.cuda.synchronize()
            by()
            torch.cuda.synchronize()
            chosen = want()
            same(kept, chosen, "kept")
            same(d.kv.w, w, "sums")
            same(d.kv.k, k.view(np.int8), "k")
            same(d.kv.v, v.view(np.int8), "v")


def test_two_streams_at_once(torch_dev):
    """Two chains and two batches of logits on two streams side by side, each with its own buffers."""
    import tritify_amd as TA

    torch = torch_dev
    ts, ss = [Chain(torch, 8), Chain(torch, 4, 128, seed=92)], [torch.cuda.Stream() for _ in range(2)]
    g = np.random.default_rng(9)
    xs = [np.round(g.normal(0, 1 << 18, size=(4, 151936))).astype(np.int32) for _ in ts]
    tok = np.array([1, 2, 3, 4], dtype=np.int32)
    bufs = []
    for x in xs:
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        bufs.append((put(torch, x), put(torch, tok), i32(4), i32(4), i32(4, 9), i32(4, 9),
                     torch.empty(TA.dec_logprobs_rows_workspace(4, 151936, 9), dtype=torch.int8, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(3):
        for t, s, (x, k, lp, ent, top, tlp, ws) in zip(ts, ss, bufs):
            t.gpu(s)
            t.cut(s)
            TA.dec_logprobs_rows(x, 4, 151936, k, TA.logit_scale(87381), lp, ws, ent, top, tlp, 9, stream=s)
    torch.cuda.synchronize()
    for t, x, b in zip(ts, xs, bufs):
        for _ in range(3):
            o = t.oracle()
            kept = t.oracle_cut()
        t.check(o, kept, "streams")
        for got, want in zip(b[2:6], O.logprobs_rows(x, 151936, tok, *TA.logit_scale(87381), 9)):
            assert np.array_equal(got.cpu().numpy(), want)


def test_wrapper_refusals(torch_dev):
    from tritify_amd.paged import PagedBatch, PagedKV

    torch = torch_dev
    c = Case(50, [(2, 40)], 4, 2, 64, 16, 8, spare=6)
    d = More(torch, c)
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    plain = Dev(torch, c).kv
    cos, sin = (put(torch, a) for a in rope_tables(64, 64))
    app = lambda **kw: d.kv.append(d.qkv, d.b, 4, cos, sin, d.o, **kw)  # noqa: E731
    for bad in (lambda: PagedKV(4, 16, 2, 64, w=z(4, 2, 16)), lambda: PagedKV(4, 16, 2, 64, w=z(4, 2, 32, dt=torch.int64)),
                lambda: PagedBatch(d.b.row_start, d.b.kv_len, d.b.table, 2, shift=z(2)),
                lambda: PagedBatch(d.b.row_start, d.b.kv_len, d.b.table, 2, shift=z(1, dt=torch.int64)),
                lambda: app(q_norm=z(64)), lambda: app(k_norm=z(32, dt=torch.int16)), lambda: app(shift=z(2)),
                lambda: app(q_norm=z(128, dt=torch.int16)[::2]), lambda: app(q_norm=z(65, dt=torch.int16)[1:]),
                lambda: d.kv.attend(d.q, d.b, 4, d.exp, d.o, d.ws, stats=z(2, 4, 1)),
                lambda: d.kv.attend(d.q, d.b, 4, d.exp, d.o, d.ws, stats=z(2, 4, 2, dt=torch.int64)),
                lambda: plain.weigh(d.q, d.b, 4, d.exp, d.stats), lambda: plain.evict(d.b, z(1, 2), 20, z(1, 2, 20)),
                lambda: d.kv.weigh(d.q, d.b, 4, d.exp, d.stats[:1]), lambda: d.kv.weigh(d.q[:1], d.b, 4, d.exp, d.stats),
                lambda: d.kv.weigh(d.q, d.b, 5, d.exp, d.stats), lambda: d.kv.weigh(d.q, d.b, 4, d.exp, d.stats, window=-1),
                lambda: d.kv.evict(d.b, z(1, 1), 20, z(1, 2, 20)), lambda: d.kv.evict(d.b, z(1, 2), 20, z(1, 2, 21)),
                lambda: d.kv.evict(d.b, z(1, 2), 0, z(1, 2, 0)), lambda: d.kv.evict(d.b, z(1, 2), 20, z(1, 2, 20), recent=18, sinks=3),
                lambda: d.kv.evict(d.b, z(1, 2), 20, z(1, 2, 20), recent=-1)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    same(d.attend(), c.attend(0, 0, FILL))
