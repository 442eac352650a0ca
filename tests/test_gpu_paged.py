"""The operators on paged caches (kt_hip_dec_*_paged, kt_hip_dec_argmax_rows) on the GPU against the oracle's value-by-value
restatement, byte for byte: whole pools, and every output row with the rows that no sequence has."""
import sys

import numpy as np
import pytest

from oracle import oracle as O
from paged_cases import Case, rope_tables

pytestmark = pytest.mark.gpu
FILL = 77


def say(*a):
    print(*a, file=sys.stderr, flush=True)


class Dev:
    """A Case's arrays on the GPU, and the calls on them."""

    def __init__(self, torch, c):
        from tritify_amd.paged import PagedBatch, PagedKV

        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.torch, self.c = torch, c
        n = (c.pages, c.nkv, -1)
        self.kv = PagedKV(c.pages, c.page, c.nkv, c.hd, c.bits, k=put(c.k.view(np.int8).reshape(n)),
                          v=put(c.v.view(np.int8).reshape(n)))
        self.b = PagedBatch(put(c.row_start), put(c.kv_len), put(c.table), c.tokens)
        self.q, self.qkv, self.exp = put(c.q), put(c.qkv), put(c.exp)
        self.o = torch.full((c.tokens, c.width), FILL, dtype=torch.int8, device="cuda")
        self.ws = self.kv.workspace(self.b, c.nh)
        self.ws.fill_(0x5A)

    def attend(self, window=0, sinks=0, stream=None):
        self.kv.attend(self.q, self.b, self.c.nh, self.exp, self.o, self.ws, window, sinks, stream)
        return self.o

    def append(self, cos, sin, stream=None):
        put = lambda a: self.torch.from_numpy(a).cuda()  # noqa: E731
        self.kv.append(self.qkv, self.b, self.c.nh, put(cos), put(sin), self.o, stream)
        return self.o


def same(got, want, what=""):
    got = got.cpu().numpy()
    want = want.reshape(got.shape)
    if not np.array_equal(got, want):
        bad = np.argwhere(got != want)
        pytest.fail(f"{what}: {len(bad)} of {got.size} differ, first at {bad[0].tolist()}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}")


def check_attend(torch, c, window=0, sinks=0):
    say(f"case: attend lens={c.lens[:6]} heads={c.nh}/{c.nkv} hd={c.hd} page={c.page} bits={c.bits} window={window}/{sinks}")
    d = Dev(torch, c)
    same(d.attend(window, sinks), c.attend(window, sinks, FILL), "attend")
    return d


HEADS = [(1, 1, 64), (14, 2, 64), (4, 4, 64), (20, 1, 64), (16, 4, 128), (9, 3, 128), (33, 1, 128)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("bits", [8, 4])
def test_attend_heads(torch_dev, nh, nkv, hd, bits):
    """Single tokens, a chunk behind a cache, a whole prompt, a sequence without rows, in one batch, at every head layout."""
    page = {1: 16, 14: 32, 4: 64, 20: 128, 16: 256, 9: 16, 33: 64}[nh]
    check_attend(torch_dev, Case(nh, [(1, 1), (1, 77), (0, 50), (13, 90), (35, 35), (1, 300)], nh, nkv, hd, page, bits, behind=3, pad=16))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 511, 513, 1025, 2500])
def test_attend_one_row_lengths(torch_dev, L, bits):
    check_attend(torch_dev, Case(L, [(1, L)], 14, 2, 64, 16, bits))


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
def test_attend_long(torch_dev, bits, hd):
    """Long enough that the positions are split over CTAs, and several times a CTA's own share."""
    check_attend(torch_dev, Case(5, [(1, 20011), (2, 9000)], 7, 1, hd, 64, bits))


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
@pytest.mark.parametrize("n,L", [(2, 2), (5, 700), (16, 16), (64, 333), (130, 130), (200, 1500)])
def test_attend_chunks(torch_dev, n, L, bits, hd):
    check_attend(torch_dev, Case(n, [(n, L), (max(1, n - 3), L + 40)], 7, 1, hd, 32, bits))


def test_attend_many_sequences(torch_dev):
    """More sequences than the 64 that one look at the row starts covers, short and long ones mixed."""
    lens = [((i * 7) % 5, (i * 7) % 5 + (i * 53) % 200) for i in range(150)]
    check_attend(torch_dev, Case(6, lens, 4, 2, 64, 16, 8))
    check_attend(torch_dev, Case(7, [(1, 40 + 3 * i) for i in range(130)], 4, 2, 64, 16, 8))


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
@pytest.mark.parametrize("seqs,nkv,window", [(150, 2, 0), (150, 2, 50), (420, 4, 0), (420, 4, 33)])
def test_attend_more_units_than_cus(torch_dev, seqs, nkv, window, bits, hd):
    """Single tokens, sequences without rows and chunks, more column tiles than CUs and many times as many."""
    lens = [(60, 90 + i) if i % 100 == 7 else (int(i % 9 > 0), 1 + (i * 53) % 140) for i in range(seqs)]
    check_attend(torch_dev, Case(60, lens, 4 * nkv if seqs < 400 else nkv, nkv, hd, 16, bits, behind=2), window, 3)


@pytest.mark.parametrize("seqs", [63, 64, 65, 4095, 4097, 9000])
def test_sequences_are_found_among_many(torch_dev, seqs):
    """Runs of sequences without rows, at the counts where the search takes another level: append and attention."""
    lens = [(0, 3) if i % 5 < 3 and i % 70 > 9 else (1 + i % 3 + 20 * (i % 61 == 0), 25 + i % 3) for i in range(seqs)]
    c = Case(62, lens, 2, 1, 64, 16, 8, behind=3)
    check_attend(torch_dev, c)
    cos, sin = rope_tables(30, 64)
    d = Dev(torch_dev, c)
    q, k, v = c.append(cos, sin, FILL)
    same(d.append(cos, sin), q, "q")
    same(d.kv.k, k.view(np.int8), "k pool")
    same(d.kv.v, v.view(np.int8), "v pool")


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
@pytest.mark.parametrize("window", [0, 2100])
def test_attend_chunk_behind_more_than_a_cta_keeps(torch_dev, window, bits, hd):
    check_attend(torch_dev, Case(61, [(160, 2600), (1, 4100), (3, 4000)], 7, 1, hd, 16, bits), window, 70)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (65, 4), (100, 20), (300, 64), (128, 1000), (5000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_attend_window(torch_dev, window, sinks, bits):
    check_attend(torch_dev, Case(8, [(1, 1), (1, 900), (30, 700), (70, 70), (150, 1000)], 7, 1, 64, 16, bits), window, sinks)


@pytest.mark.parametrize("window,sinks", [(300, 5), (4000, 0), (9000, 700)])
@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
def test_attend_window_in_a_wide_table(torch_dev, window, sinks, bits, hd):
    """Positions far behind the window: what divides the work is what the window reaches."""
    check_attend(torch_dev, Case(12, [(1, 20011), (2, 9000), (1, 100)], 7, 1, hd, 64, bits), window, sinks)


@pytest.mark.parametrize("bits", [8, 4])
def test_attend_pages_left_out(torch_dev, bits):
    """Entries outside the pool leave positions out (rows of the batch among them); a sequence without any page is zeros."""
    c = Case(9, [(1, 400), (40, 200), (1, 64), (3, 33), (1, 2000)], 4, 2, 64, 16, bits)
    c.table[0, [0, 3, 4, 20]] = [-1, c.pages, 2 ** 31 - 1, -(2 ** 31)]
    c.table[1, [1, 11, 12]] = [-7, c.pages + 5, -1]
    c.table[2] = -1
    c.table[3, 2] = c.pages
    c.table[4, :100] = -1
    d = check_attend(torch_dev, c)
    t = int(c.row_start[2])
    assert (d.o[t] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_attend_positions_outside(torch_dev, bits):
    """kv_len below the rows (the first rows are at negative positions), past the table, and extreme; row_start that starts
    late and ends early leaves the other rows as they were."""
    c = Case(10, [(5, 3), (4, 70), (2, 8), (3, 9)], 4, 2, 64, 16, bits, behind=6)
    c.kv_len = np.array([3, 2 ** 31 - 1, -(2 ** 31), 16 * c.max_pages + 1], dtype=np.int32)
    check_attend(torch_dev, c)
    c.row_start = (c.row_start + 4).astype(np.int32)
    c.kv_len = np.array([5, 70, 3, 16 * c.max_pages + 1], dtype=np.int32)
    check_attend(torch_dev, c)


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
@pytest.mark.parametrize("what", ["peaks", "flat", "zeros", "beyond", "step"])
def test_attend_tables_and_extremes(torch_dev, what, bits, hd):
    c = Case(11, [(1, 700), (33, 250), (1, 5), (1, 6000)], 7, 1, hd, 16, bits, sigma=200 if what == "peaks" else 32)
    if what == "flat":
        c.exp[:] = 32768
    if what == "zeros":
        c.exp[:] = 0
    if what == "beyond":  # clamped into [0, 2^15]
        c.exp[::3], c.exp[1::3] = 2 ** 31 - 1, -5
    if what == "step":
        c.exp[1:] = 0
    if what == "peaks":  # every value at an end of its range
        for a in (c.q, c.k.view(np.int8) if bits == 8 else c.q, c.v.view(np.int8) if bits == 8 else c.q):
            a[:] = np.where(a < 0, -128, 127)
        if bits == 4:
            c.k[:, : c.page * hd // 2], c.v[:, : c.page * hd // 2] = 0x77, 0x99
            c.k[:, c.page * hd // 2:] = c.v[:, c.page * hd // 2:] = 147
    check_attend(torch_dev, c)


@pytest.mark.parametrize("nh,nkv,hd,page", [(14, 2, 64, 16), (8, 8, 64, 64), (16, 4, 128, 32), (3, 1, 128, 256)])
@pytest.mark.parametrize("bits", [8, 4])
def test_append_and_read(torch_dev, nh, nkv, hd, page, bits):
    """Rows that fill blocks of 16 positions, begin and end inside them, at one row and at none; pools, q rows and the read
    back whole."""
    torch = torch_dev
    lens = [(1, 1), (1, 16), (1, 17), (0, 20), (16, 16), (16, 40), (15, 15), (47, 63), (1, 200), (33, 300), (0, 0)]
    c = Case(nh + bits, lens, nh, nkv, hd, page, bits, behind=2, pad=32)
    cos, sin = rope_tables(290, hd)  # the last positions of (33, 300) are past the tables
    say(f"case: append lens={lens} heads={nh}/{nkv} hd={hd} page={page} bits={bits}")
    d = Dev(torch, c)
    q, k, v = c.append(cos, sin, FILL)
    same(d.append(cos, sin), q, "q")
    same(d.kv.k, k.view(np.int8), "k pool")
    same(d.kv.v, v.view(np.int8), "v pool")
    same(d.append(cos, sin), q, "q again")
    same(d.kv.v, v.view(np.int8), "v pool again")
    for max_pos in (1, 100, 333):
        want = [np.full((len(lens), max_pos, nkv, hd), FILL, dtype=np.int8) for _ in range(2)]
        O.paged_read(c.oracle(k, v), *want)
        got = [torch.full(want[0].shape, FILL, dtype=torch.int8, device="cuda") for _ in range(2)]
        d.kv.read(d.b, *got)
        same(got[0], want[0], f"read k {max_pos}")
        same(got[1], want[1], f"read v {max_pos}")


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
def test_append_many_sequences(torch_dev, bits, hd):
    """More blocks than the chip takes at once: single tokens and chunks, begun and ended inside blocks."""
    lens = [(50, 70 + i) if i % 40 == 3 else (int(i % 7 > 0), 1 + (i * 29) % 90) for i in range(130)]
    c = Case(22, lens, 8, 4, hd, 32, bits, behind=2, pad=16)
    cos, sin = rope_tables(200, hd)
    d = Dev(torch_dev, c)
    q, k, v = c.append(cos, sin, FILL)
    same(d.append(cos, sin), q, "q")
    same(d.kv.k, k.view(np.int8), "k pool")
    same(d.kv.v, v.view(np.int8), "v pool")


@pytest.mark.parametrize("bits", [8, 4])
def test_append_outside_and_extremes(torch_dev, bits):
    torch = torch_dev
    c = Case(20, [(20, 7), (40, 60), (5, 5), (3, 50), (2, 18)], 4, 2, 64, 16, bits, behind=3)
    c.qkv[:] = np.where(c.qkv < 0, -128, 127)
    c.qkv[30:40] = 0
    c.table[1, 1], c.table[3, 3] = -1, c.pages
    c.kv_len[4] = 16 * c.max_pages + 1
    cos, sin = rope_tables(64, 64)
    d = Dev(torch, c)
    q, k, v = c.append(cos, sin, FILL)
    same(d.append(cos, sin), q, "q")
    same(d.kv.k, k.view(np.int8), "k pool")
    same(d.kv.v, v.view(np.int8), "v pool")
    want = [np.full((5, 64, 2, 64), FILL, dtype=np.int8) for _ in range(2)]
    O.paged_read(c.oracle(k, v), *want)
    got = [torch.full(want[0].shape, FILL, dtype=torch.int8, device="cuda") for _ in range(2)]
    d.kv.read(d.b, *got)
    same(got[0], want[0], "read k")
    same(got[1], want[1], "read v")


@pytest.mark.parametrize("bits", [8, 4])
def test_offsets_past_32_bits(torch_dev, bits):
    """Pools of more than 4 GiB, the pages in use at their end."""
    torch = torch_dev
    c = Case(21, [(1, 700), (20, 300)], 8, 4, 128, 256, bits)
    d = Dev(torch, c)
    part = c.k.shape[1]
    pages = (5 << 30) // (4 * part)
    say(f"case: {pages} pages of {4 * part} bytes in each pool")
    from tritify_amd.paged import PagedBatch, PagedKV

    big = [torch.empty(pages, 4, part, dtype=torch.int8, device="cuda") for _ in range(2)]
    for to, frm in zip(big, (d.kv.k, d.kv.v)):
        to[-c.pages:] = frm
    table = np.where(c.table >= 0, c.table + pages - c.pages, -1).astype(np.int32)
    kv = PagedKV(pages, 256, 4, 128, bits, k=big[0], v=big[1])
    b = PagedBatch(d.b.row_start, d.b.kv_len, torch.from_numpy(table).cuda(), c.tokens)
    kv.attend(d.q, b, 8, d.exp, d.o, d.ws)
    same(d.o, c.attend(0, 0, FILL), "attend")
    cos, sin = rope_tables(700, 128)
    q, k, v = c.append(cos, sin, FILL)
    d.o.fill_(FILL)
    kv.append(d.qkv, b, 8, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), d.o)
    same(d.o, q, "q")
    same(big[0][-c.pages:], k.view(np.int8), "k pool")
    same(big[1][-c.pages:], v.view(np.int8), "v pool")
    want = [np.zeros((2, 700, 4, 128), dtype=np.int8) for _ in range(2)]
    O.paged_read(c.oracle(k, v), *want)
    got = [torch.zeros(want[0].shape, dtype=torch.int8, device="cuda") for _ in range(2)]
    kv.read(b, *got)
    same(got[0], want[0], "read k")
    same(got[1], want[1], "read v")


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 2), (3, 97), (1, 4097), (5, 4096), (2, 151936), (64, 5000), (70, 300), (2, 65536), (3, 65537), (1, 1023), (1, 1025), (300, 70000), (1, 100000), (2, 100001), (255, 101000)])
def test_argmax_rows(torch_dev, rows, n):
    """Distinct values, ties (the first wins), all equal, both ends of int32, a stride, rows far apart."""
    import tritify_amd as TA

    torch = torch_dev
    g = np.random.default_rng(n)
    say(f"case: argmax rows={rows} n={n}")
    x = g.integers(-(2 ** 31), 2 ** 31, size=(rows, n + 5)).astype(np.int32)
    x[rows // 2] = g.integers(-2, 2, size=n + 5)
    x[-1] = -(2 ** 31)
    x[:, n:] = 2 ** 31 - 1  # past the row
    xd = torch.from_numpy(x).cuda()
    t = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    ws = torch.full((TA.dec_argmax_rows_workspace(rows, n),), 0x7F, dtype=torch.int8, device="cuda")
    for _ in range(2):
        TA.dec_argmax_rows(xd, rows, n, t, ws, stride=n + 5)
        assert t.cpu().numpy().tolist() == O.argmax_rows(x, n).tolist() + [-9]


def test_replayed_graph_follows_its_arrays(torch_dev):
    """append + attend + read + argmax captured once: each replay uses the lengths, tables and rows that the arrays then
    hold, with eager calls of other shapes between the replays."""
    import tritify_amd as TA

    torch = torch_dev
    c = Case(30, [(1, 900), (1, 30), (1, 500)], 14, 2, 64, 16, 8)
    d, other = Dev(torch, c), Dev(torch, Case(31, [(60, 90), (1, 2000)], 4, 1, 128, 32, 4))
    cos, sin = rope_tables(1000, 64)
    cd, sd = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    k, v = (torch.zeros(3, 64, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    x = torch.zeros(3, 110000, dtype=torch.int32, device="cuda")
    t, ws = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.empty(TA.dec_argmax_rows_workspace(3, 110000), dtype=torch.int8, device="cuda")

    def step(s):
        d.kv.append(d.qkv, d.b, 14, cd, sd, d.q, s)
        d.kv.attend(d.q, d.b, 14, d.exp, d.o, d.ws, 0, 0, s)
        d.kv.read(d.b, k, v, s)
        TA.dec_argmax_rows(x, 3, 110000, t, ws, stream=s)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step(s)
        torch.cuda.synchronize()
        g.capture_begin()
        step(s)
        g.capture_end()
    torch.cuda.synchronize()
    want_k, want_v = c.append(cos, sin)[1:]
    for i in range(4):
        say(f"case: replay {i}")
        c.kv_len = np.array([900 - 7 * i, 30 - i, 1 + 100 * i], dtype=np.int32)
        c.qkv = c.rows8(*c.qkv.shape)
        logits = c.g.integers(-50, 50, size=(3, 110000)).astype(np.int32)
        d.b.kv_len.copy_(torch.from_numpy(c.kv_len))
        d.qkv.copy_(torch.from_numpy(c.qkv))
        x.copy_(torch.from_numpy(logits))
        other.attend()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        c.k, c.v = want_k, want_v
        c.q, want_k, want_v = c.append(cos, sin)
        c.k, c.v = want_k, want_v
        same(d.o, c.attend(0, 0, FILL), f"attend {i}")
        same(d.kv.k, c.k.view(np.int8), f"k pool {i}")
        want = [np.zeros((3, 64, 2, 64), dtype=np.int8) for _ in range(2)]
        O.paged_read(c.oracle(), *want)
        n = [min(64, int(L)) for L in c.kv_len]
        for b in range(3):
            same(k[b, :n[b]], want[0][b, :n[b]], f"read {i}")
        assert t.cpu().numpy().tolist() == O.argmax_rows(logits, 110000).tolist()


def test_two_streams_and_two_captured_graphs(torch_dev):
    """Two batches on two streams at once, eagerly and as graphs replayed side by side, each with its own workspace."""
    torch = torch_dev
    cs = [Case(40, [(1, 5000), (1, 3000)], 14, 2, 64, 16, 8), Case(41, [(1, 4000), (150, 900)], 8, 2, 128, 32, 4)]
    ds, ss = [Dev(torch, c) for c in cs], [torch.cuda.Stream() for _ in cs]
    want = [c.attend(0, 0, FILL) for c in cs]
    torch.cuda.synchronize()
    for _ in range(3):
        for d, s in zip(ds, ss):
            for _ in range(5):
                d.attend(stream=s)
    torch.cuda.synchronize()
    for d, w in zip(ds, want):
        same(d.o, w, "eager")
    gs = []
    for d, s in zip(ds, ss):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            g.capture_begin()
            d.attend(stream=s)
            g.capture_end()
        gs.append(g)
    for _ in range(3):
        for d in ds:
            d.o.fill_(FILL)
        torch.cuda.synchronize()
        for g, s in zip(gs, ss):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for d, w in zip(ds, want):
            same(d.o, w, "replayed")


def test_wrapper_refusals(torch_dev):
    from tritify_amd.paged import PagedBatch, PagedKV

    torch = torch_dev
    c = Case(50, [(2, 40)], 4, 2, 64, 16, 8)
    d = Dev(torch, c)
    z = lambda *s, dt=torch.int8: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    for bad in (lambda: PagedKV(4, 24, 2, 64), lambda: PagedKV(4, 16, 0, 64), lambda: PagedKV(4, 16, 2, 64, k=z(4, 2, 16)),
                lambda: PagedBatch(z(3, dt=torch.int32), z(1, dt=torch.int32), z(1, 4, dt=torch.int32), 2),
                lambda: PagedBatch(z(2, dt=torch.int32), z(1, dt=torch.int64), z(1, 4, dt=torch.int32), 2),
                lambda: PagedBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                   torch.zeros(1, 4, dtype=torch.int32), 2),
                lambda: d.kv.attend(d.q[:1], d.b, 4, d.exp, d.o, d.ws),
                lambda: d.kv.attend(d.q[:, ::2], d.b, 4, d.exp, d.o, d.ws),
                lambda: d.kv.attend(z(2, 264)[:, 3:], d.b, 4, d.exp, d.o, d.ws),
                lambda: d.kv.attend(d.q, d.b, 4, d.exp[:100], d.o, d.ws),
                lambda: d.kv.attend(d.q, d.b, 4, d.exp.long(), d.o, d.ws),
                lambda: d.kv.attend(d.q, d.b, 5, d.exp, d.o, d.ws),
                lambda: d.kv.append(d.qkv, d.b, 4, z(9, 32, dt=torch.int16), z(8, 32, dt=torch.int16), d.o),
                lambda: d.kv.read(d.b, z(1, 40, 2, 64), z(1, 40, 2, 32)),
                lambda: d.kv.read(d.b, z(2, 40, 2, 64), z(2, 40, 2, 64))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    same(d.attend(), c.attend(0, 0, FILL))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("row_start", [[0, 90, 40, 60], [90, 0, 90, 30, 90], [0, 90, 89, 88, 87, 90], [-5, 200, -7, 50], [70, 10]])
def test_row_starts_that_decrease_reach_no_other_memory(torch_dev, row_start, bits):
    """Outputs between guard rows, pools with pages that no table names: only the batch's rows and its tables' pages change."""
    from tritify_amd.paged import PagedBatch

    torch = torch_dev
    say(f"case: row_start={row_start} bits={bits}")
    seqs, T, G = len(row_start) - 1, 90, 32
    c = Case(70, [(1, 200)] * seqs, 14, 2, 64, 16, bits, spare=6)
    d = Dev(torch, c)
    b = PagedBatch(torch.tensor(row_start, dtype=torch.int32, device="cuda"), d.b.kv_len, d.b.table, T)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda width: torch.randint(-127, 128, (T + 2 * G, width), generator=g, device="cuda").to(torch.int8)  # noqa: E731
    q, qkv, ws = rows(14 * 64), rows(18 * 64), d.kv.workspace(b, 14)
    o = torch.full_like(q, FILL)
    unused = [p for p in range(c.pages) if p not in c.table]
    assert len(unused) == 6
    pools = [d.kv.k.clone(), d.kv.v.clone()]
    cos, sin = rope_tables(220, 64)
    d.kv.attend(q[G:G + T], b, 14, d.exp, o[G:G + T], ws)
    assert (o[:G] == FILL).all() and (o[G + T:] == FILL).all()
    assert torch.equal(pools[0], d.kv.k) and torch.equal(pools[1], d.kv.v)
    o.fill_(FILL)
    d.kv.append(qkv[G:G + T], b, 14, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), o[G:G + T])
    assert (o[:G] == FILL).all() and (o[G + T:] == FILL).all()
    for now, was in ((d.kv.k, pools[0]), (d.kv.v, pools[1])):
        assert torch.equal(now[unused], was[unused])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("what", ["any", "most", "flat"])
def test_attend_any_byte_in_a_4_bit_pool(torch_dev, what, hd):
    """A pool is the caller's memory: codes of -8 and multipliers past the 147 that an append writes, to 255 (255 * 2^15 has no
    three balanced digits, its negative does), by the same formula. In one launch, in split passes and in chunks."""
    c = Case(71, [(1, 1), (1, 9000), (1, 700), (33, 250)] if what == "any" else [(1, 5000)], 7, 1, hd, 16, 4)
    n = c.page * hd // 2
    c.k[:, :n], c.v[:, :n] = (c.g.integers(0, 256, size=(c.pages, n)) for _ in range(2))
    if what == "any":
        c.k[:, n:], c.v[:, n:] = (c.g.choice([0, 1, 147, 148, 200, 253, 254, 255], size=(c.pages, c.page)) for _ in range(2))
    else:
        c.k[:, n:], c.v[:, n:] = 255, 255
    if what == "flat":
        c.exp[:] = 32768
    check_attend(torch_dev, c)


# sequences of one new token each, positions of the table's width: the positions split over CTAs; 8, 4 and 2 waves at their 65536
# positions each; and the waves that a wider table asks for where the number of sequences alone would take fewer
RANGE = [(1, 524288), (70, 524288), (300, 262144), (300, 524288), (1600, 131072), (1600, 262144), (1600, 524288)]


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
@pytest.mark.parametrize("seqs,positions", RANGE)
def test_attend_digit_sums_at_their_bound(torch_dev, seqs, positions, bits, hd):
    """Tables as wide as a call takes, weights all 2^15, a dimension's value the same at every position: with equal weights a row's
    answer is that value, and each digit sum is the largest its wave can have. Every page is page 0."""
    from tritify_amd.paged import PagedBatch, PagedKV, page_bytes

    torch = torch_dev
    say(f"case: {seqs} sequences, {positions} positions, bits={bits} hd={hd}")
    page, nh = 256, 7
    if bits == 8:
        codes = np.resize([127, -128, -127, 0, 1, -1, 64, -65], hd)
        value = np.clip(codes, -127, 127)
        k, v = np.full(page * hd, 127, dtype=np.int8), np.broadcast_to(codes[None, :, None], (page // 16, hd, 16)).astype(np.int8).reshape(-1)
    else:
        codes, m = np.resize([7, -8, -7, 0, 1, -1, 3, -4], hd), 255
        value = np.clip(np.sign(codes) * ((np.abs(codes) * m + 4) // 8), -127, 127)
        byte = ((codes & 15) | ((codes & 15) << 4))[None, :, None]  # all 16 positions of a dimension alike
        v = np.concatenate([np.broadcast_to(byte, (page // 16, hd, 8)).astype(np.uint8).reshape(-1), np.full(page, m, dtype=np.uint8)])
        k = np.concatenate([np.full(page * hd // 2, 0x77, dtype=np.uint8), np.full(page, m, dtype=np.uint8)]).view(np.int8)
        v = v.view(np.int8)
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    part = page_bytes(page, hd, bits)
    kv = PagedKV(1, page, 1, hd, bits, k=put(k.reshape(1, 1, part)), v=put(v.reshape(1, 1, part)))
    rows = np.ones(seqs, dtype=np.int64)
    kv_len = 1 + (np.arange(seqs) * 37) % 300
    kv_len[seqs // 2] = positions
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    b = PagedBatch(put(start), put(kv_len.astype(np.int32)), torch.zeros(seqs, positions // page, dtype=torch.int32, device="cuda"), seqs)
    q = torch.full((seqs, nh * hd), 127, dtype=torch.int8, device="cuda")
    o, exp = torch.full_like(q, FILL), torch.full((1024,), 32768, dtype=torch.int32, device="cuda")
    kv.attend(q, b, nh, exp, o, kv.workspace(b, nh))
    same(o.reshape(seqs, nh, hd), np.broadcast_to(value.astype(np.int8), (seqs, nh, hd)))


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (8, 128), (4, 128)])
def test_attend_the_longest_table(torch_dev, bits, hd):
    """524288 positions of random values, a single token and the last rows of a chunk, pages named many times over."""
    c = Case(72, [(1, 30 * 256)], 2, 1, hd, 256, bits, spare=0)
    c.table = c.g.integers(0, c.pages, size=(2, 524288 // 256)).astype(np.int32)
    c.max_pages, c.tokens, c.lens = 524288 // 256, 3, [(1, 524288), (2, 400001)]
    c.kv_len, c.row_start = np.array([524288, 400001], dtype=np.int32), np.array([0, 1, 3], dtype=np.int32)
    c.q = c.rows8(3, c.width)
    check_attend(torch_dev, c)
