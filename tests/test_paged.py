"""The paged caches' rules on the CPU: the oracle's paged functions against the contiguous decoder's (kt_dec_rope_row,
kt_dec_attend) and against closed forms, and the arguments that the C ABI refuses before any device work."""
import numpy as np
import pytest

from oracle import oracle as O
from paged_cases import Case, exp_table, part_bytes, rope_tables


@pytest.mark.parametrize("page", [16, 64, 256])
def test_eight_bits_are_the_contiguous_decoder(page):
    nh, nkv, hd, L = 4, 2, 64, 83
    c = Case(1, [(L, L), (3, 40)], nh, nkv, hd, page, 8)
    cos, sin = rope_tables(200, hd)
    q, k, v = c.append(cos, sin)
    c.q, c.k, c.v = q, k, v
    o = c.attend()
    ck, cv = (np.zeros((L, nkv, hd), dtype=np.int8) for _ in range(2))
    for p in range(L):
        row = O.dec_rope(c.qkv[p, : (nh + nkv) * hd], nh + nkv, hd, p, cos, sin).reshape(-1, hd)
        ck[p], cv[p] = row[nh:], c.qkv[p, (nh + nkv) * hd:].reshape(nkv, hd)
        assert np.array_equal(q[p].reshape(nh, hd), row[:nh])
        for h in range(nh):
            want = O.dec_attend(row[h], ck, cv, p, nkv, h // 2, hd, c.exp)
            assert np.array_equal(o[p, h * hd:(h + 1) * hd], want), (p, h)
    rk, rv = (np.full((2, L + 5, nkv, hd), 9, dtype=np.int8) for _ in range(2))
    O.paged_read(c.oracle(), rk, rv)
    assert np.array_equal(rk[0, :L], ck) and np.array_equal(rv[0, :L], cv)
    assert (rk[0, L:] == 9).all() and (rv[1, 40:] == 9).all()


def test_four_bits_hold_what_they_say():
    """Rows whose largest magnitude is at most 7 and even multiples of it survive the 4 bits; every other value is off by
    half a multiplier step at most (m / 16), and by the rounding of the read (1 / 2)."""
    hd, nkv, page = 64, 1, 16
    cos, sin = np.full((16, 32), 16384, dtype=np.int16), np.zeros((16, 32), dtype=np.int16)
    for top in (0, 1, 2, 3, 5, 7, 8, 33, 127, 128):
        c = Case(2, [(16, 16)], 1, nkv, hd, page, 4)
        x = c.g.integers(-top, min(top, 127) + 1, size=(16, 3 * hd))
        x[:, hd] = x[:, 2 * hd] = -top
        c.qkv = x.astype(np.int8)
        q, c.k, c.v = c.append(cos, sin)
        k, v = (np.zeros((1, 16, nkv, hd), dtype=np.int8) for _ in range(2))
        O.paged_read(c.oracle(), k, v)
        for got, sent in ((k, np.clip(x[:, hd:2 * hd], -127, 127)), (v, x[:, 2 * hd:])):
            m = -(-8 * np.abs(sent).max(axis=1) // 7)
            off = np.abs(got[0, :, 0].astype(int) - sent)
            assert (16 * off <= (m + 16)[:, None]).all(), top
            if top in (0, 1, 2, 3, 7):  # m / 8 is 0, 1/4, 3/8, 1/2 or 1: 8 x / m is exact or rounds back
                assert (16 * off <= m[:, None]).all() and off.max() <= (0 if top != 2 else 1)


def unpacked(c, pool, is_v):
    """Codes [page][kv head][slot][hd] and multipliers [page][kv head][slot] (1 for 8 bits) of a pool."""
    n, x = c.page * c.hd, pool.reshape(c.pages, c.nkv, -1)
    if c.bits == 8:
        codes, m = x.view(np.int8).astype(np.int64), np.ones((c.pages, c.nkv, c.page), dtype=np.int64)
    else:
        b, m = x[..., : n // 2].reshape(c.pages, c.nkv, -1, 2, 4).astype(np.int64), x[..., n // 2:].astype(np.int64)
        codes = np.stack([b & 15, b >> 4], axis=-2).reshape(c.pages, c.nkv, n)
        codes = np.where(codes > 7, codes - 16, codes)
    if is_v:
        return codes.reshape(c.pages, c.nkv, c.page // 16, c.hd, 16).swapaxes(3, 4).reshape(c.pages, c.nkv, c.page, c.hd), m
    return codes.reshape(c.pages, c.nkv, c.page, c.hd), m


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (1, 50)])
@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 64), (4, 128)])
def test_attention_is_the_formula(bits, hd, window, sinks):
    c = Case(6, [(3, 90), (1, 40)], 4, 2, hd, 32, bits)
    c.table[0, 1] = -1
    o = c.attend(window, sinks)
    (kc, km), (vc, vm) = unpacked(c, c.k, False), unpacked(c, c.v, True)
    for b, (n, L) in enumerate(c.lens):
        for i in range(n):
            p = L - n + i
            j = np.arange(p + 1)
            page = c.table[b, j // c.page]
            see = (page >= 0) & ((window == 0) | (j > p - window) | (j < sinks))
            j, page = j[see], page[see]
            for h in range(c.nh):
                t, g = c.row_start[b] + i, h * c.nkv // c.nh
                s = kc[page, g, j % c.page] @ np.maximum(c.q[t, h * hd:(h + 1) * hd].astype(np.int64), -127)
                if bits == 4:
                    s = (km[page, g, j % c.page] * s + 4) >> 3
                ix = (s.max() - s + 64) >> 7
                e = np.where(ix < 1024, c.exp[np.minimum(ix, 1023)].astype(np.int64), 0)
                num = (e * vm[page, g, j % c.page]) @ vc[page, g, j % c.page]
                den = e.sum() * (8 if bits == 4 else 1)
                want = np.sign(num) * np.minimum((2 * np.abs(num) + den) // (2 * den), 127)
                assert np.array_equal(o[t, h * hd:(h + 1) * hd], want), (b, i, h)


@pytest.mark.parametrize("bits", [8, 4])
def test_window_equals_pages_left_out(bits):
    """A window without sinks is the attention of a table whose older pages are gone, where the window ends at a page."""
    c = Case(3, [(1, 16 * 9)], 4, 2, 64, 16, bits)
    o = c.attend(window=32)
    c.table[0, :7] = [-1, 99, c.pages, -5, 2 ** 30, -1, -1]
    assert np.array_equal(c.attend(), o)
    c.table[0, :] = -1
    assert (c.attend() == 0).all()


def _lib():
    from tritify_amd import backend as B

    return B.lib()


@pytest.mark.parametrize("page,hd,bits,want", [(16, 64, 8, 1024), (16, 64, 4, 528), (256, 128, 8, 32768), (256, 128, 4, 16640),
                                               (32, 128, 4, 2080), (8, 64, 8, 0), (48, 64, 8, 0), (512, 64, 8, 0), (16, 32, 8, 0),
                                               (16, 96, 4, 0), (16, 64, 2, 0), (0, 64, 8, 0), (-16, 64, 8, 0)])
def test_page_bytes(page, hd, bits, want):
    assert _lib().kt_hip_dec_page_bytes(page, hd, bits) == want
    if want:
        assert part_bytes(page, hd, bits) == want


P = 1 << 20  # an aligned address that no call here dereferences
APPEND = dict(dev=0, qkv=P, tokens=3, qkv_stride=512, row_start=P, kv_len=P, table=P, seqs=2, max_pages=4, nh=4, nkv=2, hd=64,
              cos=P, sin=P, max_pos=64, q=P, q_stride=256, k=P, v=P, pages=8, page=16, bits=8, stream=None)
READ = dict(dev=0, k=P, v=P, pages=8, page=16, bits=8, kv_len=P, table=P, seqs=2, max_pages=4, nkv=2, hd=64, ko=P, vo=P,
            max_pos=64, stream=None)
ATTEND = dict(dev=0, q=P, tokens=3, q_stride=256, row_start=P, kv_len=P, table=P, seqs=2, max_pages=4, nh=4, nkv=2, hd=64, exp=P,
              window=0, sinks=0, k=P, v=P, pages=8, page=16, bits=8, o=P, o_stride=256, ws=P, ws_bytes=1 << 40, stream=None)
ARGMAX = dict(dev=0, logits=P, rows=3, n=1000, stride=1000, token=P, ws=P, ws_bytes=1 << 40, stream=None)
GEOMETRY = [dict(page=24), dict(page=0), dict(hd=32), dict(hd=256), dict(bits=16), dict(seqs=-1), dict(max_pages=0),
            dict(max_pages=524288 // 16 + 1), dict(nkv=0), dict(pages=-1), dict(pages=1 << 31), dict(k=P + 8), dict(v=None),
            dict(kv_len=None), dict(table=None)]
HEADS = [dict(nh=5), dict(nh=0), dict(tokens=-1), dict(tokens=1 << 30), dict(seqs=1 << 29), dict(row_start=None)]
REFUSED = (
    [("kt_hip_dec_rope_kv_paged", APPEND, x) for x in GEOMETRY + HEADS + [
        dict(qkv_stride=511), dict(qkv_stride=520), dict(q_stride=240), dict(q_stride=264), dict(qkv=P + 4), dict(q=None),
        dict(cos=P + 4), dict(sin=None), dict(max_pos=-1), dict(max_pos=1 << 31)]]
    + [("kt_hip_dec_kv_read_paged", READ, x) for x in GEOMETRY + [
        dict(ko=None), dict(vo=P + 1), dict(max_pos=-1), dict(seqs=1 << 29, max_pos=1 << 20, max_pages=1 << 14)]]
    + [("kt_hip_dec_attention_paged", ATTEND, x) for x in GEOMETRY + HEADS + [
        dict(q_stride=240), dict(q_stride=257), dict(o_stride=128), dict(o_stride=260), dict(q=None), dict(o=P + 8), dict(exp=None),
        dict(window=-1), dict(sinks=-1), dict(ws=None), dict(ws=P + 4), dict(ws_bytes=0)]]
    + [("kt_hip_dec_argmax_rows", ARGMAX, x) for x in [
        dict(rows=-1), dict(rows=65536), dict(n=0), dict(n=1 << 31), dict(stride=999), dict(logits=None), dict(token=None),
        dict(ws=None), dict(ws=P + 4), dict(ws_bytes=0)]]
)


# past a grid's threads, just
BIG = [dict(tokens=1 << 25, qkv_stride=512), dict(tokens=(1 << 25) - 32, seqs=1), dict(seqs=1 << 20), dict(nh=4098, nkv=2, q_stride=1 << 20)]
REFUSED += (
    [("kt_hip_dec_rope_kv_paged", APPEND, {**{k: v for k, v in x.items() if k in APPEND}, **({"qkv_stride": 1 << 20} if "nh" in x else {})}) for x in BIG]
    + [("kt_hip_dec_attention_paged", ATTEND, {**{k: v for k, v in x.items() if k in ATTEND}, **({"o_stride": 1 << 20} if "nh" in x else {})}) for x in BIG]
    + [("kt_hip_dec_kv_read_paged", READ, dict(seqs=1 << 20, max_pos=256, max_pages=16)), ("kt_hip_dec_kv_read_paged", READ, dict(seqs=1 << 21))]
)


@pytest.mark.parametrize("name,args,change", REFUSED, ids=[f"{n[11:]}-{'-'.join(f'{k}={v}' for k, v in x.items())}" for n, _, x in REFUSED])
def test_refused_before_any_device_work(name, args, change):
    assert getattr(_lib(), name)(*{**args, **change}.values()) == 1  # hipErrorInvalidValue


def test_empty_calls_do_nothing():
    L = _lib()
    for empty in (dict(tokens=0), dict(seqs=0)):
        assert L.kt_hip_dec_rope_kv_paged(*{**APPEND, **empty, "qkv": None, "q": None}.values()) == 0
        assert L.kt_hip_dec_attention_paged(*{**ATTEND, **empty, "q": None, "o": None}.values()) == 0
    assert L.kt_hip_dec_kv_read_paged(*{**READ, "seqs": 0, "ko": None}.values()) == 0
    assert L.kt_hip_dec_kv_read_paged(*{**READ, "max_pos": 0, "ko": None}.values()) == 0
    assert L.kt_hip_dec_argmax_rows(*{**ARGMAX, "rows": 0, "logits": None}.values()) == 0


def test_workspaces_of_refused_shapes_are_zero():
    from tritify_amd import backend as B

    L = _lib()
    assert L.kt_hip_dec_attention_paged_workspace(1, 1, 4, 16, 4, 2, 64) > 0
    for bad in ((-1, 1, 4, 16, 4, 2, 64), (1, 1, 0, 16, 4, 2, 64), (1, 1, 4, 17, 4, 2, 64), (1, 1, 4, 16, 4, 3, 64), (1, 1, 4, 16, 4, 2, 48)):
        assert L.kt_hip_dec_attention_paged_workspace(*bad) == 0
    assert L.kt_hip_dec_argmax_rows_workspace(1, 0) == 0
    with pytest.raises(ValueError):
        B.dec_argmax_rows_workspace(70000, 5)


def test_first_maximum_of_ties():
    x = np.zeros((3, 9), dtype=np.int32)
    x[1, [3, 5]] = 4
    x[2] = -(2 ** 31)
    assert O.argmax_rows(x, 9).tolist() == [0, 3, 0] and O.argmax_rows(x, 3).tolist() == [0, 0, 0]
    assert exp_table(64)[0] == 32768


def _pass(**change):
    """A decoder of 8 rows and 3 sequences without a model or buffers, and the arguments of a pass of 5 rows: what is not refused
    fails on the missing model."""
    import torch
    from types import SimpleNamespace

    from tritify_amd.paged import PagedDecoder

    d = PagedDecoder.__new__(PagedDecoder)
    d.torch, d.dev, d.max_rows, d.max_seqs = torch, -1, 8, 3  # torch's number of the CPU
    a = dict(tokens=5, seqs=3, dev=-1, ids=torch.zeros(5, dtype=torch.int32), last=torch.zeros(3, dtype=torch.int64),
             out=torch.zeros(3, dtype=torch.int32))
    a.update({k: v(torch) if callable(v) else v for k, v in change.items()})
    d.forward(a["ids"], SimpleNamespace(dev=a["dev"], tokens=a["tokens"], seqs=a["seqs"]), a["last"], a["out"])


@pytest.mark.parametrize("change", [
    dict(tokens=9, ids=lambda t: t.zeros(9, dtype=t.int32)), dict(tokens=0), dict(tokens=-1), dict(seqs=0), dict(dev=0),
    dict(seqs=4, last=lambda t: t.zeros(4, dtype=t.int64), out=lambda t: t.zeros(4, dtype=t.int32)),
    dict(tokens=2, ids=lambda t: t.zeros(2, dtype=t.int32), last=None),
    dict(ids=lambda t: t.zeros(4, dtype=t.int32)), dict(ids=lambda t: t.zeros(5, dtype=t.int64)),
    dict(ids=lambda t: t.zeros(10, dtype=t.int32)[::2]),
    dict(out=lambda t: t.zeros(2, dtype=t.int32)), dict(out=lambda t: t.zeros(3, dtype=t.int64)),
    dict(last=lambda t: t.zeros(4, dtype=t.int64)), dict(last=lambda t: t.zeros(3)), dict(last=lambda t: t.zeros(3, 1, dtype=t.int64)),
])
def test_passes_past_the_decoders_buffers_are_refused(change):
    with pytest.raises(ValueError, match="forward"):
        _pass(**change)


@pytest.mark.parametrize("change", [{}, dict(ids=lambda t: t.zeros(9, dtype=t.int32)),
                                    dict(ids=lambda t: t.zeros(5, 1, dtype=t.int32)), dict(last=lambda t: t.zeros(3, dtype=t.int32)),
                                    dict(tokens=3, last=None), dict(last=None)])
def test_passes_within_the_decoders_buffers_go_on_to_the_model(change):
    with pytest.raises(AttributeError, match="m"):
        _pass(**change)


class Counting:
    """A PagedDecoder without a model: run notes the rows of its passes and answers with each sequence's length so far."""

    def __new__(cls, max_rows, max_seqs=64):
        import torch
        from types import SimpleNamespace

        from tritify_amd.paged import PagedDecoder

        d = PagedDecoder.__new__(PagedDecoder)
        d.torch, d.device, d.m = torch, torch.device("cpu"), SimpleNamespace(V=1000)
        d.max_rows, d.max_seqs, d.page, d.sinks, d.seq, d.free, d._next = max_rows, max_seqs, 16, 0, {}, [], 0
        d.passes = []

        def run(work, stream=None):
            assert work and sum(len(t) for _, t in work) <= max_rows
            d.passes.append([len(t) for _, t in work])
            for s, t in work:
                d.seq[s]["len"] += len(t)
            return torch.tensor([d.seq[s]["len"] for s, _ in work], dtype=torch.int32)

        d.run, d._torch_stream = run, lambda stream: None
        return d


def test_generates_steps_fit_the_rows_of_a_pass():
    d = Counting(4)
    assert d.generate([[5] * n for n in (3, 1, 2, 1, 1, 6)], 3).tolist() == [[n, n + 1, n + 2] for n in (3, 1, 2, 1, 1, 6)]
    assert d.passes == [[3, 1], [2, 1, 1], [4], [2]] + [[1] * 4, [1] * 2] * 2 and not d.seq


FLOATS = [[1.5], [2.0], np.array([1.0, 7.9]), [1, float("nan")], ["12"], [None], np.array([[1, 2]]), [1, [2]]]


@pytest.mark.parametrize("tokens", FLOATS, ids=repr)
def test_host_tokens_that_are_not_integers_are_refused(tokens):
    from tritify_amd.paged import PagedDecoder

    d = Counting(100)
    s = d.add()
    with pytest.raises(ValueError, match="integers"):
        PagedDecoder.run(d, [(s, tokens)])
    with pytest.raises(ValueError, match="integers"):
        d.generate([[1, 2], tokens], 2)
    with pytest.raises(ValueError, match="vocabulary"):
        d.generate([[1, 2], [3, 1000]], 2)
    assert d.length(s) == 0 and list(d.seq) == [s] and not d.passes


def test_host_tokens_of_any_integer_type():
    import torch

    d = Counting(100)
    for ids in ([3, 999], (3, 999), np.array([3, 999], dtype=np.uint16), torch.tensor([3, 999]), [np.int64(3), torch.tensor(999)]):
        assert d._ids(ids, "") == [3, 999]


def test_generates_bounds():
    d = Counting(4, max_seqs=3)
    for bad in (dict(chunk=0), dict(chunk=-1), dict(max_new=0), dict(prompts=[[1]] * 4), dict(prompts=[[1], []])):
        with pytest.raises(ValueError, match="generate"):
            d.generate(**{**dict(prompts=[[1, 2]], max_new=2), **bad})
    assert d.generate([], 3).shape == (0, 3) and not d.passes and not d.seq
    assert d.generate([[1, 2, 3]], 1, chunk=2).tolist() == [[3]] and d.passes == [[2], [1]]
