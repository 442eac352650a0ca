"""The rules of the append with head norms, the accumulated attention weights, the eviction and the log probabilities on the CPU: the
oracle's restatement against closed forms, against real numbers with bounds, and the arguments that the C ABI refuses before any device
work."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

from oracle import oracle as O
from paged_cases import Case, rope_tables
from test_paged import APPEND, ATTEND, BIG, GEOMETRY, HEADS, _lib, unpacked


def half_away(x):
    """round(x) half away from zero of Fractions."""
    q = math.floor(abs(x) + Fraction(1, 2))
    return q if x >= 0 else -q


@pytest.mark.parametrize("hd", [64, 128])
def test_norm_is_the_formula(hd):
    c = Case(1, [(3, 20), (2, 2)], 4, 2, hd, 16, 8)
    cos, sin = rope_tables(60, hd)
    qn, kn = (c.g.integers(-9000, 9000, size=hd).astype(np.int16) for _ in range(2))
    c.qkv[1, :hd] = 0
    shift = np.array([31, 5], dtype=np.int32)
    k, v, q = c.k.copy(), c.v.copy(), np.zeros((c.tokens, c.width), dtype=np.int8)
    w = c.g.integers(1, 99, size=(c.pages, 2, 16))
    w1 = w.copy()
    O.paged_norm_append(c.oracle(k, v), c.qkv, 4, cos, sin, q, qn, kn, shift, w1)
    kc, vc = unpacked(c, k, False)[0], unpacked(c, v, True)[0]
    written = np.zeros(w.shape, dtype=bool)
    for b, (n, L) in enumerate(c.lens):
        for i in range(n):
            t, p = c.row_start[b] + i, L - n + i
            x = c.qkv[t].astype(int).reshape(-1, hd)
            page = c.table[b, p // 16]
            for h in range(6):
                norm = (qn if h < 4 else kn).astype(int)
                R = math.isqrt(int((x[h] ** 2).sum()) * 65536 // hd)
                y = [max(-16383, min(16383, half_away(Fraction(128 * int(a) * int(m), R)))) if R else 0 for a, m in zip(x[h], norm)]
                C, S = cos[p + shift[b]].astype(int), sin[p + shift[b]].astype(int)
                out = [0] * hd
                for e in range(hd // 2):
                    a, z = y[e], y[e + hd // 2]
                    out[e] = max(-127, min(127, half_away(Fraction(int(a * C[e] - z * S[e]), 1 << 20))))
                    out[e + hd // 2] = max(-127, min(127, half_away(Fraction(int(z * C[e] + a * S[e]), 1 << 20))))
                got = q[t, h * hd:(h + 1) * hd] if h < 4 else kc[page, h - 4, p % 16]
                assert got.tolist() == out, (b, i, h)
            assert np.array_equal(vc[page, :, p % 16], x[6:])
            written[page, :, p % 16] = True
    assert (w1[written] == 0).all() and np.array_equal(w1[~written], w[~written])


def test_norm_approximates_real_numbers():
    """Against the real formula: R is short of the root of the mean square by less than 1 (of 2^8 rms), n rounds to half of 1/2048, a
    table entry to half of 2^-14, and the code to half of 1/32 of a unit. Where nothing is clamped: |n| below 2^14, a code below 127."""
    hd = 64
    c = Case(2, [(40, 40)], 2, 1, hd, 16, 8)
    cos, sin = rope_tables(40, hd)
    w = np.round(4096 * (1 + 0.2 * c.g.normal(size=hd))).astype(np.int16)
    q = np.zeros((40, c.width), dtype=np.int8)
    O.paged_norm_append(c.oracle(c.k.copy(), c.v.copy()), c.qkv, 2, cos, sin, q, w, None)
    a = np.arange(40)[:, None] * 1.0e6 ** (-2.0 * np.arange(hd // 2) / hd)
    x = c.qkv[:, : 2 * hd].reshape(40, 2, hd).astype(float)
    rms = np.sqrt((x ** 2).mean(axis=2, keepdims=True))
    y = x / rms * w / 4096
    lo, hi = y[..., :32], y[..., 32:]
    C, S = np.cos(a)[:, None], np.sin(a)[:, None]
    want = np.concatenate([lo * C - hi * S, hi * C + lo * S], axis=2) * 32
    size = np.tile(np.abs(lo) + np.abs(hi), (1, 1, 2)) * 32
    # 1 / (256 rms - 1) of the size for R; sqrt(2) * 32 / 4096 for the two n; 2^-15 of the size for the tables; 1 / 2 for the code
    bound = size * (1 / (256 * rms - 1) + 2.0 ** -15) * (1 + 2.0 ** -10) + math.sqrt(2) * 32 / 4096 + 0.5 + 1e-9
    inside = (np.abs(want) < 126) & (np.tile(np.maximum(np.abs(lo), np.abs(hi)), (1, 1, 2)) < 7.9)
    assert inside.mean() > 0.9
    assert (np.abs(q[:, : 2 * hd].reshape(40, 2, hd) - want) <= bound)[inside].all()


@pytest.mark.parametrize("bits", [8, 4])
def test_without_norms_it_is_the_append(bits):
    c = Case(3, [(5, 40), (16, 16), (1, 9)], 4, 2, 64, 16, bits, behind=1)
    cos, sin = rope_tables(60, 64)
    q, k, v = c.append(cos, sin)
    q1, k1, v1 = np.full_like(q, 77), c.k.copy(), c.v.copy()
    O.paged_norm_append(c.oracle(k1, v1), c.qkv, 4, cos, sin, q1)
    assert np.array_equal(q, q1) and np.array_equal(k, k1) and np.array_equal(v, v1)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 128)])
def test_weights_are_the_formula(bits, hd, window, sinks):
    c = Case(6, [(3, 90), (1, 40)], 4, 2, hd, 32, bits)
    c.table[0, 1] = -1
    stats = O.paged_stats(c.oracle(), c.q, 4, c.exp, window, sinks)
    w = c.g.integers(0, 1 << 40, size=(c.pages, 2, 32))
    got = w.copy()
    O.paged_weigh(c.oracle(), c.q, 4, c.exp, stats, got, window, sinks)
    kc, km = unpacked(c, c.k, False)
    for b, (n, L) in enumerate(c.lens):
        for i in range(n):
            p, t = L - n + i, c.row_start[b] + i
            j = np.arange(p + 1)
            page = c.table[b, j // 32]
            see = (page >= 0) & ((window == 0) | (j > p - window) | (j < sinks))
            j, page = j[see], page[see]
            for h in range(4):
                s = kc[page, h // 2, j % 32] @ np.maximum(c.q[t, h * hd:(h + 1) * hd].astype(np.int64), -127)
                if bits == 4:
                    s = (km[page, h // 2, j % 32] * s + 4) >> 3
                ix = (s.max() - s + 64) >> 7
                e = np.where(ix < 1024, c.exp[np.minimum(ix, 1023)].astype(np.int64), 0)
                R = min((1 << 40) // int(e.sum()), 2 ** 32 - 1)
                assert stats[t, h].tolist() == [s.max(), R - (1 << 32) if R >= 1 << 31 else R]
                w[page, h // 2, j % 32] += e * R
                # a head's whole weight is 2^40, short by less than the sum of its weights
                assert 0 <= (1 << 40) - int((e * R).sum()) < int(e.sum())
    assert np.array_equal(w, got)
    O.paged_weigh(c.oracle(), c.q, 4, c.exp, stats, got, window, sinks, fresh=True)
    zero = np.zeros_like(w)
    O.paged_weigh(c.oracle(), c.q, 4, c.exp, stats, zero, window, sinks)
    live = np.zeros(w.shape, dtype=bool)
    for b, (_, L) in enumerate(c.lens):
        j = np.arange(L)[c.table[b, np.arange(L) // 32] >= 0]
        live[c.table[b, j // 32], :, j % 32] = True
    assert np.array_equal(got, np.where(live, zero, w))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("budget,recent,sinks", [(20, 5, 3), (64, 0, 0), (50, 30, 20)])
def test_eviction_is_a_sort(bits, budget, recent, sinks):
    lens = [100, 20, 19, 21, 0, 64, 65]
    need = -(-budget // 16)
    c = Case(7, [(0, L) for L in lens], 2, 2, 64, 16, bits, spare=7 * need)
    to = np.setdiff1d(np.arange(c.pages), c.table)[: 7 * need].reshape(7, need)
    w = c.g.integers(0, 12, size=(c.pages, 2, 16))  # many ties
    k, v, w1 = c.k.copy(), c.v.copy(), w.copy()
    kept = O.paged_evict(c.oracle(k, v), to, budget, recent, sinks, w1)
    now, was = [unpacked(c, p, x) for p, x in ((k, False), (v, True))], [unpacked(c, p, x) for p, x in ((c.k, False), (c.v, True))]
    moved = np.zeros(w.shape, dtype=bool)
    for b, L in enumerate(lens):
        for g in range(2):
            at = lambda j: (c.table[b, j // 16], g, j % 16)  # noqa: E731
            stay = list(range(L))
            if L > budget:
                between = sorted(range(sinks, L - recent), key=lambda j: (-w[at(j)], j))[: budget - sinks - recent]
                stay = list(range(sinks)) + sorted(between) + list(range(L - recent, L))
            assert kept[b, g].tolist() == stay + [-1] * (budget - len(stay))
            for i, j in enumerate(stay):
                there = (to[b, i // 16], g, i % 16)
                moved[there] = True
                for (nc, nm), (oc, om) in zip(now, was):
                    assert np.array_equal(nc[there], oc[at(j)]) and nm[there] == om[at(j)]
                assert w1[there] == w[at(j)]
    assert np.array_equal(w1[~moved], w[~moved])
    for (nc, nm), (oc, om) in zip(now, was):
        assert np.array_equal(nc[~moved], oc[~moved]) and np.array_equal(nm[~moved], om[~moved])


# -- log probabilities -----------------------------------------------------------------------------------------------


def real_logprobs(x, unit):
    z = x.astype(np.longdouble) / unit
    z = z - z.max(axis=1, keepdims=True)
    return z - np.log(np.exp(z).sum(axis=1, keepdims=True))


@pytest.mark.parametrize("peak", [0, 12, 20.5, 22, 26, 33])
@pytest.mark.parametrize("n,sigma", [(1, 1), (7, 2), (1000, 0.01), (3000, 3), (5000, 8), (151936, 3), (151936, 0.2)])
def test_logprobs_approximate_real_numbers(n, sigma, peak):
    """Bounds in 2^-16 of a natural unit, by the rules' own roundings: a difference of logits rounds to half of 2^-16 of a power of two
    (ln 2 / 2), an exponential's tables to 2^-31 each and its cuts to 1 of 2^30 a logit, and (mant, shift) to 2^-31 of the difference, at
    most 120 units here. A sum of positive terms is off by no more, relatively, than its terms: by ln 2 / 2 steps for the differences,
    and by 1024 / 2^30 and 2^-22 and 2^-30 a block for the cuts, 2^-19.5 in all. log2's interpolation is off by 2^-20 / 8 log2(e) at most. The
    result rounds to half. A log probability takes a difference and a sum: at most ln 2 + 0.5 + 0.1. The entropy takes a mean of t, whose
    weights are off by as much, relatively, as the terms of the sum: ln 2 / 2 steps of 2^-16 times the spread of the log probabilities,
    below 2^-16 * 20 of a step, beside its own ln 2 / 2 and the division's 1 and 2^-7."""
    g = np.random.default_rng(n)
    unit = 87381
    from tritify_amd.backend import logit_scale

    x = np.round(g.normal(0, sigma * unit, size=(3, n))).astype(np.int32)
    x[1:, n // 3] += int(peak * unit)  # one logit far above the others
    t = g.integers(0, n, size=3)
    lp, ent, top, top_lp = O.logprobs_rows(x, n, t, *logit_scale(unit), 5)
    want = real_logprobs(x, unit)
    assert (np.abs(lp - 65536 * want[np.arange(3), t]) <= math.log(2) + 0.6).all()
    assert (np.abs(ent + 65536 * (np.exp(want) * want).sum(axis=1)) <= math.log(2) + 0.5 + 1.1).all()
    for r in range(3):
        order = np.argsort(-x[r].astype(np.int64), kind="stable")[:5]
        assert top[r, : len(order)].tolist() == order.tolist() and (top[r, len(order):] == -1).all()
        assert (np.abs(top_lp[r, : len(order)] - 65536 * want[r, order]) <= math.log(2) + 0.6).all()
        assert (top_lp[r, len(order):] == -(2 ** 31)).all()


def test_logprobs_closed_forms():
    from tritify_amd.backend import logit_scale

    s = logit_scale(1000)
    x = np.full((1, 4096), 5, dtype=np.int32)
    lp, ent, top, top_lp = O.logprobs_rows(x, 4096, [9], *s, 3)
    assert lp[0] == -round(65536 * 12 * math.log(2)) and ent[0] == -lp[0] and top[0].tolist() == [0, 1, 2] and (top_lp == lp).all()
    x[0, 7] = 2 ** 31 - 1
    x[0, 8] = -(2 ** 31)
    lp, ent, top, _ = O.logprobs_rows(x, 4096, [7], *s, 2)
    assert lp[0] == 0 and ent[0] == 0 and top[0].tolist() == [7, 0]
    lp = O.logprobs_rows(x, 4096, [8], *s)[0]  # 2^32 - 1 thousandths of a unit: past 2^31 - 1 in 2^-16 of a power of two
    assert lp[0] == -((2 ** 31 - 1) * 256 * 5814540 + 2 ** 30 >> 31)
    assert O.logprobs_rows(x, 4096, [4096], *s)[0][0] == -(2 ** 31) == O.logprobs_rows(x, 4096, [-1], *s)[0][0]


def test_logit_scale():
    from tritify_amd.backend import logit_scale

    for unit in (1e-3, 0.5, 1, 8, 64, 1000, 87381, 94548.4, 1 << 20, 2.0 ** 31, 3e8):
        mant, shift = logit_scale(unit)
        assert 1 << 30 <= mant < 1 << 31 and 0 <= shift <= 62
        assert abs(mant / 2.0 ** shift * unit / (65536 * math.log2(math.e)) - 1) < 2.0 ** -31
    for bad in (0, -1, math.inf, math.nan, 1e30, 1e-9):
        with pytest.raises(ValueError):
            logit_scale(bad)


@pytest.mark.parametrize("unit", [5e-324, 1e-300, 1e300, 1.7e308])
def test_logit_scale_of_units_past_all_powers(unit):
    from tritify_amd.backend import logit_scale

    with pytest.raises(ValueError, match="logit_scale"):
        logit_scale(unit)


# -- the decoder's own checks, without a model or buffers -------------------------------------------------------------


@pytest.mark.parametrize("nh,nkv,positions", [(64, 1, 131072), (16, 1, 524288), (128, 4, 300000)])
def test_a_budget_whose_sums_may_not_hold_is_refused(nh, nkv, positions):
    from types import SimpleNamespace

    from tritify_amd.paged import PagedDecoder

    m = SimpleNamespace(nh=nh, nkv=nkv, rope_cos=np.zeros((positions, 0)))
    with pytest.raises(ValueError, match="2.23 heads"):
        PagedDecoder(m, 100, budget=64)


def test_a_pass_under_a_budget_needs_the_shifts():
    import torch
    from types import SimpleNamespace

    from tritify_amd.paged import PagedDecoder

    d = PagedDecoder.__new__(PagedDecoder)
    d.torch, d.dev, d.max_rows, d.max_seqs, d.budget, d.m = torch, -1, 8, 3, 32, SimpleNamespace(V=10)  # -1: torch's number of the CPU
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="shifts"):
        d.forward(i32, SimpleNamespace(dev=-1, tokens=2, seqs=2, shift=None), None, i32)


def test_cuts_of_many_sequences_at_a_time_are_within_what_evict_takes():
    import torch

    from tritify_amd.paged import PagedDecoder

    page, budget, n = 256, 524288 - 16, 520
    need, calls = -(-budget // page), []

    class Evict:
        def evict(self, b, to, budget, kept, recent, sinks, stream):
            calls.append(to.shape[0])
            assert to.shape == (len(b), need) and to.shape[0] * (budget // 16) < 1 << 24 and len(set(to.flatten().tolist())) == to.numel()

    class M:
        nkv = 1

    d = PagedDecoder.__new__(PagedDecoder)
    d.torch, d.device, d.m, d.page, d.budget, d.recent, d.sinks, d.most = torch, "cpu", M, page, budget, 0, 0, budget
    d.kv, d.batch = [Evict()], lambda seqs, rows: seqs
    own = 2048
    d.seq = {s: dict(len=budget + 1, cut=0, pages=list(range(s * own, (s + 1) * own)), gone=0) for s in range(n)}
    d.free, d.spare = list(range(n * own, 2 * n * own)), list(range(2 * n * own, 2 * n * own + need))
    d._cut(list(d.seq), None)
    assert sum(calls) == n and max(calls) == 512 and all(d.held(s) == budget for s in d.seq)
    pages = d.free + d.spare + [p for e in d.seq.values() for p in e["pages"]]
    assert len(pages) == len(set(pages)) == 2 * n * own + need


@pytest.mark.parametrize("fails", [0, 1, 2])
def test_a_cut_that_fails_loses_no_pages(fails):
    """Where a layer's eviction cannot run (no memory for its scratch, say), the sequences are as they were and the next pass cuts them."""
    import torch

    from tritify_amd.paged import PagedDecoder

    state = dict(calls=0, broken=True, to=[])

    class Evict:
        def evict(self, b, to, budget, kept, recent, sinks, stream):
            state["calls"] += 1
            if state["broken"] and state["calls"] > fails:
                raise RuntimeError("no memory")
            state["to"].append(to.flatten().tolist())

    class M:
        nkv = 2

    d = PagedDecoder.__new__(PagedDecoder)
    d.torch, d.device, d.m, d.page, d.budget, d.recent, d.sinks, d.most = torch, "cpu", M, 16, 40, 8, 2, 50
    d.kv, d.batch = [Evict()] * 3, lambda seqs, rows: seqs
    d.seq = {s: dict(len=60 + s, cut=0, pages=list(range(4 * s, 4 * s + 4)), gone=0) for s in range(5)}
    d.free, d.spare = list(range(40, 20, -1)), [20, 41, 42]
    before = [dict(e, pages=list(e["pages"])) for e in d.seq.values()], list(d.free), list(d.spare)
    with pytest.raises(RuntimeError, match="no memory"):
        d._cut(list(d.seq), None)
    assert (list(d.seq.values()), d.free, d.spare) == before
    state.update(broken=False, to=[])
    d._cut(list(d.seq), None)
    assert all(d.held(s) == 40 and len(d.seq[s]["pages"]) == 3 for s in d.seq) and len(state["to"]) == 3
    pages = d.free + d.spare + [p for e in d.seq.values() for p in e["pages"]]
    assert sorted(pages) == list(range(43)) and len(d.spare) == 3
    assert state["to"][0] == [20, 41, 42] + list(range(21, 33))  # the spare pages, then the free ones from the list's end


def test_scratch_is_reserved_without_a_pass():
    """No operator runs, so no weight is added; what the pass then asks for is there, and smaller shapes take it too."""
    import torch
    from types import SimpleNamespace

    from tritify_amd.paged import PagedDecoder

    class Scratch:  # no other operator to call
        def workspace_bytes(self, b, nh):
            return b.tokens * 1000 + 7

    d = PagedDecoder.__new__(PagedDecoder)
    d.torch, d.dev, d.device, d.max_rows, d.max_seqs, d.m = torch, -1, "cpu", 4096, 64, SimpleNamespace(V=200000, nh=14)
    d.kv, d._ws = [Scratch()], []
    batch = lambda tokens, seqs: SimpleNamespace(dev=-1, tokens=tokens, seqs=seqs)  # noqa: E731
    assert d.reserve_scratch(batch(2048, 64)) is None
    held = d._ws[-1].data_ptr()
    for tokens, seqs in ((2048, 64), (64, 64), (1, 1)):
        d.reserve_scratch(batch(tokens, seqs))
        ws, top = d._workspaces(batch(tokens, seqs))
        assert ws.data_ptr() == held and ws.numel() >= tokens * 1000 + 7 and top.numel() > 0 and len(d._ws) == 1
    d.reserve_scratch(batch(4096, 64))
    assert len(d._ws) == 2 and d._ws[0].data_ptr() == held  # a captured pass may hold it
    for bad in (batch(0, 1), batch(4097, 1), batch(1, 0), batch(65, 65), SimpleNamespace(dev=0, tokens=1, seqs=1)):
        with pytest.raises(ValueError, match="reserve_scratch"):
            d.reserve_scratch(bad)


# -- refusals --------------------------------------------------------------------------------------------------------

P = 1 << 20  # an aligned address that no call here dereferences
NORM = dict(dev=0, qkv=P, tokens=3, qkv_stride=512, row_start=P, kv_len=P, table=P, seqs=2, max_pages=4, nh=4, nkv=2, hd=64, cos=P, sin=P,
            max_pos=64, qn=P, kn=P, shift=P, q=P, q_stride=256, k=P, v=P, w=P, pages=8, page=16, bits=8, stream=None)
STATS = {**{k: v for k, v in ATTEND.items() if k not in ("ws", "ws_bytes", "stream")}, "stats": P, "ws": P, "ws_bytes": 1 << 40, "stream": None}
WEIGH = dict(dev=0, q=P, tokens=3, q_stride=256, row_start=P, kv_len=P, table=P, seqs=2, max_pages=4, nh=4, nkv=2, hd=64, exp=P, window=0,
             sinks=0, stats=P, fresh=0, k=P, w=P, pages=8, page=16, bits=8, stream=None)
EVICT = dict(dev=0, kv_len=P, table=P, seqs=2, max_pages=4, nkv=2, hd=64, to=P, budget=32, recent=3, sinks=2, kept=P, k=P, v=P, w=P, pages=8,
             page=16, bits=8, ws=P, ws_bytes=1 << 40, stream=None)
LOGPROBS = dict(dev=0, logits=P, rows=3, n=1000, stride=1000, token=P, mant=1 << 30, shift=30, lp=P, ent=P, k=5, top=P, top_lp=P, ws=P,
                ws_bytes=1 << 40, stream=None)


def of(args, changes):
    """The changes that name arguments of the call, with a stride that fits many heads."""
    for x in changes:
        x = {k: v for k, v in x.items() if k in args}
        if "nh" in x and x["nh"] > 4:
            x.update({s: 1 << 20 for s in ("qkv_stride", "q_stride", "o_stride") if s in args and s not in x})
        if x:
            yield x


REFUSED = (
    [("kt_hip_dec_norm_rope_kv_paged", NORM, x) for x in [*of(NORM, GEOMETRY + HEADS + BIG)] + [
        dict(qkv_stride=511), dict(qkv_stride=520), dict(q_stride=240), dict(q_stride=264), dict(qkv=P + 4), dict(q=None), dict(cos=P + 4),
        dict(sin=None), dict(max_pos=-1), dict(max_pos=1 << 31), dict(qn=P + 4), dict(kn=P + 2), dict(shift=P + 2), dict(w=P + 4)]]
    + [("kt_hip_dec_attention_paged_stats", STATS, x) for x in [*of(STATS, GEOMETRY + HEADS + BIG)] + [
        dict(q_stride=240), dict(o_stride=128), dict(q=None), dict(o=P + 8), dict(exp=None), dict(window=-1), dict(sinks=-1), dict(ws=None),
        dict(ws_bytes=0), dict(stats=None), dict(stats=P + 4)]]
    + [("kt_hip_dec_weigh_paged", WEIGH, x) for x in [*of(WEIGH, GEOMETRY + HEADS + BIG)] + [
        dict(q_stride=240), dict(q_stride=257), dict(q=None), dict(exp=None), dict(window=-1), dict(sinks=-1), dict(stats=None),
        dict(stats=P + 4), dict(w=None), dict(w=P + 4), dict(seqs=65536)]]
    + [("kt_hip_dec_evict_paged", EVICT, x) for x in [*of(EVICT, GEOMETRY)] + [
        dict(to=None), dict(kept=None), dict(kept=P + 2), dict(w=None), dict(w=P + 4), dict(budget=0), dict(budget=524289), dict(recent=-1),
        dict(sinks=-1), dict(recent=31), dict(sinks=30), dict(recent=1 << 62, sinks=1 << 62), dict(seqs=65536), dict(seqs=60000, budget=8192),
        dict(ws=None), dict(ws=P + 4), dict(ws_bytes=255)]]
    + [("kt_hip_dec_logprobs_rows", LOGPROBS, x) for x in [
        dict(rows=-1), dict(rows=65536), dict(n=0), dict(n=(1 << 20) + 1, stride=1 << 21), dict(stride=999), dict(k=-1), dict(k=33),
        dict(mant=0), dict(mant=-5), dict(mant=1 << 31), dict(shift=-1), dict(shift=63), dict(logits=None), dict(token=None), dict(lp=None),
        dict(top=None), dict(top_lp=None), dict(ws=None), dict(ws=P + 4), dict(ws_bytes=8)]]
)


@pytest.mark.parametrize("name,args,change", REFUSED, ids=[f"{n[11:]}-{'-'.join(f'{k}={v}' for k, v in x.items())}" for n, _, x in REFUSED])
def test_refused_before_any_device_work(name, args, change):
    assert set(change) <= set(args)
    assert getattr(_lib(), name)(*{**args, **change}.values()) == 1  # hipErrorInvalidValue


def test_the_calls_arguments_are_the_headers():
    L = _lib()
    for name, args in (("kt_hip_dec_norm_rope_kv_paged", NORM), ("kt_hip_dec_attention_paged_stats", STATS), ("kt_hip_dec_weigh_paged", WEIGH),
                       ("kt_hip_dec_evict_paged", EVICT), ("kt_hip_dec_logprobs_rows", LOGPROBS), ("kt_hip_dec_rope_kv_paged", APPEND)):
        f = getattr(L, name)
        assert len(f.argtypes) == len(args) and f.restype is ctypes.c_int


def test_empty_calls_do_nothing():
    L = _lib()
    for empty in (dict(tokens=0), dict(seqs=0)):
        assert L.kt_hip_dec_norm_rope_kv_paged(*{**NORM, **empty, "qkv": None, "q": None}.values()) == 0
        assert L.kt_hip_dec_attention_paged_stats(*{**STATS, **empty, "q": None, "o": None, "stats": None}.values()) == 0
        assert L.kt_hip_dec_weigh_paged(*{**WEIGH, **empty, "q": None, "stats": None}.values()) == 0
    assert L.kt_hip_dec_weigh_paged(*{**WEIGH, "pages": 0, "k": None, "w": None, "fresh": 1}.values()) == 0
    assert L.kt_hip_dec_evict_paged(*{**EVICT, "seqs": 0, "kept": None}.values()) == 0
    assert L.kt_hip_dec_logprobs_rows(*{**LOGPROBS, "rows": 0, "logits": None}.values()) == 0
    assert L.kt_hip_dec_logprobs_rows_workspace(0, 5, 0) > 0
    for bad in ((-1, 5, 0), (65536, 5, 0), (1, 0, 0), (1, (1 << 20) + 1, 0), (1, 5, 33), (1, 5, -1)):
        assert L.kt_hip_dec_logprobs_rows_workspace(*bad) == 0
    assert L.kt_hip_dec_evict_paged_workspace(1, 4, 16, 2) > 0 and L.kt_hip_dec_evict_paged_workspace(0, 4, 16, 2) > 0
    for bad in ((-1, 4, 16, 2), (65536, 4, 16, 2), (1, 0, 16, 2), (1, 4, 17, 2), (1, 4, 16, 0), (1, 524288 // 16 + 1, 16, 2)):
        assert L.kt_hip_dec_evict_paged_workspace(*bad) == 0
    from tritify_amd import backend as B

    with pytest.raises(ValueError):
        B.dec_logprobs_rows_workspace(1, 5, 40)


@pytest.mark.parametrize("page", [16, 256])
def test_no_sequences_over_a_wide_table(page):
    """A shape that the eviction takes has scratch of some bytes, whatever the table's width."""
    L, wide = _lib(), 524288 // page
    n = L.kt_hip_dec_evict_paged_workspace(0, wide, page, 2)
    assert 0 < n <= L.kt_hip_dec_evict_paged_workspace(1, wide, page, 2)
    assert L.kt_hip_dec_evict_paged(*{**EVICT, "seqs": 0, "max_pages": wide, "page": page, "ws_bytes": n}.values()) == 0


@pytest.mark.parametrize("tokens", [0, 5])
@pytest.mark.parametrize("page", [16, 256])
def test_no_sequences_attend_over_a_wide_table(page, tokens):
    L, wide = _lib(), 524288 // page
    n = L.kt_hip_dec_attention_paged_workspace(tokens, 0, wide, page, 14, 2, 64)
    assert n > 0
    empty = {**STATS, "tokens": tokens, "seqs": 0, "max_pages": wide, "page": page, "ws_bytes": n}
    assert L.kt_hip_dec_attention_paged_stats(*empty.values()) == 0
