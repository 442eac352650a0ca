"""PagedDecoder with head norms, a budget of positions, log probabilities and scores, against a decoder of one sequence whose appends,
attention, accumulated weights and evictions are the oracle's (its products, norms of rows and SiLU are the library's, which
tests/test_gpu_decoder.py checks)."""
import numpy as np
import pytest

from oracle import oracle as O
from test_gpu_paged_decoder import CFG, model, prompts, say  # noqa: F401

pytestmark = pytest.mark.gpu
UNIT = 40000


def norms(seed):
    g = np.random.default_rng(seed)
    return [np.round(4096 * (1 + 0.3 * g.normal(size=(CFG["layers"], CFG["hd"])))).astype(np.int16) for _ in range(2)]


class Slow:
    """One sequence, a pass at a time, by the rules of PagedDecoder with `page`, `bits`, and what it is given of norms and budgets."""

    def __init__(self, model, page=16, bits=8, q_norm=None, k_norm=None, budget=0, recent=0, sinks=0, most=0, pages=40):
        import torch

        self.torch, self.m, self.page, self.bits, self.pages = torch, model, page, bits, pages
        self.norms, self.cut = (q_norm, k_norm), (budget, recent, sinks, most)
        per = page * model.hd if bits == 8 else page * (model.hd // 2 + 1)
        self.k, self.v = ([np.zeros((pages, model.nkv * per), dtype=np.uint8) for _ in range(model.L)] for _ in range(2))
        self.w = [np.zeros((pages, model.nkv, page), dtype=np.int64) for _ in range(model.L)]
        self.table, self.len, self.gone, self.cuts = list(range(pages // 2)), 0, 0, 0

    def run(self, tokens):
        """The logits of every row."""
        from tritify_amd import backend as B

        torch, m, lib, P = self.torch, self.m, B.lib(), B._ptr
        T, d, ffn, nh, hd, nq = len(tokens), m.d, m.ffn, m.nh, m.hd, m.nq
        z = lambda *s, dt=torch.int8: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
        r, xn, qkv, o, h = z(T, d, dt=torch.int32), z(T, d), z(T, nq), z(T, nh * hd), z(T, ffn)
        toks = torch.tensor(list(tokens), dtype=torch.int32, device="cuda")
        cos, sin, exp = (t.cpu().numpy() for t in (m.rope_cos, m.rope_sin, m.exp_tab))
        B.check(lib.kt_hip_dec_embed(0, P(toks), T, P(m.emb16), d, P(r), 0), "slow")
        table, kv = np.array([self.table], dtype=np.int32), [self.len - self.gone + T]
        for l in range(m.L):
            B.check(lib.kt_hip_dec_rmsnorm(0, P(r), T, d, P(xn), d, 0), "slow")
            m._gemm("qkv", l, xn, T, nq, d, qkv, B.OUT_I8, 0)
            pg = O.paged(T, [0, T], kv, table, self.k[l], self.v[l], self.page, m.nkv, hd, self.bits)
            q, out = np.zeros((T, nh * hd), dtype=np.int8), np.zeros((T, nh * hd), dtype=np.int8)
            qn, kn = (None if n is None else n[l] for n in self.norms)
            O.paged_norm_append(pg, qkv.cpu().numpy(), nh, cos, sin, q, qn, kn, [self.gone], self.w[l])
            O.paged_attend(pg, q, nh, exp, out)
            O.paged_weigh(pg, q, nh, exp, O.paged_stats(pg, q, nh, exp), self.w[l])
            o.copy_(torch.from_numpy(out))
            m._gemm("o", l, o, T, d, nh * hd, r, B.OUT_I32_ADD, 0)
            lo, nib, mant, shift = m._layer_ptrs("gu", l, 2 * ffn)
            B.check(lib.kt_hip_dec_rmsnorm(0, P(r), T, d, P(xn), d, 0), "slow")
            B.check(lib.kt_hip_w12_swiglu(0, P(xn), lo, nib, T, ffn, d, mant, shift, P(m.silu), m.h_shift, P(h), ffn, 0), "slow")
            m._gemm("dn", l, h, T, d, ffn, r, B.OUT_I32_ADD, 0)
        logits = z(T, m.V, dt=torch.int32)
        B.check(lib.kt_hip_dec_rmsnorm(0, P(r), T, d, P(xn), d, 0), "slow")
        m._gemm("emb", 0, xn, T, m.V, d, logits, B.OUT_I32, 0)
        self.len += T
        budget, recent, sinks, most = self.cut
        if budget and self.len - self.gone > most:
            self.cuts += 1
            to = [p for p in range(self.pages) if p not in self.table][: -(-budget // self.page)]
            for l in range(m.L):
                pg = O.paged(0, [0, 0], [self.len - self.gone], table, self.k[l], self.v[l], self.page, m.nkv, hd, self.bits)
                O.paged_evict(pg, np.array([to]), budget, recent, sinks, self.w[l])
            rest = [p for p in range(self.pages) if p not in to]
            self.table = (to + rest)[: self.pages // 2]
            self.gone = self.len - budget
        return logits.cpu().numpy()

    def generate(self, prompt, n, chunk):
        out = []
        for at in range(0, len(prompt), chunk):
            logits = self.run(prompt[at:at + chunk])[-1]
        for _ in range(n):
            out.append(int(logits.argmax()))
            logits = self.run(out[-1:])[-1]
        return out, logits


@pytest.mark.parametrize("bits", [8, 4])
def test_head_norms(model, bits):  # noqa: F811
    from tritify_amd.paged import PagedDecoder

    q_norm, k_norm = norms(3)
    ps = prompts([37, 1, 60])
    for qn, kn in ((q_norm, k_norm), (None, k_norm)):
        say(f"case: decoder with head norms bits={bits} q={qn is not None}")
        want = [Slow(model, bits=bits, q_norm=qn, k_norm=kn).generate(p, 5, 256)[0] for p in ps]
        d = PagedDecoder(model, 60, bits=bits, q_norm=qn, k_norm=kn)
        assert d.generate(ps, 5).tolist() == want


@pytest.mark.parametrize("page,bits,budget,recent,sinks,most,chunk", [(16, 8, 40, 10, 2, 50, 256), (16, 8, 32, None, 0, None, 20), (64, 4, 48, 0, 0, 48, 30),
                                                                       (16, 4, 17, 17, 0, 30, 9)])
def test_budget(model, page, bits, budget, recent, sinks, most, chunk):  # noqa: F811
    """Sequences of different lengths cut at different passes, in one batch and by the oracle alone; chunked prompts cut as they come."""
    from tritify_amd.paged import PagedDecoder

    say(f"case: decoder with a budget page={page} bits={bits} {budget}/{recent}/{sinks} most={most} chunk={chunk}")
    ps = prompts([90, 5, 33, 120])
    kw = dict(q_norm=norms(5)[0], k_norm=norms(5)[1]) if bits == 8 else {}
    d = PagedDecoder(model, 8 * (budget // page + 1) + 40, page, bits, budget=budget, recent=recent, sinks=sinks, most=most, **kw)
    free, spare = len(d.free), len(d.spare)
    assert spare == -(-budget // page)
    slow = [Slow(model, page, bits, budget=budget, recent=d.recent, sinks=sinks, most=d.most, **kw) for _ in ps]
    want = [s.generate(p, 25, chunk) for s, p in zip(slow, ps)]
    assert sum(s.cuts for s in slow) > 4
    ids = [d.add() for _ in ps]
    last = [None] * len(ps)
    for i, (s, p) in enumerate(zip(ids, ps)):  # each prompt in its own passes, the last chunks of others beside none
        for at in range(0, len(p), chunk):
            last[i] = int(d.run([(s, p[at:at + chunk])])[0])
    got = [[t] for t in last]
    for _ in range(25):
        t = d.run([(s, [g[-1]]) for s, g in zip(ids, got)]).cpu().tolist()
        for g, x in zip(got, t):
            g.append(x)
    logits = d.logits[: len(ps)].cpu().numpy()
    for i in range(len(ps)):
        assert got[i][:25] == want[i][0], i
        assert np.array_equal(logits[i], want[i][1])
        assert d.length(ids[i]) == len(ps[i]) + 25 and d.held(ids[i]) == slow[i].len - slow[i].gone <= d.most
        for l in range(CFG["layers"]):
            k, v = (t.cpu().numpy() for t in d.read(ids[i], l))
            pg = O.paged(0, [0, 0], [slow[i].len - slow[i].gone], np.array([slow[i].table]), slow[i].k[l], slow[i].v[l], page, 2, 64, bits)
            wk, wv = (np.zeros((1,) + k.shape, dtype=np.int8) for _ in range(2))
            O.paged_read(pg, wk, wv)
            assert np.array_equal(k, wk[0]) and np.array_equal(v, wv[0])
    for s in ids:
        d.release(s)
    assert len(d.free) == free and len(set(d.free + d.spare)) == free + spare


def test_budget_with_one_cut_of_spare_pages(model):  # noqa: F811
    """No page is free but the spare ones: sequences are cut one after the other."""
    from tritify_amd.paged import PagedDecoder

    ps = prompts([64, 64, 64])
    d = PagedDecoder(model, 3 * 4 + 2, budget=32, recent=8, most=40)
    ids = [d.add() for _ in ps]
    d.run([(s, p) for s, p in zip(ids, ps)])
    assert [d.held(s) for s in ids] == [32] * 3 and len(d.free) == 12 - 6 and len(d.spare) == 2
    alone = PagedDecoder(model, 30, budget=32, recent=8, most=40)
    for s, p in zip(ids, ps):
        a = alone.add()
        alone.run([(a, p)])
        for l in range(CFG["layers"]):
            for x, y in zip(d.read(s, l), alone.read(a, l)):
                assert np.array_equal(x.cpu().numpy(), y.cpu().numpy())


def test_budget_never_reached_is_the_decoder(model):  # noqa: F811
    from tritify_amd.paged import PagedDecoder

    ps = prompts([37, 1, 100])
    assert np.array_equal(PagedDecoder(model, 80, budget=400).generate(ps, 9), PagedDecoder(model, 60).generate(ps, 9))


def test_budget_on_another_stream(model):  # noqa: F811
    import torch
    from tritify_amd.paged import PagedDecoder

    p = prompts([90])[0]
    want = Slow(model, budget=40, recent=10, sinks=2, most=50).generate(p, 20, 30)[0]
    d, s = PagedDecoder(model, 30, budget=40, recent=10, sinks=2, most=50), torch.cuda.Stream()
    a = d.add()
    for at in range(0, 90, 30):
        t = d.run([(a, p[at:at + 30])], stream=s)
    got = []
    for _ in range(20):
        s.synchronize()
        got.append(int(t.cpu()[0]))
        t = d.run([(a, t)], stream=s)
    assert got == want


def test_captured_steps_under_a_budget(model):  # noqa: F811
    """A sequence that has been cut, decoded by replays of one captured pass: tokens and accumulated weights as by eager passes."""
    import torch
    from tritify_amd.paged import PagedDecoder

    p, (qn, kn) = prompts([90])[0], norms(5)
    made = [PagedDecoder(model, 30, q_norm=qn, k_norm=kn, budget=40, recent=10, sinks=2, most=50) for _ in range(2)]
    (d, a), (e, _) = [(d, d.add()) for d in made]
    toks = [d.run([(a, p)]) for d in made]
    assert d.held(a) == 40 and d.length(a) == 90
    d._reserve([(a, 98)])
    b = d.batch([a], [1])
    x, out = toks[0].clone(), torch.empty_like(toks[0])
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        before = [kv.w.clone() for kv in d.kv]
        d.forward(x, b, None, out, s)  # the shape's workspace; what it adds to the weights is taken back
        for kv, w in zip(d.kv, before):
            kv.w.copy_(w)
        torch.cuda.synchronize()
        g.capture_begin()
        d.forward(x, b, None, out, s)
        g.capture_end()
    torch.cuda.synchronize()
    t = toks[1]
    for step in range(8):
        say(f"case: replay {step}")
        g.replay()
        torch.cuda.synchronize()
        t = e.run([(a, t)])
        torch.cuda.synchronize()
        assert torch.equal(out, t)
        for l in range(model.L):
            assert torch.equal(d.kv[l].w, e.kv[l].w) and torch.equal(d.kv[l].k, e.kv[l].k) and torch.equal(d.kv[l].v, e.kv[l].v)
        x.copy_(out)
        b.kv_len.add_(1)
        torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_steps_by_the_documented_calls(model, bits):  # noqa: F811
    """Scratch reserved, a step captured and replayed, nothing taken back by hand: tokens, caches and accumulated weights as by eager
    passes, and after the cuts that follow the same positions are held."""
    import torch
    from tritify_amd.paged import PagedDecoder

    p = prompts([90])[0]
    made = [PagedDecoder(model, 30, bits=bits, budget=40, recent=10, sinks=2, most=50) for _ in range(2)]
    (d, a), (e, _) = [(d, d.add()) for d in made]
    toks = [d.run([(a, p)]) for d in made]
    d._reserve([(a, 98)])
    b = d.batch([a], [1])
    x, out = toks[0].clone(), torch.empty_like(toks[0])
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        d.reserve_scratch(b)
        held = len(d._ws)
        torch.cuda.synchronize()
        g.capture_begin()
        d.forward(x, b, None, out, s)
        g.capture_end()
    torch.cuda.synchronize()
    assert len(d._ws) == held
    t = toks[1]
    for step in range(8):
        say(f"case: replay {step} bits={bits}")
        g.replay()
        torch.cuda.synchronize()
        t = e.run([(a, t)])
        torch.cuda.synchronize()
        assert torch.equal(out, t)
        for l in range(model.L):
            assert torch.equal(d.kv[l].w, e.kv[l].w) and torch.equal(d.kv[l].k, e.kv[l].k) and torch.equal(d.kv[l].v, e.kv[l].v)
        x.copy_(out)
        b.kv_len.add_(1)
        torch.cuda.synchronize()
    d.seq[a]["len"] += 8  # the replays' tokens; two more passes cut both sequences
    for _ in range(3):
        x, t = d.run([(a, x)]), e.run([(a, t)])
        assert torch.equal(x, t) and d.held(a) == e.held(a)
    assert d.length(a) == e.length(a) == 101 and d.held(a) == 40
    for l in range(model.L):
        for u, v in zip(d.read(a, l), e.read(a, l)):
            assert torch.equal(u, v)


def test_a_batch_without_shifts_under_a_budget(model):  # noqa: F811
    import torch
    from tritify_amd.paged import PagedBatch, PagedDecoder

    d = PagedDecoder(model, 30, budget=40)
    a = d.add()
    t = d.run([(a, prompts([20])[0])])
    d._reserve([(a, 21)])
    b = d.batch([a], [1])
    with pytest.raises(ValueError, match="shifts"):
        d.forward(t, PagedBatch(b.row_start, b.kv_len, b.table, 1), None, torch.empty_like(t))


@pytest.mark.parametrize("k", [0, 5])
def test_logprobs_of_a_pass(model, k):  # noqa: F811
    import torch
    from tritify_amd import backend as B
    from tritify_amd.paged import PagedDecoder

    ps = prompts([9, 30, 2])
    d = PagedDecoder(model, 30)
    t = d.run([(d.add(), p) for p in ps])
    logits = d.logits[:3].cpu().numpy()
    for tok in (t, torch.tensor([5, 999, 1000], dtype=torch.int32, device="cuda")):
        got = d.logprobs(tok, UNIT, k)
        want = O.logprobs_rows(logits, 1000, tok.cpu().numpy(), *B.logit_scale(UNIT), k)
        assert (got[2] is None) == (k == 0)
        for g, w in zip(got, want):
            assert g is None or np.array_equal(g.cpu().numpy(), w)
    if k:
        assert np.array_equal(d.logprobs(t, UNIT, k)[2][:, 0].cpu().numpy(), t.cpu().numpy())  # the greedy choice is the likeliest
    for bad in (t.long(), t.cpu(), torch.zeros(65, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError, match="logprobs"):
            d.logprobs(bad, UNIT)


@pytest.mark.parametrize("k,max_seqs,kw", [(0, 64, {}), (3, 4, {}), (2, 7, dict(bits=4)), (1, 64, dict(budget=24, recent=8, most=30))])
def test_score(model, k, max_seqs, kw):  # noqa: F811
    """Each token's log probability given those before it, whatever the texts share their passes with; then a second chunk."""
    from tritify_amd import backend as B
    from tritify_amd.paged import PagedDecoder

    say(f"case: score k={k} max_seqs={max_seqs} {kw}")
    ps = prompts([20, 1, 33])
    d = PagedDecoder(model, 60, max_seqs=max_seqs, **kw)
    slow = [Slow(model, bits=kw.get("bits", 8), budget=kw.get("budget", 0), recent=d.recent, sinks=0, most=d.most) for _ in ps]
    ids = [d.add() for _ in ps]
    for more in range(2):
        got = d.score(list(zip(ids, ps)), UNIT, k)
        for s, p, g in zip(slow, ps, got):
            logits = s.run(p)
            want = O.logprobs_rows(logits, 1000, list(p[1:]) + [-1], *B.logit_scale(UNIT), k)
            for x, w in zip(g, want):
                assert (x is None and k == 0) or np.array_equal(x.cpu().numpy(), w)
            assert int(g[0][-1]) == -(2 ** 31)
        ps = [p[::-1].copy() for p in ps]
    assert [d.length(s) for s in ids] == [2 * len(p) for p in ps]


def test_refusals(model):  # noqa: F811
    from tritify_amd.paged import PagedDecoder

    for kw in (dict(budget=-1), dict(budget=32, window=64), dict(budget=32, sinks=20, recent=13), dict(budget=32, most=31),
               dict(budget=16 * 41), dict(budget=32, recent=-1), dict(q_norm=np.zeros((2, 64), dtype=np.int32)),
               dict(k_norm=np.zeros((3, 64), dtype=np.int16)), dict(q_norm=np.zeros((2, 32), dtype=np.int16))):
        with pytest.raises(ValueError, match="PagedDecoder"):
            PagedDecoder(model, 40, **kw)
    d = PagedDecoder(model, 40, max_rows=16)
    s = d.add()
    for bad in ([], [(s, [])], [(s, [1] * 17)], [(s, [1]), (s, [2])], [(s + 1, [1])], [(s, [1000])]):
        with pytest.raises(ValueError, match="run"):
            d.score(bad, UNIT)
    for unit in (0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="unit"):
            d.score([(s, [1, 2])], unit)
