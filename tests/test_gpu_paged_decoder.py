"""The paged decoder (tritify_amd.paged.PagedDecoder) against DecoderModel, which runs one sequence from contiguous caches and
is itself checked against the oracle (tests/test_gpu_decoder.py): the same tokens and logits for every sequence, whatever it
shares its passes with. With 4-bit pages, where no contiguous decoder exists, a batch against its sequences alone."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
CFG = dict(d=128, ffn=256, nh=4, nkv=2, hd=64, layers=2, vocab=1000)


def say(*a):
    print(*a, file=sys.stderr, flush=True)


@pytest.fixture(scope="module")
def model(torch_dev):
    from tritify_amd import workloads as W
    from tritify_amd.decoder import DecoderModel

    m = DecoderModel(CFG, 400, 256)
    for l in range(CFG["layers"]):
        m.set_layer(l, *W.decoder_layer_codes(l, CFG, 500))
    m.set_embedding(*W.decoder_embedding_codes(CFG, 500))
    m.set_tables(*W.rope_tables(400, CFG["hd"]), W.exp_table(), W.silu_table())
    return m


def prompts(lens):
    from tritify_amd import workloads as W

    return [W.decoder_prompt(600 + i, n, CFG["vocab"]) for i, n in enumerate(lens)]


@pytest.mark.parametrize("page,chunk", [(16, 256), (64, 50), (16, 7)])
def test_generate_equals_the_contiguous_decoder(model, page, chunk):
    from tritify_amd.paged import PagedDecoder

    ps = prompts([37, 1, 100, 16, 250, 5])
    say(f"case: paged generate, page {page}, passes of {chunk} rows")
    want = np.array([model.generate(p, 12)[0] for p in ps])
    d = PagedDecoder(model, 60 * 16 // page + 10, page, max_rows=256)
    free = len(d.free)
    assert np.array_equal(d.generate(ps, 12, chunk), want)
    assert len(d.free) == free and sorted(d.free) == list(range(free)) and not d.seq


@pytest.mark.parametrize("max_rows", [1, 4, 5, 6])
def test_generate_for_more_prompts_than_a_pass_has_rows(model, max_rows):
    from tritify_amd.paged import PagedDecoder

    ps = prompts([7, 1, 20, 16, 3, 5])
    want = np.array([model.generate(p, 4)[0] for p in ps])
    d = PagedDecoder(model, 40, max_rows=max_rows)
    assert np.array_equal(d.generate(ps, 4), want)
    assert len(d.free) == 40 and not d.seq


@pytest.mark.parametrize("seqs", [17, 64, 130])
def test_many_sequences_in_a_step(model, torch_dev, seqs):
    """Steps of more rows than the norms are fused for and than the lm_head's one-pass product takes: tokens and logits of each
    sequence, prompts of a few kinds, are the contiguous decoder's."""
    from tritify_amd.paged import PagedDecoder

    kinds = prompts([5, 1, 12, 33, 16])
    ref = [model.generate(p, 4) for p in kinds]
    of = [(7 * i) % 5 for i in range(seqs)]
    say(f"case: {seqs} sequences in a step")
    d = PagedDecoder(model, 6 * seqs, max_seqs=seqs, max_rows=33 * seqs)
    ids = [d.add() for _ in of]
    t = d.run([(s, kinds[k]) for s, k in zip(ids, of)])
    for step in range(4):
        got = d.logits[:seqs].cpu().numpy()
        for i, k in enumerate(of):
            assert np.array_equal(got[i], ref[k][1][step]), (step, i)
        assert t.cpu().numpy().tolist() == [ref[k][0][step] for k in of], step
        # host tokens, one tensor of the device a sequence
        t = d.run([(s, [int(t[i])] if step == 1 else t[i:i + 1]) for i, s in enumerate(ids)])
    if seqs == 64:
        d = PagedDecoder(model, 6 * seqs, max_seqs=seqs, max_rows=100)
        want = np.array([ref[k][0] for k in of])
        assert np.array_equal(d.generate([kinds[k] for k in of], 4), want)


def test_sequences_come_and_go(model, torch_dev):
    """Sequences that join and leave between passes, prompts beside single tokens: logits of every pass as the contiguous
    decoder records them."""
    from tritify_amd.paged import PagedDecoder

    ps = prompts([20, 64, 3, 90])
    ref = [model.generate(p, 10) for p in ps]
    d = PagedDecoder(model, 40, max_rows=256)
    made = {}

    def go(work):
        t = d.run([(made[i]["id"], x) for i, x in work])
        for r, (i, _) in enumerate(work):
            n = made[i]["n"]
            assert np.array_equal(d.logits[r].cpu().numpy(), ref[i][1][n]), (i, n)
            made[i]["n"], made[i]["t"] = n + 1, t[r:r + 1]
            assert int(t[r]) == ref[i][0][n]

    def join(i):
        made[i] = dict(id=d.add(), n=0)
        return (i, ps[i])

    def on(*ii):
        return [(i, made[i]["t"]) for i in ii]

    go([join(0)])
    go([join(1)] + on(0))
    go(on(0, 1))
    go(on(1) + [join(2), join(3)] + on(0))
    d.release(made[1]["id"])
    for _ in range(4):
        go(on(3, 0, 2))
    k, v = d.read(made[3]["id"], 1)
    assert k.shape == (d.length(made[3]["id"]), 2, 64) and d.length(made[3]["id"]) == 94
    model.generate(ps[3], 5)  # leaves the same positions in its own caches
    n = 400 * 2 * 64
    assert torch_dev.equal(k.reshape(-1), model.kc[n:n + k.numel()]) and torch_dev.equal(v.reshape(-1), model.vc[n:n + v.numel()])


@pytest.mark.parametrize("bits,window,sinks", [(4, 0, 0), (8, 40, 4), (4, 33, 0), (4, 20, 18)])
def test_a_batch_equals_its_sequences_alone(model, bits, window, sinks):
    """And in other chunks; with a window, the pages that it leaves behind are free again on the way."""
    from tritify_amd.paged import PagedDecoder

    ps = prompts([37, 1, 120, 16])
    say(f"case: paged generate alone and together, bits={bits} window={window} sinks={sinks}")
    mk = lambda pages: PagedDecoder(model, pages, bits=bits, max_rows=200, window=window, sinks=sinks)  # noqa: E731
    want = np.concatenate([mk(30).generate([p], 20, 11) for p in ps])
    assert np.array_equal(mk(60).generate(ps, 20), want)
    if window:
        d = mk(8)  # 8 pages of 16: the 140 positions of the longest need 9
        assert np.array_equal(d.generate([ps[2]], 20, 11), want[2:3])
        assert sorted(d.free) == list(range(8))


def test_refusals_leave_the_decoder_as_it_was(model):
    from tritify_amd.paged import PagedDecoder

    d = PagedDecoder(model, 6, max_seqs=2, max_rows=100)
    a, b = d.add(), d.add()
    d.run([(a, [1, 2, 3])])
    for bad in ([], [(a, [])], [(a, [1]), (a, [2])], [(99, [1])], [(a, [1000])], [(a, [-1])], [(a, [1] * 101)],
                [(a, [1] * 94), (b, [1] * 6)], [(a, [0] * 98)], [(a, [1]), (b, [1]), (d.add(), [1])]):
        with pytest.raises(ValueError):
            d.run(bad)
        assert d.length(a) == 3 and len(d.free) == 5 and d.length(b) == 0
    with pytest.raises(ValueError):
        d.generate([[1], []], 2)
    for kw in (dict(max_rows=0), dict(max_seqs=0), dict(window=-1), dict(page=20), dict(bits=3)):
        with pytest.raises(ValueError):
            PagedDecoder(model, 6, **kw)


def test_tokens_as_tensors(model, torch_dev):
    """Host lists, host tensors and tensors of the device of either width are the same; ids outside the vocabulary on the device
    count as the nearest inside; matrices and floats are refused."""
    from tritify_amd.paged import PagedDecoder

    torch = torch_dev
    d = PagedDecoder(model, 64, max_rows=100)
    got = []
    for ids in ([0, 7, 999], torch.tensor([0, 7, 999]), torch.tensor([0, 7, 999], dtype=torch.int32),
                torch.tensor([0, 7, 999], device="cuda"), torch.tensor([-5, 7, 2 ** 40], device="cuda"),
                torch.tensor([[0, 1], [7, 1], [999, 1]], device="cuda", dtype=torch.int32)[:, 0]):
        s = d.add()
        d.run([(s, ids)])
        got.append(d.logits[0].cpu().numpy())
        d.release(s)
    assert all(np.array_equal(g, got[0]) for g in got)
    s = d.add()
    for bad in (torch.tensor([[1, 2]], device="cuda"), torch.tensor([1.0], device="cuda"), torch.tensor([1000]), torch.tensor([True])):
        with pytest.raises(ValueError):
            d.run([(s, bad)])
        assert d.length(s) == 0


def test_passes_and_reads_on_another_stream(model, torch_dev):
    from tritify_amd.paged import PagedDecoder

    torch = torch_dev
    ps = prompts([60, 9])
    want = [model.generate(p, 4)[0] for p in ps]
    s = torch.cuda.Stream()
    torch.cuda._sleep(20_000_000)  # the null stream is behind: a decoder made on it is whole all the same
    d = PagedDecoder(model, 64, max_rows=100)
    ids = [d.add() for _ in ps]
    t, got = d.run(list(zip(ids, ps)), stream=s), []
    for _ in range(3):
        got.append(t)
        t = d.run([(ids[0], t[:1]), (ids[1], t[1:])], stream=s)
    k, _ = d.read(ids[0], 0, stream=s)
    s.synchronize()
    assert np.array_equal(torch.stack(got + [t]).cpu().numpy().T, np.array(want))
    model.generate(ps[0], 4)
    assert torch.equal(k[:62].reshape(-1), model.kc[: 62 * 2 * 64])


def test_generate_within_another_stream(model, torch_dev):
    """The passes, made longer here, are on the null stream, torch's current stream is another: the tokens are read after them."""
    from tritify_amd.paged import PagedDecoder

    torch = torch_dev
    ps = prompts([60, 9])
    want = np.array([model.generate(p, 4)[0] for p in ps])
    d = PagedDecoder(model, 64, max_rows=100)
    forward = d.forward

    def late(*a):
        torch.cuda._sleep(20_000_000)
        forward(*a)

    d.forward = late
    with torch.cuda.stream(torch.cuda.Stream()):
        got = d.generate(ps, 4)
    torch.cuda.synchronize()
    assert np.array_equal(got, want)


def test_captured_decode_steps(model, torch_dev):
    """A decode step of a batch as one graph: the tables and lengths move on the device arrays between the replays."""
    from tritify_amd.paged import PagedDecoder

    torch = torch_dev
    ps = prompts([37, 5, 100])
    want = np.array([model.generate(p, 9)[0] for p in ps])
    d = PagedDecoder(model, 40, max_rows=256)
    ids = [d.add() for _ in ps]
    tok = d.run(list(zip(ids, ps)))
    got = [tok.cpu().numpy()]
    d._reserve([(s, d.length(s) + 8) for s in ids])
    b = d.batch(ids, [1, 1, 1])
    x, out = tok.clone(), torch.empty_like(tok)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        d.forward(x, b, None, out, s)  # the shape's workspace; the positions are written again by the first replay
        torch.cuda.synchronize()
        g.capture_begin()
        d.forward(x, b, None, out, s)
        g.capture_end()
    torch.cuda.synchronize()
    for step in range(8):
        g.replay()
        torch.cuda.synchronize()
        got.append(out.cpu().numpy())
        x.copy_(out)
        b.kv_len.add_(1)
        torch.cuda.synchronize()
    assert np.array_equal(np.array(got).T, want)


def test_captured_steps_of_two_shapes_and_passes_between(model, torch_dev):
    """Two captured steps whose batches differ, replayed in turn, with eager passes of other shapes between: the scratch that a
    graph holds stays its own."""
    from tritify_amd.paged import PagedDecoder

    torch = torch_dev
    ps = prompts([37, 5, 100, 250])
    want = [model.generate(p, 9)[0] for p in ps]
    d = PagedDecoder(model, 4096, max_rows=512)
    ids = [d.add() for _ in ps]
    tok = d.run(list(zip(ids, ps)))
    d._reserve([(s, d.length(s) + 8) for s in ids])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    steps = []
    for part in ([0, 1, 2], [3]):
        b = d.batch([ids[i] for i in part], [1] * len(part))
        if part == [3]:  # a table long enough for split passes
            wide = torch.full((1, 1024), -1, dtype=torch.int32, device="cuda")
            wide[:, : b.max_pages] = b.table
            from tritify_amd.paged import PagedBatch
            b = PagedBatch(b.row_start, b.kv_len, wide, 1)
        x = tok[part[0]: part[-1] + 1].clone()
        out, g = torch.empty_like(x), torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            d.forward(x, b, None, out, s)
            torch.cuda.synchronize()
            g.capture_begin()
            d.forward(x, b, None, out, s)
            g.capture_end()
        steps.append((part, b, x, out, g))
    other = d.add()
    torch.cuda.synchronize()
    for n in range(1, 9):
        for part, b, x, out, g in steps:
            g.replay()
            torch.cuda.synchronize()
            assert out.cpu().numpy().tolist() == [want[i][n] for i in part], (n, part)
            x.copy_(out)
            b.kv_len.add_(1)
            junk = [torch.full((1 << 16,), 0x55, dtype=torch.int8, device="cuda") for _ in range(20)]
            d.run([(other, [1] * (3 * n))])
            del junk
            torch.cuda.synchronize()


def test_a_pass_larger_than_the_buffers_is_refused(model, torch_dev):
    """A caller's own batch of more rows, or of more sequences, than the decoder was made for; a pass within them goes on."""
    from tritify_amd.paged import PagedBatch, PagedDecoder

    torch = torch_dev
    d = PagedDecoder(model, 20, max_seqs=2, max_rows=16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for rows in ([17], [1, 1, 1], [1, 16]):
        start = np.concatenate([[0], np.cumsum(rows)])
        b = PagedBatch(i32(*start), i32(*rows), torch.arange(2 * len(rows), dtype=torch.int32, device="cuda").reshape(-1, 2), int(start[-1]))
        with pytest.raises(ValueError):
            d.forward(torch.zeros(b.tokens, dtype=torch.int32, device="cuda"), b, b.row_start[1:].long() - 1, i32(*[0] * b.seqs))
    p, = prompts([16])
    s = d.add()
    assert int(d.run([(s, p)])[0]) == model.generate(p, 1)[0][0]


def test_a_step_padded_with_rows_of_no_sequence(model, torch_dev):
    """Three sequences of one row each in a pass of five and of twenty rows: the rows behind them change nothing."""
    from tritify_amd.paged import PagedBatch, PagedDecoder

    torch = torch_dev
    ps = prompts([9, 30, 4])
    ref = [model.generate(p, 4) for p in ps]
    d = PagedDecoder(model, 20, max_rows=64)
    ids = [d.add() for _ in ps]
    t = d.run(list(zip(ids, ps)))
    for step, rows in ((1, 5), (2, 20), (3, 3)):
        d._reserve([(s, d.length(s) + 1) for s in ids])
        b = d.batch(ids, [1, 1, 1])
        x = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
        x[:3] = t
        t = torch.full((rows,), -3, dtype=torch.int32, device="cuda")
        d.forward(x, PagedBatch(b.row_start, b.kv_len, b.table, rows), None, t)
        assert t.cpu().numpy().tolist() == [r[0][step] for r in ref] + [-3] * (rows - 3)
        assert np.array_equal(d.logits[:3].cpu().numpy(), [r[1][step] for r in ref])
        t = t[:3].clone()
        for s in ids:
            d.seq[s]["len"] += 1
