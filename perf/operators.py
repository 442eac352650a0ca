"""Timed cases of the int8 decoder's paged serving operators, beside their plain forms in elementary torch.

Four operators, all with integer results that the rules fix, so every output is compared exactly:

  append   RoPE of a batch's new rows, k and v written to their pages (8 bits)
  cache    the same write and the read back of every sequence as contiguous rows (8 bits, or quantised to 4)
  attend   attention of the new rows over the pages: chunks and single tokens, 8 or 4 bits, windows with sinks
  argmax   the greedy choice of each row of a batch's logits

A batch is ragged: sequence b has rows row_start[b] .. row_start[b + 1] - 1 and kv_len[b] positions, its rows the last of
them; position j is slot j % page of page table[b][j // page]. The rules are those of the contiguous caches (rotate-half
RoPE by int16 tables, e = T[(max - s + 64) >> 7], rounding half away from zero). In 4 bits a row x of one position and
kv head is held as a multiplier m = ceil(8 max|x| / 7) and codes c = clamp(round(8 x / m), +-7), and stands for c m / 8;
its score is (m (q . c) + 4) >> 3.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"


def _case(name, kind, **kw):
    c = dict(name=name, kind=kind)
    if kind == "argmax":
        c.update(kw)
        return c
    c.update(seqs=1, prompts=0, rows=1, past=0, ragged=False, nh=14, nkv=2, hd=64, page=16, bits=8)
    if kind == "attend":
        c.update(window=0, sinks=0)
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of a batch: a new position in each sequence's last page
        _case("append_batch", "append", seqs=64, past=1000, ragged=True),
        # prompts of a few sequences admitted together, behind a shared system prompt
        _case("append_prompts", "append", seqs=4, prompts=4, rows=512, past=77, page=64),
        # one decode step into 4-bit pages and the sequences handed over as contiguous rows
        _case("cache4_batch", "cache", seqs=24, past=200, ragged=True, bits=4),
        # a prompt stored in 4 bits and read back, head_dim 128
        _case("cache4_prompt", "cache", prompts=1, rows=2048, nh=16, nkv=4, hd=128, page=32, bits=4),
        # a single user's decode step: latency
        _case("attend_one", "attend", past=640),
        # the decode step of a served batch with long histories: the cache's bytes are the work
        _case("attend_batch", "attend", seqs=128, past=8191, ragged=True),
        # one very long document on 4-bit pages, a token at a time
        _case("attend_long4", "attend", past=131000, bits=4, page=64),
        # a chunk of a long prompt behind what is cached of it (chunked prefill)
        _case("attend_chunk", "attend", prompts=1, rows=1024, past=7777),
        # whole prompts of odd lengths, nothing cached
        _case("attend_prompts", "attend", seqs=3, prompts=3, rows=1021, page=32),
        # a sliding window with sinks: chunks and single tokens in one batch, head_dim 128
        _case("attend_window", "attend", seqs=12, prompts=2, rows=200, past=6000, ragged=True, nh=16, nkv=4, hd=128,
              window=1024, sinks=4),
        # the choice of a single sequence's next token
        _case("argmax_one", "argmax", n=151936, batch=1),
        # the choice of a served batch's next tokens
        _case("argmax_batch", "argmax", n=151936, batch=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "cache", "cache", "attend", "attend", "attend", "attend", "attend", "argmax"])
    if kind == "argmax":
        return dict(kind=kind, n=_log(rng, 97, 200000), batch=_log(rng, 1, 64))
    nkv = rng.choice([1, 2, 2, 4])
    c = _case("", kind, nkv=nkv, nh=nkv * rng.choice([1, 4, 7, 7, 8, 12]), hd=rng.choice([64, 64, 64, 128]),
              page=rng.choice([16, 16, 32, 64, 128]), bits=8 if kind == "append" else rng.choice([8, 4]),
              ragged=rng.random() < 0.7)
    del c["name"]
    if rng.random() < 0.5:  # single tokens
        c.update(seqs=_log(rng, 1, 64), past=_log(rng, 1, 8000 if kind == "attend" else 1500))
    else:  # chunks, some of them beside single tokens
        c.update(rows=_log(rng, 2, 600), past=rng.choice([0, _log(rng, 1, 3000)]))
        c["seqs"] = rng.randint(1, 4)
        c["prompts"] = rng.randint(1, c["seqs"])
    if kind == "attend" and rng.random() < 0.3:
        c.update(window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 100]))
    while work(c)["flops"] > 3e10 or work(c)["bytes"] > 2e8:  # no more than the largest of the listed ones
        key = "rows" if c["prompts"] and c["rows"] > c["past"] // 8 else "past"
        c[key] //= 2
    return c


# -- inputs ----------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _lengths(case):
    """(new rows, positions with them) of each sequence."""
    out = []
    for i in range(case["seqs"]):
        n = case["rows"] if i < case["prompts"] else 1
        past = case["past"]
        if case["ragged"]:
            past -= (i * 40503 + 17) % (past // 2 + 1)
            n -= (i * 97) % (n // 3 + 1)
        out.append((n, past + n))
    return out


def _rows8(g, *shape):
    """Int8 activations at 32 codes per unit."""
    return torch.randn(*shape, generator=g, device=DEV).mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def _exp_table(hd):
    """round(2^15 exp(-i / w)), w the entries of one unit of logit at head_dim hd (64 at 64)."""
    i = torch.arange(1024, dtype=torch.float64)
    return (32768.0 * torch.exp(-i / (8.0 * math.sqrt(hd)))).round().to(torch.int32).to(DEV)


def _rope_tables(n, hd):
    f = 1.0e6 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * f
    return tuple((16384.0 * t).round().to(torch.int16) for t in (torch.cos(a), torch.sin(a)))


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "argmax":
        x = torch.randn(case["batch"], case["n"], generator=g, device=DEV).mul_(1 << 18).round_().to(torch.int32)
        st = dict(case=case, logits=x, tokens=torch.zeros(case["batch"], dtype=torch.int32, device=DEV))
        if own:
            _handles(st)
        return st
    lens = _lengths(case)
    page, nkv, nh, hd, seqs = (case[k] for k in ("page", "nkv", "nh", "hd", "seqs"))
    need = [-(-L // page) for _, L in lens]
    max_pages, pages = max(need), sum(need) + 3
    row_start = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).to(DEV)
    kv_len = torch.tensor([L for _, L in lens], dtype=torch.int32, device=DEV)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((seqs, max_pages), -1, dtype=torch.int32, device=DEV)
    used = torch.arange(max_pages, device=DEV) < torch.tensor(need, device=DEV)[:, None]
    table[used] = order[: sum(need)]
    tokens = sum(n for n, _ in lens)
    st = dict(case=case, tokens=tokens, max_pages=max_pages, pages=pages, row_start=row_start, kv_len=kv_len, table=table)
    kp, vp = _rows8(g, pages, nkv, page, hd), _rows8(g, pages, nkv, page, hd)
    if case["bits"] == 8:
        kp, vp = kp.reshape(pages, nkv, -1), _blocks(vp).reshape(pages, nkv, -1)
    else:
        (kc, km), (vc, vm) = _quant4(kp), _quant4(vp)
        kp = torch.cat([_pack4(kc).reshape(pages, nkv, -1), km.to(torch.uint8).view(torch.int8)], dim=2)
        vp = torch.cat([_pack4(_blocks(vc)).reshape(pages, nkv, -1), vm.to(torch.uint8).view(torch.int8)], dim=2)
    st.update(k=kp.contiguous(), v=vp.contiguous())
    if case["kind"] == "attend":
        st.update(q=_rows8(g, tokens, nh * hd), exp=_exp_table(hd),
                  o=torch.zeros(tokens, nh * hd, dtype=torch.int8, device=DEV))
    else:
        cap = max(L for _, L in lens)
        cos, sin = _rope_tables(cap, hd)
        st.update(qkv=_rows8(g, tokens, (nh + 2 * nkv) * hd), cos=cos, sin=sin,
                  q=torch.zeros(tokens, nh * hd, dtype=torch.int8, device=DEV))
        if case["kind"] == "cache":
            st.update(ko=torch.zeros(seqs, cap, nkv, hd, dtype=torch.int8, device=DEV),
                      vo=torch.zeros(seqs, cap, nkv, hd, dtype=torch.int8, device=DEV))
    if own:
        _handles(st)
    return st


def _handles(st):
    """The framework's handles of the same buffers, which a program makes once."""
    from tritify_amd import backend as B
    from tritify_amd.paged import PagedBatch, PagedKV

    c = st["case"]
    if c["kind"] == "argmax":
        st["ws"] = torch.empty(B.dec_argmax_rows_workspace(c["batch"], c["n"]), dtype=torch.int8, device=DEV)
        return
    st["batch"] = PagedBatch(st["row_start"], st["kv_len"], st["table"], st["tokens"])
    st["kv"] = PagedKV(st["pages"], c["page"], c["nkv"], c["hd"], bits=c["bits"], k=st["k"], v=st["v"])
    if c["kind"] == "attend":
        st["ws"] = st["kv"].workspace(st["batch"], c["nh"])


# -- one pass --------------------------------------------------------------------------------------------------------


def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    if kind == "argmax":
        n = st["logits"].shape[1]  # the first maximum: the largest (value, -index)
        key = st["logits"].long() * (1 << 32) + torch.arange(n - 1, -1, -1, device=DEV)
        return (n - 1 - (key.amax(dim=1) & 0xFFFFFFFF)).to(torch.int32)
    if kind == "attend":
        return _plain_attend(st)
    q = _plain_append(st)
    if kind == "append":
        return q, st["k"], st["v"]
    return (q,) + _plain_read(st)


def _own(st, kind):
    if kind == "argmax":
        from tritify_amd import backend as B

        B.dec_argmax_rows(st["logits"], st["logits"].shape[0], st["logits"].shape[1], st["tokens"], st["ws"])
        return st["tokens"]
    kv, batch, c = st["kv"], st["batch"], st["case"]
    if kind == "attend":
        kv.attend(st["q"], batch, c["nh"], st["exp"], st["o"], st["ws"], window=c["window"], sinks=c["sinks"])
        return st["o"]
    kv.append(st["qkv"], batch, c["nh"], st["cos"], st["sin"], st["q"])
    if kind == "append":
        return st["q"], st["k"], st["v"]
    kv.read(batch, st["ko"], st["vo"])
    return st["q"], st["ko"], st["vo"]


# -- the plain forms -------------------------------------------------------------------------------------------------


def _div_round(a, b):
    """round(a / b) half away from zero, b > 0."""
    return torch.sign(a) * torch.div(2 * a.abs() + b, 2 * b, rounding_mode="floor")


def _blocks(v):
    """[..., page, hd] -> [..., page / 16, hd, 16]: each dimension's 16 positions side by side."""
    return v.unflatten(-2, (-1, 16)).transpose(-1, -2).contiguous()


def _unblocks(v):
    return v.transpose(-1, -2).flatten(-3, -2)


def _quant4(x):
    """Codes and multipliers of the rows x (last axis)."""
    x = x.to(torch.int32)
    m = torch.div(8 * x.abs().amax(dim=-1) + 6, 7, rounding_mode="floor")
    return _div_round(8 * x, m.clamp(min=1)[..., None]).clamp(-7, 7), m


def _pack4(c):
    """16 codes in 8 bytes: byte 4 h + r holds code 8 h + r in its low half and code 8 h + 4 + r in its high half."""
    c = (c & 15).unflatten(-1, (-1, 2, 2, 4))
    return (c[..., 0, :] | (c[..., 1, :] << 4)).to(torch.uint8).view(torch.int8).flatten(-3)


def _unpack4(b):
    b = b.view(torch.uint8).to(torch.int32).unflatten(-1, (-1, 2, 4))
    c = torch.stack([b & 15, b >> 4], dim=-2).flatten(-4)
    return torch.where(c > 7, c - 16, c)


def _pages(st):
    """Codes [page][kv head][slot][hd] of both pools as int32 or int8, and the rows' multipliers (4 bits)."""
    c = st["case"]
    page, hd, n = c["page"], c["hd"], c["page"] * c["hd"]
    k, v = st["k"], st["v"]
    if c["bits"] == 8:
        return k.unflatten(2, (page, hd)), _unblocks(v.unflatten(2, (page // 16, hd, 16))), None, None
    kc = _unpack4(k[..., : n // 2]).unflatten(2, (page, hd))
    vc = _unblocks(_unpack4(v[..., : n // 2]).unflatten(2, (page // 16, hd, 16)))
    return kc, vc, k[..., n // 2:].view(torch.uint8).to(torch.int32), v[..., n // 2:].view(torch.uint8).to(torch.int32)


def _by_sequence(x, table):
    """[page][kv head][slot] ... -> [sequence][kv head][position] ..."""
    return x[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)


def _row_places(st):
    """(sequence, position) of every row."""
    t = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(st["row_start"][1:].contiguous(), t.to(torch.int32), right=True)
    return b, st["kv_len"][b].long() - st["row_start"][b + 1].long() + t


def _plain_append(st):
    c = st["case"]
    nh, nkv, hd, page = (c[k] for k in ("nh", "nkv", "hd", "page"))
    b, p = _row_places(st)
    x = st["qkv"].to(torch.int32).unflatten(1, (-1, hd))
    lo, hi = x[:, : nh + nkv, : hd // 2], x[:, : nh + nkv, hd // 2:]
    C, S = st["cos"][p].to(torch.int32)[:, None], st["sin"][p].to(torch.int32)[:, None]
    turn = torch.cat([lo * C - hi * S, hi * C + lo * S], dim=2)
    turn = (torch.sign(turn) * ((turn.abs() + (1 << 13)) >> 14)).clamp(-127, 127).to(torch.int8)
    k, v = turn[:, nh:], x[:, nh + nkv:].to(torch.int8)
    pid, off = st["table"][b, p // page].long(), p % page
    if c["bits"] == 8:
        st["k"].unflatten(2, (page, hd))[pid, :, off] = k
        st["v"].unflatten(2, (page // 16, hd, 16))[pid, :, off // 16, :, off % 16] = v
    else:
        n = page * hd // 2
        (kc, km), (vc, vm) = _quant4(k), _quant4(v)
        st["k"][..., :n].unflatten(2, (page, hd // 2))[pid, :, off] = _pack4(kc)
        st["k"][..., n:][pid, :, off] = km.to(torch.uint8).view(torch.int8)
        st["v"][..., n:][pid, :, off] = vm.to(torch.uint8).view(torch.int8)
        # two positions share a byte of v: the codes are unpacked, written and packed again
        blk = _unpack4(st["v"][..., :n]).unflatten(2, (page // 16, hd, 16))
        blk[pid, :, off // 16, :, off % 16] = vc
        st["v"][..., :n] = _pack4(blk).flatten(2)
    return turn[:, :nh].flatten(1)


def _plain_read(st):
    cap = st["ko"].shape[1]
    kc, vc, km, vm = _pages(st)
    live = torch.arange(cap, device=DEV) < st["kv_len"][:, None]
    out = []
    for x, m in ((kc, km), (vc, vm)):
        x = _by_sequence(x, st["table"])
        if m is not None:
            x = _div_round(x * _by_sequence(m, st["table"])[..., None], 8).clamp(-127, 127).to(torch.int8)
        out.append(torch.where(live[:, :, None, None], x[:, :, :cap].transpose(1, 2), 0))
    return tuple(out)


def _plain_attend(st):
    c = st["case"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    rep = nh // nkv
    b, p = _row_places(st)
    most = int(max(n for n, _ in _lengths(c)))
    i = torch.arange(st["tokens"], device=DEV) - st["row_start"][b].long()
    q = torch.zeros(c["seqs"], most, nkv, rep, hd, device=DEV)
    q[b, i] = st["q"].float().unflatten(1, (nkv, rep, hd))
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)  # sequence, kv head, (row, head of the group), dimension
    pos = torch.full((c["seqs"], most), -1, dtype=torch.int64, device=DEV)
    pos[b, i] = p
    pos = pos.repeat_interleave(rep, dim=1)[:, None, :, None]
    kc, vc, km, vm = _pages(st)
    k, v = _by_sequence(kc, st["table"]).float(), _by_sequence(vc, st["table"])
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).to(torch.int32)  # exact: at most 2^21
    if km is not None:
        s = (s * _by_sequence(km, st["table"])[:, :, None] + 4) >> 3
    j = torch.arange(s.shape[3], device=DEV)
    seen = j <= pos
    if c["window"]:
        seen &= (j > pos - c["window"]) | (j < c["sinks"])
    low = torch.iinfo(torch.int32).min // 2
    s = torch.where(seen, s, low)
    at = ((s.amax(dim=3, keepdim=True) - s + 64) >> 7).clamp(0, 1024)
    e = torch.cat([st["exp"], st["exp"].new_zeros(1)])[at]
    e = torch.where(seen, e, 0)
    del s, at, seen
    den = e.sum(dim=3, keepdim=True)  # 64 bits
    w = e.double()
    if vm is not None:
        w = w * _by_sequence(vm, st["table"])[:, :, None]
        den = 8 * den
    top = torch.matmul(w, v.double()).to(torch.int64)  # exact: sums of integers below 2^53
    o = _div_round(top, den.clamp(min=1)).clamp(-127, 127).to(torch.int8)
    o = o.unflatten(2, (most, rep)).permute(0, 2, 1, 3, 4)
    return o[b, i].flatten(1)


# -- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "argmax":
        return dict(bytes=4 * case["batch"] * (case["n"] + 1), flops=case["batch"] * case["n"])
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    lens = _lengths(case)
    tokens = sum(n for n, _ in lens)
    held = nkv * (hd if case["bits"] == 8 else hd // 2 + 1)  # bytes of one position in one pool
    if case["kind"] == "attend":
        pairs = places = 0
        for n, L in lens:
            first = L - n
            w, s = case["window"], case["sinks"]
            if not w:
                places += L
                pairs += n * first + n * (n + 1) // 2
            else:
                lo = max(0, first - w + 1)
                places += L - lo + min(s, lo)
                pairs += sum(min(p + 1, w) + min(s, max(0, p + 1 - w)) for p in range(first, L))
        return dict(bytes=2 * held * places + 2 * tokens * nh * hd, flops=4 * hd * nh * pairs)
    b = tokens * ((nh + 2 * nkv) * hd + nh * hd + 2 * held) + 2 * hd * max(n for n, _ in lens)
    if case["kind"] == "cache":
        b += sum(L for _, L in lens) * 2 * (held + nkv * hd)
    return dict(bytes=b, flops=tokens * (nh + nkv) * hd * 3)


# -- the definition, in 64 bits --------------------------------------------------------------------------------------


def _slot(st, pool, pid, g, off):
    """What positions (page ids pid, slots off) of kv head g hold, from the layout alone: codes and multipliers, int64."""
    c = st["case"]
    page, hd = c["page"], c["hd"]
    d = torch.arange(hd, device=DEV)
    raw = st[pool][pid, g].long() & 255  # positions x bytes of a page
    if pool == "k":
        place = off[:, None] * hd + d
        sub = d % 16 + 0 * off[:, None]
    else:
        place = (off[:, None] // 16) * (16 * hd) + d * 16 + off[:, None] % 16
        sub = off[:, None] % 16 + 0 * d
    if c["bits"] == 8:
        x = raw.gather(1, place)
        return torch.where(x > 127, x - 256, x), None
    chunk = place // 16  # of 16 codes, 8 bytes
    x = raw.gather(1, chunk * 8 + (sub // 8) * 4 + sub % 4)
    x = torch.where(sub % 8 >= 4, x // 16, x % 16)
    return torch.where(x > 7, x - 16, x), raw.gather(1, page * hd // 2 + off[:, None])[:, 0]


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "argmax":
        x = st["logits"].cpu().numpy()
        return torch.from_numpy(x.argmax(axis=1)).to(torch.int32)
    nh, nkv, hd, page = (case[k] for k in ("nh", "nkv", "hd", "page"))
    lens, at = _lengths(case), 0
    if case["kind"] != "attend":
        q = torch.zeros(st["tokens"], nh * hd, dtype=torch.int8, device=DEV)
        ko, vo = ((st["ko"].long(), st["vo"].long()) if case["kind"] == "cache" else (None, None))
        half = hd // 2
        for b, (n, L) in enumerate(lens):
            p = torch.arange(L - n, L, device=DEV)
            x = st["qkv"][at:at + n].double().view(n, -1, hd)
            C, S = st["cos"][p].double()[:, None], st["sin"][p].double()[:, None]
            y = x.clone()
            y[..., :half] = x[..., :half] * C - x[..., half:] * S
            y[..., half:] = x[..., half:] * C + x[..., :half] * S
            y = (torch.sign(y) * torch.floor(y.abs() / 16384 + 0.5)).clamp(-127, 127)
            q[at:at + n] = y[:, :nh].reshape(n, -1).to(torch.int8)
            k, v = y[:, nh:nh + nkv].long(), x[:, nh + nkv:].long()
            if case["kind"] == "append":
                pid = st["table"][b, (p // page)].long()
                for g in range(nkv):
                    d = torch.arange(hd, device=DEV)
                    off = (p % page)[:, None]
                    st["k"][pid[:, None], g, off * hd + d] = k[:, g].to(torch.int8)
                    st["v"][pid[:, None], g, (off // 16) * 16 * hd + d * 16 + off % 16] = v[:, g].to(torch.int8)
            else:
                j = torch.arange(L, device=DEV)
                pid = st["table"][b, j // page].long()
                for g in range(nkv):
                    for pool, new, to in (("k", k, ko), ("v", v, vo)):
                        c, m = _slot(st, pool, pid, g, j % page)
                        c = c.double()
                        if m is not None:
                            c = (torch.sign(c) * torch.floor(c.abs() * m[:, None] / 8 + 0.5)).clamp(-127, 127)
                            r = new[:, g].double()
                            mm = torch.ceil(8 * r.abs().amax(dim=1, keepdim=True) / 7)
                            cc = (torch.sign(r) * torch.floor(8 * r.abs() / mm.clamp(min=1) + 0.5)).clamp(-7, 7)
                            c[L - n:] = (torch.sign(cc) * torch.floor(cc.abs() * mm / 8 + 0.5)).clamp(-127, 127)
                        else:
                            c[L - n:] = new[:, g].double()
                        to[b, :L, g] = c.long()
            at += n
        return (q, st["k"], st["v"]) if case["kind"] == "append" else (q, ko.to(torch.int8), vo.to(torch.int8))
    o = torch.zeros(st["tokens"], nh, hd, dtype=torch.int8, device=DEV)
    T = torch.cat([st["exp"].double(), torch.zeros(1, dtype=torch.float64, device=DEV)])
    for b, (n, L) in enumerate(lens):
        j = torch.arange(L, device=DEV)
        pid = st["table"][b, j // page].long()
        p = torch.arange(L - n, L, device=DEV)[:, None]
        seen = j <= p
        if case["window"]:
            seen = seen & ((p - j < case["window"]) | (j < case["sinks"]))
        for g in range(nkv):
            kc, km = _slot(st, "k", pid, g, j % page)
            vc, vm = _slot(st, "v", pid, g, j % page)
            for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                q = st["q"][at:at + n, h * hd:(h + 1) * hd].double()
                s = q @ kc.double().t().contiguous()
                if km is not None:
                    s = torch.floor((s * km + 4) / 8)
                s = s.masked_fill(~seen, -math.inf)
                i = torch.floor((s.amax(dim=1, keepdim=True) - s + 64) / 128).clamp(max=1024).long()
                w = T[i]
                den = w.sum(dim=1, keepdim=True)
                if vm is not None:
                    w, den = w * vm, 8 * den
                y = w @ vc.double()
                # |y| / den half away from zero, the floor in whole numbers
                y = torch.sign(y) * torch.div(2 * y.abs().long() + den.long(), 2 * den.long(), rounding_mode="floor")
                o[at:at + n, h] = y.clamp(-127, 127).to(torch.int8)
        at += n
    return o.view(st["tokens"], -1)
