"""Timed cases of the paged int8 decoder's further operators, beside their plain forms in elementary torch.

Four operators, all with integer results that the rules fix, so every output is compared exactly:

  norm      the new rows' q and k normed head by head, rotated, k and v written to their pages (8 bits, or 4)
  weigh     each held position's share of the rows' attention, added up per kv head (what an eviction goes by)
  evict     a sequence cut down to its heaviest positions, which move to other pages
  logprobs  log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits

A batch is ragged: sequence b has rows row_start[b] .. row_start[b + 1] - 1 and kv_len[b] positions, its rows the last of
them; position j is slot j % page of page table[b][j // page]. 8-bit pages hold int8 codes; in 4 bits a row x of one
position and kv head is held as a multiplier m = ceil(8 max|x| / 7) and codes c = clamp(round(8 x / m), +-7), for c m / 8.

norm      V = sum x^2 over a head, R = isqrt(V 2^16 / hd), n = clamp(round(128 x w / R), +-16383) with w at 2^12, then rotate-half by
          the int16 tables of position p + shift[b]: clamp(round((n C - n' S) / 2^20), +-127). v goes as it is.
weigh     of a row and head, top = max s and R = min(floor(2^40 / sum e), 2^32 - 1) are known; e = T[(top - s + 64) >> 7],
          s = q . k (4 bits: (m (q . c) + 4) >> 3); W[kv head][position] = sum over rows and heads of e R.
evict     of more than `budget` positions the first `sinks`, the last `recent` and, of the others, those with the largest W stay (ties: the
          first), in order.
logprobs  t(d) = (d mant + 2^(shift - 1)) >> shift, in 2^-16 of a power of two. For blocks of 1024 logits with maxima M_B:
          t = min(t(M_B - x), 31 2^16), e = 2^30 2^(-t / 2^16) (product of two tables, cut), S_B = sum e, W_B = sum e t. Joined to M =
          max M_B by the same tables (t at most 41 2^16), log2 by a table of 1025, outputs in 2^-16 nats.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"


def _case(name, kind, **kw):
    c = dict(name=name, kind=kind)
    if kind != "logprobs":
        c.update(seqs=1, prompts=0, rows=1, past=0, ragged=False, nh=14, nkv=2, hd=64, page=16, bits=8)
    if kind == "weigh":
        c.update(window=0, sinks=0)
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of a batch whose sequences have been cut down before: positions apart from slots
        _case("norm_batch", "norm", seqs=64, past=1000, ragged=True),
        # prompts of a few sequences admitted together, behind a shared system prompt
        _case("norm_prompts", "norm", seqs=4, prompts=4, rows=512, past=77, nh=16, nkv=4, hd=128, page=64),
        # a long prompt into 4-bit pages
        _case("norm_prompt4", "norm", prompts=1, rows=2048, nh=16, nkv=4, hd=128, page=32, bits=4),
        # a single user's decode step: latency
        _case("weigh_one", "weigh", past=640),
        # the decode step of a served batch with long histories: K's bytes are the work
        _case("weigh_batch", "weigh", seqs=128, past=8191, ragged=True),
        # the last rows of a long prompt, before it is cut down
        _case("weigh_chunk", "weigh", prompts=1, rows=1024, past=7777),
        # one very long document on 4-bit pages, a token at a time
        _case("weigh_long4", "weigh", past=131000, bits=4, page=64),
        # a served batch past its budget, most of its sequences at once
        _case("evict_batch", "evict", seqs=64, past=2200, ragged=True, budget=1024, recent=256, sinks=4),
        # one very long document on 4-bit pages cut to an eighth
        _case("evict_long4", "evict", past=131000, bits=4, page=64, budget=16384, recent=1024, sinks=16),
        # what a single user asks of a token: its probability and five others
        _case("logprobs_one", "logprobs", n=151936, rows=1, k=5),
        # the same for a served batch, with twenty alternatives
        _case("logprobs_batch", "logprobs", n=151936, rows=64, k=20),
        # a text of odd length scored: no alternatives
        _case("logprobs_text", "logprobs", n=151936, rows=1021, k=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "weigh", "weigh", "weigh", "evict", "evict", "logprobs", "logprobs"])
    if kind == "logprobs":
        c = dict(kind=kind, n=_log(rng, 97, 200000), rows=_log(rng, 1, 700), k=rng.choice([0, 1, 5, 20, 32]))
    else:
        nkv = rng.choice([1, 2, 2, 4])
        c = _case("", kind, nkv=nkv, nh=nkv * rng.choice([1, 4, 7, 7, 8, 12]), hd=rng.choice([64, 64, 64, 128]),
                  page=rng.choice([16, 16, 32, 64, 128]), bits=rng.choice([8, 4]), ragged=rng.random() < 0.7)
        del c["name"]
        if kind == "evict":
            c.update(seqs=_log(rng, 1, 64), past=_log(rng, 40, 30000))
            c["budget"] = max(1, int(c["past"] * rng.uniform(0.05, 0.9)))
            c["sinks"] = rng.choice([0, 1, 4, min(16, c["budget"] // 4)]) if c["budget"] >= 16 else 0
            c["recent"] = int((c["budget"] - c["sinks"]) * rng.choice([0.0, 0.25, 0.5, 1.0]))
        elif rng.random() < 0.5:  # single tokens
            c.update(seqs=_log(rng, 1, 64), past=_log(rng, 1, 8000 if kind == "weigh" else 1500))
        else:  # chunks, some of them beside single tokens
            c.update(rows=_log(rng, 2, 600), past=rng.choice([0, _log(rng, 1, 3000)]))
            c["seqs"] = rng.randint(1, 4)
            c["prompts"] = rng.randint(1, c["seqs"])
        if kind == "weigh" and rng.random() < 0.3:
            c.update(window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 100]))
    while work(c)["flops"] > 1.5e10 or work(c)["bytes"] > 6e8:  # no more than the largest of the listed ones
        key = "rows" if kind == "logprobs" or (kind != "evict" and c["prompts"] and c["rows"] > c["past"] // 8) else "past"
        c[key] //= 2
    return c


# -- inputs ----------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _lengths(case):
    """(new rows, positions with them) of each sequence; an eviction has no new rows."""
    out = []
    for i in range(case["seqs"]):
        n = case["rows"] if i < case["prompts"] else 1
        past = case["past"]
        if case["ragged"]:
            past -= (i * 40503 + 17) % (past // 2 + 1)
            n -= (i * 97) % (n // 3 + 1)
        out.append((0, past) if case["kind"] == "evict" else (n, past + n))
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


UNIT = 87381  # codes of a logit's natural unit: at a standard deviation of 2^18, three units


def _scale():
    """(mant, shift) of UNIT: logits to 2^-16 of a power of two."""
    r = 65536.0 * math.log2(math.e) / UNIT
    shift = 30 - math.floor(math.log2(r))
    return round(r * 2.0 ** shift), shift


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "logprobs":
        rows, n, k = (case[x] for x in ("rows", "n", "k"))
        x = torch.randn(rows, n, generator=g, device=DEV).mul_(1 << 18).round_().to(torch.int32)
        sure = torch.rand(rows, 2, generator=g, device=DEV)  # most rows have a token that stands out, and most ask for it
        tok = torch.randint(0, n, (rows,), generator=g, device=DEV)
        x[torch.arange(rows, device=DEV), tok] += (sure[:, 0] * (20 * UNIT)).to(torch.int32)
        tok = torch.where(sure[:, 1] < 0.7, tok, torch.randint(0, n, (rows,), generator=g, device=DEV)).to(torch.int32)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
        st = dict(case=case, logits=x, tokens=tok, lp=i32(rows), ent=i32(rows), top=i32(rows, k), top_lp=i32(rows, k),
                  tables=_tables())
        if own:
            _handles(st)
        return st
    lens = _lengths(case)
    kind, page, nkv, nh, hd, seqs = (case[k] for k in ("kind", "page", "nkv", "nh", "hd", "seqs"))
    need = [-(-L // page) for _, L in lens]
    after = [-(-min(L, case["budget"]) // page) for _, L in lens] if kind == "evict" else []
    max_pages, pages = max(need), sum(need) + sum(after) + 3
    row_start = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).to(DEV)
    kv_len = torch.tensor([L for _, L in lens], dtype=torch.int32, device=DEV)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)

    def table_of(counts, first):
        t = torch.full((seqs, max(counts)), -1, dtype=torch.int32, device=DEV)
        used = torch.arange(max(counts), device=DEV) < torch.tensor(counts, device=DEV)[:, None]
        t[used] = order[first: first + sum(counts)]
        return t

    tokens = sum(n for n, _ in lens)
    st = dict(case=case, tokens=tokens, max_pages=max_pages, pages=pages, row_start=row_start, kv_len=kv_len,
              table=table_of(need, 0))
    kp, vp = _rows8(g, pages, nkv, page, hd), _rows8(g, pages, nkv, page, hd)
    if case["bits"] == 8:
        kp, vp = kp.reshape(pages, nkv, -1), _blocks(vp).reshape(pages, nkv, -1)
    else:
        (kc, km), (vc, vm) = _quant4(kp), _quant4(vp)
        kp = torch.cat([_pack4(kc).reshape(pages, nkv, -1), km.to(torch.uint8).view(torch.int8)], dim=2)
        vp = torch.cat([_pack4(_blocks(vc)).reshape(pages, nkv, -1), vm.to(torch.uint8).view(torch.int8)], dim=2)
    st.update(k=kp.contiguous(), v=vp.contiguous())
    if kind == "norm":
        shift = torch.randint(0, 400, (seqs,), generator=g, device=DEV).to(torch.int32)
        cos, sin = _rope_tables(max(L for _, L in lens) + 400, hd)
        wt = lambda: (4096 * (1 + 0.3 * torch.randn(hd, generator=g, device=DEV))).round().to(torch.int16)  # noqa: E731
        st.update(qkv=_rows8(g, tokens, (nh + 2 * nkv) * hd), cos=cos, sin=sin, shift=shift, q_norm=wt(), k_norm=wt(),
                  q=torch.zeros(tokens, nh * hd, dtype=torch.int8, device=DEV))
    elif kind == "weigh":
        st.update(q=_rows8(g, tokens, nh * hd), exp=_exp_table(hd), w=torch.zeros(pages, nkv, page, dtype=torch.int64, device=DEV))
        top, den, _ = _softmax(st)
        R = torch.div(1 << 40, den.clamp(min=1), rounding_mode="floor").clamp(max=(1 << 32) - 1) * (den > 0)
        st["stats"] = torch.stack([top, torch.where(R >= 1 << 31, R - (1 << 32), R).to(torch.int32)], dim=-1).contiguous()
    else:
        # sums of weights over many rows: a few positions hold most, many were never looked at
        w = torch.exp(2.5 * torch.randn(pages, nkv, page, generator=g, device=DEV)).mul_(1 << 38).to(torch.int64)
        w[torch.rand(pages, nkv, page, generator=g, device=DEV) < 0.2] = 0
        st.update(w=w, to=table_of(after, sum(need)),
                  kept=torch.zeros(seqs, nkv, case["budget"], dtype=torch.int32, device=DEV))
    if own:
        _handles(st)
    return st


def _handles(st):
    """The framework's handles of the same buffers, which a program makes once."""
    from tritify_amd import backend as B
    from tritify_amd.paged import PagedBatch, PagedKV

    c = st["case"]
    if c["kind"] == "logprobs":
        st["ws"] = torch.empty(B.dec_logprobs_rows_workspace(c["rows"], c["n"], c["k"]), dtype=torch.int8, device=DEV)
        st["scale"] = B.logit_scale(UNIT)
        return
    st["batch"] = PagedBatch(st["row_start"], st["kv_len"], st["table"], st["tokens"])
    st["kv"] = PagedKV(st["pages"], c["page"], c["nkv"], c["hd"], bits=c["bits"], k=st["k"], v=st["v"], w=st.get("w"))


# -- one pass --------------------------------------------------------------------------------------------------------


def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    if kind == "norm":
        return _plain_norm(st), st["k"], st["v"]
    if kind == "weigh":
        _plain_weigh(st)
        return st["w"]
    if kind == "evict":
        _plain_evict(st)
        return st["kept"], st["k"], st["v"], st["w"]
    return _plain_logprobs(st)


def _own(st, kind):
    c = st["case"]
    if kind == "logprobs":
        from tritify_amd import backend as B

        B.dec_logprobs_rows(st["logits"], c["rows"], c["n"], st["tokens"], st["scale"], st["lp"], st["ws"], entropy_dev=st["ent"],
                            top_dev=st["top"] if c["k"] else None, top_lp_dev=st["top_lp"] if c["k"] else None, k=c["k"])
        return (st["lp"], st["ent"], st["top"], st["top_lp"]) if c["k"] else (st["lp"], st["ent"])
    kv, batch = st["kv"], st["batch"]
    if kind == "norm":
        kv.append(st["qkv"], batch, c["nh"], st["cos"], st["sin"], st["q"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                  shift=st["shift"])
        return st["q"], st["k"], st["v"]
    if kind == "weigh":
        kv.weigh(st["q"], batch, c["nh"], st["exp"], st["stats"], window=c["window"], sinks=c["sinks"], fresh=True)
        return st["w"]
    kv.evict(batch, st["to"], c["budget"], st["kept"], recent=c["recent"], sinks=c["sinks"])
    return st["kept"], st["k"], st["v"], st["w"]


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


def _by_sequence(x, table):
    """[page][kv head][slot] ... -> [sequence][kv head][position] ..."""
    return x[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)


def _row_places(st):
    """(sequence, position) of every row."""
    t = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(st["row_start"][1:].contiguous(), t.to(torch.int32), right=True)
    return b, st["kv_len"][b].long() - st["row_start"][b + 1].long() + t


def _write(st, pid, heads, off, k, v):
    """Rows k and v (.. x hd codes; 4 bits: (codes, multipliers)) to slots `off` of pages pid, kv heads `heads`."""
    c = st["case"]
    page, hd = c["page"], c["hd"]
    if c["bits"] == 8:
        st["k"].unflatten(2, (page, hd))[pid, heads, off] = k
        st["v"].unflatten(2, (page // 16, hd, 16))[pid, heads, off // 16, :, off % 16] = v
        return
    n = page * hd // 2
    st["k"][..., :n].unflatten(2, (page, hd // 2))[pid, heads, off] = _pack4(k[0])
    st["k"][..., n:][pid, heads, off] = k[1].to(torch.uint8).view(torch.int8)
    st["v"][..., n:][pid, heads, off] = v[1].to(torch.uint8).view(torch.int8)
    # two positions share a byte of v: the codes are unpacked, written and packed again
    blk = _unpack4(st["v"][..., :n]).unflatten(2, (page // 16, hd, 16))
    blk[pid, heads, off // 16, :, off % 16] = v[0]
    st["v"][..., :n] = _pack4(blk).flatten(2)


def _plain_norm(st):
    c = st["case"]
    nh, nkv, hd, page = (c[k] for k in ("nh", "nkv", "hd", "page"))
    b, p = _row_places(st)
    x = st["qkv"].to(torch.int64).unflatten(1, (-1, hd))
    h = x[:, : nh + nkv]
    V = (h * h).sum(dim=2, keepdim=True) * (65536 // hd)  # below 2^31: the root of its double is off by less than one
    R = torch.sqrt(V.double()).to(torch.int64)
    R = R - (R * R > V).long()
    R = R + ((R + 1) * (R + 1) <= V).long()
    w = torch.cat([st["q_norm"].expand(nh, hd), st["k_norm"].expand(nkv, hd)]).to(torch.int64)
    n = torch.where(R > 0, _div_round(128 * h * w, R.clamp(min=1)), 0).clamp(-16383, 16383)
    at = p + st["shift"][b].long()
    C, S = st["cos"][at].to(torch.int64)[:, None], st["sin"][at].to(torch.int64)[:, None]
    lo, hi = n[..., : hd // 2], n[..., hd // 2:]
    turn = torch.cat([lo * C - hi * S, hi * C + lo * S], dim=2)
    turn = (torch.sign(turn) * ((turn.abs() + (1 << 19)) >> 20)).clamp(-127, 127).to(torch.int8)
    k, v = turn[:, nh:], x[:, nh + nkv:].to(torch.int8)
    if c["bits"] == 4:
        k, v = _quant4(k), _quant4(v)
    pid, off = st["table"][b, p // page].long()[:, None], (p % page)[:, None]
    _write(st, pid, torch.arange(nkv, device=DEV)[None], off, k, v)
    return turn[:, :nh].flatten(1)


def _softmax(st):
    """Of every row and head the largest score and the sum of weights, and the scores: sequence, kv head, (row, head), position."""
    c = st["case"]
    nh, nkv, hd, page = (c[k] for k in ("nh", "nkv", "hd", "page"))
    rep = nh // nkv
    b, p = _row_places(st)
    most = int(max(n for n, _ in _lengths(c)))
    i = torch.arange(st["tokens"], device=DEV) - st["row_start"][b].long()
    q = torch.zeros(c["seqs"], most, nkv, rep, hd, device=DEV)
    q[b, i] = st["q"].float().unflatten(1, (nkv, rep, hd))
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)
    pos = torch.full((c["seqs"], most), -1, dtype=torch.int64, device=DEV)
    pos[b, i] = p
    pos = pos.repeat_interleave(rep, dim=1)[:, None, :, None]
    n = page * hd
    k, m = st["k"], None
    if c["bits"] == 8:
        k = k.unflatten(2, (page, hd))
    else:
        k, m = _unpack4(k[..., : n // 2]).unflatten(2, (page, hd)), k[..., n // 2:].view(torch.uint8).to(torch.int32)
    k = _by_sequence(k, st["table"]).float()
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).to(torch.int32)  # exact: at most 2^21
    if m is not None:
        s = (s * _by_sequence(m, st["table"])[:, :, None] + 4) >> 3
    j = torch.arange(s.shape[3], device=DEV)
    seen = j <= pos
    if c["window"]:
        seen &= (j > pos - c["window"]) | (j < c["sinks"])
    s = torch.where(seen, s, -(1 << 30))
    top = s.amax(dim=3, keepdim=True)
    den = _exp_of(st, top, s).sum(dim=3)
    by_row = lambda x: x.unflatten(2, (most, rep)).permute(0, 2, 1, 3)[b, i].flatten(1)  # noqa: E731
    return by_row(top[..., 0]), by_row(den), s


def _exp_of(st, top, s):
    e = torch.cat([st["exp"], st["exp"].new_zeros(1)])[((top - s + 64) >> 7).clamp(0, 1024)]
    return torch.where(s > -(1 << 30), e, 0)


def _plain_weigh(st):
    c = st["case"]
    nh, nkv = c["nh"], c["nkv"]
    rep = nh // nkv
    b, _ = _row_places(st)
    most = int(max(n for n, _ in _lengths(c)))
    i = torch.arange(st["tokens"], device=DEV) - st["row_start"][b].long()
    s = _softmax(st)[2]
    x = torch.zeros(c["seqs"], most, nkv, rep, 2, dtype=torch.int64, device=DEV)
    x[b, i] = st["stats"].long().unflatten(1, (nkv, rep))
    top, R = x.permute(0, 2, 1, 3, 4).flatten(2, 3).unbind(dim=-1)
    w = (_exp_of(st, top[..., None].to(torch.int32), s).long() * (R & 0xFFFFFFFF)[..., None]).sum(dim=2)
    live = torch.arange(w.shape[2], device=DEV) < st["kv_len"][:, None]
    sq, j = live.nonzero(as_tuple=True)
    st["w"][st["table"][sq, j // c["page"]].long(), :, j % c["page"]] = w[sq, :, j]


def _plain_evict(st):
    c = st["case"]
    nkv, hd, page, budget = c["nkv"], c["hd"], c["page"], c["budget"]
    cap = st["max_pages"] * page
    w = _by_sequence(st["w"], st["table"])[..., :cap]
    j = torch.arange(cap, device=DEV)
    L = st["kv_len"].long()[:, None, None]
    # by weight, then by the lower position: protected ones first, those past the length last
    rank = torch.where((j < c["sinks"]) | (j >= L - c["recent"]), 1 << 62, w)
    rank = torch.where(j < L, rank, -1)
    order = torch.sort(rank, dim=2, descending=True, stable=True)[1][..., :budget]
    order = torch.sort(torch.where(order < L, order, cap), dim=2)[0]
    kept = torch.full_like(st["kept"], -1)
    kept[..., : order.shape[2]] = torch.where(order < cap, order, -1).to(torch.int32)
    st["kept"].copy_(kept)
    b, g, i = (kept >= 0).nonzero(as_tuple=True)
    src = kept[b, g, i].long()
    sp, so, tp, to = st["table"][b, src // page].long(), src % page, st["to"][b, i // page].long(), i % page
    n = page * hd
    if c["bits"] == 8:
        k = st["k"].unflatten(2, (page, hd))[sp, g, so]
        v = st["v"].unflatten(2, (page // 16, hd, 16))[sp, g, so // 16, :, so % 16]
    else:
        k = (_unpack4(st["k"][..., : n // 2]).unflatten(2, (page, hd))[sp, g, so], st["k"][..., n // 2:][sp, g, so])
        v = (_unpack4(st["v"][..., : n // 2]).unflatten(2, (page // 16, hd, 16))[sp, g, so // 16, :, so % 16],
             st["v"][..., n // 2:][sp, g, so])
        k, v = (k[0], k[1].view(torch.uint8)), (v[0], v[1].view(torch.uint8))
    _write(st, tp, g, to, k, v)
    st["w"][tp, g, to] = st["w"][sp, g, so]


def _tables():
    """2^31 2^(-i / 2^8), 2^31 2^(-i / 2^16), 2^24 log2(1 + i / 2^10)."""
    i = torch.arange(256, dtype=torch.float64, device=DEV)
    j = torch.arange(1025, dtype=torch.float64, device=DEV)
    return tuple(x.round().to(torch.int64) for x in (2147483648.0 * torch.exp2(-i / 256), 2147483648.0 * torch.exp2(-i / 65536),
                                                     16777216.0 * torch.log2(1 + j / 1024)))


def _bits(d, most):
    """t(d), at most `most`."""
    mant, shift = _scale()
    end = ((most + 1) << shift) // mant + 1  # past it t is past `most`
    return ((d.clamp(max=end) * mant + ((1 << shift) >> 1)) >> shift).clamp(max=most)


MOST, FAR = 31 << 16, 41 << 16
LN2 = 5814540  # 2^23 ln 2


def _plain_logprobs(st):
    c, x = st["case"], st["logits"].long()
    rows, n, k = c["rows"], c["n"], c["k"]
    A, F, G = st["tables"]
    pad = torch.full((rows, -n % 1024), -(1 << 40), dtype=torch.int64, device=DEV)
    x = torch.cat([x, pad], dim=1).unflatten(1, (-1, 1024))
    mb = x.amax(dim=2, keepdim=True)
    t = _bits(mb - x, MOST)
    e = (A[(t & 65535) >> 8] * F[t & 255] >> 32) >> (t >> 16)
    S, W = e.sum(dim=2), (e * t).sum(dim=2)
    del e, t
    mb = mb[..., 0]
    M = mb.amax(dim=1, keepdim=True)
    u = _bits(M - mb, FAR)
    m = A[(u & 65535) >> 8] * F[u & 255] >> 32
    W = ((((W + u * S) >> 21) * (m >> 8)) >> (22 + (u >> 16))).sum(dim=1)
    S = (((S >> 8) * m) >> (22 + (u >> 16))).sum(dim=1)
    a = (torch.log2(S.double()) + 1e-12).floor().long()  # S is below 2^51: a power of two or off it by 2^-51 at least
    a = a - ((1 << a) > S).long()
    y = torch.where(a >= 31, S >> (a - 31).clamp(min=0), S << (31 - a).clamp(min=0)) - (1 << 31)
    i = y >> 21
    L = ((a - 30) << 24) + G[i] + (((G[i + 1] - G[i]) * (y & ((1 << 21) - 1))) >> 21)
    ent = ((((torch.div(W << 18, S >> 3, rounding_mode="floor")) << 8) + L) * LN2 + (1 << 30)) >> 31
    x = x.flatten(1)[:, :n]

    def lp(v):
        return -((((_bits(M - v, (1 << 31) - 1) << 8) + L[:, None]) * LN2 + (1 << 30)) >> 31).to(torch.int32)

    out = [lp(x.gather(1, st["tokens"].long()[:, None]))[:, 0], ent.to(torch.int32)]
    if k == 0:
        return tuple(out)
    top = torch.full((rows, k), -1, dtype=torch.int32, device=DEV)
    top_lp = torch.full((rows, k), -(1 << 31), dtype=torch.int32, device=DEV)
    key = x * (1 << 32) + torch.arange(n - 1, -1, -1, device=DEV)  # the largest (value, -index)
    for r in range(min(k, n)):
        best = key.amax(dim=1, keepdim=True)
        top[:, r] = (n - 1 - (best[:, 0] & 0xFFFFFFFF)).to(torch.int32)
        top_lp[:, r] = lp(best >> 32)[:, 0]
        key.scatter_(1, top[:, r:r + 1].long(), -(1 << 63))
    return tuple(out + [top, top_lp])


# -- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "logprobs":
        return dict(bytes=4 * case["rows"] * (case["n"] + 3 + 2 * case["k"]), flops=6 * case["rows"] * case["n"])
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    lens = _lengths(case)
    tokens = sum(n for n, _ in lens)
    held = nkv * (hd if case["bits"] == 8 else hd // 2 + 1)  # bytes of one position in one pool
    if case["kind"] == "evict":
        kept = sum(min(L, case["budget"]) for _, L in lens)
        # the weights of all positions; the kept ones' k, v and weight moved, and their positions
        held = sum(8 * nkv * L for _, L in lens) + kept * (4 * held + 12 * nkv)
        return dict(bytes=held, flops=sum(nkv * L for _, L in lens))
    if case["kind"] == "weigh":
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
        return dict(bytes=held * places + 8 * nkv * sum(L for _, L in lens) + tokens * nh * (hd + 8), flops=2 * hd * nh * pairs)
    b = tokens * ((nh + 2 * nkv) * hd + nh * hd + 2 * held) + 2 * hd * max(n for n, _ in lens)
    return dict(bytes=b, flops=tokens * (nh + nkv) * hd * 8)


# -- the definition, in 64 bits --------------------------------------------------------------------------------------


def _places(case, pool, off):
    """Byte places (and which half of the byte, 4 bits) of slots `off` in a part of a page: slots x hd."""
    hd = case["hd"]
    d = torch.arange(hd, device=DEV)
    place = off[:, None] * hd + d if pool == "k" else (off[:, None] // 16) * (16 * hd) + d * 16 + off[:, None] % 16
    if case["bits"] == 8:
        return place, None
    sub = place % 16
    return (place // 16) * 8 + (sub // 8) * 4 + sub % 4, sub % 8 >= 4


def _get(st, pool, pid, g, off):
    """What slots `off` of pages pid hold for kv head g, from the layout alone: codes and multipliers, int64."""
    c = st["case"]
    raw = st[pool][pid, g].long() & 255
    place, high = _places(c, pool, off)
    x = raw.gather(1, place)
    if high is None:
        return torch.where(x > 127, x - 256, x), None
    x = torch.where(high, x // 16, x % 16)
    return torch.where(x > 7, x - 16, x), raw.gather(1, c["page"] * c["hd"] // 2 + off[:, None])[:, 0]


def _put(st, pool, pid, g, off, x, m):
    """Codes x (and multipliers m) to slots `off`, half bytes one after the other."""
    c = st["case"]
    place, high = _places(c, pool, off)
    if high is None:
        st[pool][pid[:, None], g, place] = x.to(torch.int8)
        return
    for half in (False, True):
        at = (high == half).nonzero(as_tuple=True)
        p, w = pid[at[0]], place[at]
        old = st[pool][p, g, w].long() & 255
        new = (old % 16 + 16 * (x[at] & 15)) if half else (old // 16 * 16 + (x[at] & 15))
        st[pool][p, g, w] = torch.where(new > 127, new - 256, new).to(torch.int8)
    m = torch.where(m > 127, m - 256, m)
    st[pool][pid, g, c["page"] * c["hd"] // 2 + off] = m.to(torch.int8)


def _held4(r):
    """Codes and multipliers that hold the rows r (float64 whole numbers) in 4 bits."""
    m = torch.ceil(8 * r.abs().amax(dim=1, keepdim=True) / 7)
    x = (torch.sign(r) * torch.floor(8 * r.abs() / m.clamp(min=1) + 0.5)).clamp(-7, 7)
    return x.long(), m[:, 0].long()


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(st)
    nh, nkv, hd, page = (case[k] for k in ("nh", "nkv", "hd", "page"))
    lens, at = _lengths(case), 0
    if case["kind"] == "norm":
        q = torch.zeros(st["tokens"], nh, hd, dtype=torch.int8, device=DEV)
        for b, (n, L) in enumerate(lens):
            p = torch.arange(L - n, L, device=DEV)
            x = st["qkv"][at:at + n].double().view(n, -1, hd)
            C, S = (st[t][p + st["shift"][b].long()].double() for t in ("cos", "sin"))
            pid = st["table"][b, p // page].long()
            for h in range(nh + nkv):
                w = (st["q_norm"] if h < nh else st["k_norm"]).double()
                R = torch.floor(torch.sqrt((x[:, h] ** 2).mean(dim=1, keepdim=True) * 65536))
                y = 128 * x[:, h] * w
                y = torch.sign(y) * torch.div(2 * y.abs() + R, 2 * R.clamp(min=0.5), rounding_mode="floor")
                y = torch.where(R > 0, y, 0).clamp(-16383, 16383)
                a, c = y[:, : hd // 2], y[:, hd // 2:]
                y = torch.cat([a * C - c * S, c * C + a * S], dim=1) / 1048576
                y = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127)
                if h < nh:
                    q[at:at + n, h] = y.to(torch.int8)
                    continue
                for pool, r in (("k", y), ("v", x[:, h + nkv])):
                    codes, m = _held4(r) if case["bits"] == 4 else (r.long(), None)
                    _put(st, pool, pid, h - nh, p % page, codes, m)
            at += n
        return q.flatten(1), st["k"], st["v"]
    if case["kind"] == "weigh":
        T = torch.cat([st["exp"].double(), torch.zeros(1, dtype=torch.float64, device=DEV)])
        for b, (n, L) in enumerate(lens):
            j = torch.arange(L, device=DEV)
            pid = st["table"][b, j // page].long()
            p = torch.arange(L - n, L, device=DEV)[:, None]
            seen = j <= p
            if case["window"]:
                seen = seen & ((p - j < case["window"]) | (j < case["sinks"]))
            for g in range(nkv):
                kc, km = _get(st, "k", pid, g, j % page)
                total = torch.zeros(L, dtype=torch.int64, device=DEV)
                for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                    s = st["q"][at:at + n, h * hd:(h + 1) * hd].double() @ kc.double().t().contiguous()
                    if km is not None:
                        s = torch.floor((s * km + 4) / 8)
                    top, R = st["stats"][at:at + n, h].double().t()
                    R = torch.where(R < 0, R + 4294967296.0, R)
                    i = torch.floor((top[:, None] - s + 64) / 128).clamp(0, 1024).long()
                    w = T[i] * R[:, None]  # exact: below 2^47
                    total += torch.where(seen, w, 0).long().sum(dim=0)
                st["w"][pid, g, j % page] = total
            at += n
        return st["w"]
    if case["kind"] == "evict":
        src = {k: st[k].clone() for k in ("k", "v", "w")}
        src["case"] = case
        st["kept"].fill_(-1)
        for b, (_, L) in enumerate(lens):
            for g in range(nkv):
                j = torch.arange(L, device=DEV)
                if L > case["budget"]:
                    s, r = case["sinks"], case["recent"]
                    w = src["w"][st["table"][b, j // page].long(), g, j % page][s:L - r].cpu().numpy()
                    best = np.sort(s + np.lexsort((np.arange(len(w)), -w))[: case["budget"] - s - r])
                    j = torch.from_numpy(np.concatenate([np.arange(s), best, np.arange(L - r, L)])).to(DEV)
                i = torch.arange(len(j), device=DEV)
                st["kept"][b, g, i] = j.to(torch.int32)
                pid, to = st["table"][b, j // page].long(), st["to"][b, i // page].long()
                for pool in ("k", "v"):
                    _put(st, pool, to, g, i % page, *_get(src, pool, pid, g, j % page))
                st["w"][to, g, i % page] = src["w"][pid, g, j % page]
        return st["kept"], st["k"], st["v"], st["w"]


def _exact_logprobs(st):
    """Row by row, the products in floating point of 64 bits where they fit its 53 and in Python's whole numbers elsewhere."""
    c = st["case"]
    n, k = c["n"], c["k"]
    mant, shift = _scale()
    A = [round(2.0 ** 31 * 2.0 ** (-i / 256)) for i in range(256)]
    F = [round(2.0 ** 31 * 2.0 ** (-i / 65536)) for i in range(256)]
    G = [round(2.0 ** 24 * math.log2(1 + i / 1024)) for i in range(1025)]
    two = torch.tensor([a * f >> 32 for a in A for f in F], dtype=torch.int64, device=DEV)  # of every fraction of a power
    half = 1 << (shift - 1)

    def power(d, most):
        return min((d * mant + half) >> shift, most)

    out = [[], [], [], []]
    order = torch.sort(st["logits"], dim=1, descending=True, stable=True)[1][:, :k].cpu() if k else None
    for r in range(c["rows"]):
        x = st["logits"][r].long()
        M, S, W = int(x.max()), 0, 0
        xs = torch.nn.functional.pad(x, (0, -n % 1024), value=-(1 << 33)).view(-1, 1024)
        mb = xs.max(dim=1)[0]
        d = mb[:, None] - xs
        t = torch.where(d < (1 << 22) * 64, (d.clamp(max=1 << 28) * mant + half) >> shift, MOST).clamp(max=MOST)
        e = two[t % 65536] // (2 ** (t // 65536))
        for m_b, s_b, w_b in zip(mb.tolist(), e.sum(dim=1).tolist(), (e * t).sum(dim=1).tolist()):
            u = power(M - m_b, FAR)
            m = A[u % 65536 // 256] * F[u % 256] // 2 ** 32
            S += (s_b // 256 * m) // 2 ** (22 + u // 65536)
            W += ((w_b + u * s_b) // 2 ** 21 * (m // 256)) // 2 ** (22 + u // 65536)
        a = S.bit_length() - 1
        y = (S * 2 ** 31 >> a) - 2 ** 31
        i = y >> 21
        L = (a - 30) * 2 ** 24 + G[i] + ((G[i + 1] - G[i]) * (y % 2 ** 21) >> 21)
        nats = lambda t: ((t * 256 + L) * LN2 + 2 ** 30) // 2 ** 31  # noqa: E731
        lp = lambda v: -nats(power(M - v, 2 ** 31 - 1))  # noqa: E731
        out[0].append(lp(int(x[int(st["tokens"][r])])))
        out[1].append(nats((W << 18) // (S >> 3)))
        if k:
            top = order[r].tolist()
            vals = x[order[r].to(DEV)].tolist()
            out[2].append(top + [-1] * (k - len(top)))
            out[3].append([lp(v) for v in vals] + [-2 ** 31] * (k - len(top)))
    return tuple(torch.tensor(o, dtype=torch.int32) for o in (out if k else out[:2]))
