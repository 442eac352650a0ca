"""The int8 decoder for many sequences at once: KV caches in pages (8 bits, or quantised to 4), attention of chunks and
single tokens over them, and the greedy choice of a batch, over the C ABI (kt_hip_dec_*_paged, include/kt_hip.h).

The reference decodes one sequence from contiguous caches (crates/01-engine/kt-core/src/model.rs:290-353,
generate.rs:82-111); `DecoderModel` mirrors that. `PagedKV` holds one layer's pools and offers the operators on them;
`PagedDecoder` runs a DecoderModel's layers over them for a batch whose sequences come and go. With 8-bit pages every
sequence gets the integers that DecoderModel gives it alone. torch allocates the buffers, copies, and bounds token ids; it computes nothing else.
"""
from __future__ import annotations

import operator

import numpy as np

from . import backend as B

PAGES = (16, 32, 64, 128, 256)
MAX_POS = 524288  # KT_PAGED_MAX_POS


def page_bytes(page: int, hd: int, bits: int = 8) -> int:
    """Bytes of one kv head's part of a page in one pool."""
    n = B.lib().kt_hip_dec_page_bytes(page, hd, bits)
    if n == 0:
        raise ValueError(f"no page layout for page={page} hd={hd} bits={bits}: page in {PAGES}, hd 64 or 128, bits 8 or 4")
    return n


def _need(t, what: str, dtype, dev: int, shape) -> None:
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor of shape {tuple(shape)} on GPU {dev} is needed, not "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


class PagedBatch:
    """A ragged batch on the device: row_start (seqs + 1 int32), kv_len (seqs int32, the new rows counted) and table
    (seqs x max_pages int32, -1 where a sequence has no page); `tokens` new rows in all. The tensors are read when the
    kernels run, so a captured call follows what is copied into them."""

    def __init__(self, row_start, kv_len, table, tokens: int):
        import torch

        if not table.is_cuda:
            raise ValueError("PagedBatch: the tensors live on the GPU")
        if table.dim() != 2 or not 0 <= tokens <= 1 << 30:
            raise ValueError("PagedBatch: table is seqs x max_pages, tokens a count of rows")
        self.seqs, self.max_pages, self.tokens, self.dev = table.shape[0], table.shape[1], int(tokens), table.get_device()
        _need(table, "table", torch.int32, self.dev, table.shape)
        _need(row_start, "row_start", torch.int32, self.dev, (self.seqs + 1,))
        _need(kv_len, "kv_len", torch.int32, self.dev, (self.seqs,))
        self.row_start, self.kv_len, self.table = row_start, kv_len, table
        self.ptrs = (row_start.data_ptr(), kv_len.data_ptr(), table.data_ptr())


class PagedKV:
    """One layer's K and V pools: `pages` pages of `page` positions for `nkv` kv heads of `hd` values, in 8 or 4 bits. k
    and v (pages x nkv x page_bytes int8) are allocated as zeros unless given. Every call is asynchronous on `stream` (None:
    the null stream)."""

    def __init__(self, pages: int, page: int, nkv: int, hd: int, bits: int = 8, k=None, v=None, dev: int = 0):
        import torch

        part = page_bytes(page, hd, bits)
        if pages < 0 or nkv < 1:
            raise ValueError("PagedKV: pages >= 0 and nkv >= 1")
        self.pages, self.page, self.nkv, self.hd, self.bits, self.dev = pages, page, nkv, hd, bits, dev
        self.device = torch.device("cuda", dev)
        self._i8, self._i16, self._i32 = torch.int8, torch.int16, torch.int32
        shape = (pages, nkv, part)
        self.k = torch.zeros(shape, dtype=torch.int8, device=self.device) if k is None else k
        self.v = torch.zeros(shape, dtype=torch.int8, device=self.device) if v is None else v
        if k is None or v is None:  # zeros before any stream writes
            torch.cuda.current_stream(self.device).synchronize()
        _need(self.k, "k", torch.int8, dev, shape)
        _need(self.v, "v", torch.int8, dev, shape)
        self._pools = (self.k.data_ptr(), self.v.data_ptr(), pages, page, bits)  # as every call passes them

    def _batch(self, batch: PagedBatch) -> None:
        if batch.dev != self.dev:
            raise ValueError(f"the batch is on GPU {batch.dev}, the pools on GPU {self.dev}")
        if not 1 <= batch.max_pages <= MAX_POS // self.page:
            raise ValueError(f"a table of {batch.max_pages} pages of {self.page}: 1 to {MAX_POS} positions")

    def _rows(self, t, what: str, batch: PagedBatch, width: int) -> tuple[int, int]:
        """The address and stride of `t`, whose rows hold at least `width` int8 values for every row of the batch."""
        if t.dtype is not self._i8 or t.get_device() != self.dev or t.dim() != 2:
            raise ValueError(f"{what}: an int8 matrix on GPU {self.dev} is needed")
        (rows, cols), (stride, by), at = t.shape, t.stride(), t.data_ptr()
        if rows <= 1 and stride < cols:
            stride = cols
        if rows < batch.tokens or cols < width or (by != 1 and cols > 1) or stride < cols:
            raise ValueError(f"{what}: {tuple(t.shape)} with strides {t.stride()}: {batch.tokens} rows of {width} side by side")
        if stride % 16 or at % 16:
            raise ValueError(f"{what}: rows must start at multiples of 16 bytes")
        return at, stride

    def append(self, qkv, batch: PagedBatch, nh: int, cos, sin, q, stream=None) -> None:
        """The rows of qkv (q heads, k heads, v heads; read only): their rotated q heads to q, their rotated k and their v
        to the pages. cos / sin: int16 tables of max_pos x hd / 2 at 2^14."""
        self._batch(batch)
        hd, nkv = self.hd, self.nkv
        shape = cos.shape
        n = shape[0] if len(shape) == 2 and shape[1] == hd // 2 else -1
        _need(cos, "cos", self._i16, self.dev, shape if n >= 0 else (n, hd // 2))
        _need(sin, "sin", self._i16, self.dev, shape)
        at, stride = self._rows(qkv, "qkv", batch, (nh + 2 * nkv) * hd)
        to, q_stride = self._rows(q, "q", batch, nh * hd)
        B.check(B.lib().kt_hip_dec_rope_kv_paged(
            self.dev, at, batch.tokens, stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, nkv, hd, cos.data_ptr(),
            sin.data_ptr(), n, to, q_stride, *self._pools, B._stream(stream)), "dec rope + paged append")

    def read(self, batch: PagedBatch, k, v, stream=None) -> None:
        """Every sequence's positions as contiguous rows: k / v seqs x max_pos x nkv x hd int8, positions from
        min(kv_len, max_pos) on left as they are."""
        self._batch(batch)
        n = k.shape[1] if k.dim() == 4 else -1
        shape = (batch.seqs, n, self.nkv, self.hd)
        _need(k, "k", self._i8, self.dev, shape)
        _need(v, "v", self._i8, self.dev, shape)
        B.check(B.lib().kt_hip_dec_kv_read_paged(
            self.dev, *self._pools, batch.ptrs[1], batch.ptrs[2], batch.seqs, batch.max_pages, self.nkv, self.hd,
            k.data_ptr(), v.data_ptr(), n, B._stream(stream)), "dec paged read")

    def workspace_bytes(self, batch: PagedBatch, nh: int) -> int:
        """Scratch bytes of attend for `nh` q heads over this batch's shape (a smaller batch may need more)."""
        self._batch(batch)
        n = B.lib().kt_hip_dec_attention_paged_workspace(batch.tokens, batch.seqs, batch.max_pages, self.page, nh,
                                                         self.nkv, self.hd)
        if n == 0:
            raise ValueError(f"attend: {batch.tokens} rows, {batch.seqs} sequences, {nh} heads over {self.nkv} kv heads")
        return n

    def workspace(self, batch: PagedBatch, nh: int):
        """A workspace for attend; calls that may overlap need one each."""
        import torch

        return torch.empty(self.workspace_bytes(batch, nh), dtype=torch.int8, device=self.device)

    def attend(self, q, batch: PagedBatch, nh: int, exp_tab, o, ws, window: int = 0, sinks: int = 0,
               stream=None) -> None:
        """The rows' attention over their sequences' pages (after the append of the rows' own k and v), q and o rows of
        nh * hd. window >= 1: a row at p sees positions past p - window and the first `sinks`; 0: all up to its own."""
        self._batch(batch)
        _need(exp_tab, "exp_tab", self._i32, self.dev, (1024,))
        if ws.get_device() != self.dev or not ws.is_contiguous():
            raise ValueError(f"ws: a contiguous tensor on GPU {self.dev} is needed")
        at, q_stride = self._rows(q, "q", batch, nh * self.hd)
        to, o_stride = self._rows(o, "o", batch, nh * self.hd)
        B.check(B.lib().kt_hip_dec_attention_paged(
            self.dev, at, batch.tokens, q_stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, self.nkv, self.hd,
            exp_tab.data_ptr(), window, sinks, *self._pools, to, o_stride, ws.data_ptr(), ws.nbytes, B._stream(stream)),
            "dec paged attention")


class PagedDecoder:
    """A DecoderModel's layers over paged caches, for sequences that come and go. `model` gives the weights, scales and
    tables (its own caches and activations are not touched); `pages` pages of `page` positions serve every layer, and a
    pass takes at most max_rows new rows of at most max_seqs sequences.

        d = PagedDecoder(model, pages=4096)
        a, b = d.add(), d.add()
        tokens = d.run([(a, prompt_a), (b, prompt_b)])          # one pass, ragged: the next token of each
        tokens = d.run([(a, tokens[:1]), (b, tokens[1:])])      # a decode step of both
        d.release(a)
    """

    def __init__(self, model, pages: int, page: int = 16, bits: int = 8, max_seqs: int = 64, max_rows: int = 2048,
                 window: int = 0, sinks: int = 0):
        import torch

        if max_rows < 1 or not 1 <= max_seqs <= 65535 or window < 0 or sinks < 0:
            raise ValueError("PagedDecoder: max_rows >= 1, 1 <= max_seqs <= 65535, window >= 0, sinks >= 0")
        self.torch, self.m, self.dev, self.device = torch, model, model.dev, model.device
        self.page, self.bits, self.max_seqs, self.max_rows = page, bits, max_seqs, max_rows
        self.window, self.sinks = window, sinks
        self.kv = [PagedKV(pages, page, model.nkv, model.hd, bits, dev=model.dev) for _ in range(model.L)]
        self.max_pos = min(int(model.rope_cos.shape[0]), MAX_POS)
        self.max_pages = max(1, -(-self.max_pos // page))
        if not window:  # a sequence holds each of its positions; with a window it gives pages back as it goes
            self.max_pages = max(1, min(self.max_pages, pages))
        self.free = list(range(pages - 1, -1, -1))
        self.seq: dict[int, dict] = {}
        self._next = 0

        def zeros(*shape, dt=torch.int8):
            return torch.zeros(shape, dtype=dt, device=self.device)

        R, m = max_rows, model
        self.r, self.xn, self.h = zeros(R, m.d, dt=torch.int32), zeros(R, m.d), zeros(R, m.ffn)
        self.qkv, self.q, self.o = zeros(R, m.nq), zeros(R, m.nh * m.hd), zeros(R, m.nh * m.hd)
        self.r_last, self.x_last = zeros(max_seqs, m.d, dt=torch.int32), zeros(max_seqs, m.d)
        self.logits = zeros(max_seqs, m.V, dt=torch.int32)
        self._ws = []
        torch.cuda.current_stream(self.device).synchronize()  # the buffers are zeros before a pass on any stream

    # sequences -----------------------------------------------------------------------------------------------------

    def add(self) -> int:
        """A new, empty sequence."""
        s = self._next
        self._next += 1
        self.seq[s] = dict(len=0, pages=[], gone=-(-self.sinks // self.page))
        return s

    def release(self, s: int) -> None:
        """The sequence ends: its pages are free again."""
        self.free += [p for p in self.seq.pop(s)["pages"] if p >= 0]

    def length(self, s: int) -> int:
        return self.seq[s]["len"]

    def _reserve(self, lens: list) -> None:
        """Pages for sequence s up to new positions, all or none."""
        want = {s: -(-n // self.page) - len(self.seq[s]["pages"]) for s, n in lens}
        for s, n in lens:
            if n > self.max_pos or n > self.max_pages * self.page:
                raise ValueError(f"sequence {s}: {n} positions, {min(self.max_pos, self.max_pages * self.page)} at most")
        if sum(max(0, w) for w in want.values()) > len(self.free):
            raise ValueError(f"out of pages: {sum(max(0, w) for w in want.values())} needed, {len(self.free)} free")
        for s, w in want.items():
            self.seq[s]["pages"] += [self.free.pop() for _ in range(w)]

    def _trim(self, s: int) -> None:
        """Pages that the window has left behind, and no sink is in, are free again."""
        e = self.seq[s]
        gone = max(0, e["len"] + 1 - self.window) // self.page  # pages that no later row's window reaches
        for i in range(e["gone"], gone):
            self.free.append(e["pages"][i])
            e["pages"][i] = -1
        e["gone"] = max(e["gone"], gone)

    # a pass --------------------------------------------------------------------------------------------------------

    def batch(self, seqs: list, rows: list) -> PagedBatch:
        """The batch of `rows` new rows for each of `seqs`, whose positions are reserved."""
        torch = self.torch
        # as wide as the longest needs, to a power of two: the attention divides its work by the table's width
        need = max([1] + [len(self.seq[s]["pages"]) for s in seqs])
        table = np.full((len(seqs), min(self.max_pages, 1 << (need - 1).bit_length())), -1, dtype=np.int32)
        for i, s in enumerate(seqs):
            table[i, : len(self.seq[s]["pages"])] = self.seq[s]["pages"]
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        kv = np.array([self.seq[s]["len"] + n for s, n in zip(seqs, rows)], dtype=np.int32)
        put = lambda a: torch.from_numpy(a).to(self.device)  # noqa: E731
        return PagedBatch(put(start), put(kv), put(table), int(start[-1]))

    def run(self, work: list, stream=None):
        """One pass over (sequence, its new tokens) pairs: prompts, chunks of prompts and single tokens alike. Returns the
        greedy next token of each (int32, on the device); their logits are self.logits[: len(work)]. The tokens may be
        host integers, which are checked, or a tensor of the device, whose ids outside the vocabulary count as the nearest
        one inside. Asynchronous on `stream` (None: the null stream); other streams' work is the caller's to order."""
        torch = self.torch
        seqs = [s for s, _ in work]
        rows = [len(t) for _, t in work]
        if not work or len(set(seqs)) != len(seqs) or len(seqs) > self.max_seqs or any(s not in self.seq for s in seqs):
            raise ValueError("run: between 1 and max_seqs sequences, each known and named once")
        if min(rows) < 1 or sum(rows) > self.max_rows:
            raise ValueError(f"run: at least one token each, {self.max_rows} in all at most")
        ids = []  # of host tokens; a tensor of the device as it is
        for s, t in work:
            if torch.is_tensor(t) and (t.dim() != 1 or t.dtype not in (torch.int32, torch.int64)):
                raise ValueError(f"run: sequence {s}: tokens are a vector of int32 or int64")
            ids.append(t if self._on_gpu(t) else self._ids(t, f"run: sequence {s}"))
        self._reserve([(s, self.seq[s]["len"] + n) for s, n in zip(seqs, rows)])
        with torch.cuda.stream(self._torch_stream(stream)):
            b = self.batch(seqs, rows)
            toks = [t.clamp(0, self.m.V - 1).to(device=self.device, dtype=torch.int32) if self._on_gpu(t) else
                    torch.tensor(t, dtype=torch.int32, device=self.device) for t in ids]
            toks = torch.cat(toks) if len(toks) > 1 else toks[0].contiguous()
            last = None
            if b.tokens != b.seqs:
                last = (b.row_start[1:] - 1).long()
            out = torch.empty(b.seqs, dtype=torch.int32, device=self.device)
            self.forward(toks, b, last, out, stream)
        for s, n in zip(seqs, rows):
            self.seq[s]["len"] += n
            if self.window:
                self._trim(s)
        return out

    def _ids(self, t, what: str) -> list:
        """Host tokens as integers of the vocabulary."""
        try:
            ids = [operator.index(x) for x in t]
        except TypeError:
            raise ValueError(f"{what}: tokens are integers") from None
        if not all(0 <= x < self.m.V for x in ids):
            raise ValueError(f"{what} has a token outside the vocabulary")
        return ids

    def _on_gpu(self, t) -> bool:
        return self.torch.is_tensor(t) and t.is_cuda

    def _torch_stream(self, stream):
        torch = self.torch
        if stream is None or stream == 0:
            return torch.cuda.default_stream(self.device)
        return torch.cuda.ExternalStream(stream, device=self.device) if isinstance(stream, int) else stream

    def _workspaces(self, b: PagedBatch) -> tuple:
        """Scratch of the attention and of the choice. What a captured pass may hold is kept when a larger one is made."""
        n, top = self.kv[0].workspace_bytes(b, self.m.nh), B.dec_argmax_rows_workspace(b.seqs, self.m.V)
        n = -(-n // 256) * 256
        if not self._ws or self._ws[-1].numel() < n + top:
            size = max(n + top, 2 * self._ws[-1].numel() if self._ws else 1 << 16)
            self._ws.append(self.torch.empty(size, dtype=self.torch.int8, device=self.device))
        return self._ws[-1][:n], self._ws[-1][n:]

    def _check_pass(self, tokens_dev, b: PagedBatch, last, out) -> None:
        """What a pass reads and writes lies within its tensors and the decoder's buffers."""
        if b.dev != self.dev or not 1 <= b.tokens <= self.max_rows or not 1 <= b.seqs <= self.max_seqs:
            raise ValueError(f"forward: a batch on GPU {self.dev} of 1 to {self.max_rows} rows and 1 to {self.max_seqs} sequences "
                             f"is needed, not {b.tokens} rows of {b.seqs} on GPU {b.dev}")
        i32 = self.torch.int32
        for t, what, n in ((tokens_dev, "tokens", b.tokens), (out, "out", b.seqs)):
            if t.dtype is not i32 or t.get_device() != self.dev or t.numel() < n or not t.is_contiguous():
                raise ValueError(f"forward: {what}: a contiguous tensor of at least {n} int32 on GPU {self.dev} is needed, not "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        if last is None:
            if b.tokens < b.seqs:  # (rows behind the sequences' are a padded batch's)
                raise ValueError(f"forward: {b.tokens} rows of {b.seqs} sequences need the indexes of the last rows")
        elif last.dtype not in (i32, self.torch.int64) or last.get_device() != self.dev or last.shape != (b.seqs,):
            raise ValueError(f"forward: last: {b.seqs} int32 or int64 on GPU {self.dev} are needed, not {tuple(last.shape)} "
                             f"{last.dtype} on {last.device}")

    def forward(self, tokens_dev, b: PagedBatch, last, out, stream=None) -> None:
        """The layers over the batch's rows, whose ids (tokens_dev, int32) are within the vocabulary; the logits of each
        sequence's last row (`last`: their indexes among the rows, None where every sequence has one row) to self.logits, the
        greedy choice of each to out (int32). Asynchronous on `stream`, which torch's current stream has to be; capturable
        after a call of the batch's shape. Passes of one decoder, captured or not, share its buffers: they follow one
        another."""
        self._check_pass(tokens_dev, b, last, out)
        m, lib, dev, s, P = self.m, B.lib(), self.dev, B._stream(stream), B._ptr
        T, d, ffn, nh, hd, nq = b.tokens, m.d, m.ffn, m.nh, m.hd, m.nq
        ws, ws_top = self._workspaces(b)
        B.check(lib.kt_hip_dec_embed(dev, P(tokens_dev), T, P(m.emb16), d, P(self.r), s), "dec embed")
        fuse = m.fuse_norm and T <= B.NORM_MAX_M
        for l in range(m.L):
            if fuse:
                m._gemm_norm("qkv", l, self.r, T, nq, d, self.qkv, B.OUT_I8, s)
            else:
                B.check(lib.kt_hip_dec_rmsnorm(dev, P(self.r), T, d, P(self.xn), d, s), "dec rmsnorm")
                m._gemm("qkv", l, self.xn, T, nq, d, self.qkv, B.OUT_I8, s)
            self.kv[l].append(self.qkv, b, nh, m.rope_cos, m.rope_sin, self.q, stream)
            self.kv[l].attend(self.q, b, nh, m.exp_tab, self.o, ws, self.window, self.sinks, stream)
            m._gemm("o", l, self.o, T, d, nh * hd, self.r, B.OUT_I32_ADD, s)
            lo, nib, mant, shift = m._layer_ptrs("gu", l, 2 * ffn)
            if fuse:
                B.check(lib.kt_hip_w12_swiglu_norm(dev, P(self.r), lo, nib, T, ffn, d, mant, shift, P(m.silu), m.h_shift,
                                                   P(self.h), ffn, s), "dec gate/up")
            else:
                B.check(lib.kt_hip_dec_rmsnorm(dev, P(self.r), T, d, P(self.xn), d, s), "dec rmsnorm")
                B.check(lib.kt_hip_w12_swiglu(dev, P(self.xn), lo, nib, T, ffn, d, mant, shift, P(m.silu), m.h_shift,
                                              P(self.h), ffn, s), "dec gate/up")
            m._gemm("dn", l, self.h, T, d, ffn, self.r, B.OUT_I32_ADD, s)
        r = self.r
        if last is not None:
            self.torch.index_select(self.r, 0, last, out=self.r_last[: b.seqs])
            r = self.r_last
        B.check(lib.kt_hip_dec_rmsnorm(dev, P(r), b.seqs, d, P(self.x_last), d, s), "dec rmsnorm")
        m._gemm("emb", 0, self.x_last, b.seqs, m.V, d, self.logits, B.OUT_I32, s)
        B.dec_argmax_rows(self.logits, b.seqs, m.V, out, ws_top, stream=stream, dev=dev)

    def read(self, s: int, layer: int, max_pos: int | None = None, stream=None):
        """Sequence s's K and V of a layer as contiguous rows (max_pos x nkv x hd int8, zeros past its length and where a window
        has left pages behind): the caches that DecoderModel continues from. On `stream`, as the passes are."""
        torch = self.torch
        n = self.seq[s]["len"] if max_pos is None else max_pos
        with torch.cuda.stream(self._torch_stream(stream)):
            k, v = (torch.zeros(1, n, self.m.nkv, self.m.hd, dtype=torch.int8, device=self.device) for _ in range(2))
            self.kv[layer].read(self.batch([s], [0]), k, v, stream)
        return k[0], v[0]

    def generate(self, prompts: list, max_new: int, chunk: int | None = None) -> np.ndarray:
        """generate_greedy_by (crates/01-engine/kt-core/src/generate.rs:82-111) for a batch of prompts with no stop
        tokens: max_new tokens each (len(prompts) x max_new). Prompts go in passes of at most `chunk` rows (max_rows by
        default), shared by as many sequences as fit; a step of more sequences than max_rows takes several passes."""
        chunk = self.max_rows if chunk is None else min(chunk, self.max_rows)
        if max_new < 1 or chunk < 1 or len(prompts) > self.max_seqs or any(len(p) < 1 for p in prompts):
            raise ValueError("generate: at least one token to make, no empty prompt, max_seqs prompts at most")
        todo = [(i, self._ids(p, f"generate: prompt {i}")) for i, p in enumerate(prompts)]
        out = np.zeros((len(prompts), max_new), dtype=np.int32)

        def choose(work):
            t = self.run(work)
            with self.torch.cuda.stream(self._torch_stream(None)):  # the passes' stream, whatever torch's current one is
                return t.cpu().numpy()

        ids = [self.add() for _ in prompts]
        try:
            while todo:
                room, work, left = chunk, [], []
                for i, p in todo:
                    n = min(room, len(p))
                    if n:
                        work.append((i, p[:n], n == len(p)))
                    if n < len(p):
                        left.append((i, p[n:]))
                    room -= n
                t = choose([(ids[i], p) for i, p, _ in work])
                for (i, _, done), x in zip(work, t):
                    if done:
                        out[i, 0] = x
                todo = left
            for step in range(1, max_new):
                for at in range(0, len(ids), self.max_rows):
                    now = range(at, min(at + self.max_rows, len(ids)))
                    out[now.start:now.stop, step] = choose([(ids[i], out[i, step - 1:step]) for i in now])
        finally:
            for s in ids:
                self.release(s)
        return out
