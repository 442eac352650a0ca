"""The int8 decoder for many sequences at once: KV caches in pages (8 bits, or quantised to 4), attention of chunks and
single tokens over them, the greedy choice of a batch and its log probabilities, head norms, and sequences cut down to the
positions that attention looks at, over the C ABI (kt_hip_dec_*_paged, kt_hip_dec_*_rows, include/kt_hip.h).

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


def _torch_stream(stream, device):
    """torch's name for `stream` (None: the null stream)."""
    import torch

    if stream is None or stream == 0:
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream


class PagedBatch:
    """A ragged batch on the device: row_start (seqs + 1 int32), kv_len (seqs int32, the new rows counted) and table
    (seqs x max_pages int32, -1 where a sequence has no page); `tokens` new rows in all. shift (seqs int32, or None: zeros):
    how far each sequence's rotations are ahead of its positions, where it has been cut down. The tensors are read when the
    kernels run, so a captured call follows what is copied into them."""

    def __init__(self, row_start, kv_len, table, tokens: int, shift=None):
        import torch

        if not table.is_cuda:
            raise ValueError("PagedBatch: the tensors live on the GPU")
        if table.dim() != 2 or not 0 <= tokens <= 1 << 30:
            raise ValueError("PagedBatch: table is seqs x max_pages, tokens a count of rows")
        self.seqs, self.max_pages, self.tokens, self.dev = table.shape[0], table.shape[1], int(tokens), table.get_device()
        _need(table, "table", torch.int32, self.dev, table.shape)
        _need(row_start, "row_start", torch.int32, self.dev, (self.seqs + 1,))
        _need(kv_len, "kv_len", torch.int32, self.dev, (self.seqs,))
        if shift is not None:
            _need(shift, "shift", torch.int32, self.dev, (self.seqs,))
        self.row_start, self.kv_len, self.table, self.shift = row_start, kv_len, table, shift
        self.ptrs = (row_start.data_ptr(), kv_len.data_ptr(), table.data_ptr())


class PagedKV:
    """One layer's K and V pools: `pages` pages of `page` positions for `nkv` kv heads of `hd` values, in 8 or 4 bits. k
    and v (pages x nkv x page_bytes int8) are allocated as zeros unless given; w (pages x nkv x page int64), the slots' accumulated
    attention weights, if given or, as zeros, with `weights`. Every call is asynchronous on `stream` (None: the null stream)."""

    def __init__(self, pages: int, page: int, nkv: int, hd: int, bits: int = 8, k=None, v=None, dev: int = 0, w=None,
                 weights: bool = False):
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
        self.w = torch.zeros((pages, nkv, page), dtype=torch.int64, device=self.device) if w is None and weights else w
        if k is None or v is None or (w is None and weights):  # zeros before any stream writes
            torch.cuda.current_stream(self.device).synchronize()
        _need(self.k, "k", torch.int8, dev, shape)
        _need(self.v, "v", torch.int8, dev, shape)
        if self.w is not None:
            _need(self.w, "w", torch.int64, dev, (pages, nkv, page))
            self._no_ws = torch.empty(256, dtype=torch.int8, device=self.device)  # of calls that need none
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

    def append(self, qkv, batch: PagedBatch, nh: int, cos, sin, q, stream=None, q_norm=None, k_norm=None, shift=None) -> None:
        """The rows of qkv (q heads, k heads, v heads; read only): their rotated q heads to q, their rotated k and their v
        to the pages. cos / sin: int16 tables of max_pos x hd / 2 at 2^14. q_norm / k_norm (hd int16 at 2^12): the heads are brought
        to a root mean square of 1 (32 codes) and weighted before the rotation. shift (seqs int32; None: the batch's): added to
        the positions that the tables are read at. The accumulated weights of the written slots, if there are any, become 0."""
        self._batch(batch)
        hd, nkv = self.hd, self.nkv
        shape = cos.shape
        n = shape[0] if len(shape) == 2 and shape[1] == hd // 2 else -1
        _need(cos, "cos", self._i16, self.dev, shape if n >= 0 else (n, hd // 2))
        _need(sin, "sin", self._i16, self.dev, shape)
        at, stride = self._rows(qkv, "qkv", batch, (nh + 2 * nkv) * hd)
        to, q_stride = self._rows(q, "q", batch, nh * hd)
        if shift is None:
            shift = batch.shift
        if q_norm is None and k_norm is None and shift is None and self.w is None:
            B.check(B.lib().kt_hip_dec_rope_kv_paged(
                self.dev, at, batch.tokens, stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, nkv, hd, cos.data_ptr(),
                sin.data_ptr(), n, to, q_stride, *self._pools, B._stream(stream)), "dec rope + paged append")
            return
        qn = kn = ahead = 0
        if q_norm is not None:
            _need(q_norm, "q_norm", self._i16, self.dev, (hd,))
            qn = q_norm.data_ptr()
        if k_norm is not None:
            _need(k_norm, "k_norm", self._i16, self.dev, (hd,))
            kn = k_norm.data_ptr()
        if shift is not None:
            if shift is not batch.shift:  # (which was looked at)
                _need(shift, "shift", self._i32, self.dev, (batch.seqs,))
            ahead = shift.data_ptr()
        k, v, pages, page, bits = self._pools
        B.check(B.lib().kt_hip_dec_norm_rope_kv_paged(
            self.dev, at, batch.tokens, stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, nkv, hd, cos.data_ptr(),
            sin.data_ptr(), n, qn, kn, ahead, to, q_stride, k, v, 0 if self.w is None else self.w.data_ptr(), pages, page, bits,
            B._stream(stream)), "dec norm + rope + paged append")

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
               stream=None, stats=None) -> None:
        """The rows' attention over their sequences' pages (after the append of the rows' own k and v), q and o rows of
        nh * hd. window >= 1: a row at p sees positions past p - window and the first `sinks`; 0: all up to its own. stats
        (tokens x nh x 2 int32, or None) takes each row's and head's largest score and the reciprocal of its weights' sum, which
        weigh needs."""
        self._batch(batch)
        _need(exp_tab, "exp_tab", self._i32, self.dev, (1024,))
        if ws.get_device() != self.dev or not ws.is_contiguous():
            raise ValueError(f"ws: a contiguous tensor on GPU {self.dev} is needed")
        at, q_stride = self._rows(q, "q", batch, nh * self.hd)
        to, o_stride = self._rows(o, "o", batch, nh * self.hd)
        args = (self.dev, at, batch.tokens, q_stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, self.nkv, self.hd,
                exp_tab.data_ptr(), window, sinks, *self._pools, to, o_stride)
        if stats is None:
            B.check(B.lib().kt_hip_dec_attention_paged(*args, ws.data_ptr(), ws.nbytes, B._stream(stream)), "dec paged attention")
            return
        _need(stats, "stats", self._i32, self.dev, (batch.tokens, nh, 2))
        B.check(B.lib().kt_hip_dec_attention_paged_stats(*args, stats.data_ptr(), ws.data_ptr(), ws.nbytes, B._stream(stream)),
                "dec paged attention with its statistics")

    def weigh(self, q, batch: PagedBatch, nh: int, exp_tab, stats, window: int = 0, sinks: int = 0, fresh: bool = False,
              stream=None) -> None:
        """Each position's share of the rows' attention, per kv head, added to w: 2^40 for a head's whole weight. q, exp_tab, window and
        sinks as attend took them, stats as it left them. fresh: the sums of the batch's sequences start from 0."""
        self._batch(batch)
        if self.w is None:
            raise ValueError("weigh: the pools were made without accumulated weights")
        _need(exp_tab, "exp_tab", self._i32, self.dev, (1024,))
        _need(stats, "stats", self._i32, self.dev, (batch.tokens, nh, 2))
        at, q_stride = self._rows(q, "q", batch, nh * self.hd)
        k, _, pages, page, bits = self._pools
        B.check(B.lib().kt_hip_dec_weigh_paged(
            self.dev, at, batch.tokens, q_stride, *batch.ptrs, batch.seqs, batch.max_pages, nh, self.nkv, self.hd,
            exp_tab.data_ptr(), window, sinks, stats.data_ptr(), int(fresh), k, self.w.data_ptr(), pages, page, bits,
            B._stream(stream)), "dec paged weigh")

    def evict_workspace_bytes(self, batch: PagedBatch) -> int:
        """Scratch bytes of evict for this batch's shape; 256 where it needs none."""
        self._batch(batch)
        n = B.lib().kt_hip_dec_evict_paged_workspace(batch.seqs, batch.max_pages, self.page, self.nkv)
        if n == 0:
            raise ValueError(f"evict: {batch.seqs} sequences")
        return n

    def evict(self, batch: PagedBatch, to, budget: int, kept, recent: int = 0, sinks: int = 0, stream=None, ws=None) -> None:
        """The batch's sequences cut down to at most `budget` positions, each kv head by itself: the first `sinks`, the last `recent`
        and, of the others, those with the largest w (ties: the lower position). They move, in order, to the pages `to`
        (seqs x ceil(budget / page) int32: pages of no table, each once); kept (seqs x nkv x budget int32) says which they
        were, -1 past the last. The caller takes `to` for the tables, min(kv_len, budget) for the lengths, and adds what went to the shifts;
        the old pages are free. ws: scratch of evict_workspace_bytes, one for each call that may overlap; None: of the call's own, from torch's
        allocator for `stream`."""
        n = self.evict_workspace_bytes(batch)
        if self.w is None:
            raise ValueError("evict: the pools were made without accumulated weights")
        if not 1 <= budget <= MAX_POS:
            raise ValueError(f"evict: a budget of {budget}: 1 to {MAX_POS} positions")
        _need(to, "to", self._i32, self.dev, (batch.seqs, -(-budget // self.page)))
        _need(kept, "kept", self._i32, self.dev, (batch.seqs, self.nkv, budget))
        if ws is None:
            ws = self._no_ws if n <= 256 else self._scratch(n, stream)
        elif ws.get_device() != self.dev or not ws.is_contiguous():
            raise ValueError(f"ws: a contiguous tensor on GPU {self.dev} is needed")
        k, v, pages, page, bits = self._pools
        B.check(B.lib().kt_hip_dec_evict_paged(
            self.dev, batch.ptrs[1], batch.ptrs[2], batch.seqs, batch.max_pages, self.nkv, self.hd, to.data_ptr(), budget, recent,
            sinks, kept.data_ptr(), k, v, self.w.data_ptr(), pages, page, bits, ws.data_ptr(), ws.nbytes, B._stream(stream)),
            "dec paged evict")

    def _scratch(self, n: int, stream):
        """n bytes that are this stream's until what it has been given is done."""
        import torch

        if torch.cuda.current_stream(self.device).cuda_stream == B._stream(stream):  # (the context below is 15 us)
            return torch.empty(n, dtype=torch.int8, device=self.device)
        with torch.cuda.stream(_torch_stream(stream, self.device)):
            return torch.empty(n, dtype=torch.int8, device=self.device)


class PagedDecoder:
    """A DecoderModel's layers over paged caches, for sequences that come and go. `model` gives the weights, scales and
    tables (its own caches and activations are not touched); `pages` pages of `page` positions serve every layer, and a
    pass takes at most max_rows new rows of at most max_seqs sequences.

        d = PagedDecoder(model, pages=4096)
        a, b = d.add(), d.add()
        tokens = d.run([(a, prompt_a), (b, prompt_b)])          # one pass, ragged: the next token of each
        tokens = d.run([(a, tokens[:1]), (b, tokens[1:])])      # a decode step of both
        lp, entropy, ids, lps = d.logprobs(tokens, unit, k=5)   # of these two, among the likeliest five
        d.release(a)

    q_norm / k_norm (layers x hd int16 at 2^12): the model norms its q and k heads before the rotation. budget >= 1: a sequence that holds
    more than `most` positions (budget + half of it by default) after a pass is cut down to `budget` of them, in every layer and kv head the
    first `sinks`, the last `recent` (budget // 2 by default, as far as the sinks leave room) and those that the rows so far have attended to
    most. The pages for one such cut are set aside.
    """

    def __init__(self, model, pages: int, page: int = 16, bits: int = 8, max_seqs: int = 64, max_rows: int = 2048,
                 window: int = 0, sinks: int = 0, q_norm=None, k_norm=None, budget: int = 0, recent: int | None = None,
                 most: int | None = None):
        import torch

        if max_rows < 1 or not 1 <= max_seqs <= 65535 or window < 0 or sinks < 0:
            raise ValueError("PagedDecoder: max_rows >= 1, 1 <= max_seqs <= 65535, window >= 0, sinks >= 0")
        recent = min(budget // 2, max(0, budget - sinks)) if recent is None else recent
        most = budget + budget // 2 if most is None else most
        if budget and (not 1 <= budget <= MAX_POS or window or recent < 0 or sinks + recent > budget or most < budget):
            raise ValueError(f"PagedDecoder: a budget of {budget} positions (1 to {MAX_POS}) needs no window, sinks + recent within "
                             f"it (not {sinks} + {recent}) and most not below it (not {most})")
        if budget and min(int(model.rope_cos.shape[0]), MAX_POS) * (model.nh // model.nkv) >= 1 << 23:
            raise ValueError(f"PagedDecoder: a budget: {model.rope_cos.shape[0]} positions of {model.nh // model.nkv} q heads to a kv head may "
                             "put more weight on one position than its sum holds, that of 2^23 heads")
        spare = -(-budget // page)
        if budget and pages < spare:
            raise ValueError(f"PagedDecoder: {pages} pages, {spare} of them set aside to cut a sequence to {budget} positions")
        self.torch, self.m, self.dev, self.device = torch, model, model.dev, model.device
        self.page, self.bits, self.max_seqs, self.max_rows = page, bits, max_seqs, max_rows
        self.window, self.sinks, self.budget, self.recent, self.most = window, sinks, budget, recent, most
        self.kv = [PagedKV(pages, page, model.nkv, model.hd, bits, dev=model.dev, weights=budget > 0) for _ in range(model.L)]
        self.q_norm, self.k_norm = (self._norms(t, what) for t, what in ((q_norm, "q_norm"), (k_norm, "k_norm")))
        self.max_pos = min(int(model.rope_cos.shape[0]), MAX_POS)
        self.max_pages = max(1, -(-self.max_pos // page))
        if not window:  # a sequence holds each of its positions; with a window it gives pages back as it goes
            self.max_pages = max(1, min(self.max_pages, pages))
        self.free = list(range(pages - 1, -1, -1))
        self.spare = [self.free.pop() for _ in range(spare)] if budget else []
        self.seq: dict[int, dict] = {}
        self._next = 0

        def zeros(*shape, dt=torch.int8):
            return torch.zeros(shape, dtype=dt, device=self.device)

        R, m = max_rows, model
        self.r, self.xn, self.h = zeros(R, m.d, dt=torch.int32), zeros(R, m.d), zeros(R, m.ffn)
        self.qkv, self.q, self.o = zeros(R, m.nq), zeros(R, m.nh * m.hd), zeros(R, m.nh * m.hd)
        self.r_last, self.x_last = zeros(max_seqs, m.d, dt=torch.int32), zeros(max_seqs, m.d)
        self.logits = zeros(max_seqs, m.V, dt=torch.int32)
        self.stats = zeros(R, m.nh, 2, dt=torch.int32) if budget else None
        self._ws = []
        torch.cuda.current_stream(self.device).synchronize()  # the buffers are zeros before a pass on any stream

    def _norms(self, t, what: str):
        """The layers' weights on the device, or None."""
        if t is None:
            return None
        t = self.torch.as_tensor(t)
        if t.dtype is not self.torch.int16 or t.shape != (self.m.L, self.m.hd):
            raise ValueError(f"PagedDecoder: {what}: {self.m.L} x {self.m.hd} int16 are needed, not {tuple(t.shape)} {t.dtype}")
        return t.to(self.device).contiguous().clone()

    # sequences -----------------------------------------------------------------------------------------------------

    def add(self) -> int:
        """A new, empty sequence."""
        s = self._next
        self._next += 1
        self.seq[s] = dict(len=0, cut=0, pages=[], gone=-(-self.sinks // self.page))
        return s

    def release(self, s: int) -> None:
        """The sequence ends: its pages are free again."""
        self.free += [p for p in self.seq.pop(s)["pages"] if p >= 0]

    def length(self, s: int) -> int:
        return self.seq[s]["len"]

    def held(self, s: int) -> int:
        """The positions of s that its pages hold: all, but for those that a budget has cut (a window's are counted)."""
        return self.seq[s]["len"] - self.seq[s]["cut"]

    def _reserve(self, lens: list) -> None:
        """Pages for sequence s up to new positions, all or none."""
        want = {s: -(-(n - self.seq[s]["cut"]) // self.page) - len(self.seq[s]["pages"]) for s, n in lens}
        for s, n in lens:
            if n > self.max_pos or n - self.seq[s]["cut"] > self.max_pages * self.page:
                raise ValueError(f"sequence {s}: {n} positions, {self.seq[s]['cut']} of them cut: {self.max_pos} at most, "
                                 f"{self.max_pages * self.page} held")
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

    def _cut(self, seqs: list, stream) -> None:
        """Those of `seqs` that hold more than `most` positions cut down to the budget, as many at a time as there are pages for. After
        the pass, on its stream (torch's current one)."""
        torch = self.torch
        seqs, need = [s for s in seqs if self.held(s) > self.most], len(self.spare)
        while seqs:
            n = min(len(seqs), 1 + len(self.free) // need, ((1 << 24) - 1) // -(-self.budget // 16))
            now, seqs = seqs[:n], seqs[n:]
            more = (n - 1) * need  # from the list's end, and off it once all layers have been cut
            pages = self.spare + self.free[-1:-1 - more:-1]
            to = torch.tensor(pages, dtype=torch.int32).reshape(n, need).to(self.device)
            b = self.batch(now, [0] * n)
            kept = torch.empty(n, self.m.nkv, self.budget, dtype=torch.int32, device=self.device)
            for kv in self.kv:
                kv.evict(b, to, self.budget, kept, self.recent, self.sinks, stream)
            del self.free[len(self.free) - more:]
            for i, s in enumerate(now):
                e = self.seq[s]
                self.free += e["pages"]
                e["pages"], e["cut"] = pages[i * need:(i + 1) * need], e["len"] - self.budget
            self.spare = [self.free.pop() for _ in range(need)]

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
        kv = np.array([self.held(s) + n for s, n in zip(seqs, rows)], dtype=np.int32)
        put = lambda a: torch.from_numpy(a).to(self.device)  # noqa: E731
        shift = put(np.array([self.seq[s]["cut"] for s in seqs], dtype=np.int32)) if self.budget else None
        return PagedBatch(put(start), put(kv), put(table), int(start[-1]), shift)

    def run(self, work: list, stream=None):
        """One pass over (sequence, its new tokens) pairs: prompts, chunks of prompts and single tokens alike. Returns the
        greedy next token of each (int32, on the device); their logits are self.logits[: len(work)]. The tokens may be
        host integers, which are checked, or a tensor of the device, whose ids outside the vocabulary count as the nearest
        one inside. Asynchronous on `stream` (None: the null stream); other streams' work is the caller's to order."""
        seqs, rows, ids = self._work(work)
        with self.torch.cuda.stream(self._torch_stream(stream)):
            b, toks = self._tokens(seqs, rows, ids)
            last = None
            if b.tokens != b.seqs:
                last = (b.row_start[1:] - 1).long()
            out = self.torch.empty(b.seqs, dtype=self.torch.int32, device=self.device)
            self.forward(toks, b, last, out, stream)
            self._advance(seqs, rows, stream)
        return out

    def _work(self, work: list) -> tuple:
        """The sequences of a pass, their rows, and their tokens checked; their positions are reserved."""
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
        return seqs, rows, ids

    def _tokens(self, seqs: list, rows: list, ids: list) -> tuple:
        """The batch and its tokens on the device."""
        torch = self.torch
        b = self.batch(seqs, rows)
        toks = [t.clamp(0, self.m.V - 1).to(device=self.device, dtype=torch.int32) if self._on_gpu(t) else
                torch.tensor(t, dtype=torch.int32, device=self.device) for t in ids]
        return b, torch.cat(toks) if len(toks) > 1 else toks[0].contiguous()

    def _advance(self, seqs: list, rows: list, stream) -> None:
        """The sequences after a pass: what a window or a budget leaves of them."""
        for s, n in zip(seqs, rows):
            self.seq[s]["len"] += n
            if self.window:
                self._trim(s)
        if self.budget:
            self._cut(seqs, stream)

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
        return _torch_stream(stream, self.device)

    def _workspaces(self, b: PagedBatch) -> tuple:
        """Scratch of the attention and of the choice. What a captured pass may hold is kept when a larger one is made."""
        n, top = self.kv[0].workspace_bytes(b, self.m.nh), B.dec_argmax_rows_workspace(b.seqs, self.m.V)
        n = -(-n // 256) * 256
        if not self._ws or self._ws[-1].numel() < n + top:
            size = max(n + top, 2 * self._ws[-1].numel() if self._ws else 1 << 16)
            self._ws.append(self.torch.empty(size, dtype=self.torch.int8, device=self.device))
        return self._ws[-1][:n], self._ws[-1][n:]

    def reserve_scratch(self, b: PagedBatch) -> None:
        """Scratch for `forward` of batches of b's shape (rows, sequences, table width), so that the pass can be captured. Nothing runs
        and nothing of the decoder changes. On the stream of the passes, which torch's current one has to be, before the capture."""
        self._check_batch(b, "reserve_scratch")
        self._workspaces(b)

    def _check_batch(self, b: PagedBatch, what: str) -> None:
        if b.dev != self.dev or not 1 <= b.tokens <= self.max_rows or not 1 <= b.seqs <= self.max_seqs:
            raise ValueError(f"{what}: a batch on GPU {self.dev} of 1 to {self.max_rows} rows and 1 to {self.max_seqs} sequences "
                             f"is needed, not {b.tokens} rows of {b.seqs} on GPU {b.dev}")

    def _check_pass(self, tokens_dev, b: PagedBatch, last, out) -> None:
        """What a pass reads and writes lies within its tensors and the decoder's buffers."""
        self._check_batch(b, "forward")
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
        after reserve_scratch of the batch's shape. Passes of one decoder, captured or not, share its buffers: they follow one
        another. Under a budget the batch has its sequences' shifts, as `batch` gives them, and no sequence is cut. Each pass then adds
        the weights that its rows attend with to those held: the same rows passed twice (a trial before a capture, say) count
        twice in the cuts that follow, where without a budget the second pass leaves everything as the first did."""
        self._check_pass(tokens_dev, b, last, out)
        vocab = self.m.V
        if self.budget and b.shift is None:
            raise ValueError("forward: a decoder with a budget needs the batch's shifts")
        self._layers(tokens_dev, b, stream)
        r = self.r
        if last is not None:
            self.torch.index_select(self.r, 0, last, out=self.r_last[: b.seqs])
            r = self.r_last
        self._head(r, b.seqs, stream)
        B.dec_argmax_rows(self.logits, b.seqs, vocab, out, self._workspaces(b)[1], stream=stream, dev=self.dev)

    def _layers(self, tokens_dev, b: PagedBatch, stream) -> None:
        """The layers over the batch's rows: their residual to self.r."""
        m, lib, dev, s, P = self.m, B.lib(), self.dev, B._stream(stream), B._ptr
        T, d, ffn, nh, hd, nq = b.tokens, m.d, m.ffn, m.nh, m.hd, m.nq
        ws, _ = self._workspaces(b)
        stats = self.stats[:T] if self.budget else None
        B.check(lib.kt_hip_dec_embed(dev, P(tokens_dev), T, P(m.emb16), d, P(self.r), s), "dec embed")
        fuse = m.fuse_norm and T <= B.NORM_MAX_M
        for l in range(m.L):
            if fuse:
                m._gemm_norm("qkv", l, self.r, T, nq, d, self.qkv, B.OUT_I8, s)
            else:
                B.check(lib.kt_hip_dec_rmsnorm(dev, P(self.r), T, d, P(self.xn), d, s), "dec rmsnorm")
                m._gemm("qkv", l, self.xn, T, nq, d, self.qkv, B.OUT_I8, s)
            norms = {} if self.q_norm is None else dict(q_norm=self.q_norm[l])
            if self.k_norm is not None:
                norms["k_norm"] = self.k_norm[l]
            self.kv[l].append(self.qkv, b, nh, m.rope_cos, m.rope_sin, self.q, stream, **norms)
            if self.budget:  # (sinks are what a cut leaves here, not a window's)
                self.kv[l].attend(self.q, b, nh, m.exp_tab, self.o, ws, 0, 0, stream, stats=stats)
                self.kv[l].weigh(self.q, b, nh, m.exp_tab, stats, stream=stream)
            else:
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

    def _head(self, r, rows: int, stream) -> None:
        """The logits of the first `rows` rows (at most max_seqs) of the residual r to self.logits."""
        m, s, P = self.m, B._stream(stream), B._ptr
        B.check(B.lib().kt_hip_dec_rmsnorm(self.dev, P(r), rows, m.d, P(self.x_last), m.d, s), "dec rmsnorm")
        m._gemm("emb", 0, self.x_last, rows, m.V, m.d, self.logits, B.OUT_I32, s)

    def logprobs(self, tokens, unit: float, k: int = 0, stream=None):
        """Of the rows that the last pass left in self.logits, the log probability of tokens[r] in row r (int32 on the device, one for
        each sequence of the pass, in its order), the entropy, and the k likeliest tokens with theirs (None where k is 0), in
        2^-16 of a natural unit, which is `unit` codes of a logit. On `stream`, as the pass was."""
        torch = self.torch
        n = tokens.numel()
        if tokens.dtype is not torch.int32 or tokens.get_device() != self.dev or not tokens.is_contiguous() or n > self.max_seqs:
            raise ValueError(f"logprobs: a contiguous tensor of at most {self.max_seqs} int32 on GPU {self.dev} is needed, not "
                             f"{tuple(tokens.shape)} {tokens.dtype} on {tokens.device}")
        with torch.cuda.stream(self._torch_stream(stream)):
            i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=self.device)  # noqa: E731
            out = (i32(n), i32(n), *((i32(n, k), i32(n, k)) if k else (None, None)))
            ws = torch.empty(B.dec_logprobs_rows_workspace(n, self.m.V, k), dtype=torch.int8, device=self.device)
            B.dec_logprobs_rows(self.logits, n, self.m.V, tokens, B.logit_scale(unit), out[0], ws, *out[1:], k, stream=stream,
                                dev=self.dev)
        return out

    def score(self, work: list, unit: float, k: int = 0, stream=None):
        """One pass over (sequence, its new tokens) pairs, as run's, for the log probabilities of the tokens themselves: row i of a
        sequence's tokens gives that of its token i + 1, the last row the entropy and alternatives alone (its log probability is that
        of no token: -2^31). Returns, for each pair, what logprobs does, one row a token. The logits are made max_seqs rows at a time (1021
        tokens of the Qwen2.5-0.5B shape: 3.5 ms with 256, 4.8 with 64, 42 with 1)."""
        torch = self.torch
        B.logit_scale(unit), B.dec_logprobs_rows_workspace(self.max_seqs, self.m.V, k)  # refused before anything is reserved
        seqs, rows, ids = self._work(work)
        with torch.cuda.stream(self._torch_stream(stream)):
            b, toks = self._tokens(seqs, rows, ids)
            self._layers(toks, b, stream)
            want = torch.full_like(toks, -1)
            want[:-1] = toks[1:]
            want[(b.row_start[1:] - 1).long()] = -1
            got = []
            for at in range(0, b.tokens, self.max_seqs):
                n = min(self.max_seqs, b.tokens - at)
                self._head(self.r[at:at + n], n, stream)
                got.append(self.logprobs(want[at:at + n], unit, k, stream))
            got = [torch.cat(t) if t[0] is not None else None for t in zip(*got)]
            self._advance(seqs, rows, stream)
        parts = [t.split(rows) if t is not None else [None] * len(rows) for t in got]
        return list(zip(*parts))

    def read(self, s: int, layer: int, max_pos: int | None = None, stream=None):
        """Sequence s's K and V of a layer as contiguous rows (max_pos x nkv x hd int8, zeros past its length and where a window
        has left pages behind; of a sequence that a budget has cut, what it holds): the caches that DecoderModel continues from. On
        `stream`, as the passes are."""
        torch = self.torch
        n = self.held(s) if max_pos is None else max_pos
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
