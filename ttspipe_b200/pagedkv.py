"""Paged key-value cache of a batch of streams (sm_100a kernels).

The reference keeps one dense cache of one stream
(app/engine/fusedlayer.py:212-269); here many streams share pools of fixed-size
pages, so memory follows their real lengths and they decode together. Three
operators work on the pools:

``write``      q/k norm + rotary + scatter of any number of tokens into their pages
               (one per stream in a decode step, a whole prompt in a prefill), with
               the bits ``nf4b_qk_rope_kv`` gives a dense cache
``attention``  one new token of each stream over its own rows; with ``weight`` every
               row's received attention weight is added up
``evict``      each KV head keeps its ``budget`` most attended rows (the first ``sink``
               tokens and the ``recent`` newest always among them), in place

Pools are [n_pages, n_kv, page_size, 128] bf16 or fp16; ``weight`` (fp32) and
``position`` (int32) are [n_pages, n_kv, page_size]; ``block_table`` is int32
[n_seqs, max_pages] (-1: not assigned); lengths, rows and positions are int32. All
of them stay on the device and are read there, so a CUDA graph of a step serves
every state of the cache. ``PagedKVCache`` holds the pools of all layers and hands
out pages; ``decode_block`` is a transformer block's decode step for a batch of streams.

A tensor of a wrong type, shape, layout or device (all on the current one) is refused with ValueError,
what the library refuses (head groups over 16, page sizes that are not a multiple of 16,
...) with ``Nf4bError``, in both cases before anything is launched.

Workspaces: one for each stream, grown as calls need it, by capacity (max_pages * page_size) and not
by length: a tracked attention takes 4 * n_head bytes a row. A captured graph has its own, from its own memory,
so captures need no warm-up here and graphs may be replayed side by side; the linears of
``decode_block`` share one workspace a device (``nf4gemv``), so steps of blocks may not.
"""

from __future__ import annotations

import ctypes

import torch

from ttspipe_b200 import _lib

HEAD_DIM = 128
_stats = {"write": 0, "attention": 0, "evict": 0, "block": 0}
# (kind, device, stream): (tensor, address, bytes, capture); calls on other streams may overlap, and so may a captured
# graph's replays: those of a capture (its id, 0 for none) are the capture's own, from its graph's memory
_NONE = (None, None, 0, 0)
_workspaces: dict = {}
_captured: dict = {}  # of the latest capture on each stream, to be dropped once it is over
_native = None

#: The current stream's handle, without the Stream object (2 us a call) torch.cuda.current_stream makes.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _bound():
    """The binding (csrc/pagedkv_bind.cpp), handed the library's functions. Raises if it has not been built."""
    global _native
    if _native is None:
        lib = _lib.lib()
        try:
            from ttspipe_b200 import _pagedkv
        except ImportError as exc:
            from ttspipe_b200 import build

            why = f"does not load ({exc})" if build.BIND.exists() else "is not built"
            raise RuntimeError(f"_pagedkv.so {why}; run `python -m ttspipe_b200.build`") from exc
        _pagedkv.bind(*(ctypes.cast(getattr(lib, f"nf4b_{name}"), ctypes.c_void_p).value
                        for name in ("paged_write", "paged_attention", "paged_evict", "capture_id")))
        _native = _pagedkv
    return _native


def stats() -> dict:
    return dict(_stats)


def _capture_id(stream: int) -> int:
    return _lib.lib().nf4b_capture_id(stream)


def _empty(size: int, device: int):
    return torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device))


def _workspace(kind: str, device: int, stream: int, need: int):
    """The workspace of a call that the stream's usual one does not serve: a larger one for the stream, or, in a
    graph capture, the capture's own. What has to be zero in a new one is zeroed (in a capture, by every replay)."""
    key, capture = (kind, device, stream), _capture_id(stream)
    kept = _captured if capture else _workspaces
    got = kept.get(key, _NONE)
    if got[3] != capture or got[2] < need:
        size = need if capture else max(need, 2 * got[2], 1 << 20)
        ws = _empty(size, device)
        if kind == "attention":
            ws[:_lib.PAGED_COUNTER_BYTES].zero_()
        got = kept[key] = (ws, ws.data_ptr(), size, capture)
    return got


def _raise(status: int):
    raise _lib.Nf4bError(status, _lib.last_error())


def write(qkv, k, v, block_table, rows, positions, freqs, *, n_head: int, seqs=None, q_norm=None, k_norm=None,
          eps: float = 1e-6, weight=None, position=None, out=None):
    """The tokens of `qkv` [T, (n_head + 2 n_kv) * 128] enter the cache; returns
    their rotated queries [T, n_head, 128].

    Token t has the rotary row `freqs`[positions[t]] (a (rows, 64, 2) table of cos,
    sin in fp32, fp16 or bf16) and becomes row `rows`[t] of sequence `seqs`[t]
    (None: of sequence t). `q_norm` / `k_norm` are the heads' RMSNorm weights [128].
    `weight` is set to 0 and `position` to the token's position at the new rows. A
    token whose row or position is out of range (-1, say) is padding: nothing of it
    enters the cache. No two tokens of a call may name the same row."""
    got = (_native or _bound()).write(qkv, k, v, block_table, rows, positions, freqs, n_head, seqs, q_norm, k_norm, eps,
                                      weight, position, out, _stream(k.get_device()) if k.is_cuda else 0)
    if type(got) is int:
        _raise(got)
    _stats["write"] += 1
    return got


def attention(q, k, v, block_table, lens, *, mask=None, scale: float | None = None, weight=None, out=None):
    """softmax(`scale` q k^T) v of one new token of each sequence, `q` [n_seqs, n_head,
    128], over its rows [0, lens[s]); returns [n_seqs, n_head, 128] of q's type.

    `mask` (bool or uint8 [n_seqs, max_pages * page_size], True = visible) hides rows,
    whatever they hold; a sequence that sees none gets zeros. `out` must not overlap an input. `scale` defaults to
    128 ** -0.5. `weight` receives every visible row's weight, summed over the query
    heads of its KV head. Up to 16 query heads to a KV head."""
    call, dev = (_native or _bound()).attention, k.get_device()
    stream = _stream(dev) if dev >= 0 else 0
    scale = HEAD_DIM ** -0.5 if scale is None else scale
    _, ws, size, capture = _workspaces.get(("attention", dev, stream), _NONE)
    got = call(q, k, v, block_table, lens, mask, scale, weight, out, ws, size, capture, stream)
    if type(got) is int:
        if got != _lib.NF4B_ERR_WORKSPACE:
            _raise(got)
        _, ws, size, capture = _workspace("attention", dev, stream, _lib.lib().nf4b_paged_attention_workspace_size(
            q.shape[0], q.shape[1], k.shape[1], block_table.shape[1], k.shape[2], weight is not None))
        got = call(q, k, v, block_table, lens, mask, scale, weight, out, ws, size, capture, stream)
        if type(got) is int:
            _raise(got)
    elif _captured:
        _captured.clear()
    _stats["attention"] += 1
    return got


def evict(k, v, weight, position, block_table, lens, *, budget: int, recent: int = 0, sink: int = 0,
          weight_out=None, position_out=None, lens_out=None):
    """Each KV head of each sequence keeps min(lens[s], `budget`) rows; returns the new
    lengths (`lens_out`, or `lens` itself).

    The rows of the first `sink` token positions and of the `recent` newest ones stay,
    then those with the greatest `weight`, equal ones by rising row. Kept rows at or past the budget
    move into the places below it that fall free (k, v in place), so rows
    [0, new length) hold the sequence - in another order, which attention does not
    see - and the pages after them are free. `weight_out`, `position_out` and
    `lens_out` receive the rows' weights and positions and the new lengths; None: in place.
    The sequences must not share pages. Rows of unassigned pages are not there: those below the
    new length are no places, so as many fewer of the others stay."""
    call, dev = (_native or _bound()).evict, k.get_device()
    stream = _stream(dev) if dev >= 0 else 0
    args = (k, v, weight, position, block_table, lens, budget, recent, sink,
            weight if weight_out is None else weight_out, position if position_out is None else position_out,
            lens if lens_out is None else lens_out)
    _, ws, size, capture = _workspaces.get(("evict", dev, stream), _NONE)
    got = call(*args, ws, size, capture, stream)
    if type(got) is int:
        if got != _lib.NF4B_ERR_WORKSPACE:
            _raise(got)
        _, ws, size, capture = _workspace("evict", dev, stream, _lib.lib().nf4b_paged_evict_workspace_size(
            block_table.shape[0], k.shape[1], block_table.shape[1], k.shape[2], budget))
        got = call(*args, ws, size, capture, stream)
        if type(got) is int:
            _raise(got)
    elif _captured:
        _captured.clear()
    _stats["evict"] += 1
    return got


class PagedKVCache:
    """The paged caches of `n_seqs` streams for `n_layers` blocks: each layer's pools, one
    block table and one set of lengths for all of them (an eviction leaves every
    head and layer of a stream equally many rows), and the pages' bookkeeping on the host.

    A decode step: ``reserve(streams)`` for every stream that takes part (its next row needs a
    page), ``begin_step()``, the blocks (``decode_block``), ``end_step()``; between steps
    ``evict`` where streams grow past a budget. Rows can be reserved for several steps ahead. A
    stream whose reserved rows are used up, whose next position is past the rotary table, or without
    ``active``, is passed over: its rows, weights, length and next position stay as they are.
    A prompt: ``reserve(stream, rows, prompt=True)``, ``prefill_block`` through the layers,
    ``prefilled(stream, rows)``; steps in between pass the stream over.
    Everything but ``reserve``, ``prefilled``, ``trim`` and ``release`` runs on the device and can be captured."""

    def __init__(self, n_layers: int, n_seqs: int, max_len: int, n_pages: int, n_kv: int, *, page_size: int = 64,
                 device, dtype=torch.bfloat16, track: bool = True):
        self.n_layers, self.n_seqs, self.page_size, self.n_pages = n_layers, n_seqs, page_size, n_pages
        self.max_pages = -(-max_len // page_size)
        pool = (n_pages, n_kv, page_size, HEAD_DIM)

        def per_layer(shape, dt):
            return [torch.zeros(shape, dtype=dt, device=device) for _ in range(n_layers)]

        self.k, self.v = per_layer(pool, dtype), per_layer(pool, dtype)
        self.weight = per_layer(pool[:3], torch.float32) if track else [None] * n_layers
        self.position = per_layer(pool[:3], torch.int32) if track else [None] * n_layers
        self.block_table = torch.full((n_seqs, self.max_pages), -1, dtype=torch.int32, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        # a stream takes part in a step where its three numbers in _at, its length, its next token's position and 0,
        # are below those in _below: the rows promised to it, the rotary table's and `active`
        self._at, self._below, self._is_below = (torch.zeros(3, n_seqs, **i32) for _ in range(3))
        self.lens = self._at[0]                       # rows of each stream
        self.next_pos = self._at[1]                   # position of its next token
        self.active = self._below[2]                  # 1: takes part in the steps that it has rows for
        self._below[1] = 2**31 - 1
        self._positions = None       # what _below[1] is set to, where the host knows
        self._step_positions = None  # rows of the shortest rotary table of this step so far
        self._promised = self._below[0].unbind()
        self.part = torch.zeros(n_seqs, **i32)        # of a step: 1 for each stream that takes part
        self.rows = torch.full((n_seqs,), -1, **i32)  # of a step: the new row of each stream, -1 for none
        self.live = torch.zeros(n_seqs, **i32)        # of a step: the rows its token attends to, 0 for none
        self._left = torch.zeros(n_seqs, **i32)
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: list = [[] for _ in range(n_seqs)]
        self._rows = [0] * n_seqs  # rows promised to each stream
        self._prompt = [0] * n_seqs  # those of them that a prompt has not filled yet

    def free_pages(self) -> int:
        return len(self._free)

    def reserved(self, seq: int) -> int:
        """The rows promised to a stream, those that it has among them."""
        return self._rows[seq]

    def reserve(self, seqs, rows: int = 1, *, prompt: bool = False) -> None:
        """Pages for `rows` more rows of a stream, which becomes active, or of each of several (64 in one call: 40 us on the
        host and one transfer; one by one 300 us and a launch each). Refuses (ValueError) what is past a stream's capacity
        and (RuntimeError) what the free pages do not hold, changing nothing.
        `prompt`: the rows are filled by ``prefill_block``, and the stream is passed over until ``prefilled`` has
        counted them (otherwise each step takes the next of them for its token)."""
        one = not hasattr(seqs, "__iter__")
        every = (seqs,) if one else tuple(seqs)
        if len(set(every)) < len(every):
            raise ValueError(f"a stream twice in {every}")
        free = len(self._free)
        for seq in every:
            want = self._rows[seq] + rows
            need = -(-want // self.page_size)
            if rows < 0 or need > self.max_pages:
                raise ValueError(f"{want} rows of stream {seq}: at most {self.max_pages * self.page_size}")
            new = max(0, need - len(self._pages[seq]))
            if new > free:
                raise RuntimeError(f"stream {seq} needs {new} pages, {free} are free")
            free -= new
        for seq in every:
            want = self._rows[seq] + rows
            held, need = self._pages[seq], -(-want // self.page_size)
            if need > len(held):
                new = [self._free.pop() for _ in range(need - len(held))]
                self.block_table[seq, len(held):need] = torch.tensor(new, dtype=torch.int32).to(self.block_table.device)
                held += new
            if prompt and rows:
                self._prompt[seq] += rows
                self.active[seq] = 0
            elif self._rows[seq] == 0 and rows:
                self.active[seq] = 1
            self._rows[seq] = want
        if one:
            self._promised[seqs].fill_(self._rows[seqs])
        elif every:
            self._below[0].copy_(torch.tensor(self._rows, dtype=torch.int32), non_blocking=True)

    def prefilled(self, seq: int, rows: int) -> None:
        """`rows` tokens of a prompt have passed through every layer's ``prefill_block``: they count as rows of the
        stream and as positions, and with the last of those reserved the stream takes part in steps."""
        if not 0 <= rows <= self._prompt[seq]:
            raise ValueError(f"{rows} rows of stream {seq}, {self._prompt[seq]} are reserved for its prompt")
        self._prompt[seq] -= rows
        self.lens[seq] += rows
        self.next_pos[seq] += rows
        if rows and not self._prompt[seq]:
            self.active[seq] = 1

    def trim(self, seq: int, rows: int) -> None:
        """A stream has `rows` rows left (after an eviction): later pages become free. Refused (RuntimeError) while
        its prompt is still being filled in."""
        if self._prompt[seq]:
            raise RuntimeError(f"{self._prompt[seq]} rows of stream {seq} are reserved for its prompt")
        if rows < self._rows[seq]:
            self._rows[seq] = rows
            self._promised[seq].fill_(rows)
        keep = -(-self._rows[seq] // self.page_size)
        held = self._pages[seq]
        if keep < len(held):
            self.block_table[seq, keep:len(held)] = -1
            self._free += held[keep:][::-1]
            del held[keep:]

    def release(self, seq: int) -> None:
        """A stream has ended: its pages become free and its place can be used again."""
        self._prompt[seq] = 0
        self.trim(seq, 0)
        self.lens[seq] = 0
        self.next_pos[seq] = 0
        self.active[seq] = 0

    def begin_step(self) -> None:
        """Rows and lengths of one new token of each stream that takes part; the others have no row and length 0, so
        that nothing is written for them, attended to or weighed."""
        self._step_positions = None
        self._take_part()

    def _take_part(self) -> None:
        torch.lt(self._at, self._below, out=self._is_below)
        torch.amin(self._is_below, 0, out=self.part)
        torch.addcmul(self.part, self.part, self.lens, out=self.live)
        torch.sub(self.live, 1, out=self.rows)

    def end_step(self) -> None:
        self._at[:2].add_(self.part)

    def _bound_positions(self, n: int) -> None:
        """A step's rotary table has `n` rows: streams whose next position is past it take no part, in this step
        if its first layer says so, else (another layer's table is shorter) from the next one on."""
        first = self._step_positions is None
        if not first and n >= self._step_positions:
            return
        self._step_positions = n
        known, captured = self._positions == n, self.lens.is_cuda and torch.cuda.is_current_stream_capturing()
        if known and not captured:
            return
        self._below[1].fill_(n)  # by every replay too: steps with another table may run in between
        self._positions = None if captured else n
        if first and not known:
            self._take_part()

    def write(self, layer: int, qkv, rows, positions, freqs, *, n_head: int, **kw):
        """``write`` into one layer's pools; of a step's tokens where `positions` is ``next_pos``."""
        if positions is self.next_pos:
            self._bound_positions(freqs.shape[0])
        return write(qkv, self.k[layer], self.v[layer], self.block_table, rows, positions, freqs, n_head=n_head,
                     weight=self.weight[layer], position=self.position[layer], **kw)

    def attention(self, layer: int, q, **kw):
        """``attention`` of a step's tokens over one layer's pools."""
        return attention(q, self.k[layer], self.v[layer], self.block_table, self.live, weight=self.weight[layer], **kw)

    def evict(self, budget: int, *, recent: int = 0, sink: int = 0) -> None:
        """``evict`` in every layer (each head by its own weights); afterwards ``trim`` frees the pages. Refused
        (RuntimeError) while a prompt is still being filled in: its rows lie past the lengths."""
        if any(self._prompt):
            raise RuntimeError(f"the prompt of stream {next(s for s, n in enumerate(self._prompt) if n)} is not filled in")
        for i in range(self.n_layers):
            evict(self.k[i], self.v[i], self.weight[i], self.position[i], self.block_table, self.lens, budget=budget,
                  recent=recent, sink=sink, lens_out=self._left)
        self.lens.copy_(self._left)

    def evict_and_trim(self, budget: int, *, recent: int = 0, sink: int = 0) -> None:
        """``evict``, and the pages that it leaves free are taken back (on the host, from its own count of
        rows): after ``end_step``, before rows are reserved for the next step."""
        self.evict(budget, recent=recent, sink=sink)
        for seq in range(self.n_seqs):
            self.trim(seq, budget)

    def rows_of(self, layer: int, seq: int, rows: int):
        """(k, v) [1, n_kv, rows, 128]: a copy of a stream's first `rows` rows."""
        pages = self.block_table[seq, : -(-rows // self.page_size)].long()
        return tuple(t[pages].transpose(0, 1).flatten(1, 2)[None, :, :rows] for t in (self.k[layer], self.v[layer]))


def _norms(a):
    qn, kn = (a.q_norm, a.k_norm) if a.attention_qk_norm else (None, None)
    eps = float(qn.eps if qn is not None and qn.eps is not None else 1e-6)
    return dict(q_norm=None if qn is None else qn.weight, k_norm=None if kn is None else kn.weight, eps=eps)


def _linear(module, x, *, norm=None, epi: int = 0, operand=None):
    """``nf4gemv.matmul``, with the bias of a linear that has one: added, as its own forward does, to the rounded
    product, and the epilogue then applied to that. None where `norm` cannot be fused."""
    from ttspipe_b200 import nf4gemv

    if getattr(module, "_nf4_fast", None) is None:
        nf4gemv.prepare(module)
    bias = getattr(module, "bias", None)
    y = nf4gemv.matmul(module, x, norm=norm, epi=epi if bias is None else nf4gemv.EPI_NONE,
                       operand=operand if bias is None else None)
    if y is None:
        if norm is None:
            raise ValueError(f"the block's {module} does not run on the NF4 kernels for {tuple(x.shape)} {x.dtype}")
        return None
    if bias is None:
        return y
    y = (y + bias).to(y.dtype)
    if epi == nf4gemv.EPI_RESIDUAL:
        return operand + y
    return torch.nn.functional.silu(operand) * y if epi == nf4gemv.EPI_SILU_GATE else y


def _normed_linear(norm, module, x):
    """norm, then the linear: in one launch where the kernel serves that."""
    from ttspipe_b200 import fusedops

    y = _linear(module, x, norm=(norm.weight, norm.eps))
    return _linear(module, fusedops.rms_norm(x, norm.weight, norm.eps)) if y is None else y


def _feed_forward(block, h):
    from ttspipe_b200 import fusedops, nf4gemv

    ff, norm = block.feed_forward, block.ffn_norm
    for module in (ff.w1, ff.w3):
        if getattr(module, "_nf4_fast", None) is None:
            nf4gemv.prepare(module)
    gated = all(getattr(module, "bias", None) is None for module in (ff.w1, ff.w3))  # the one launch adds none
    g = nf4gemv.matmul_gated(ff.w1, ff.w3, h, norm=(norm.weight, norm.eps)) if gated else None
    if g is None:
        hn = fusedops.rms_norm(h, norm.weight, norm.eps)
        g = nf4gemv.matmul_gated(ff.w1, ff.w3, hn) if gated else None
        if g is None:
            g = _linear(ff.w3, hn, epi=nf4gemv.EPI_SILU_GATE, operand=_linear(ff.w1, hn))
    return _linear(ff.w2, g, epi=nf4gemv.EPI_RESIDUAL, operand=h)


def decode_block(block, x, freqs, cache: PagedKVCache, layer: int):
    """One token of every stream through a transformer block: ``fusedlayer.decode_block``
    for a batch, over a paged cache. `x` is [n_seqs, 1, dim], `freqs` the whole rotary
    table (rows, 64, 2); between ``cache.begin_step()`` and ``cache.end_step()``. The
    rows of streams that take no part (``cache.part``) are computed and mean nothing."""
    from ttspipe_b200 import nf4gemv

    a = block.attention
    qkv = _normed_linear(block.attention_norm, a.wqkv, x)
    q = cache.write(layer, qkv.view(cache.n_seqs, -1), cache.rows, cache.next_pos, freqs, n_head=a.n_head, **_norms(a))
    y = cache.attention(layer, q).view(cache.n_seqs, 1, -1)
    h = _linear(a.wo, y, epi=nf4gemv.EPI_RESIDUAL, operand=x)
    out = _feed_forward(block, h)
    _stats["block"] += 1
    return out


def prefill_block(block, x, freqs, cache: PagedKVCache, layer: int, seq: int, rows: int = 0, position: int = 0):
    """The tokens `x` [1, T, dim] of one stream through a transformer block, entering the
    cache after its `rows` rows, from token position `position` on (both on the host;
    ``reserve`` T rows with ``prompt`` first, and ``prefilled`` after the last layer).
    Each attends to the rows before it and to itself, by the grouped torch formulation
    of ``fastpath``: over copies of the stream's rows, with its roundings of scores and
    probabilities to the activation type, which ``attention`` does not make, and
    n_head x T x rows of scores. Weights are not accumulated here: a prompt's rows start with
    weight 0 and gather it from the tokens decoded after it, so an eviction that comes soon
    keeps mostly the lowest of them, besides `sink` and `recent`."""
    from ttspipe_b200 import fastpath, nf4gemv

    a, n = block.attention, x.shape[1]
    if rows < 0 or rows + n > cache.reserved(seq):
        raise ValueError(f"rows {rows} to {rows + n} of stream {seq}: {cache.reserved(seq)} are reserved")
    if position < 0 or position + n > freqs.shape[0]:
        raise ValueError(f"positions {position} to {position + n}: the rotary table has {freqs.shape[0]} rows")
    dev = x.device
    qkv = _normed_linear(block.attention_norm, a.wqkv, x)
    at = torch.arange(n, dtype=torch.int32, device=dev)
    q = cache.write(layer, qkv.view(n, -1), at + rows, at + position, freqs, n_head=a.n_head,
                    seqs=torch.full_like(at, seq), **_norms(a))
    k, v = cache.rows_of(layer, seq, rows + n)
    mask = (torch.arange(rows + n, device=dev)[None] <= at[:, None] + rows)[None, None]
    y = fastpath._grouped_torch(q.transpose(0, 1)[None], k, v, mask, a.n_head, a.n_local_heads, HEAD_DIM)
    h = _linear(a.wo, y.transpose(1, 2).reshape(1, n, -1), epi=nf4gemv.EPI_RESIDUAL, operand=x)
    return _feed_forward(block, h)
