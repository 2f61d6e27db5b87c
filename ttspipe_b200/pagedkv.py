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
every state of the cache. ``PagedKVCache`` holds one layer's pools and hands out
pages; ``decode_block`` is a transformer block's decode step for a batch of streams.

A tensor of a wrong type, shape, layout or device is refused with ValueError,
what the library refuses (head groups over 16, page sizes that are not a multiple of 16,
...) with ``Nf4bError``, in both cases before anything is launched.
"""

from __future__ import annotations

import ctypes

import torch

from ttspipe_b200 import _lib

HEAD_DIM = 128
_stats = {"write": 0, "attention": 0, "evict": 0, "block": 0}
_workspaces: dict = {}  # (kind, device, stream): (tensor, address, bytes); calls on other streams may overlap
_retired: list = []  # replaced workspaces: a captured graph may still name them
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
            raise RuntimeError("_pagedkv.so is not built; run `python -m ttspipe_b200.build`") from exc
        _pagedkv.bind(*(ctypes.cast(getattr(lib, f"nf4b_paged_{name}"), ctypes.c_void_p).value
                        for name in ("write", "attention", "evict")))
        _native = _pagedkv
    return _native


def stats() -> dict:
    return dict(_stats)


def _grow(kind: str, device, stream: int, need: int):
    """A larger zeroed workspace for a device and stream, outside graph capture only."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"paged {kind} workspace must be sized before graph capture")
    old = _workspaces.get((kind, device, stream))
    if old is not None:
        _retired.append(old[0])
    ws = torch.zeros(max(need, 2 * old[2] if old else 1 << 20), dtype=torch.uint8, device=torch.device("cuda", device))
    got = _workspaces[(kind, device, stream)] = (ws, ws.data_ptr(), ws.numel())
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
    whatever they hold; a sequence that sees none gets zeros. `scale` defaults to
    128 ** -0.5. `weight` receives every visible row's weight, summed over the query
    heads of its KV head. Up to 16 query heads to a KV head."""
    call, dev = (_native or _bound()).attention, k.get_device()
    stream = _stream(dev) if dev >= 0 else 0
    scale = HEAD_DIM ** -0.5 if scale is None else scale
    _, ws, size = _workspaces.get(("attention", dev, stream)) or (None, None, 0)
    got = call(q, k, v, block_table, lens, mask, scale, weight, out, ws, size, stream)
    if type(got) is int:
        if got != _lib.NF4B_ERR_WORKSPACE:
            _raise(got)
        _, ws, size = _grow("attention", dev, stream, _lib.lib().nf4b_paged_attention_workspace_size(
            q.shape[0], q.shape[1], k.shape[1], block_table.shape[1], k.shape[2], weight is not None))
        got = call(q, k, v, block_table, lens, mask, scale, weight, out, ws, size, stream)
        if type(got) is int:
            _raise(got)
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
    The sequences must not share pages."""
    call, dev = (_native or _bound()).evict, k.get_device()
    stream = _stream(dev) if dev >= 0 else 0
    args = (k, v, weight, position, block_table, lens, budget, recent, sink,
            weight if weight_out is None else weight_out, position if position_out is None else position_out,
            lens if lens_out is None else lens_out)
    _, ws, size = _workspaces.get(("evict", dev, stream)) or (None, None, 0)
    got = call(*args, ws, size, stream)
    if type(got) is int:
        if got != _lib.NF4B_ERR_WORKSPACE:
            _raise(got)
        _, ws, size = _grow("evict", dev, stream, _lib.lib().nf4b_paged_evict_workspace_size(
            block_table.shape[0], k.shape[1], block_table.shape[1], k.shape[2], budget))
        got = call(*args, ws, size, stream)
        if type(got) is int:
            _raise(got)
    _stats["evict"] += 1
    return got
