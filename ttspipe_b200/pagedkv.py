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
_FTYPE = {torch.float32: _lib.NF4B_F32, torch.float16: _lib.NF4B_F16, torch.bfloat16: _lib.NF4B_BF16}
_ACT = {torch.bfloat16: _lib.NF4B_BF16, torch.float16: _lib.NF4B_F16}
_stats = {"write": 0, "attention": 0, "evict": 0, "block": 0}
_workspaces: dict = {}  # (kind, device, stream): (tensor, address, bytes); calls on other streams may overlap
_retired: list = []  # replaced workspaces: a captured graph may still name them


#: The current stream's handle, without the Stream object (2 us a call) torch.cuda.current_stream makes.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


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


def _take(name: str, t, dtype, shape, device: int):
    """The tensor's address; refused if it is not of this type, shape and device, or not contiguous."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} {tuple(shape)} on cuda:{device} needed, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")
    return t.data_ptr()


def _cache(k, v, block_table, weight=None, position=None):
    """The library's description of a paged cache, the shape of its rows and its device, after their checks."""
    dtype, shape, device = k.dtype, k.shape, k.get_device()
    dt = _ACT.get(dtype)
    if dt is None or device < 0:
        raise ValueError(f"pools of {dtype} on {k.device} are not served")
    table = block_table.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or len(table) != 2 or 0 in shape or 0 in table:
        raise ValueError(f"pools [n_pages, n_kv, page_size, {HEAD_DIM}] and a table [n_seqs, max_pages] needed, got "
                         f"{tuple(shape)} and {tuple(table)}")
    slots = shape[:3]
    return _lib.PagedKv(
        _take("k", k, dtype, shape, device), _take("v", v, dtype, shape, device),
        _take("block_table", block_table, torch.int32, table, device),
        None if weight is None else _take("weight", weight, torch.float32, slots, device),
        None if position is None else _take("position", position, torch.int32, slots, device),
        *table, *slots, dt), slots, device


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
    c, (_, n_kv, _), dev = _cache(k, v, block_table, weight, position)
    dtype, width = k.dtype, (n_head + 2 * n_kv) * HEAD_DIM
    if qkv.dim() != 2 or n_head < 1:
        raise ValueError(f"qkv: [tokens, {width}] and n_head >= 1 needed, got {tuple(qkv.shape)} and {n_head}")
    n = qkv.shape[0]
    ft = _FTYPE.get(freqs.dtype)
    if ft is None or freqs.dim() != 3:
        raise ValueError(f"freqs: (rows, 64, 2) of fp32, fp16 or bf16 needed, got {freqs.dtype} {tuple(freqs.shape)}")
    n_freqs = freqs.shape[0]
    if out is None:
        out = qkv.new_empty((n, n_head, HEAD_DIM))
    _lib.check(_lib.lib().nf4b_paged_write(
        c, _take("qkv", qkv, dtype, (n, width), dev), None if seqs is None else _take("seqs", seqs, torch.int32, (n,), dev),
        _take("rows", rows, torch.int32, (n,), dev), _take("positions", positions, torch.int32, (n,), dev),
        _take("freqs", freqs, freqs.dtype, (n_freqs, HEAD_DIM // 2, 2), dev), ft, n_freqs,
        None if q_norm is None else _take("q_norm", q_norm, dtype, (HEAD_DIM,), dev),
        None if k_norm is None else _take("k_norm", k_norm, dtype, (HEAD_DIM,), dev), eps,
        _take("out", out, dtype, (n, n_head, HEAD_DIM), dev), n, n_head, _stream(dev)))
    _stats["write"] += 1
    return out


def attention(q, k, v, block_table, lens, *, mask=None, scale: float | None = None, weight=None, out=None):
    """softmax(`scale` q k^T) v of one new token of each sequence, `q` [n_seqs, n_head,
    128], over its rows [0, lens[s]); returns [n_seqs, n_head, 128] of q's type.

    `mask` (bool or uint8 [n_seqs, max_pages * page_size], True = visible) hides rows,
    whatever they hold; a sequence that sees none gets zeros. `scale` defaults to
    128 ** -0.5. `weight` receives every visible row's weight, summed over the query
    heads of its KV head. Up to 16 query heads to a KV head."""
    c, (_, n_kv, page_size), dev = _cache(k, v, block_table, weight)
    dtype, shape = k.dtype, q.shape
    if len(shape) != 3 or shape[0] != c.n_seqs or shape[2] != HEAD_DIM:
        raise ValueError(f"q: [{c.n_seqs}, n_head, {HEAD_DIM}] needed, got {tuple(shape)}")
    if out is None:
        out = torch.empty_like(q)
    if mask is not None and mask.dtype is torch.bool:
        mask = mask.view(torch.uint8)
    n_head, stream, lib = shape[1], _stream(dev), _lib.lib()
    args = (_take("q", q, dtype, shape, dev), _take("lens", lens, torch.int32, (shape[0],), dev),
            None if mask is None else _take("mask", mask, torch.uint8, (shape[0], c.max_pages * page_size), dev),
            HEAD_DIM ** -0.5 if scale is None else scale, _take("out", out, dtype, shape, dev), n_head)
    _, ws, size = _workspaces.get(("attention", dev, stream)) or (None, None, 0)
    status = lib.nf4b_paged_attention(c, *args, ws, size, stream)
    if status == _lib.NF4B_ERR_WORKSPACE:
        _, ws, size = _grow("attention", dev, stream, lib.nf4b_paged_attention_workspace_size(
            shape[0], n_head, n_kv, c.max_pages, page_size, weight is not None))
        status = lib.nf4b_paged_attention(c, *args, ws, size, stream)
    _lib.check(status)
    _stats["attention"] += 1
    return out


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
    c, slots, dev = _cache(k, v, block_table, weight, position)
    weight_out = weight if weight_out is None else weight_out
    position_out = position if position_out is None else position_out
    lens_out = lens if lens_out is None else lens_out
    n, stream, lib = c.n_seqs, _stream(dev), _lib.lib()
    args = (_take("lens", lens, torch.int32, (n,), dev), budget, recent, sink,
            _take("weight_out", weight_out, torch.float32, slots, dev),
            _take("position_out", position_out, torch.int32, slots, dev),
            _take("lens_out", lens_out, torch.int32, (n,), dev))
    _, ws, size = _workspaces.get(("evict", dev, stream)) or (None, None, 0)
    status = lib.nf4b_paged_evict(c, *args, ws, size, stream)
    if status == _lib.NF4B_ERR_WORKSPACE:
        _, ws, size = _grow("evict", dev, stream, lib.nf4b_paged_evict_workspace_size(
            n, c.n_kv, c.max_pages, c.page_size, budget))
        status = lib.nf4b_paged_evict(c, *args, ws, size, stream)
    _lib.check(status)
    _stats["evict"] += 1
    return lens_out
