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
_stats = {"write": 0, "attention": 0, "evict": 0, "block": 0}
_workspaces: dict = {}
_retired: list = []  # replaced workspaces: a captured graph may still name them


def stats() -> dict:
    return dict(_stats)


def _workspace(kind: str, device, stream: int, need: int):
    """Zeroed workspace of a device and stream (calls on other streams may run at
    the same time), grown outside graph capture only."""
    key = (kind, device.index, stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"paged {kind} workspace must be sized before graph capture")
        if ws is not None:
            _retired.append(ws)
        ws = torch.zeros(max(need, 2 * ws.numel() if ws is not None else 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def _take(name: str, t, dtype, shape, device):
    """Refuse a tensor that is not of this type, shape and device, or not contiguous."""
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} {tuple(shape)} on {device} needed, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")
    return t.data_ptr()


def _cache(k, v, block_table, weight=None, position=None):
    """The library's description of a paged cache, after its checks."""
    dt = _lib.act_type(k.dtype)
    if dt is None or not k.is_cuda:
        raise ValueError(f"pools of {k.dtype} on {k.device} are not served")
    if k.dim() != 4 or k.shape[3] != HEAD_DIM or block_table.dim() != 2 or not k.numel() or not block_table.numel():
        raise ValueError(f"pools [n_pages, n_kv, page_size, {HEAD_DIM}] and a table [n_seqs, max_pages] needed, got "
                         f"{tuple(k.shape)} and {tuple(block_table.shape)}")
    n_pages, n_kv, page_size, _ = k.shape
    n_seqs, max_pages = block_table.shape
    dev, slots = k.device, k.shape[:3]
    return _lib.PagedKv(
        _take("k", k, k.dtype, k.shape, dev), _take("v", v, k.dtype, k.shape, dev),
        _take("block_table", block_table, torch.int32, block_table.shape, dev),
        None if weight is None else _take("weight", weight, torch.float32, slots, dev),
        None if position is None else _take("position", position, torch.int32, slots, dev),
        n_seqs, max_pages, n_pages, n_kv, page_size, dt)


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
    c = _cache(k, v, block_table, weight, position)
    dev = k.device
    width = (n_head + 2 * c.n_kv) * HEAD_DIM
    if qkv.dim() != 2 or not qkv.shape[0]:
        raise ValueError(f"qkv: [tokens, {width}] with at least one token needed, got {tuple(qkv.shape)}")
    n = qkv.shape[0]
    ft = _FTYPE.get(freqs.dtype)
    if ft is None or freqs.dim() != 3:
        raise ValueError(f"freqs: (rows, 64, 2) of fp32, fp16 or bf16 needed, got {freqs.dtype} {tuple(freqs.shape)}")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm are given together or not at all")
    if out is None:
        out = torch.empty((n, n_head, HEAD_DIM), dtype=k.dtype, device=dev)
    _lib.check(_lib.lib().nf4b_paged_write(
        c, _take("qkv", qkv, k.dtype, (n, width), dev),
        None if seqs is None else _take("seqs", seqs, torch.int32, (n,), dev),
        _take("rows", rows, torch.int32, (n,), dev), _take("positions", positions, torch.int32, (n,), dev),
        _take("freqs", freqs, freqs.dtype, (freqs.shape[0], HEAD_DIM // 2, 2), dev), ft, freqs.shape[0],
        None if q_norm is None else _take("q_norm", q_norm, k.dtype, (HEAD_DIM,), dev),
        None if k_norm is None else _take("k_norm", k_norm, k.dtype, (HEAD_DIM,), dev), eps,
        _take("out", out, k.dtype, (n, n_head, HEAD_DIM), dev), n, n_head,
        torch.cuda.current_stream(dev).cuda_stream))
    _stats["write"] += 1
    return out


def attention(q, k, v, block_table, lens, *, mask=None, scale: float | None = None, weight=None, out=None):
    """softmax(`scale` q k^T) v of one new token of each sequence, `q` [n_seqs, n_head,
    128], over its rows [0, lens[s]); returns [n_seqs, n_head, 128] of q's type.

    `mask` (bool or uint8 [n_seqs, max_pages * page_size], True = visible) hides rows,
    whatever they hold; a sequence that sees none gets zeros. `scale` defaults to
    128 ** -0.5. `weight` receives every visible row's weight, summed over the query
    heads of its KV head. Up to 16 query heads to a KV head."""
    c = _cache(k, v, block_table, weight)
    dev = k.device
    if q.dim() != 3:
        raise ValueError(f"q: [{c.n_seqs}, n_head, {HEAD_DIM}] needed, got {tuple(q.shape)}")
    n_head = q.shape[1]
    shape = (c.n_seqs, n_head, HEAD_DIM)
    if out is None:
        out = torch.empty(shape, dtype=k.dtype, device=dev)
    if mask is not None and mask.dtype is torch.bool:
        mask = mask.view(torch.uint8)
    stream = torch.cuda.current_stream(dev).cuda_stream
    lib = _lib.lib()
    need = lib.nf4b_paged_attention_workspace_size(c.n_seqs, n_head, c.n_kv, c.max_pages, c.page_size,
                                                   weight is not None)
    ws = _workspace("attention", dev, stream, need)
    _lib.check(lib.nf4b_paged_attention(
        c, _take("q", q, k.dtype, shape, dev), _take("lens", lens, torch.int32, (c.n_seqs,), dev),
        None if mask is None else _take("mask", mask, torch.uint8, (c.n_seqs, c.max_pages * c.page_size), dev),
        HEAD_DIM ** -0.5 if scale is None else scale, _take("out", out, k.dtype, shape, dev), n_head,
        ws.data_ptr(), ws.numel(), stream))
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
    c = _cache(k, v, block_table, weight, position)
    dev, slots = k.device, k.shape[:3]
    weight_out = weight if weight_out is None else weight_out
    position_out = position if position_out is None else position_out
    lens_out = lens if lens_out is None else lens_out
    stream = torch.cuda.current_stream(dev).cuda_stream
    lib = _lib.lib()
    need = lib.nf4b_paged_evict_workspace_size(c.n_seqs, c.n_kv, c.max_pages, c.page_size, budget)
    ws = _workspace("evict", dev, stream, need)
    _lib.check(lib.nf4b_paged_evict(
        c, _take("lens", lens, torch.int32, (c.n_seqs,), dev), budget, recent, sink,
        _take("weight_out", weight_out, torch.float32, slots, dev),
        _take("position_out", position_out, torch.int32, slots, dev),
        _take("lens_out", lens_out, torch.int32, (c.n_seqs,), dev), ws.data_ptr(), ws.numel(), stream))
    _stats["evict"] += 1
    return lens_out
