"""What the paged KV cache refuses, on the host and before anything is launched
(runs without a GPU), and the oracle's own rules."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from ttspipe_b200 import _lib, pagedkv

ARG, SHAPE, ALIGN, DTYPE, WORKSPACE = -1, -2, -3, -4, -5


class Host:
    """Host memory that stands in for device pointers: the calls fail before any launch."""

    def __init__(self):
        self.buf = ctypes.create_string_buffer(1 << 16)
        self.at = (ctypes.addressof(self.buf) + 255) // 256 * 256

    def cache(self, **kw):
        c = _lib.PagedKv(self.at, self.at, self.at, self.at, self.at, 2, 4, 8, 2, 16, _lib.NF4B_BF16)
        for name, value in kw.items():
            setattr(c, name, value)
        return c

    def write(self, c=None, **kw):
        a = dict(qkv=self.at, seqs=None, rows=self.at, positions=self.at, freqs=self.at, ftype=_lib.NF4B_BF16,
                 freqs_rows=10, qw=None, kw=None, eps=1e-6, q=self.at, n=2, n_head=4)
        a.update(kw)
        return _lib.lib().nf4b_paged_write(self.cache() if c is None else c, *a.values(), None)

    def attention(self, c=None, **kw):
        a = dict(q=self.at, lens=self.at, mask=None, scale=0.1, out=self.at, n_head=4, ws=self.at, bytes=1 << 40)
        a.update(kw)
        return _lib.lib().nf4b_paged_attention(self.cache() if c is None else c, *a.values(), None)

    def evict(self, c=None, **kw):
        a = dict(lens=self.at, budget=8, recent=2, sink=1, w=self.at, p=self.at, l=self.at, ws=self.at, bytes=1 << 40)
        a.update(kw)
        return _lib.lib().nf4b_paged_evict(self.cache() if c is None else c, *a.values(), None)


@pytest.fixture()
def host():
    return Host()


CACHE_FAULTS = [
    ("k", None, ARG), ("v", None, ARG), ("block_table", None, ARG),
    ("dtype", _lib.NF4B_F32, DTYPE), ("dtype", 7, DTYPE),
    ("n_seqs", 0, SHAPE), ("n_seqs", 4097, SHAPE), ("n_kv", 0, SHAPE), ("n_kv", 40000, SHAPE),
    ("page_size", 0, SHAPE), ("page_size", 8, SHAPE), ("page_size", 40, SHAPE), ("page_size", -16, SHAPE),
    ("n_pages", 0, SHAPE), ("max_pages", 0, SHAPE), ("max_pages", 1 << 28, SHAPE),
]


@pytest.mark.parametrize("call", ["write", "attention", "evict"])
@pytest.mark.parametrize("field,value,status", CACHE_FAULTS)
def test_every_call_refuses_a_cache_it_does_not_serve(host, call, field, value, status):
    assert getattr(host, call)(host.cache(**{field: value})) == status
    assert _lib.last_error()


@pytest.mark.parametrize("call", ["write", "attention", "evict"])
@pytest.mark.parametrize("field,off", [("k", 8), ("v", 2), ("block_table", 2), ("weight", 2), ("position", 1)])
def test_every_call_refuses_a_misaligned_cache(host, call, field, off):
    assert getattr(host, call)(host.cache(**{field: host.at + off})) == ALIGN


def test_no_cache(host):
    L = _lib.lib()
    assert L.nf4b_paged_attention(None, host.at, host.at, None, 1.0, host.at, 4, host.at, 1 << 30, None) == ARG
    assert L.nf4b_paged_evict(None, host.at, 8, 0, 0, host.at, host.at, host.at, host.at, 1 << 30, None) == ARG


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), ARG), (dict(rows=None), ARG), (dict(positions=None), ARG), (dict(freqs=None), ARG),
    (dict(q=None), ARG), (dict(ftype=3), DTYPE), (dict(freqs_rows=0), SHAPE), (dict(n=0), SHAPE),
    (dict(n=-4), SHAPE), (dict(n=3), SHAPE),  # three tokens of two sequences without seqs
    (dict(n_head=3), SHAPE), (dict(n_head=0), SHAPE),
])
def test_write_refusals(host, kw, status):
    assert host.write(**kw) == status


def test_write_refuses_half_a_norm_and_misalignment(host):
    assert host.write(qw=host.at) == ARG
    assert host.write(qw=host.at, kw=host.at, eps=-1.0) == ARG
    assert host.write(qw=host.at, kw=host.at, eps=float("nan")) == ARG
    for name, off in (("qkv", 8), ("q", 4), ("rows", 2), ("positions", 1), ("seqs", 2), ("freqs", 1)):
        assert host.write(**{name: host.at + off}) == ALIGN


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), ARG), (dict(lens=None), ARG), (dict(out=None), ARG), (dict(scale=float("nan")), ARG),
    (dict(scale=float("inf")), ARG), (dict(n_head=3), SHAPE), (dict(n_head=0), SHAPE), (dict(n_head=34), SHAPE),
    (dict(ws=None), WORKSPACE), (dict(bytes=1000), WORKSPACE),
])
def test_attention_refusals(host, kw, status):
    assert host.attention(**kw) == status


def test_attention_misalignment(host):
    for name, off in (("q", 8), ("out", 2), ("lens", 2), ("ws", 16)):
        assert host.attention(**{name: host.at + off}) == ALIGN


@pytest.mark.parametrize("kw,status", [
    (dict(lens=None), ARG), (dict(w=None), ARG), (dict(p=None), ARG), (dict(l=None), ARG), (dict(budget=0), ARG),
    (dict(budget=-1), ARG), (dict(recent=-1), ARG), (dict(sink=-1), ARG), (dict(recent=7, sink=2), ARG),
    (dict(recent=2**31 - 1, sink=2**31 - 1), ARG), (dict(ws=None), WORKSPACE), (dict(bytes=10), WORKSPACE),
])
def test_evict_refusals(host, kw, status):
    assert host.evict(**kw) == status


def test_evict_needs_weights_and_positions_and_alignment(host):
    assert host.evict(host.cache(weight=None)) == ARG
    assert host.evict(host.cache(position=None)) == ARG
    for name, off in (("lens", 2), ("w", 1), ("p", 2), ("l", 2), ("ws", 128)):
        assert host.evict(**{name: host.at + off}) == ALIGN


def test_workspace_sizes():
    L = _lib.lib()
    att = L.nf4b_paged_attention_workspace_size
    assert att(0, 32, 8, 10, 64, 0) == 0 and att(1, 31, 8, 10, 64, 0) == 0
    assert 0 < att(1, 32, 8, 10, 64, 0) < att(1, 32, 8, 10, 64, 1)
    ev = L.nf4b_paged_evict_workspace_size
    assert ev(1, 0, 10, 64, 5) == 0 and ev(2, 8, 10, 64, 0) == 0 and ev(2, 8, 10, 64, 100) > 0


def test_python_refuses_tensors_on_the_host():
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    t = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="not served"):
        pagedkv.attention(torch.zeros(1, 4, 128, dtype=torch.bfloat16), k, k, t, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="not served"):
        pagedkv.evict(k.float(), k.float(), k[..., 0].float(), k[..., 0].int(), t, t[0], budget=1)


def test_oracle_attention_is_a_softmax():
    """The oracle against itself: weights sum to the group's heads, and one row gives its value."""
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((3, 1, 16, 128)), rng.standard_normal((3, 1, 16, 128))
    table = np.array([[2, 0, -1]])
    out, added, _ = po.attention(rng.standard_normal((1, 2, 128)), k, v, table, [20], scale=0.1)
    assert abs(added.sum() - 2) < 1e-12 and added[1].sum() == 0
    out, _, _ = po.attention(rng.standard_normal((1, 2, 128)), k, v, table, [1], scale=0.1)
    assert np.allclose(out[0], v[2, 0, 0])


def test_oracle_kept_rows():
    w = np.array([5, 1, 1, 9, np.nan, 0, 1], np.float32)
    pos = np.arange(7)
    assert po.kept(w, pos, 3, 0, 0).nonzero()[0].tolist() == [0, 1, 3]
    assert po.kept(w, pos, 3, 1, 1).nonzero()[0].tolist() == [0, 3, 6]
    to, src = po.moves(po.kept(w, pos, 3, 1, 1), 3)
    assert to.tolist() == [1, 2] and src.tolist() == [3, 6]


# ---- the cache's pages on the host -------------------------------------------


def make_cache(n_pages=6, **kw):
    return pagedkv.PagedKVCache(2, 3, 64, n_pages, 2, page_size=16, device="cpu", **kw)


def test_pages_are_handed_out_and_taken_back():
    c = make_cache()
    c.reserve(0, 17)
    c.reserve(1)
    assert c.free_pages() == 3 and c.active.tolist() == [1, 1, 0]
    own = [p for s in range(2) for p in c.block_table[s].tolist() if p >= 0]
    assert len(set(own)) == 3 and (c.block_table[2] == -1).all()
    for _ in range(15):
        c.reserve(1)  # rows 2 to 16 share the page of the first
    assert c.free_pages() == 3
    c.reserve(1)
    assert c.free_pages() == 2 and (c.block_table[1] >= 0).sum() == 2
    c.trim(0, 16)
    assert c.free_pages() == 3 and (c.block_table[0] >= 0).tolist() == [True, False, False, False]
    c.lens[1] = 17
    c.release(1)
    assert c.free_pages() == 5 and c.lens[1] == 0 and c.active[1] == 0 and (c.block_table[1] == -1).all()


def test_a_reservation_that_does_not_fit_changes_nothing():
    c = make_cache()
    c.reserve(0, 64)
    before = c.block_table.clone()
    with pytest.raises(ValueError, match="at most 64"):
        c.reserve(0)
    with pytest.raises(RuntimeError, match="2 are free"):
        c.reserve(1, 33)
    assert torch.equal(c.block_table, before) and c.free_pages() == 2 and c.active.tolist() == [1, 0, 0]
    c.reserve(1, 32)
    assert c.free_pages() == 0


def test_a_step_counts_the_active_streams_only():
    c = make_cache(track=False)
    c.reserve(0, 5)
    c.reserve(2, 1)
    c.lens.copy_(torch.tensor([4, 0, 0]))
    c.next_pos.copy_(torch.tensor([9, 0, 0]))
    c.begin_step()
    assert c.rows.tolist() == [4, -1, 0] and c.live.tolist() == [5, 0, 1]
    c.end_step()
    assert c.lens.tolist() == [5, 0, 1] and c.next_pos.tolist() == [10, 0, 1]
    assert c.weight == [None, None]


def test_rows_come_back_in_sequence_order():
    c = make_cache()
    c.reserve(0, 16)
    c.reserve(1, 16)
    c.reserve(0, 10)
    for r in range(26):
        c.k[1][int(c.block_table[0, r // 16]), :, r % 16] = r
    k, v = c.rows_of(1, 0, 26)
    assert k.shape == (1, 2, 26, 128) and k[0, 1, :, 5].tolist() == list(range(26)) and not v.any()
