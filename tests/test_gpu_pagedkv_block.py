"""Batched decode through transformer blocks over a paged cache: each stream against the
oracle's block of that stream alone, at the dense block's own bar (B200 only)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import nf4_oracle as orc
from tests.helpers import randn_bf16, to_bits
from tests.test_gpu_block import BLOCK_TOL, _oracle_weights
from ttspipe_b200 import fusedlayer, fusedops, model, nf4gemv, pagedkv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def installed():
    assert nf4gemv.install() and fusedops.install() and fusedlayer.install()


def _cfg(qk):
    return model.ModelArgs(dim=512, n_head=8, n_local_heads=2, intermediate_size=1024, max_seq_len=128,
                           attention_qk_norm=qk)


class Alone:
    """One stream's block in the oracle, token after token."""

    def __init__(self, blk, cfg, freqs):
        self.w, self.cfg, self.freqs, self.pos = _oracle_weights(blk), cfg, orc.bf16_to_f32(to_bits(freqs)), 0
        shape = (cfg.n_local_heads, cfg.max_seq_len, cfg.head_dim)
        self.k, self.v = np.zeros(shape, np.uint16), np.zeros(shape, np.uint16)

    def error(self, x, y):
        """How far y is from the block of the next token x: max|err| / max|ref|."""
        c = self.cfg
        want = orc.decode_block(to_bits(x).reshape(-1), self.w, self.k, self.v, self.pos, self.freqs[self.pos],
                                c.n_head, c.n_local_heads, c.head_dim, c.norm_eps, c.norm_eps)
        self.pos += 1
        return orc.relative_error(orc.bf16_to_f32(to_bits(y)).ravel(), orc.bf16_to_f32(want).ravel())


@pytest.mark.parametrize("qk,n_seqs", [(False, 3), (True, 12)])
def test_streams_decode_as_each_alone(qk, n_seqs):
    """Streams that join and leave at different steps; 12 of them take the GEMM."""
    cfg = _cfg(qk)
    blk = model.random_block(cfg, device="cuda", seed=3)
    freqs = model.precompute_freqs_cis(128, 128, 1e6, device="cuda")
    cache = pagedkv.PagedKVCache(1, n_seqs, 128, 3 * n_seqs, 2, page_size=16, device="cuda")
    steps = [(s, s + 12 + 4 * (s % 3)) for s in range(n_seqs)]  # each stream's first step and the one it ends before
    got = {}
    with torch.inference_mode():
        for t in range(24):
            x = randn_bf16((n_seqs, 1, cfg.dim), seed=100 + t, device="cuda")
            for s, (first, last) in enumerate(steps):
                if first <= t < last:
                    cache.reserve(s)
                elif t == last:
                    cache.release(s)
            cache.begin_step()
            y = pagedkv.decode_block(blk, x, freqs, cache, 0)
            cache.end_step()
            for s, (first, last) in enumerate(steps):
                if first <= t < last:
                    got[s, t - first] = (x[s : s + 1], y[s : s + 1].clone())
        assert cache.lens.tolist() == [24 - first if last > 23 else 0 for first, last in steps]
        for s, (first, last) in enumerate(steps):
            alone = Alone(blk, cfg, freqs)
            for pos in range(min(24, last) - first):
                assert alone.error(*got[s, pos]) < BLOCK_TOL, (s, pos)


def test_prefill_then_decode_as_the_stream_alone():
    cfg = _cfg(False)
    blk = model.random_block(cfg, device="cuda", seed=5)
    freqs = model.precompute_freqs_cis(128, 128, 1e6, device="cuda")
    cache = pagedkv.PagedKVCache(1, 2, 128, 16, 2, page_size=32, device="cuda")
    x = randn_bf16((1, 50, cfg.dim), seed=6, device="cuda")
    alone = Alone(blk, cfg, freqs)
    with torch.inference_mode():
        cache.reserve(0, 50)
        y = torch.cat([pagedkv.prefill_block(blk, x[:, :33], freqs, cache, 0, 0),
                       pagedkv.prefill_block(blk, x[:, 33:], freqs, cache, 0, 0, rows=33, position=33)], 1)
        cache.lens[0] += 50
        cache.next_pos[0] += 50
        for t in range(50):
            assert alone.error(x[:, t], y[:, t]) < BLOCK_TOL, t
        cache.reserve(0)
        cache.begin_step()
        xs = randn_bf16((2, 1, cfg.dim), seed=7, device="cuda")
        got = pagedkv.decode_block(blk, xs, freqs, cache, 0)
        cache.end_step()
        assert alone.error(xs[:1], got[:1]) < BLOCK_TOL
        assert cache.lens.tolist() == [51, 0]


def test_a_bounded_cache_keeps_decoding():
    """Two layers under a budget for 80 steps: rows stay bounded, pages come back, sinks and the newest
    rows are kept, and a head's weights sum to what its tokens gave out less what was evicted."""
    cfg = _cfg(False)
    blocks = [model.random_block(cfg, device="cuda", seed=8 + i) for i in range(2)]
    freqs = model.precompute_freqs_cis(128, 128, 1e6, device="cuda")
    cache = pagedkv.PagedKVCache(2, 2, 128, 10, 2, page_size=16, device="cuda")
    with torch.inference_mode():
        for t in range(80):
            for s in range(2):
                cache.reserve(s)
            cache.begin_step()
            x = randn_bf16((2, 1, cfg.dim), seed=200 + t, device="cuda")
            for i, blk in enumerate(blocks):
                x = pagedkv.decode_block(blk, x, freqs, cache, i)
            cache.end_step()
            assert torch.isfinite(x.float()).all()
            if (t + 1) % 40 == 0:
                cache.evict_and_trim(24, recent=8, sink=2)
                assert cache.lens.tolist() == [24, 24] and cache.free_pages() == 10 - 4
    assert cache.next_pos.tolist() == [80, 80]
    for i in range(2):
        for s in range(2):
            pages = cache.block_table[s, :2].long()
            pos = cache.position[i][pages].transpose(0, 1).flatten(1)[:, :24]
            assert all({0, 1, *range(72, 80)} <= set(h.tolist()) for h in pos)
            w = cache.weight[i][pages].transpose(0, 1).flatten(1)[:, :24]
            assert (w > 0).all() and w.sum() <= 80 * cfg.n_head + 1e-2
    cache.release(0)
    cache.release(1)
    assert cache.free_pages() == 10


def test_a_step_replays_from_a_cuda_graph():
    cfg = _cfg(False)
    blk = model.random_block(cfg, device="cuda", seed=11)
    freqs = model.precompute_freqs_cis(128, 128, 1e6, device="cuda")
    caches = [pagedkv.PagedKVCache(1, 4, 128, 12, 2, page_size=16, device="cuda") for _ in range(2)]
    x = randn_bf16((4, 1, cfg.dim), seed=12, device="cuda")
    out = torch.empty_like(x)

    def step(cache):
        cache.begin_step()
        out.copy_(pagedkv.decode_block(blk, x, freqs, cache, 0))
        cache.end_step()

    want = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(side):
        for t in range(20):
            x.copy_(randn_bf16((4, 1, cfg.dim), seed=300 + t))
            caches[0].reserve(1)
            caches[0].reserve(3)
            step(caches[0])
            want.append(out[[1, 3]].clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    for t in range(20):
        x.copy_(randn_bf16((4, 1, cfg.dim), seed=300 + t))
        caches[1].reserve(1)
        caches[1].reserve(3)
        graph.replay()
        assert torch.equal(out[[1, 3]], want[t])
    assert caches[1].lens.tolist() == [0, 20, 0, 20]
    del graph
