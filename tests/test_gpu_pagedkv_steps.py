"""Blocks over a paged cache on the B200: linears with biases, streams that pause."""

from __future__ import annotations

import pytest
import torch

from tests.helpers import randn_bf16
from tests.test_gpu_block import BLOCK_TOL
from ttspipe_b200 import fusedlayer, fusedops, model, nf4gemv, pagedkv

pytestmark = pytest.mark.gpu

CFG = model.ModelArgs(dim=512, n_head=8, n_local_heads=2, intermediate_size=1024, max_seq_len=128)


@pytest.fixture(scope="module", autouse=True)
def installed():
    assert nf4gemv.install() and fusedops.install() and fusedlayer.install()


def freqs(rows=128):
    return model.precompute_freqs_cis(rows, 128, 1e6, device="cuda")


def biased_block(seed):
    blk = model.random_block(CFG, device="cuda", seed=seed)
    a, ff = blk.attention, blk.feed_forward
    for i, lin in enumerate((a.wqkv, a.wo, ff.w1, ff.w3, ff.w2)):
        lin.bias = torch.nn.Parameter(randn_bf16((lin.out_features,), seed=seed + i, device="cuda"), requires_grad=False)
    return blk


def own_forward(blk, x, first):
    """The block's own forward of tokens from position `first` on of one stream, over its dense cache."""
    at = torch.arange(first, first + x.shape[1], device="cuda")
    mask = torch.ones(128, 128, dtype=torch.bool, device="cuda").tril()[None, None, at, : first + x.shape[1]]
    return blk(x, freqs()[at], mask, at)


def near(got, want):
    """Two computations that each stay within BLOCK_TOL of the exact block."""
    return float((got - want).float().abs().max() / want.float().abs().max()) < 2 * BLOCK_TOL


@pytest.mark.parametrize("n", [3, 12])  # decode GEMVs, then the GEMM
def test_decode_of_a_block_with_biases(n):
    blk = biased_block(20)
    cache = pagedkv.PagedKVCache(1, n, 128, 2 * n, 2, page_size=16, device="cuda")
    with torch.inference_mode():
        x = randn_bf16((n, 4, CFG.dim), seed=5, device="cuda")
        got = []
        for t in range(4):
            for s in range(n):
                cache.reserve(s)
            cache.begin_step()
            got.append(pagedkv.decode_block(blk, x[:, t : t + 1].contiguous(), freqs(), cache, 0))
            cache.end_step()
        for s in range(n):
            for t in range(4):
                assert near(got[t][s : s + 1], own_forward(blk, x[s : s + 1, t : t + 1], t)), (s, t)


def test_prefill_of_a_block_with_biases():
    blk = biased_block(30)
    cache = pagedkv.PagedKVCache(1, 2, 128, 8, 2, page_size=16, device="cuda")
    with torch.inference_mode():
        x = randn_bf16((1, 40, CFG.dim), seed=6, device="cuda")
        cache.reserve(1, 40)
        assert near(pagedkv.prefill_block(blk, x, freqs(), cache, 0, 1), own_forward(blk, x, 0))


def step(blk, cache, x, table):
    cache.begin_step()
    out = pagedkv.decode_block(blk, x, table, cache, 0)
    cache.end_step()
    return out


def held_by(cache, seq):
    pages = cache.block_table[seq]
    pages = pages[pages >= 0].long()
    pools = (cache.k[0], cache.v[0], cache.weight[0], cache.position[0])
    return [t[pages].clone() for t in pools] + [cache.lens[seq].clone(), cache.next_pos[seq].clone()]


def unchanged(cache, seq, before):
    return all(torch.equal(a, b) for a, b in zip(held_by(cache, seq), before))


def test_a_stream_that_is_not_active_is_passed_over():
    """NaN in its slot of x: its rows, weights and lengths stay, and it goes on as one that never paused."""
    blk, table = model.random_block(CFG, device="cuda", seed=40), freqs()
    x = randn_bf16((2, 24, CFG.dim), seed=41, device="cuda")
    caches = [pagedkv.PagedKVCache(1, 2, 128, 8, 2, page_size=16, device="cuda") for _ in range(2)]
    with torch.inference_mode():
        want = []
        for t in range(24):
            for s in range(2):
                caches[0].reserve(s)
            want.append(step(blk, caches[0], x[:, t : t + 1].contiguous(), table)[1])
        cache, at = caches[1], 0
        for t in range(34):
            paused = 8 <= t < 18
            if t == 8:
                cache.active[1] = 0
                before = held_by(cache, 1)
            if t == 18:
                cache.active[1] = 1
            cache.reserve(0)
            if not paused:
                cache.reserve(1)
            xt = torch.stack([x[0, min(t, 23)], torch.full_like(x[1, 0], float("nan")) if paused else x[1, at]])[:, None]
            got = step(blk, cache, xt, table)
            if paused:
                assert unchanged(cache, 1, before)
            else:
                assert torch.equal(got[1], want[at]), t
                at += 1
        assert at == 24 and cache.lens.tolist() == [34, 24]


def test_replayed_steps_pass_over_streams_that_are_not_reserved():
    """One captured step: streams join, wait at a full page and in the middle of one, and go on."""
    blk, table = model.random_block(CFG, device="cuda", seed=50), freqs()
    x = randn_bf16((3, 40, CFG.dim), seed=51, device="cuda")
    waits = [set(), set(range(16, 20)) | set(range(25, 28)), set(range(5))]
    caches = [pagedkv.PagedKVCache(1, 3, 128, 12, 2, page_size=16, device="cuda") for _ in range(2)]
    xt, out = torch.empty(3, 1, CFG.dim, dtype=torch.bfloat16, device="cuda"), None
    side = torch.cuda.Stream()
    with torch.inference_mode():
        want = []
        with torch.cuda.stream(side):
            for t in range(40):
                for s in range(3):
                    caches[0].reserve(s)
                want.append(step(blk, caches[0], x[:, t : t + 1].contiguous(), table)[:, 0].clone())
            graph, cache = torch.cuda.CUDAGraph(), caches[1]
            with torch.cuda.graph(graph, stream=side):
                out = step(blk, cache, xt, table)
        torch.cuda.synchronize()
        at = [0, 0, 0]
        for t in range(40):
            parts = [t not in w for w in waits]
            before = [held_by(cache, s) for s in range(3)]
            for s in range(3):
                xt[s, 0] = x[s, at[s]] if parts[s] else float("nan")
                if parts[s]:
                    cache.reserve(s)
            graph.replay()
            for s in range(3):
                if parts[s]:
                    assert torch.equal(out[s, 0], want[at[s]][s]), (s, t)
                    at[s] += 1
                else:
                    assert torch.equal(cache.lens[s], before[s][4]) and torch.equal(cache.next_pos[s], before[s][5])
                    assert all(torch.equal(a[: len(b)], b) for a, b in zip(held_by(cache, s)[:4], before[s][:4]))
        assert cache.lens.tolist() == at == [40, 33, 35]
        del graph


@pytest.mark.parametrize("captured", [False, True])
def test_positions_past_the_rotary_table_are_passed_over(captured):
    """A bounded stream runs on until its positions reach the table's end and stops there, unchanged."""
    blk, table = model.random_block(CFG, device="cuda", seed=60), freqs(40)
    caches = [pagedkv.PagedKVCache(1, 2, 64, 8, 2, page_size=16, device="cuda") for _ in range(2)]
    x = randn_bf16((2, 1, CFG.dim), seed=61, device="cuda")
    side, cache = torch.cuda.Stream(), caches[1]
    with torch.inference_mode(), torch.cuda.stream(side):
        step(blk, caches[0], x, table)
        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph, stream=side):
                step(blk, cache, x, table)
        for t in range(50):
            cache.reserve(0)
            before = held_by(cache, 0)
            graph.replay() if captured else step(blk, cache, x, table)
            assert t < 40 or unchanged(cache, 0, before)
            if cache.lens[0] >= 30 and t < 40:
                cache.evict_and_trim(16, recent=4, sink=1)
            if t >= 40:
                cache.trim(0, int(cache.lens[0]))
        assert cache.next_pos.tolist() == [40, 0] and cache.part.tolist() == [0, 0]
        del graph
    torch.cuda.synchronize()


def test_steps_of_streams_reserved_together():
    """The host runs ahead: each step goes by the reservations made before it, none by a later one."""
    cache = pagedkv.PagedKVCache(1, 4, 256, 64, 2, page_size=16, device="cuda", track=False)
    g = torch.Generator().manual_seed(3)
    parts, seen = [], []
    torch.cuda._sleep(int(2e8))
    for _ in range(100):
        seqs = [s for s in range(4) if torch.rand((), generator=g) < 0.5]
        cache.reserve(seqs)
        cache.begin_step()
        cache.end_step()
        parts.append([int(s in seqs) for s in range(4)])
        seen.append(cache.part.clone())
    assert torch.stack(seen).tolist() == parts
    assert cache.lens.tolist() == [sum(p[s] for p in parts) for s in range(4)]
