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
