"""The transformer block over a paged cache, its launches replaced by the products and copies that they
are documented to be (runs without a GPU): what the block makes of its linears and of the cache."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from ttspipe_b200 import fastpath, fusedops, model, nf4gemv, pagedkv

DIM, HEADS, KV = 64, 2, 1
CFG = model.ModelArgs(dim=DIM, n_head=HEADS, n_local_heads=KV, intermediate_size=96, max_seq_len=64)


def _matmul(module, x, *, epi=nf4gemv.EPI_NONE, operand=None, prefetch=None, norm=None):
    if norm is not None:
        x = _rms_norm(x, *norm)
    y = x @ module.dense.T
    if epi == nf4gemv.EPI_RESIDUAL:
        return operand + y
    return F.silu(operand) * y if epi == nf4gemv.EPI_SILU_GATE else y


def _rms_norm(x, weight, eps):
    xf = x.float()
    return (xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)).to(x.dtype) * weight


def _write(qkv, k, v, block_table, rows, positions, freqs, *, n_head, seqs=None, weight=None, position=None, **_):
    heads = qkv.view(len(rows), -1, 128)
    for t in range(len(rows)):
        s, r, pos = t if seqs is None else int(seqs[t]), int(rows[t]), int(positions[t])
        if r < 0 or not 0 <= pos < len(freqs) or r >= block_table.shape[1] * k.shape[2]:
            continue
        page, at = int(block_table[s, r // k.shape[2]]), r % k.shape[2]
        if page < 0:
            continue
        k[page, :, at], v[page, :, at] = heads[t, n_head:n_head + k.shape[1]], heads[t, n_head + k.shape[1]:]
        if weight is not None:
            weight[page, :, at], position[page, :, at] = 0.0, pos
    return heads[:, :n_head].clone()


def _attention(q, k, v, block_table, lens, *, weight=None, **_):
    """The mean of the rows; each of them is attended to equally."""
    out = torch.zeros_like(q)
    for s, n in enumerate(lens.tolist()):
        for r in range(n):
            page, at = int(block_table[s, r // k.shape[2]]), r % k.shape[2]
            out[s] += v[page, :, at].repeat_interleave(q.shape[1] // k.shape[1], 0) / n
            if weight is not None:
                weight[page, :, at] += q[s].sum() * 0 + q.shape[1] / k.shape[1] / n
    return out


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    monkeypatch.setattr(nf4gemv, "prepare", lambda module: setattr(module, "_nf4_fast", {}) or True)
    monkeypatch.setattr(nf4gemv, "matmul", _matmul)
    monkeypatch.setattr(nf4gemv, "matmul_gated", lambda w1, w3, x, *, prefetch=None, norm=None: _matmul(
        w3, x, norm=norm, epi=nf4gemv.EPI_SILU_GATE, operand=_matmul(w1, x, norm=norm)))
    monkeypatch.setattr(fusedops, "rms_norm", _rms_norm)
    monkeypatch.setattr(pagedkv, "write", _write)
    monkeypatch.setattr(pagedkv, "attention", _attention)


def make_block(biases=()):
    g = torch.Generator().manual_seed(1)
    blk = model.TransformerBlock(CFG)
    for norm in (blk.attention_norm, blk.ffn_norm):
        norm.weight = torch.nn.Parameter(torch.ones(DIM), requires_grad=False)
    a, ff = blk.attention, blk.feed_forward
    for name, lin in (("wqkv", a.wqkv), ("wo", a.wo), ("w1", ff.w1), ("w3", ff.w3), ("w2", ff.w2)):
        lin.dense = torch.randn(lin.out_features, lin.in_features, generator=g) / lin.in_features ** 0.5
        bias = torch.randn(lin.out_features, generator=g)
        lin.bias = torch.nn.Parameter(bias, requires_grad=False) if name in biases else None
    return blk


def make_cache(n_seqs=2, **kw):
    return pagedkv.PagedKVCache(1, n_seqs, 64, 8, KV, page_size=16, device="cpu", dtype=torch.float32, **kw)


def block_alone(blk, x):
    """The block's own formula for tokens of one stream, each attending to all so far by the mean."""
    def linear(lin, y):
        return y @ lin.dense.T + (0 if lin.bias is None else lin.bias)

    v = linear(blk.attention.wqkv, _rms_norm(x, blk.attention_norm.weight, CFG.norm_eps))[..., -128 * KV:]
    mean = v.cumsum(-2) / torch.arange(1, x.shape[-2] + 1)[:, None]
    h = x + linear(blk.attention.wo, mean.repeat(1, HEADS // KV))
    hn, ff = _rms_norm(h, blk.ffn_norm.weight, CFG.norm_eps), blk.feed_forward
    return h + linear(ff.w2, F.silu(linear(ff.w1, hn)) * linear(ff.w3, hn))


FREQS = torch.zeros(64, 64, 2)
BIASES = [(), ("wqkv",), ("wo",), ("w1",), ("w3",), ("w2",), ("wqkv", "wo", "w1", "w3", "w2")]


@pytest.mark.parametrize("biases", BIASES)
def test_decode_adds_the_biases(biases):
    blk, cache = make_block(biases), make_cache()
    x = torch.randn(2, 3, DIM, generator=torch.Generator().manual_seed(2))
    want = torch.stack([block_alone(blk, x[s]) for s in range(2)])
    for t in range(3):
        for s in range(2):
            cache.reserve(s)
        cache.begin_step()
        got = pagedkv.decode_block(blk, x[:, t:t + 1], FREQS, cache, 0)
        cache.end_step()
        assert torch.allclose(got[:, 0], want[:, t], atol=1e-4)


@pytest.mark.parametrize("biases", BIASES)
def test_prefill_adds_the_biases(biases, monkeypatch):
    def mean(q, k, v, mask, n_head, n_kv, d):
        m = mask[0, 0].float()
        return (m @ v / m.sum(-1, keepdim=True)).repeat_interleave(n_head // n_kv, 1)

    monkeypatch.setattr(fastpath, "_grouped_torch", mean)
    blk, cache = make_block(biases), make_cache()
    x = torch.randn(1, 5, DIM, generator=torch.Generator().manual_seed(3))
    cache.reserve(1, 5)
    got = pagedkv.prefill_block(blk, x, FREQS, cache, 0, 1)
    assert torch.allclose(got[0], block_alone(blk, x[0]), atol=1e-4)


def step(blk, cache, x):
    cache.begin_step()
    out = pagedkv.decode_block(blk, x, FREQS, cache, 0)
    cache.end_step()
    return out


def held_by(cache, seq):
    """Everything the cache holds of a stream."""
    pages = [p for p in cache.block_table[seq].tolist() if p >= 0]
    pools = (cache.k[0], cache.v[0], cache.weight[0], cache.position[0])
    return [t[pages].clone() for t in pools] + [cache.lens[seq].clone(), cache.next_pos[seq].clone()]


def unchanged(cache, seq, before):
    return all(torch.equal(a, b) for a, b in zip(held_by(cache, seq), before))


def test_a_stream_that_is_not_active_is_passed_over():
    """Whatever its slot of x holds: no row, no weight, no length of it changes, and it goes on as if nothing had been."""
    blk, cache = make_block(), make_cache()
    x = torch.randn(2, 9, DIM, generator=torch.Generator().manual_seed(4))
    for t in range(3):
        for s in range(2):
            cache.reserve(s)
        step(blk, cache, x[:, t:t + 1])
    cache.active[1] = 0
    before = held_by(cache, 1)
    for t in range(3, 6):
        cache.reserve(0)
        mixed = x[:, t:t + 1].clone()
        mixed[1] = float("nan")
        got = step(blk, cache, mixed)
        assert torch.allclose(got[0, 0], block_alone(blk, x[0])[t], atol=1e-4)
        assert cache.live[1] == 0 and unchanged(cache, 1, before)
    cache.active[1] = 1
    cache.reserve(1)
    got = step(blk, cache, x[:, 3:4])
    assert torch.allclose(got[1, 0], block_alone(blk, x[1])[3], atol=1e-4) and cache.lens.tolist()[1] == 4


def test_a_stream_that_is_not_reserved_is_passed_over():
    """A stream of 16 rows, its page full, then steps that reserve only the other one; and one in the middle of a page."""
    blk, cache = make_block(), make_cache()
    x = torch.randn(2, 40, DIM, generator=torch.Generator().manual_seed(5))
    alone = [block_alone(blk, x[s]) for s in range(2)]
    n = [0, 0]
    for t in range(40):
        parts = [True, not (16 <= t < 20 or 25 <= t < 28)]
        before = held_by(cache, 1)
        for s in range(2):
            if parts[s]:
                cache.reserve(s)
        got = step(blk, cache, torch.stack([x[s, min(n[s], 39)] for s in range(2)])[:, None])
        assert cache.part.tolist() == [int(p) for p in parts]
        for s in range(2):
            if parts[s]:
                assert torch.allclose(got[s, 0], alone[s][n[s]], atol=1e-4), (s, t)
                n[s] += 1
        assert parts[1] or unchanged(cache, 1, before)
        assert cache.lens.tolist() == n and cache.next_pos.tolist() == n
        assert all(cache.lens[s] <= cache._rows[s] for s in range(2))


def test_rows_reserved_ahead_last_for_as_many_steps():
    blk, cache = make_block(), make_cache()
    x = torch.randn(2, 7, DIM, generator=torch.Generator().manual_seed(6))
    cache.reserve(0, 5)
    cache.reserve(1, 7)
    for t in range(7):
        got = step(blk, cache, x[:, t:t + 1])
        assert torch.allclose(got[1, 0], block_alone(blk, x[1])[t], atol=1e-4)
    assert cache.lens.tolist() == [5, 7]


def test_a_prompt_is_filled_in_while_others_decode(monkeypatch):
    def mean(q, k, v, mask, n_head, n_kv, d):
        m = mask[0, 0].float()
        return (m @ v / m.sum(-1, keepdim=True)).repeat_interleave(n_head // n_kv, 1)

    monkeypatch.setattr(fastpath, "_grouped_torch", mean)
    blk, cache = make_block(), make_cache()
    x = torch.randn(2, 30, DIM, generator=torch.Generator().manual_seed(7))
    alone = [block_alone(blk, x[s]) for s in range(2)]
    at = 0

    def decode(both=False):
        nonlocal at
        cache.reserve(0)
        if both:
            cache.reserve(1)
        got = step(blk, cache, torch.stack([x[0, at], x[1, int(cache.lens[1]) if both else 0]])[:, None])
        assert torch.allclose(got[0, 0], alone[0][at], atol=1e-4)
        at += 1
        return got[1, 0]

    decode()
    cache.reserve(1, 20, prompt=True)
    decode()
    got = pagedkv.prefill_block(blk, x[1:, :13], FREQS, cache, 0, 1)
    assert torch.allclose(got[0], alone[1][:13], atol=1e-4)
    decode()
    cache.prefilled(1, 13)
    decode()
    got = pagedkv.prefill_block(blk, x[1:, 13:20], FREQS, cache, 0, 1, rows=13, position=13)
    assert torch.allclose(got[0], alone[1][13:20], atol=1e-4)
    decode()
    cache.prefilled(1, 7)
    assert cache.lens.tolist() == [5, 20] and cache.next_pos.tolist() == [5, 20]
    decode()  # nothing is reserved for its next token yet
    for t in range(20, 25):
        assert torch.allclose(decode(both=True), alone[1][t], atol=1e-4)
    assert cache.lens.tolist() == [11, 25]


def test_while_a_prompt_is_filled_in_nothing_takes_its_rows():
    cache = make_cache()
    cache.reserve(0, 20)
    cache.reserve(1, 20, prompt=True)
    for call in (lambda: cache.evict(8), lambda: cache.evict_and_trim(8), lambda: cache.trim(1, 8)):
        with pytest.raises(RuntimeError, match="prompt"):
            call()
    for rows in (21, -1):
        with pytest.raises(ValueError, match="20 are reserved"):
            cache.prefilled(1, rows)
    with pytest.raises(ValueError, match="0 are reserved"):
        cache.prefilled(0, 1)
    assert cache.active.tolist() == [1, 0] and cache.lens.tolist() == [0, 0]
    cache.release(1)
    cache.trim(0, 8)
    cache.reserve(1)
    assert cache.active.tolist() == [1, 1] and cache.free_pages() == 6


def test_rows_taken_back_by_a_trim_are_not_stepped_into():
    cache = make_cache(track=False)
    cache.reserve(0, 40)  # ahead
    cache.lens[0] = 30
    cache.lens[0] = 20  # an eviction
    cache.trim(0, 20)
    cache.begin_step()
    assert cache.rows.tolist() == [-1, -1] and cache.part.tolist() == [0, 0]
    cache.reserve(0)
    cache.begin_step()
    assert cache.rows.tolist() == [20, -1] and cache.live.tolist() == [21, 0]


@pytest.mark.parametrize("rows,position", [(0, 0), (10, 10), (-1, 0)])
def test_prefill_refuses_rows_that_are_not_reserved(rows, position):
    blk, cache = make_block(), make_cache()
    cache.reserve(0, 20, prompt=True)
    cache.reserve(1, 20, prompt=True)
    before = cache.k[0].clone()
    with pytest.raises(ValueError, match="reserved"):
        pagedkv.prefill_block(blk, torch.randn(1, 21, DIM), FREQS, cache, 0, 1, rows=rows, position=position)
    assert torch.equal(cache.k[0], before)


def test_positions_past_the_rotary_table_are_passed_over():
    """An evicted stream's positions run ahead of its rows: at the table's end it stops, with nothing changed."""
    blk, cache = make_block(), make_cache()
    x = torch.randn(2, 9, DIM, generator=torch.Generator().manual_seed(8))
    cache.reserve(0)
    step(blk, cache, x[:, :1])  # the longer table is seen first
    cache.next_pos[0] = 3
    cache.reserve(0, 4)
    cache.reserve(1, 9)
    for t in range(8):
        if t >= 3:
            before = held_by(cache, 0)
        cache.begin_step()
        pagedkv.decode_block(blk, x[:, t:t + 1], FREQS[:6], cache, 0)
        cache.end_step()
        assert t < 3 or unchanged(cache, 0, before)
    assert cache.lens.tolist() == [4, 6] and cache.next_pos.tolist() == [6, 6]
    assert cache.part.tolist() == [0, 0] and cache.live.tolist() == [0, 0]
    cache.release(0)
    cache.reserve(0)
    cache.begin_step()
    assert cache.part.tolist() == [1, 0]


@pytest.mark.parametrize("rows,position", [(0, 2), (0, -1)])
def test_prefill_refuses_positions_outside_the_rotary_table(rows, position):
    blk, cache = make_block(), make_cache()
    cache.reserve(0, 5, prompt=True)
    with pytest.raises(ValueError, match="rotary"):
        pagedkv.prefill_block(blk, torch.randn(1, 5, DIM), FREQS[:6], cache, 0, 0, rows=rows, position=position)


def test_streams_reserved_together_are_reserved_as_one_after_the_other():
    caches = [make_cache(4, track=False) for _ in range(2)]
    rng = torch.Generator().manual_seed(9)
    for t in range(30):
        seqs = [s for s in range(4) if torch.rand((), generator=rng) < 0.6]
        rows = 1 + t % 2
        try:
            caches[0].reserve(seqs, rows)
        except RuntimeError:
            break
        for s in seqs:
            caches[1].reserve(s, rows)
        for c in caches:
            c.begin_step()
            c.end_step()
        for name in ("lens", "next_pos", "active", "block_table", "part", "rows", "_below", "_at"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
        assert caches[0]._pages == caches[1]._pages and caches[0]._rows == caches[1]._rows
    assert t > 10 and caches[0].free_pages() < 3


def test_a_joint_reservation_that_does_not_fit_changes_nothing():
    c = make_cache(4, track=False)
    c.reserve([0, 2], 30)
    state = [c.block_table.clone(), c._below.clone(), list(c._rows), list(c._free)]
    for seqs, rows, error, match in (([1, 3, 0], 33, RuntimeError, "stream 3 needs 3 pages, 1 are free"),
                                     ([1, 0], 35, ValueError, "stream 0: at most 64"), ([1, 1], 1, ValueError, "twice"),
                                     ([1, 2], -1, ValueError, "at most")):
        with pytest.raises(error, match=match):
            c.reserve(seqs, rows)
        assert torch.equal(c.block_table, state[0]) and torch.equal(c._below, state[1])
        assert c._rows == state[2] and c._free == state[3]
    c.reserve([], 5)
    c.reserve(range(4))
    assert c._rows == [31, 1, 31, 1]


def test_only_a_steps_own_table_bounds_its_positions():
    """Rows written with positions of one's own, from part of the table, say nothing about the steps."""
    blk, cache = make_block(), make_cache()
    at = torch.arange(5, dtype=torch.int32)
    cache.reserve(0, 5, prompt=True)
    cache.write(0, torch.randn(5, (HEADS + 2 * KV) * 128), at, at, FREQS[:5], n_head=HEADS, seqs=torch.zeros_like(at))
    cache.prefilled(0, 5)
    cache.reserve([0, 1])
    step(blk, cache, torch.randn(2, 1, DIM))
    assert cache.part.tolist() == [1, 1] and cache.lens.tolist() == [6, 1]


def test_a_longer_rotary_table_lets_streams_go_on():
    blk, cache = make_block(), make_cache()
    cache.reserve([0, 1], 20)

    def steps(n, table):
        for _ in range(n):
            cache.begin_step()
            pagedkv.decode_block(blk, torch.randn(2, 1, DIM), table, cache, 0)
            cache.end_step()

    steps(8, FREQS[:6])
    assert cache.lens.tolist() == [6, 6]
    steps(4, FREQS)
    assert cache.lens.tolist() == [10, 10] and cache.next_pos.tolist() == [10, 10]
    steps(2, FREQS[:7])
    assert cache.lens.tolist() == [10, 10]


def test_a_prompt_that_fills_the_rotary_table_is_not_stepped_past():
    """The cache learns of the table with the step's first layer, and the step goes by it all the same."""
    blk, cache = make_block(), make_cache()
    cache.reserve(0, 6, prompt=True)
    cache.prefilled(0, 6)
    cache.reserve([0, 1])
    before = held_by(cache, 0)
    cache.begin_step()
    pagedkv.decode_block(blk, torch.randn(2, 1, DIM), FREQS[:6], cache, 0)
    cache.end_step()
    assert unchanged(cache, 0, before) and cache.part.tolist() == [0, 1] and cache.lens.tolist() == [6, 1]
