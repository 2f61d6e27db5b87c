"""The paged KV cache's operators where inputs are not finite or tables have gaps, against NumPy in
64 bits, with the bounds of test_gpu_pagedkv.py (B200 only)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from tests.test_gpu_pagedkv import DT, Pool, attend, f64, one_rounding
from ttspipe_b200 import nf4gemv, pagedkv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def available():
    assert nf4gemv.available()


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(8, 2), (16, 1)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("val", [np.nan, np.inf])
def test_a_score_that_is_not_finite_reaches_the_weights_of_visible_rows_only(val, masked, heads, name):
    """Sequence 0 has 20 rows, the other 12 rows of its second page are sequence 1's; rows 7 and 18 may be masked."""
    p = Pool([20, 48, 40, 700], n_kv=heads[1], page=16, dtype=DT[name], seed=3)
    shared, g = int(p.table[0, 1]), torch.Generator().manual_seed(2)
    p.table[1, 1] = shared
    for t in (p.k, p.v):
        t[shared] = torch.randn(heads[1], 16, 128, generator=g).to(DT[name]).cuda()
    p.k[int(p.table[0, 0]), 0, 2, 5] = float(val)
    p.k[int(p.table[3, 40]), 0, 1, 9] = float(val)
    q = torch.randn(4, heads[0], 128, generator=g).abs().to(DT[name]).cuda()
    mask = None
    if masked:
        mask = torch.ones(4, p.table.shape[1] * 16, dtype=torch.bool, device="cuda")
        mask[0, 7] = mask[0, 18] = mask[3, 5] = mask[3, 699] = False
    got = attend(p, q, weight=p.weight, mask=mask)
    want, added, _ = po.attention(f64(q), f64(p.k), f64(p.v), p.table.cpu().numpy(), p.lens_host, scale=128 ** -0.5,
                                  mask=None if mask is None else mask.cpu().numpy())
    w, nan = p.weight.cpu().numpy(), np.isnan(added)
    assert nan.any() and np.array_equal(np.isnan(w), nan)
    assert np.all(np.abs(w - added)[~nan] <= 2.0 ** -13 * added[~nan])
    assert np.array_equal(np.isnan(f64(got)), np.isnan(want))


@pytest.mark.parametrize("n,page,gone,budget,recent,sink", [
    (96, 16, [1], 48, 16, 0),          # a gap below the budget
    (96, 16, [0, 4], 48, 16, 3),       # the first page, and one that would move
    (96, 16, [5], 48, 16, 0),          # the newest rows are not there
    (70, 16, [1, 2], 40, 40, 0),       # the budget ends in a page that is assigned, all places protected
    (70, 16, [2], 40, 4, 2),           # the budget ends inside the gap
    (70, 16, [0, 1, 2, 3, 4], 30, 3, 1),  # nothing is there
    (3000, 48, [3, 7, 20, 61], 1111, 200, 5),
    (9001, 64, list(range(10, 40)), 4000, 64, 4),
    (40000, 128, [1, 2, 100, 200, 311], 20001, 2000, 16),
])
@pytest.mark.parametrize("inplace", [False, True])
def test_evict_of_a_table_with_unassigned_pages(n, page, gone, budget, recent, sink, inplace):
    """The places below the budget that have a page go to the best of the rows that have one."""
    p = Pool([n, 50], n_kv=2, page=page, dtype=torch.bfloat16, seed=n)
    tab = p.table.cpu().numpy()
    tab[0, gone] = [-1 if i % 2 else p.n_pages + i for i in range(len(gone))]
    p.table.copy_(torch.from_numpy(tab))
    rng = np.random.default_rng(n)
    k0, v0, left = p.k.clone(), p.v.clone(), min(n, budget)
    pg, at = po.slots(tab[0], np.arange(n), p.n_pages, page)
    there = np.nonzero(pg >= 0)[0]
    w, pos = rng.random((2, n)).astype(np.float32).round(2), np.stack([rng.permutation(n) for _ in range(2)])
    for h in range(2):
        p.weight[pg[there], h, at[there]] = torch.as_tensor(w[h, there], device="cuda")
        p.position[pg[there], h, at[there]] = torch.as_tensor(pos[h, there], dtype=torch.int32, device="cuda")
    outs = (p.weight, p.position, p.lens) if inplace else \
        (torch.full_like(p.weight, -7.0), torch.full_like(p.position, -7), torch.full_like(p.lens, -7))
    pagedkv.evict(p.k, p.v, p.weight, p.position, p.table, p.lens, budget=budget, recent=recent, sink=sink,
                  weight_out=outs[0], position_out=outs[1], lens_out=outs[2])
    assert outs[2].tolist() == [left, min(50, budget)]
    inside = there[there < left]
    k1, v1 = k0.clone(), v0.clone()
    for h in range(2):
        keep = np.zeros(n, bool)
        if len(inside):
            keep[there] = po.kept(w[h, there], pos[h, there], len(inside), recent, sink)
        to, src = inside[~keep[inside]], there[(there >= left) & keep[there]]
        assert len(to) == len(src)
        k1[pg[to], h, at[to]], v1[pg[to], h, at[to]] = k0[pg[src], h, at[src]], v0[pg[src], h, at[src]]
        new = np.arange(n)
        new[to] = src
        assert np.array_equal(outs[0][pg[inside], h, at[inside]].cpu().numpy(), w[h, new[inside]])
        assert np.array_equal(outs[1][pg[inside], h, at[inside]].cpu().numpy(), pos[h, new[inside]])
    mine = np.zeros(p.n_pages, bool)
    mine[pg[there]] = True
    for now, want in ((p.k, k1), (p.v, v1)):
        now, want = now[torch.from_numpy(mine).cuda()], want[torch.from_numpy(mine).cuda()]
        assert torch.equal(now.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(8, 2), (16, 1)])
@pytest.mark.parametrize("n", [300, 9000])
def test_attention_of_infinite_values(n, heads, name):
    """An infinity in a visible value is one of the output's, opposite ones are NaN; no other dimension notices."""
    p = Pool([n, 40], n_kv=heads[1], page=16, dtype=DT[name], seed=5)
    q = torch.randn(2, heads[0], 128, generator=torch.Generator().manual_seed(4)).to(DT[name]).cuda()
    for s, r, d, val in ((0, 3, 7, np.inf), (0, n - 100, 9, -np.inf), (0, 5, 11, np.inf), (0, n - 10, 11, -np.inf),
                         (0, n - 1, 127, np.nan), (1, 39, 0, np.inf), (1, 0, 0, np.inf)):
        p.v[int(p.table[s, r // 16]), :, r % 16, d] = float(val)
    with np.errstate(invalid="ignore"):
        want, _, size = po.attention(f64(q), f64(p.k), f64(p.v), p.table.cpu().numpy(), p.lens_host, scale=128 ** -0.5)
    got = attend(p, q, weight=p.weight)
    odd = ~np.isfinite(want)
    assert odd[0].sum(0).any() and np.array_equal(f64(got)[odd], want[odd], equal_nan=True)
    want[odd], size[odd] = 0.0, 0.0
    assert one_rounding(got.masked_fill(torch.from_numpy(odd).cuda(), 0), want, 2.0 ** -14 * size)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_attention_of_an_infinite_value_of_the_largest_and_of_a_small_weight(name):
    """Weight 1 exactly, and 2^-20 exactly, leave nothing when they are cut to 16 bits; a score of -inf has no weight."""
    p = Pool([3, 3], n_kv=1, page=16, dtype=DT[name], seed=6)
    q = torch.zeros(2, 1, 128, dtype=DT[name], device="cuda")
    q[..., 0] = 1.0
    for s in range(2):
        pg = int(p.table[s, 0])
        p.k[pg, 0, :3] = 0.0
        p.k[pg, 0, :3, 0] = torch.tensor([0.0, -20.0, -20.0], dtype=DT[name])
        p.v[pg, 0, :3] = 1.0
        p.v[pg, 0, 0, 0] = p.v[pg, 0, 1, 1] = float("inf")
    got = attend(p, q, scale=float(np.log(2.0)))
    assert torch.isinf(got[:, 0, :2]).all() and (got[:, 0, 2:] == 1).all()
    p.k[int(p.table[0, 0]), 0, 0, 0] = float("-inf")  # its value is infinite: 0 * inf, as the formula
    got = attend(p, q, scale=float(np.log(2.0)))
    assert torch.isnan(got[0, 0, 0]) and torch.isinf(got[0, 0, 1]) and (got[0, 0, 2:] == 1).all()
