"""The paged KV cache's operators where inputs are not finite or tables have gaps, against NumPy in
64 bits, with the bounds of test_gpu_pagedkv.py (B200 only)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from tests.test_gpu_pagedkv import DT, Pool, attend, f64
from ttspipe_b200 import nf4gemv

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
