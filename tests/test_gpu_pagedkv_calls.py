"""The paged KV cache's Python calls on the B200: what they refuse of tensors, with the cache left as it was."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_pagedkv import Pool
from ttspipe_b200 import _lib, model, nf4gemv, pagedkv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def available():
    assert nf4gemv.available()


def arguments():
    """Of each call, all served; `name` of one is replaced by a test."""
    p = Pool([40, 9], n_kv=2, page=16, dtype=torch.bfloat16, seed=1)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = dict(k=p.k, v=p.v, block_table=p.table, weight=p.weight)
    return {
        "write": dict(cache, position=p.position, qkv=torch.zeros(3, 12 * 128, dtype=torch.bfloat16, device="cuda"),
                      rows=torch.zeros(3, **i32), positions=torch.zeros(3, **i32), seqs=torch.zeros(3, **i32),
                      freqs=model.precompute_freqs_cis(20, 128, 1e6, device="cuda"), n_head=8),
        "attention": dict(cache, q=torch.zeros(2, 8, 128, dtype=torch.bfloat16, device="cuda"), lens=p.lens,
                          mask=torch.ones(2, p.table.shape[1] * 16, dtype=torch.bool, device="cuda")),
        "evict": dict(cache, position=p.position, lens=p.lens, budget=8),
    }


TENSORS = [("write", n) for n in ("k", "v", "block_table", "weight", "position", "qkv", "rows", "positions", "seqs",
                                  "freqs")] + \
          [("attention", n) for n in ("v", "block_table", "weight", "q", "lens", "mask")] + \
          [("evict", n) for n in ("v", "block_table", "weight", "position", "lens")]


@pytest.mark.parametrize("call,name", TENSORS)
def test_tensors_of_another_shape_type_layout_or_device_are_refused(call, name):
    a = arguments()[call]
    before = {n: t.clone() for n, t in a.items() if isinstance(t, torch.Tensor)}
    t = a[name]
    wrong = [t.unsqueeze(0), t.double(), t.cpu()]
    if name in ("k", "freqs"):
        wrong.append(t[..., :1].contiguous())
    elif (call, name) != ("write", "block_table"):  # there any number of sequences is one
        wrong.append(t[:-1])
    if t.dim() > 1:
        wrong.append(t.transpose(0, 1).contiguous().transpose(0, 1))
    else:
        wrong.append(t.repeat_interleave(2)[::2])
    for w in wrong:
        with pytest.raises(ValueError, match=r"needed, got|not served|\(\d+, \d+"):
            getattr(pagedkv, call)(**dict(a, **{name: w}))
    with pytest.raises(TypeError):
        getattr(pagedkv, call)(**dict(a, **{name: 5})) if name != "k" else pagedkv._bound().write(5)
    torch.cuda.synchronize()
    for n, t in before.items():
        assert torch.equal(a[n].view(torch.uint8), t.view(torch.uint8))


def test_what_the_library_refuses_names_the_numbers():
    a = arguments()
    with pytest.raises(_lib.Nf4bError, match="17 query heads"):
        pagedkv.attention(**dict(a["attention"], q=torch.zeros(2, 34, 128, dtype=torch.bfloat16, device="cuda")))
    with pytest.raises(_lib.Nf4bError, match="budget 8"):
        pagedkv.evict(**dict(a["evict"], recent=9))
    with pytest.raises(ValueError, match="out of range"):
        pagedkv.evict(**dict(a["evict"], budget=2**31))
    for call in a:  # as they are, they are served
        getattr(pagedkv, call)(**a[call])
    torch.cuda.synchronize()
