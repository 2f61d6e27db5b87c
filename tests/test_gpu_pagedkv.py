"""The paged KV cache's operators on the B200, against NumPy in 64 bits
(oracle/paged_oracle.py) and against the dense cache's kernels.

Bounds. Before the attention's one rounding: a score is a sum of 128 products in fp32,
8 MMA steps that may each truncate at 2^-23 of the running size, so |ds| <= 16 * 2^-23 *
sum|q k| * scale, and with N(0, 1) entries sum|q k| * scale is about 8, below 16: 2^-15;
exp2 and the fp32 sums add less than 2^-20, the weights' two 16-bit parts 2^-17. All
scale with sum p|v|: 2^-14 of it is allowed. The rounding itself is checked exactly: an output
lies between the roundings of the exact value less and plus that slack. A row's
accumulated weight carries the scores' error twice (numerator and sum): 2^-13 of it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from tests.helpers import randn_bf16
from ttspipe_b200 import _lib, fastpath, model, nf4gemv, pagedkv

pytestmark = pytest.mark.gpu

FTYPE = {torch.float32: _lib.NF4B_F32, torch.float16: _lib.NF4B_F16, torch.bfloat16: _lib.NF4B_BF16}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}  # one rounding to nearest, relative


@pytest.fixture(scope="module", autouse=True)
def available():
    assert nf4gemv.available()


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


class Pool:
    """A cache of random rows whose sequences own scattered pages; every row outside
    the sequences holds NaN."""

    def __init__(self, lens, *, n_kv, page, dtype, width=None, seed=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens_host, self.page, self.n_kv = list(lens), page, n_kv
        need = [-(-max(n, 0) // page) for n in lens]
        width = width or max(1, max(need))
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at : at + n].int()
            at += n
        shape = (self.n_pages, n_kv, page, 128)
        k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
        live = torch.zeros(self.n_pages, page, dtype=torch.bool)
        for s, n in enumerate(lens):
            for r in range(max(n, 0)):
                live[table[s, r // page], r % page] = True
        for t in (k, v):
            t.transpose(1, 2)[~live] = float("nan")
        self.table, self.k, self.v = table.cuda(), k.cuda(), v.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.weight = torch.zeros(shape[:3], device="cuda")
        self.position = torch.zeros(shape[:3], dtype=torch.int32, device="cuda")
        self.dtype = dtype


def attend(p, q, **kw):
    return pagedkv.attention(q, p.k, p.v, p.table, p.lens, **kw)


def one_rounding(got, want, slack):
    """`got` is a rounding of something within `slack` of `want`."""
    lo, hi = (f64(torch.from_numpy(x).to(got.dtype)) for x in (want - slack, want + slack))
    return bool(np.all((lo <= f64(got)) & (f64(got) <= hi)))


def check_attention(p, q, name, *, mask=None, scale=None, got=None, weight=None):
    want, added, size = po.attention(f64(q), f64(p.k), f64(p.v), p.table.cpu().numpy(), p.lens_host,
                                     scale=128 ** -0.5 if scale is None else scale,
                                     mask=None if mask is None else mask.cpu().numpy())
    assert got.dtype == DT[name] and one_rounding(got, want, 2.0 ** -14 * size)
    if weight is not None:
        assert np.all(np.abs(weight.cpu().numpy() - added) <= 2.0 ** -13 * added), "weights"
    return want


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("lens", [[1], [16], [17, 0, 1], [129, 128, 127, 0, 33], [2049, 5]])
def test_attention_at_the_lengths_where_tiles_and_pages_end(lens, page, name):
    p = Pool(lens, n_kv=2, page=page, dtype=DT[name], seed=sum(lens) + page, width=-(-max(lens) // page) + 1)
    q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(7)).to(DT[name]).cuda()
    got = attend(p, q, weight=p.weight)
    check_attention(p, q, name, got=got, weight=p.weight)
    assert torch.equal(got, attend(p, q))  # the same with and without weights


@pytest.mark.parametrize("n_head,n_kv", [(8, 8), (3, 1), (12, 2), (8, 1), (9, 1), (26, 2), (16, 1), (32, 8)])
def test_attention_for_every_kind_of_head_group(n_head, n_kv):
    p = Pool([700, 65], n_kv=n_kv, page=64, dtype=torch.bfloat16, seed=n_head)
    q = randn_bf16((2, n_head, 128), seed=n_head, device="cuda")
    check_attention(p, q, "bf16", got=attend(p, q, weight=p.weight), weight=p.weight)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(8, 2), (16, 1)])
def test_attention_masks_hide_rows_whatever_they_hold(name, heads):
    p = Pool([300, 40, 64, 17], n_kv=heads[1], page=32, dtype=DT[name], seed=3)
    g = torch.Generator().manual_seed(9)
    width = p.table.shape[1] * p.page
    mask = (torch.rand(4, width, generator=g) < 0.6).cuda()
    mask[1] = False  # sees nothing
    mask[2] = False
    mask[2, 63] = True  # sees one row
    mask[3, :16] = False  # its first tile is hidden
    mask[3, 16] = True
    for s in range(4):
        for r in range(p.lens_host[s]):
            if not mask[s, r]:
                pg = int(p.table[s, r // p.page])
                p.k[pg, :, r % p.page] = float("nan") if r % 2 else float("inf")
                p.v[pg, :, r % p.page] = float("inf") if r % 2 else float("nan")
    q = torch.randn(4, heads[0], 128, generator=g).to(DT[name]).cuda()
    got = attend(p, q, mask=mask, weight=p.weight)
    check_attention(p, q, name, mask=mask, got=got, weight=p.weight)
    assert not got[1].any() and torch.equal(got, attend(p, q, mask=mask.to(torch.uint8)))


def test_attention_sharp_scores_and_scale():
    """A scale that lets one row win, and one that makes all equal: the running maximum
    and the fp16 weights' range."""
    for name in ("bf16", "fp16"):
        p = Pool([5000, 90], n_kv=1, page=16, dtype=DT[name], seed=21)
        q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(2)).to(DT[name]).cuda()
        for scale in (0.0, 1e-3):
            w = torch.zeros_like(p.weight)
            check_attention(p, q, name, scale=scale, got=attend(p, q, scale=scale, weight=w), weight=w)
        # scores of about +-45: |ds| is 45 / 4 times what the bounds above assume
        want, _, size = po.attention(f64(q), f64(p.k), f64(p.v), p.table.cpu().numpy(), p.lens_host, scale=1.0)
        assert one_rounding(attend(p, q, scale=1.0), want, 2.0 ** -10 * size)


def test_attention_small_weights_of_many_rows_count_in_fp16():
    """One row 17 above 60000 equal ones (e^17 = 2.4e7): those hold 0.25% of the sum, each
    below fp16's smallest number (2^-24) relative to the first."""
    n = 60001
    p = Pool([n], n_kv=1, page=16, dtype=torch.float16, seed=5)
    k, v = torch.zeros(n, 128), torch.ones(n, 128)
    k[12345, 0] = 17.0
    v[12345] = 3.0
    rows = torch.arange(n)
    tab = p.table[0].cpu().long()
    p.k[tab[rows // 16], 0, rows % 16] = k.half().cuda()
    p.v[tab[rows // 16], 0, rows % 16] = v.half().cuda()
    q = torch.zeros(1, 1, 128, dtype=torch.float16, device="cuda")
    q[0, 0, 0] = 1.0
    got = attend(p, q, scale=1.0)
    check_attention(p, q, "fp16", scale=1.0, got=got)


def test_attention_infinite_scores():
    """-inf scores are rows without weight (all of them: zeros); +inf and NaN give NaN,
    as the formula does."""
    p = Pool([40, 40, 40, 40], n_kv=1, page=16, dtype=torch.bfloat16, seed=8)
    q = torch.ones(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    for s, (rows, val) in enumerate([(range(40), -np.inf), (range(0, 40, 3), -np.inf), ([39], np.inf), ([0], np.nan)]):
        for r in rows:
            p.k[int(p.table[s, r // 16]), 0, r % 16, 5] = float(val)
    got = attend(p, q, weight=p.weight)
    assert not got[0].any() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    want, _, size = po.attention(f64(q)[:2], f64(p.k), f64(p.v), p.table.cpu().numpy()[:2], [40, 40], scale=128 ** -0.5)
    assert one_rounding(got[1], want[1], 2.0 ** -14 * size[1])
    first = p.table[0].cpu().long()
    assert not p.weight[first[0]].any()


def test_attention_lengths_and_tables_out_of_range():
    """Lengths past the capacity and below zero, and pages that are not assigned."""
    p = Pool([96, 96, 96], n_kv=2, page=32, dtype=torch.bfloat16, seed=4)
    q = randn_bf16((3, 8, 128), seed=5, device="cuda")
    p.table[1, 1] = -1
    p.table[2, 2] = p.n_pages
    p.lens_host = [1000, 96, 96]
    p.lens = torch.tensor(p.lens_host, dtype=torch.int32, device="cuda")
    check_attention(p, q, "bf16", got=attend(p, q, weight=p.weight), weight=p.weight)
    p.lens_host = [-5, 0, 1]
    p.lens = torch.tensor(p.lens_host, dtype=torch.int32, device="cuda")
    check_attention(p, q, "bf16", got=attend(p, q))


@pytest.mark.parametrize("n", [400, 4096])
def test_attention_many_short_sequences(n):
    lens = [(37 * i) % 70 for i in range(n)]
    p = Pool(lens, n_kv=2, page=16, dtype=torch.bfloat16, seed=6)
    q = randn_bf16((n, 8, 128), seed=6, device="cuda")
    check_attention(p, q, "bf16", got=attend(p, q, weight=p.weight), weight=p.weight)


@pytest.mark.parametrize("heads,lens", [((16, 1), [30000]), ((13, 1), [17, 12001, 12002]), ((4, 1), [70001]),
                                        ((32, 2), [9000, 1, 20000])])
def test_attention_of_sequences_in_very_many_parts(heads, lens):
    """Few heads of long sequences: so many parts that they are joined in two steps. Twice,
    with the counters back at zero in between."""
    p = Pool(lens, n_kv=heads[1], page=128, dtype=torch.bfloat16, seed=len(lens) + heads[0])
    q = randn_bf16((len(lens), heads[0], 128), seed=31, device="cuda")
    got = attend(p, q, weight=p.weight)
    check_attention(p, q, "bf16", got=got, weight=p.weight)
    assert torch.equal(got, attend(p, q))


def test_attention_pages_shared_by_two_sequences_collect_both_weights():
    p = Pool([64, 64], n_kv=1, page=32, dtype=torch.bfloat16, seed=12)
    p.table[1, 0] = p.table[0, 0]  # a common prefix
    q = randn_bf16((2, 4, 128), seed=13, device="cuda")
    check_attention(p, q, "bf16", got=attend(p, q, weight=p.weight), weight=p.weight)


def test_attention_repeats_bit_for_bit_and_adds_up():
    p = Pool([3000, 1, 517], n_kv=8, page=64, dtype=torch.bfloat16, seed=14)
    q = randn_bf16((3, 32, 128), seed=15, device="cuda")
    one = torch.zeros_like(p.weight)
    first = attend(p, q, weight=one)
    twice = torch.zeros_like(one)
    for _ in range(2):
        assert torch.equal(first, attend(p, q, weight=twice))
    assert torch.equal(twice, one + one)


def test_attention_equals_the_dense_cache_kernel_closely():
    """The dense kernel rounds scores to bf16 first: 2^-9 of a score of up to about 5."""
    p = Pool([2048], n_kv=8, page=64, dtype=torch.bfloat16, seed=16)
    q = randn_bf16((1, 32, 128), seed=17, device="cuda")
    tab = p.table[0].long()
    k, v = (t[tab].transpose(0, 1).reshape(1, 8, 2048, 128) for t in (p.k, p.v))
    mask = torch.ones(1, 1, 1, 2048, dtype=torch.bool, device="cuda")
    dense = fastpath.decode_attention(q.view(1, 32, 1, 128), k, v, mask, 32, 8, 128).view(1, 32, 128)
    got = attend(p, q)
    rel = (got.float() - dense.float()).norm() / dense.float().norm()
    assert rel < 1e-2


def test_attention_past_32_bit_offsets():
    """Pools of more than 2^32 bytes and 2^31 elements, the sequence in their last pages."""
    n_pages, n_kv, page = 2100, 8, 1024
    k = torch.empty(n_pages, n_kv, page, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    weight = torch.zeros(n_pages, n_kv, page, device="cuda")
    small = Pool([1500], n_kv=n_kv, page=page, dtype=torch.bfloat16, seed=18)
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    for i in range(2):
        k[n_pages - 1 - i], v[n_pages - 1 - i] = (t[int(small.table[0, i])] for t in (small.k, small.v))
    q = randn_bf16((1, 32, 128), seed=19, device="cuda")
    got = pagedkv.attention(q, k, v, table, small.lens, weight=weight)
    want = attend(small, q, weight=small.weight)
    assert torch.equal(got, want)
    assert torch.equal(weight[n_pages - 1], small.weight[int(small.table[0, 0])])
    position = torch.zeros(n_pages, n_kv, page, dtype=torch.int32, device="cuda")
    position[n_pages - 1] = torch.arange(page, dtype=torch.int32, device="cuda")
    position[n_pages - 2] = page + torch.arange(page, dtype=torch.int32, device="cuda")
    small.position[small.table[0].long()] = position[table[0].long()]
    a = pagedkv.evict(k, v, weight, position, table, small.lens.clone(), budget=700, recent=64, sink=1)
    b = pagedkv.evict(small.k, small.v, small.weight, small.position, small.table, small.lens.clone(), budget=700,
                      recent=64, sink=1)
    assert torch.equal(a, b) and int(a) == 700
    first, want = k[n_pages - 1, :, :700], small.k[int(small.table[0, 0]), :, :700]
    assert torch.equal(first, want) and torch.equal(v[n_pages - 1, :, :700], small.v[int(small.table[0, 0]), :, :700])


def test_attention_on_two_streams_at_once():
    p = Pool([4000] * 4, n_kv=8, page=64, dtype=torch.bfloat16, seed=23)
    qs = [randn_bf16((4, 32, 128), seed=30 + i, device="cuda") for i in range(2)]
    want = [attend(p, q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(attend(p, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


# ---- write ------------------------------------------------------------------


def _write_inputs(n_tokens, n_head, n_kv, dtype, seed, freqs_dtype=torch.bfloat16, rows=600):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n_tokens, (n_head + 2 * n_kv) * 128, generator=g).to(dtype).cuda()
    w = [(1 + 0.1 * torch.randn(128, generator=g)).to(dtype).cuda() for _ in range(2)]
    freqs = model.precompute_freqs_cis(rows, 128, 1e6).to(freqs_dtype).cuda()
    return qkv, w, freqs


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("freqs_dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_write_has_the_bits_of_the_dense_cache(name, norm, freqs_dtype):
    nh, nkv, page, n = 32, 8, 16, 37
    qkv, (qw, kw), freqs = _write_inputs(n, nh, nkv, DT[name], 40, freqs_dtype)
    p = Pool([n, 20], n_kv=nkv, page=page, dtype=DT[name], seed=41)
    rows = torch.arange(n, dtype=torch.int32, device="cuda")
    pos = rows * 7 + 3
    q = pagedkv.write(qkv, p.k, p.v, p.table, rows, pos, freqs, n_head=nh, seqs=torch.zeros_like(rows),
                      q_norm=qw if norm else None, k_norm=kw if norm else None, weight=p.weight, position=p.position)
    kc, vc = (torch.zeros(nkv, n, 128, dtype=DT[name], device="cuda") for _ in range(2))
    qd = torch.empty(n, nh, 128, dtype=DT[name], device="cuda")
    for t in range(n):
        at = torch.tensor([t], device="cuda")
        _lib.check(_lib.lib().nf4b_qk_rope_kv_ex(
            qkv[t].data_ptr(), qw.data_ptr() if norm else None, kw.data_ptr() if norm else None, 1e-6,
            freqs[int(pos[t])].data_ptr(), FTYPE[freqs_dtype], at.data_ptr(), qd[t].data_ptr(),
            kc.data_ptr(), vc.data_ptr(), nh, nkv, 128, n, _lib.act_type(DT[name]),
            torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    tab, r = p.table[0].long(), rows.long()
    assert torch.equal(q, qd)
    assert torch.equal(p.k[tab[r // page], :, r % page], kc.transpose(0, 1))
    assert torch.equal(p.v[tab[r // page], :, r % page], vc.transpose(0, 1))
    assert torch.equal(p.position[tab[r // page], :, r % page], pos[:, None].expand(-1, nkv))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("n_head,n_kv,n", [(3, 1, 1), (8, 8, 5), (16, 1, 200), (32, 8, 333)])
def test_write_against_64_bits(name, n_head, n_kv, n):
    """Two roundings to the type (norm, rotary), each of values no larger than the row's
    rotated pair; their product, and the fp32 steps between, below 2^-14 of it."""
    qkv, (qw, kw), freqs = _write_inputs(n, n_head, n_kv, DT[name], 50 + n)
    seqs = torch.arange(n, dtype=torch.int32) % 3
    rows = (torch.arange(n) // 3).int() + 5
    p = Pool([int(rows.max()) + 1] * 3, n_kv=n_kv, page=32, dtype=DT[name], seed=51)
    p.weight.fill_(2.0)
    pos = (torch.arange(n, dtype=torch.int32) * 3) % 600
    before = (p.k.clone(), p.v.clone())
    q = pagedkv.write(qkv, p.k, p.v, p.table, rows.cuda(), pos.cuda(), freqs, n_head=n_head, seqs=seqs.cuda(),
                      q_norm=qw, k_norm=kw, weight=p.weight, position=p.position)
    want_q, written = po.write(f64(qkv), p.table.cpu().numpy(), rows.numpy(), pos.numpy(), f64(freqs), n_head=n_head,
                               n_kv=n_kv, page=32, n_pages=p.n_pages, seqs=seqs.numpy(), q_norm=f64(qw), k_norm=f64(kw))

    def near(got, want):
        pair = np.repeat(np.hypot(want[..., 0::2], want[..., 1::2]), 2, axis=-1)
        return np.all(np.abs(got - want) <= (2 * U[name] + 2.0 ** -14) * pair + 2.0 ** -24)

    assert near(f64(q), want_q)
    k, v, w, ps = f64(p.k), f64(p.v), p.weight.cpu().numpy(), p.position.cpu().numpy()
    touched = np.zeros(w.shape, bool)
    for (pg, at), (kt, vt, position) in written.items():
        assert near(k[pg, :, at], kt) and np.array_equal(v[pg, :, at], vt)
        assert (ps[pg, :, at] == position).all() and (w[pg, :, at] == 0).all()
        touched[pg, :, at] = True
    assert touched.sum() == n * n_kv and (w[~touched] == 2.0).all()
    for now, old in zip((p.k, p.v), before):  # nothing else was written (bits: the rest holds NaN)
        same = (now.view(torch.int16) == old.view(torch.int16)).all(-1).cpu().numpy()
        assert same[~touched].all()


def test_write_of_padding_and_rows_out_of_range():
    nh, nkv = 8, 2
    qkv, _, freqs = _write_inputs(7, nh, nkv, torch.bfloat16, 60, rows=100)
    p = Pool([64, 64], n_kv=nkv, page=32, dtype=torch.bfloat16, seed=61)
    p.table[1, 1] = -1
    before = (p.k.clone(), p.v.clone())
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rows, pos, seqs = i32([-1, 64, 3, 4, 5, 6, 40]), i32([1, 2, 100, -1, 3, 4, 5]), i32([0, 0, 0, 0, 2, -1, 1])
    q = pagedkv.write(qkv, p.k, p.v, p.table, rows, pos, freqs, n_head=nh, seqs=seqs)
    for now, old in zip((p.k, p.v), before):
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))
    assert not q[2].any() and not q[3].any() and all(q[i].any() for i in (0, 1, 4, 5, 6))


# ---- evict ------------------------------------------------------------------


def check_evict(p, w, pos, budget, recent, sink, inplace):
    """`w`, `pos` [n_seqs][n_kv, rows]: put into the pools, evicted, compared."""
    k0, v0 = p.k.clone(), p.v.clone()
    tab, page = p.table.cpu().numpy(), p.page
    for s, n in enumerate(p.lens_host):
        for h in range(p.n_kv):
            pg, at = po.slots(tab[s], np.arange(n), p.n_pages, page)
            p.weight[pg, h, at] = torch.as_tensor(w[s][h], dtype=torch.float32, device="cuda")
            p.position[pg, h, at] = torch.as_tensor(pos[s][h], dtype=torch.int32, device="cuda")
    outs = (p.weight, p.position, p.lens) if inplace else \
        (torch.full_like(p.weight, -7.0), torch.full_like(p.position, -7), torch.full_like(p.lens, -7))
    got = pagedkv.evict(p.k, p.v, p.weight, p.position, p.table, p.lens, budget=budget, recent=recent, sink=sink,
                        weight_out=outs[0], position_out=outs[1], lens_out=outs[2])
    assert got is outs[2] and got.tolist() == [min(n, budget) for n in p.lens_host]
    k1, v1 = k0.clone(), v0.clone()
    for s, n in enumerate(p.lens_host):
        left = min(n, budget)
        if not n:
            continue
        pg, at = po.slots(tab[s], np.arange(n), p.n_pages, page)
        for h in range(p.n_kv):
            wh, ph = np.asarray(w[s][h], np.float32), np.asarray(pos[s][h])
            to, src = po.moves(po.kept(wh, ph, budget, recent, sink), budget)
            k1[pg[to], h, at[to]], v1[pg[to], h, at[to]] = k0[pg[src], h, at[src]], v0[pg[src], h, at[src]]
            new = np.arange(left)
            new[to] = src
            assert np.array_equal(outs[0][pg[:left], h, at[:left]].cpu().numpy(), wh[new], equal_nan=True)
            assert np.array_equal(outs[1][pg[:left], h, at[:left]].cpu().numpy(), ph[new])
    for now, want in ((p.k, k1), (p.v, v1)):
        assert torch.equal(now.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens,page,budget,recent,sink", [
    ([1, 0, 5], 16, 1, 0, 0),
    ([17, 16, 15], 16, 16, 4, 2),
    ([300, 40, 129], 48, 64, 64, 0),
    ([2000, 1025, 1024], 64, 1000, 100, 4),
    ([3000], 128, 2999, 0, 7),
    ([3000], 128, 7, 3, 4),
])
def test_evict_keeps_what_was_attended_to(lens, page, budget, recent, sink, inplace, name):
    p = Pool(lens, n_kv=2, page=page, dtype=DT[name], seed=70 + sum(lens))
    rng = np.random.default_rng(71)
    w = [[np.where(rng.random(n) < 0.3, 0.0, np.exp(2 * rng.standard_normal(n))) for _ in range(2)] for n in lens]
    pos = [[rng.permutation(n) * 2 for _ in range(2)] for n in lens]
    check_evict(p, w, pos, budget, recent, sink, inplace)


def test_evict_ties_signs_nan_and_infinities():
    """Equal weights, zeros of both signs, NaN, infinities and subnormals in one order."""
    n = 600
    p = Pool([n, n], n_kv=2, page=32, dtype=torch.bfloat16, seed=80)
    rng = np.random.default_rng(81)
    values = np.array([0.0, -0.0, np.nan, np.inf, -np.inf, 1.0, 1.0, -1.0, 1e-42, 3.5], np.float32)
    w = [[values[rng.integers(0, len(values), n)], np.full(n, 0.25)] for _ in range(2)]
    pos = [[rng.permutation(n) for _ in range(2)] for _ in range(2)]
    for budget in (500, 333, 60, 1):
        check_evict(p, w, pos, budget, 0, 0, False)


@pytest.mark.parametrize("n", [6001, 20000, 70001, 140000])
def test_evict_of_a_long_cache(n):
    """One CTA, clusters of several, and more rows than a cluster holds at once."""
    p = Pool([n], n_kv=1, page=16, dtype=torch.bfloat16, seed=82)
    rng = np.random.default_rng(83)
    check_evict(p, [[rng.random(n).astype(np.float32).round(3)]], [[np.arange(n)]], n // 2 - 1, 1000, 16, True)


def test_evict_of_many_lists():
    """More lists than SMs, of a capacity that takes 512 threads each."""
    lens = [(977 * i) % 5000 for i in range(80)]
    p = Pool(lens, n_kv=2, page=64, dtype=torch.bfloat16, seed=86, width=96)
    rng = np.random.default_rng(87)
    w = [[rng.random(n).astype(np.float32).round(2) for _ in range(2)] for n in lens]
    check_evict(p, w, [[rng.permutation(n) for _ in range(2)] for n in lens], 1200, 100, 4, False)


def test_evict_then_attention_is_attention_over_the_kept_rows():
    """The rows that stay, in whatever places, give the attention of a cache that never held the others."""
    p = Pool([900, 300], n_kv=2, page=64, dtype=torch.bfloat16, seed=84)
    q = randn_bf16((2, 8, 128), seed=85, device="cuda")
    attend(p, q, weight=p.weight)
    tab = p.table.cpu().numpy()
    for s, n in enumerate(p.lens_host):
        pg, at = po.slots(tab[s], np.arange(n), p.n_pages, 64)
        p.position[pg, :, at] = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].expand(-1, 2)
    mask = torch.zeros(2, p.table.shape[1] * 64, dtype=torch.bool, device="cuda")
    keep = []
    for s, n in enumerate(p.lens_host):
        pg, at = po.slots(tab[s], np.arange(n), p.n_pages, 64)
        keep.append([po.kept(p.weight[pg, h, at].cpu().numpy(), np.arange(n), 256, 32, 4) for h in range(2)])
    outs = []
    for h in range(2):  # the dense answer: each head masks its own rows
        for s, n in enumerate(p.lens_host):
            mask[s, :n] = torch.from_numpy(keep[s][h]).cuda()
        outs.append(attend(p, q, mask=mask)[:, 4 * h : 4 * h + 4])
    lens = pagedkv.evict(p.k, p.v, p.weight, p.position, p.table, p.lens, budget=256, recent=32, sink=4)
    assert lens.tolist() == [256, 256]
    got, want = attend(p, q).float(), torch.cat(outs, 1).float()
    # the same rows in another order: each one rounding, and 2^-14 of sum p|v| (about 0.8), from the exact value
    assert ((got - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 2.0 ** -12).all()


def test_calls_replay_from_a_cuda_graph_as_the_cache_grows():
    nh, nkv, page = 8, 2, 16
    p = Pool([64, 64], n_kv=nkv, page=page, dtype=torch.bfloat16, seed=90)
    p.k.zero_(), p.v.zero_()
    qkv, _, freqs = _write_inputs(2, nh, nkv, torch.bfloat16, 91)
    lens = torch.tensor([3, 30], dtype=torch.int32, device="cuda")
    out = torch.empty(2, nh, 128, dtype=torch.bfloat16, device="cuda")

    def step():
        q = pagedkv.write(qkv, p.k, p.v, p.table, lens, lens, freqs, n_head=nh, weight=p.weight, position=p.position)
        lens.add_(1)
        pagedkv.attention(q, p.k, p.v, p.table, lens, weight=p.weight, out=out)
        pagedkv.evict(p.k, p.v, p.weight, p.position, p.table, lens, budget=32, recent=8, sink=1)

    want, graph = [], torch.cuda.CUDAGraph()
    state = [t.clone() for t in (p.k, p.v, p.weight, p.position, lens)]

    def reset():
        for t, s in zip((p.k, p.v, p.weight, p.position, lens), state):
            t.copy_(s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # workspaces belong to a stream: sized on the one that captures
        for i in range(6):
            qkv.fill_(0.5).mul_(i + 1)
            step()
            want.append((out.clone(), lens.clone()))
        reset()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    reset()
    for i in range(6):
        qkv.fill_(0.5).mul_(i + 1)
        graph.replay()
        assert torch.equal(out, want[i][0]) and torch.equal(lens, want[i][1])
    assert lens.tolist() == [9, 32]
    del graph
