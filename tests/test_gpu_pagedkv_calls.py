"""The paged KV cache's Python calls on the B200: what they refuse of tensors, with the cache left as it was."""

from __future__ import annotations

import pytest
import torch

from tests.helpers import randn_bf16
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


class Work:
    """Attention of long sequences (joined from many parts), with weights, and an eviction of copies."""

    def __init__(self, seed):
        self.p = Pool([4000, 1, 2500, 3999], n_kv=8, page=64, dtype=torch.bfloat16, seed=seed)
        self.p.position[self.p.table.clamp(min=0).long()] = 1
        self.q = randn_bf16((4, 32, 128), seed=seed, device="cuda")
        self.out, self.weight = torch.empty_like(self.q), torch.zeros_like(self.p.weight)
        self.evicted = [torch.zeros_like(t) for t in (self.p.weight, self.p.position, self.p.lens)]
        self.k, self.v = self.p.k.clone(), self.p.v.clone()

    def run(self):
        p = self.p
        self.weight.zero_()
        for _ in range(3):
            pagedkv.attention(self.q, p.k, p.v, p.table, p.lens, weight=self.weight, out=self.out)
        self.k.copy_(p.k), self.v.copy_(p.v)
        pagedkv.evict(self.k, self.v, self.weight, p.position, p.table, p.lens, budget=1111, recent=0, sink=0,
                      weight_out=self.evicted[0], position_out=self.evicted[1], lens_out=self.evicted[2])

    def result(self):
        torch.cuda.synchronize()
        return [t.clone().view(torch.uint8) for t in (self.out, self.weight, self.k, self.v, *self.evicted)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_capture_needs_no_warm_up():
    """The usual form: on torch's own capture stream, where nothing of this kind has run."""
    work = Work(1)
    work.run()
    want = work.result()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work.run()
    for t in (work.out, work.weight, *work.evicted):
        t.zero_()
    for _ in range(3):
        graph.replay()
        assert same(work.result(), want)
    del graph


def test_graphs_of_one_capture_stream_replay_side_by_side():
    """Two graphs captured on one stream, replayed on two others, with calls on that stream in between."""
    works = [Work(2), Work(3), Work(4)]
    side, lanes = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs, want = [torch.cuda.CUDAGraph() for _ in lanes], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for work in works:
            work.run()
            want.append(work.result())
        for graph, work in zip(graphs, works):
            with torch.cuda.graph(graph, stream=side):
                work.run()
    torch.cuda.synchronize()
    for _ in range(20):
        for _ in range(5):
            for lane, graph in zip(lanes, graphs):
                with torch.cuda.stream(lane):
                    graph.replay()
            with torch.cuda.stream(side):
                works[2].run()
        for work, w in zip(works, want):
            assert same(work.result(), w)
    del graphs


def test_streams_of_one_capture_do_not_share_a_workspace():
    works = [Work(5), Work(6)]
    want = []
    for work in works:
        work.run()
        want.append(work.result())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        works[0].run()
        with torch.cuda.stream(side):
            works[1].run()
        main.wait_stream(side)
    for _ in range(20):
        graph.replay()
        for work, w in zip(works, want):
            assert same(work.result(), w)
    del graph
