"""The operators of the paged key-value cache as measured cases: ``write`` (q/k norm, rotary and the scatter into
pages), ``attention`` (one new token of each sequence over its pages, the rows' weights accumulated) and ``evict``
(each head keeps the rows that were attended to most).

``run`` makes the calls of ``ttspipe_b200.pagedkv`` where ``own`` is true and computes the plain torch forms where it
is false. Pools are [n_pages, n_kv, page_size, 128]; a sequence's rows lie in the pages its block-table row names.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = ((32, 8), (16, 8), (8, 8), (16, 1), (24, 8), (32, 4))
EPS = 1e-6


def _attention(name, batch, length, *, lens="ragged", heads=(32, 8), page=64, dtype="bf16", track=False, mask=False):
    return {"name": name, "op": "attention", "batch": batch, "len": length, "lens": lens, "n_head": heads[0],
            "n_kv": heads[1], "page": page, "dtype": dtype, "track": track, "mask": mask}


def _write(name, seqs, tokens, *, heads=(32, 8), page=64, dtype="bf16", norm=True):
    return {"name": name, "op": "write", "batch": seqs, "tokens": tokens, "n_head": heads[0], "n_kv": heads[1],
            "page": page, "dtype": dtype, "norm": norm}


def _evict(name, batch, length, budget, recent, sink, *, lens="full", heads=(32, 8), page=64, dtype="bf16"):
    return {"name": name, "op": "evict", "batch": batch, "len": length, "lens": lens, "budget": budget,
            "recent": recent, "sink": sink, "n_head": heads[0], "n_kv": heads[1], "page": page, "dtype": dtype}


def listed():
    return [
        # the first tokens of one stream: launch latency alone
        _attention("attn 1x19", 1, 19, lens="full", page=16),
        # one stream with a full cache of the slow stack's 2048 rows (32 query and 8 KV heads)
        _attention("attn 1x2048", 1, 2048, lens="full"),
        # 32 streams that started at different times, weights kept for a later eviction
        _attention("attn 32x4096 tracked", 32, 4096, track=True),
        # one stream of a very long context, pages of 16, fp16
        _attention("attn 1x65521 fp16", 1, 65521, lens="full", page=16, dtype="fp16"),
        # many query heads on one KV head, with rows masked out (padding inside the prompt), odd lengths
        _attention("attn 5x3001 16/1 masked", 5, 3001, heads=(16, 1), page=32, dtype="fp16", mask=True, track=True),
        # a full server: 64 streams of 8192 rows
        _attention("attn 64x8192 tracked", 64, 8192, lens="full", page=128, track=True),
        # one stream's decode step
        _write("write 1 token", 1, 1, norm=False),
        # the decode step of 64 streams
        _write("write 64x1", 64, 1),
        # prompts and reference clips of four streams entering their pages
        _write("write 4x2047 fp16", 4, 2047, page=16, dtype="fp16"),
        # one stream's cache of 2048 rows halved
        _evict("evict 1x2048", 1, 2048, 1024, 128, 4),
        # ragged streams, some of them still under the budget
        _evict("evict 32x4096 ragged fp16", 32, 4096, 1500, 257, 1, lens="ragged", page=32, dtype="fp16"),
        # long contexts halved on a full server
        _evict("evict 8x32768", 8, 32768, 16384, 1024, 16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "write", "evict"))
    heads, page, dtype = rng.choice(HEADS), rng.choice((16, 32, 64, 128)), rng.choice(("bf16", "fp16"))
    if op == "write":
        seqs = _log_int(rng, 1, 64)
        c = _write("", seqs, _log_int(rng, 1, max(1, 8192 // seqs)), heads=heads, page=page, dtype=dtype,
                   norm=rng.random() < 0.5)
    elif op == "attention":
        batch = _log_int(rng, 1, 64)
        c = _attention("", batch, _log_int(rng, 1, min(65536, 64 * 8192 // batch)), lens=rng.choice(("full", "ragged")),
                       heads=heads, page=page, dtype=dtype, track=rng.random() < 0.5, mask=rng.random() < 0.3)
    else:
        batch = _log_int(rng, 1, 32)
        length = _log_int(rng, 2, min(32768, 8 * 32768 // batch))
        budget = rng.randint(1, length)
        recent = rng.randint(0, budget)
        c = _evict("", batch, length, budget, recent, rng.randint(0, min(16, budget - recent)),
                   lens=rng.choice(("full", "ragged")), heads=heads, page=page, dtype=dtype)
    del c["name"]
    return c


def _lens(case):
    """Each sequence's rows: all of them, or lengths anywhere up to it, with the longest, one row and (from three
    sequences on) none among them."""
    batch, length = case["batch"], case["len"]
    if case["lens"] == "full":
        return [length] * batch
    rng = random.Random(1000003 * batch + length)
    lens = [rng.randint(1, length) for _ in range(batch)]
    lens[0] = length
    if batch > 1:
        lens[1] = 1
    if batch > 2:
        lens[2] = 0
    return lens


VISIBLE = 0.75  # share of the rows that a mask leaves visible


def work(case):
    nh, nkv, op = case["n_head"], case["n_kv"], case["op"]
    if op == "write":
        t = case["batch"] * case["tokens"]
        # qkv in, q and the cache rows out; rotary rows (bf16 cos, sin); position, weight; row, position and sequence in
        return {"bytes": t * (2 * (nh + 2 * nkv) * D * 2 + 8 * nkv + 12) + min(t, case["tokens"]) * D * 2,
                "flops": t * (nh + nkv) * D * (7 if case["norm"] else 3)}
    rows = sum(_lens(case))
    if op == "attention":
        seen = rows * (VISIBLE if case["mask"] else 1.0)
        per = 2 * D * 2 + (8 if case["track"] else 0)
        return {"bytes": seen * nkv * per + 2 * case["batch"] * nh * D * 2 + (rows if case["mask"] else 0),
                "flops": seen * nh * 4 * D}
    moved = sum(case["budget"] * (n - case["budget"]) / n for n in _lens(case) if n > case["budget"])
    kept = sum(min(n, case["budget"]) for n in _lens(case))
    return {"bytes": nkv * (rows * 8 + kept * 8 + moved * 2 * 2 * D * 2), "flops": nkv * rows * 4}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _table(g, lens, page, length):
    """A block table whose sequences own pages spread over the pool, -1 where none is assigned, and the pool's size."""
    need = [-(-n // page) for n in lens]
    width = max(1, -(-length // page))
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    own_pages = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[own_pages] = order[: sum(need)]
    return table, n_pages


def _rotary_table(rows):
    """(rows, 64, 2) = (cos, sin) in bf16, base 1e6."""
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").double() / D))
    ang = torch.outer(torch.arange(rows, device="cuda").double(), inv)
    return torch.stack([ang.cos(), ang.sin()], -1).to(torch.bfloat16)


def prepare(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    nh, nkv, page, batch = case["n_head"], case["n_kv"], case["page"], case["batch"]
    s = {"op": case["op"], "n_head": nh, "n_kv": nkv, "page": page}
    if case["op"] == "write":
        t, n = batch * case["tokens"], case["tokens"]
        start = 37  # rows that are in the cache already
        s["table"], n_pages = _table(g, [start + n] * batch, page, start + n)
        s["qkv"] = _normal(g, t, (nh + 2 * nkv) * D, dtype=dt)
        s["seqs"] = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(n)
        s["rows"] = (start + torch.arange(n, device="cuda", dtype=torch.int32)).repeat(batch)
        s["positions"] = s["rows"] + 211  # rows were evicted before: positions run ahead of them
        s["freqs"] = _rotary_table(start + n + 211)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = (1 + 0.1 * _normal(g, D, dtype=torch.float32)).to(dt)
            s["k_norm"] = (1 + 0.1 * _normal(g, D, dtype=torch.float32)).to(dt)
        s["k"], s["v"] = (torch.zeros(n_pages, nkv, page, D, dtype=dt, device="cuda") for _ in range(2))
        s["weight"] = torch.ones(n_pages, nkv, page, device="cuda")
        s["position"] = torch.zeros(n_pages, nkv, page, dtype=torch.int32, device="cuda")
        return s
    lens = _lens(case)
    s["table"], n_pages = _table(g, lens, page, case["len"])
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["k"], s["v"] = _normal(g, n_pages, nkv, page, D, dtype=dt), _normal(g, n_pages, nkv, page, D, dtype=dt)
    if case["op"] == "attention":
        s["q"] = _normal(g, batch, nh, D, dtype=dt)
        s["mask"] = None
        if case["mask"]:
            s["mask"] = torch.rand(batch, s["table"].shape[1] * page, generator=g, device="cuda") < VISIBLE
            s["mask"][-1] = False  # a sequence that sees nothing
            s["v"][:, :, ::7] = torch.where(_seen(s)[:, None, ::7, None], s["v"][:, :, ::7], float("nan"))
        s["weight"] = torch.zeros(n_pages, nkv, page, device="cuda") if case["track"] else None
        return s
    # accumulated weights spread over decades, new rows at exactly 0; the first `budget` rows hold what earlier
    # evictions left, in any order, the others came one after another
    width = s["table"].shape[1] * page
    w = torch.exp(2.5 * torch.randn(batch, nkv, width, generator=g, device="cuda")) / case["len"]
    w = w * (torch.rand(batch, nkv, width, generator=g, device="cuda") < 0.95)
    head = min(case["budget"], width)
    pos = torch.arange(width, device="cuda").repeat(batch, nkv, 1)
    pos[..., :head] = torch.rand(batch, nkv, head, generator=g, device="cuda").argsort(-1)
    s["weight"] = _scattered(s, w, torch.zeros(n_pages, nkv, page, device="cuda"))
    s["position"] = _scattered(s, pos.to(torch.int32), torch.zeros(n_pages, nkv, page, dtype=torch.int32, device="cuda"))
    s["weight_out"], s["position_out"] = torch.zeros_like(s["weight"]), torch.zeros_like(s["position"])
    s["lens_out"] = torch.zeros_like(s["lens"])
    s["rule"] = {k: case[k] for k in ("budget", "recent", "sink")}
    return s


def _pages_of(s, x):
    """[batch, n_kv, width] -> [batch, pages, n_kv, page]."""
    b, h, _ = x.shape
    return x.view(b, h, -1, s["page"]).permute(0, 2, 1, 3)


def _scattered(s, x, pool):
    used = s["table"] >= 0
    pool[s["table"][used].long()] = _pages_of(s, x)[used]
    return pool


def _seen(s):
    """[n_pages, page]: whether a pool row is visible to its sequence."""
    seen = _visible(s).view(s["table"].shape[0], -1, s["page"])
    used = s["table"] >= 0
    pool = torch.zeros(s["k"].shape[0], s["page"], dtype=torch.bool, device="cuda")
    pool[s["table"][used].long()] = seen[used]
    return pool


def _visible(s):
    """[batch, width]: whether a row takes part."""
    width = s["table"].shape[1] * s["page"]
    seen = torch.arange(width, device="cuda")[None] < s["lens"][:, None]
    return seen if s.get("mask") is None else seen & s["mask"]


def _gathered(s, pool):
    """[batch, n_kv, width, ...] rows of a pool in sequence order; unassigned pages read page 0."""
    x = pool[s["table"].clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _plain_attention(s):
    b, nh, _ = s["q"].shape
    nkv = s["n_kv"]
    seen = _visible(s)[:, None, None]
    k = _gathered(s, s["k"]).float()
    q = s["q"].float().view(b, nkv, nh // nkv, D)
    score = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    del k
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = torch.where(_visible(s)[:, None, :, None], _gathered(s, s["v"]).float(), 0.0)
    out = torch.matmul(p, v).view(b, nh, D).to(s["q"].dtype)
    if s["weight"] is None:
        return {"out": out}
    add = _pages_of(s, p.sum(2))
    s["weight"].index_add_(0, s["table"].clamp(min=0).long().view(-1), add.reshape(-1, nkv, s["page"]))
    return {"out": out, "weight": s["weight"]}


def _rotated(x, cs):
    a, b = x[..., 0::2], x[..., 1::2]
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain_write(s):
    nh, nkv, page = s["n_head"], s["n_kv"], s["page"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, D)
    cs = s["freqs"][s["positions"].long()].float()
    q = _rotated(_normed(x[:, :nh], s["q_norm"]), cs).to(s["qkv"].dtype)
    k = _rotated(_normed(x[:, nh : nh + nkv], s["k_norm"]), cs).to(s["qkv"].dtype)
    pages = s["table"][s["seqs"].long(), s["rows"].long() // page].long()
    rows = s["rows"].long() % page
    s["k"][pages, :, rows] = k
    s["v"][pages, :, rows] = s["qkv"].view(-1, nh + 2 * nkv, D)[:, nh + nkv :]
    s["weight"][pages, :, rows] = 0.0
    s["position"][pages, :, rows] = s["positions"][:, None].expand(-1, nkv)
    return {"q": q, "k": s["k"], "v": s["v"], "weight": s["weight"], "position": s["position"]}


def _plain_evict(s):
    page, nkv = s["page"], s["n_kv"]
    budget, recent, sink = (s["rule"][k] for k in ("budget", "recent", "sink"))
    w, pos = _gathered(s, s["weight"]), _gathered(s, s["position"])
    r = torch.arange(w.shape[-1], device="cuda")
    live = (r < s["lens"][:, None, None]).expand_as(w)
    newest = torch.where(live, pos, -1).amax(-1, keepdim=True)
    guarded = (pos < sink) | (pos > newest - recent)
    rank_class = torch.where(live, torch.where(guarded, 0, 1), 2)
    key = torch.where(rank_class == 1, torch.where(torch.isnan(w), -math.inf, w), 0.0)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank_class.gather(-1, order), dim=-1, stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, r.expand_as(order))
    left = s["lens"].clamp(max=budget)
    kept = rank < left[:, None, None]
    inside = r < left[:, None, None]
    table = s["table"].clamp(min=0).long()

    def places(which):  # flat pool rows of the chosen rows, by sequence, head and row
        b, h, i = which.nonzero(as_tuple=True)
        return (table[b, i // page] * nkv + h) * page + i % page

    to, src = places(~kept & inside), places(kept & ~inside)
    for pool in (s["k"], s["v"]):
        flat = pool.view(-1, D)
        flat[to] = flat[src]
    stay = places(kept & inside)
    for pool, out in ((s["weight"], s["weight_out"]), (s["position"], s["position_out"])):
        out.view(-1)[stay] = pool.view(-1)[stay]
        out.view(-1)[to] = pool.view(-1)[src]
    s["lens_out"].copy_(left)
    return {"k": s["k"], "v": s["v"], "weight": s["weight_out"], "position": s["position_out"], "lens": s["lens_out"]}


def run(s):
    if not own:
        return {"attention": _plain_attention, "write": _plain_write, "evict": _plain_evict}[s["op"]](s)
    from ttspipe_b200 import pagedkv

    if s["op"] == "attention":
        out = pagedkv.attention(s["q"], s["k"], s["v"], s["table"], s["lens"], mask=s["mask"], weight=s["weight"])
        return {"out": out} if s["weight"] is None else {"out": out, "weight": s["weight"]}
    if s["op"] == "write":
        q = pagedkv.write(s["qkv"], s["k"], s["v"], s["table"], s["rows"], s["positions"], s["freqs"],
                          n_head=s["n_head"], seqs=s["seqs"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                          weight=s["weight"], position=s["position"])
        return {"q": q, "k": s["k"], "v": s["v"], "weight": s["weight"], "position": s["position"]}
    pagedkv.evict(s["k"], s["v"], s["weight"], s["position"], s["table"], s["lens"], **s["rule"],
                  weight_out=s["weight_out"], position_out=s["position_out"], lens_out=s["lens_out"])
    return {"k": s["k"], "v": s["v"], "weight": s["weight_out"], "position": s["position_out"], "lens": s["lens_out"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "write": _exact_write, "evict": _exact_evict}[case["op"]](s)


def _exact_attention(s):
    """softmax(q k / sqrt(128)) v one sequence after another, over the rows that take part."""
    b, nh, _ = s["q"].shape
    nkv, page = s["n_kv"], s["page"]
    out = torch.zeros(b, nh, D, dtype=torch.float64, device="cuda")
    weight = None if s["weight"] is None else s["weight"].double()
    for i, n in enumerate(s["lens"].tolist()):
        rows = torch.arange(n, device="cuda")
        if s["mask"] is not None:
            rows = rows[s["mask"][i, :n]]
        if not rows.numel():
            continue
        pages, at = s["table"][i].long()[rows // page], rows % page
        k, v = s["k"][pages, :, at].double(), s["v"][pages, :, at].double()  # [rows, n_kv, 128]
        score = torch.einsum("hgd,rhd->hgr", s["q"][i].double().view(nkv, -1, D), k) / math.sqrt(D)
        p = torch.softmax(score, -1)
        out[i] = torch.einsum("hgr,rhd->hgd", p, v).reshape(nh, D)
        if weight is not None:
            weight[pages, :, at] += p.sum(1).T
    return {"out": out} if weight is None else {"out": out, "weight": weight}


def _exact_write(s):
    nh, nkv, page = s["n_head"], s["n_kv"], s["page"]
    heads = s["qkv"].double().view(-1, nh + 2 * nkv, D)
    f = torch.view_as_complex(s["freqs"].double()[s["positions"].long()].contiguous())[:, None]  # [tokens, 1, 64]

    def turned(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous()) * f).flatten(-2)

    k, v, weight = s["k"].double(), s["v"].double(), s["weight"].double()
    where = (s["table"].long()[s["seqs"].long(), s["rows"].long() // page], slice(None), s["rows"].long() % page)
    k[where], v[where], weight[where] = turned(heads[:, nh:-nkv], s["k_norm"]), heads[:, -nkv:], 0.0
    return {"q": turned(heads[:, :nh], s["q_norm"]), "k": k, "v": v, "weight": weight, "position": None}


def _exact_evict(s):
    """One head after another on the host: the rows to keep by (guarded, weight, row), then the moves."""
    page, nkv = s["page"], s["n_kv"]
    w, pos, table = (s[k].cpu().numpy() for k in ("weight", "position", "table"))
    weight, moves = np.zeros(w.shape), []
    for b, n in enumerate(s["lens"].tolist()):
        pages = table[b, : -(-n // page)]
        left = min(n, s["rule"]["budget"])
        if not n:
            continue
        for h in range(nkv):
            wh, ph = w[pages, h].reshape(-1)[:n], pos[pages, h].reshape(-1)[:n]
            guarded = (ph < s["rule"]["sink"]) | (ph > ph.max() - s["rule"]["recent"])
            order = np.lexsort((np.arange(n), -wh.astype(np.float64), ~guarded))
            keep = np.zeros(n, bool)
            keep[order[:left]] = True
            to, src = np.nonzero(~keep[:left])[0], left + np.nonzero(keep[left:])[0]
            new = wh[:left].copy()
            new[to] = wh[src]
            r = np.arange(left)
            weight[pages[r // page], h, r % page] = new
            flat = lambda i: (pages[i // page].astype(np.int64) * nkv + h) * page + i % page  # noqa: E731
            moves.append(np.stack([flat(to), flat(src)]))
    to, src = torch.from_numpy(np.concatenate(moves, 1)).cuda()
    k, v = s["k"].double(), s["v"].double()
    for pool in (k, v):
        pool.view(-1, D)[to] = pool.view(-1, D)[src]
    return {"k": k, "v": v, "weight": torch.from_numpy(weight), "position": None, "lens": None}
