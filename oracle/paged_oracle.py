"""The paged KV cache's operators in NumPy and 64 bits, one sequence and head after
another (for the tests, never the product). Pools are [n_pages, n_kv, page_size, ...]
arrays of values, not bit patterns."""

from __future__ import annotations

import numpy as np


def slots(table_row, rows, n_pages: int, page: int):
    """(page, row in the page) of cache rows; page -1 where none is assigned."""
    rows = np.asarray(rows, dtype=np.int64)
    pg = np.asarray(table_row, dtype=np.int64)[rows // page]
    return np.where((pg >= 0) & (pg < n_pages), pg, -1), rows % page


def attention(q, k, v, table, lens, *, scale, mask=None, weight=None):
    """(out [n_seqs, n_head, 128], the weights added [n_pages, n_kv, page], and
    sum p |v| of every output, the size its errors go by)."""
    q = np.asarray(q, np.float64)
    n_seqs, n_head, d = q.shape
    n_pages, n_kv, page, _ = k.shape
    groups = n_head // n_kv
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    added = np.zeros((n_pages, n_kv, page))
    for s in range(n_seqs):
        n = min(max(int(lens[s]), 0), table.shape[1] * page)
        pg, at = slots(table[s], np.arange(n), n_pages, page)
        see = pg >= 0
        if mask is not None:
            see &= np.asarray(mask[s][:n], bool)
        pg, at = pg[see], at[see]
        if not len(pg):
            continue
        for h in range(n_kv):
            ks, vs = np.asarray(k[pg, h, at], np.float64), np.asarray(v[pg, h, at], np.float64)
            for g in range(groups):
                head = h * groups + g
                sc = scale * (ks @ q[s, head])
                top = sc.max()
                if top == -np.inf:
                    continue
                with np.errstate(invalid="ignore"):
                    p = np.exp(sc - top)
                p /= p.sum()
                out[s, head] = p @ vs
                size[s, head] = p @ np.abs(vs)
                np.add.at(added[:, h], (pg, at), p)
    return out, added, size


def rotated(x, cs):
    """Interleaved-pair rotary of [..., 128] by (cos, sin) rows [..., 64, 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cs[..., 0], cs[..., 1]
    return np.stack([a * c - b * s, b * c + a * s], -1).reshape(x.shape)


def normed(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def write(qkv, table, rows, positions, freqs, *, n_head, n_kv, page, n_pages, seqs=None, q_norm=None, k_norm=None,
          eps=1e-6):
    """(q [T, n_head, 128], {(page, row in it): (k [n_kv, 128], v, position)})."""
    x = np.asarray(qkv, np.float64).reshape(len(rows), n_head + 2 * n_kv, 128)
    q, written = np.zeros((len(rows), n_head, 128)), {}
    for t in range(len(rows)):
        pos = int(positions[t])
        if not 0 <= pos < len(freqs):
            continue
        cs = np.asarray(freqs[pos], np.float64)
        qt, kt, vt = x[t, :n_head], x[t, n_head : n_head + n_kv], x[t, n_head + n_kv :]
        if q_norm is not None:
            qt, kt = normed(qt, np.asarray(q_norm, np.float64), eps), normed(kt, np.asarray(k_norm, np.float64), eps)
        q[t] = rotated(qt, cs)
        s, r = (t if seqs is None else int(seqs[t])), int(rows[t])
        if not (0 <= s < table.shape[0] and 0 <= r < table.shape[1] * page):
            continue
        pg, at = slots(table[s], [r], n_pages, page)
        if pg[0] >= 0:
            written[(int(pg[0]), int(at[0]))] = (rotated(kt, cs), vt, pos)
    return q, written


def kept(weight, position, budget: int, recent: int, sink: int):
    """Which rows of one head stay: bool [rows]. Protected ones first, then by falling
    weight (NaN as -inf), then by rising row."""
    n = len(weight)
    newest = int(position.max()) if n else 0
    guarded = (position < sink) | (position > newest - recent)
    w = np.where(np.isnan(weight), -np.inf, np.asarray(weight, np.float64))
    order = sorted(range(n), key=lambda i: (not guarded[i], -w[i] if not guarded[i] else 0.0, i))
    keep = np.zeros(n, bool)
    keep[order[: min(n, budget)]] = True
    return keep


def moves(keep, budget: int):
    """(rows that are overwritten, rows that move there) of one head."""
    left = min(len(keep), budget)
    return np.nonzero(~keep[:left])[0], left + np.nonzero(keep[left:])[0]
