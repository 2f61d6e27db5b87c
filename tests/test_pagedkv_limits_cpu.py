"""The largest caches that the paged calls take (runs without a GPU)."""

from __future__ import annotations

import pytest

from tests.test_pagedkv_cpu import SHAPE, Host


@pytest.mark.parametrize("call", ["write", "attention", "evict"])
def test_work_whose_count_would_pass_32_bits_is_refused(call):
    """32 heads of 2^26 - 9 tiles of 16 rows, 8 more counted for each: 2^31 - 32, which the kernels' steps of up to 64
    would carry past 2^31 - 1."""
    host = Host()
    assert getattr(host, call)(host.cache(n_seqs=1, n_kv=32, max_pages=2**26 - 9, n_pages=8, page_size=16),
                               **(dict(n_head=32, n=1) if call == "write" else dict(n_head=32) if call == "attention"
                                  else {})) == SHAPE
    fits = getattr(host, call)(host.cache(n_seqs=1, n_kv=32, max_pages=2**26 - 12, n_pages=8, page_size=16),
                               **(dict(n_head=32, n=1) if call == "write" else dict(n_head=32) if call == "attention"
                                  else {}))
    assert fits != SHAPE
