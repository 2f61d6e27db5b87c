"""The paged KV cache's Python binding by itself (runs without a GPU)."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_refusal_that_names_numbers_is_an_exception():
    """In a process of its own: a crash is a failure here, not the end of the tests."""
    code = ("from ttspipe_b200 import pagedkv\n"
            "for call in ('write', 'attention', 'evict'):\n"
            "    try:\n        getattr(pagedkv._bound(), call)(1)\n"
            "    except TypeError as exc:\n        print(exc)\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.splitlines() == [f"{n} arguments needed, got 1" for n in (16, 12, 15)]
