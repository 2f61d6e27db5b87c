"""The paged KV cache's Python binding by itself (runs without a GPU)."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

from ttspipe_b200 import pagedkv

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


def test_pools_of_another_device_than_the_current_one_are_refused():
    """Launched all the same, a kernel would run on the current GPU with the other one's addresses."""
    check = pagedkv._bound().check_device
    for device, current in ((1, 0), (0, 1), (7, 3)):
        with pytest.raises(ValueError, match=f"pools on cuda:{device}, the current device is cuda:{current}"):
            check(device, current)
    assert check(0, 0) is None and check(5, 5) is None
