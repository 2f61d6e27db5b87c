"""The paged KV cache's Python binding by itself (runs without a GPU)."""

from __future__ import annotations

import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from ttspipe_b200 import _lib, pagedkv

ROOT = Path(__file__).resolve().parent.parent


def test_a_refusal_that_names_numbers_is_an_exception():
    """In a process of its own: a crash is a failure here, not the end of the tests."""
    code = ("from ttspipe_b200 import pagedkv\n"
            "for call in ('write', 'attention', 'evict'):\n"
            "    try:\n        getattr(pagedkv._bound(), call)(1)\n"
            "    except TypeError as exc:\n        print(exc)\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.splitlines() == [f"{n} arguments needed, got 1" for n in (16, 13, 16)]


def test_pools_of_another_device_than_the_current_one_are_refused():
    """Launched all the same, a kernel would run on the current GPU with the other one's addresses."""
    check = pagedkv._bound().check_device
    for device, current in ((1, 0), (0, 1), (7, 3)):
        with pytest.raises(ValueError, match=f"pools on cuda:{device}, the current device is cuda:{current}"):
            check(device, current)
    assert check(0, 0) is None and check(5, 5) is None


class Calls:
    """The binding's attention and eviction, which need workspaces of `need` bytes, and a stream that captures or not."""

    def __init__(self, monkeypatch):
        self.need, self.capture, self.seen = 100, 0, []
        monkeypatch.setattr(pagedkv, "_native", types.SimpleNamespace(attention=self.call, evict=self.call))
        monkeypatch.setattr(pagedkv, "_workspaces", {})
        monkeypatch.setattr(pagedkv, "_captured", {})
        monkeypatch.setattr(pagedkv, "_stream", lambda device: self.stream)
        monkeypatch.setattr(pagedkv, "_capture_id", lambda stream: self.capture)
        monkeypatch.setattr(pagedkv, "_empty", lambda size, device: torch.full((size,), 7, dtype=torch.uint8))
        sizes = types.SimpleNamespace(nf4b_paged_attention_workspace_size=lambda *a: self.need,
                                      nf4b_paged_evict_workspace_size=lambda *a: self.need)
        monkeypatch.setattr(_lib, "lib", lambda: sizes)

    def call(self, *args):
        ws, size, capture = args[-4:-1]
        if ws is None or capture != self.capture or size < self.need:
            return _lib.NF4B_ERR_WORKSPACE
        self.seen.append((ws, size))
        return "done"

    def __call__(self, kind, stream, capture=0, need=100):
        self.stream, self.capture, self.need = stream, capture, need
        t = types.SimpleNamespace(get_device=lambda: 0, shape=(4, 2, 16, 128))
        got = pagedkv.attention(t, t, t, t, t) if kind == "attention" else pagedkv.evict(t, t, t, t, t, t, budget=1)
        assert got == "done"
        return self.seen[-1]


def test_every_capture_has_workspaces_of_its_own(monkeypatch):
    run = Calls(monkeypatch)
    eager = {(kind, s): run(kind, s)[0] for kind in ("attention", "evict") for s in (0, 5, 6)}
    assert len(set(eager.values())) == 6
    first = {(kind, s): run(kind, s, capture=31) for kind in ("attention", "evict") for s in (5, 6)}
    kept = [w[0] for w in pagedkv._captured.values()]
    assert first == {key: run(*key, capture=31) for key in first}  # the same for all calls of a capture
    second = {key: run(*key, capture=32) for key in first}
    # (an address may come again once the first capture's are let go: kept alive here)
    places = [w[0] for w in (*first.values(), *second.values())] + list(eager.values())
    assert len(set(places)) == len(places) and len(kept) == 4
    assert run("attention", 5, capture=32, need=300)[1] == 300
    assert {key: run(*key)[0] for key in eager} == eager and not pagedkv._captured


def test_a_new_workspace_is_zero_where_it_has_to_be(monkeypatch):
    run = Calls(monkeypatch)
    need = _lib.PAGED_COUNTER_BYTES + 64
    run("attention", 5, capture=3, need=need)
    (ws, *_), = pagedkv._captured.values()
    assert ws.numel() == need and not ws[: _lib.PAGED_COUNTER_BYTES].any()
    run("attention", 5, need=need)
    first = pagedkv._workspaces["attention", 0, 5]
    assert first[2] == 1 << 20 and not first[0][: _lib.PAGED_COUNTER_BYTES].any()
    run("attention", 5, need=(1 << 20) + 1)
    assert pagedkv._workspaces["attention", 0, 5][2] == 2 << 20


def test_the_counters_are_what_the_header_says():
    text = (ROOT / "include" / "nf4b200.h").read_text()
    assert f"#define NF4B_PAGED_COUNTER_BYTES {_lib.PAGED_COUNTER_BYTES}u" in text
    assert _lib.lib().nf4b_capture_id(None) == 0
