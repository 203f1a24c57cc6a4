"""Calls of the operators of a served layer as their wrappers make them, without a GPU: a library that records in the place of the native one."""
import weakref

import pytest
import torch

from jarvis_b200 import ops
from tests.test_block_operators_cpu import BF16, F32, _on


class Library:
    """Stands for the native library; `seen`: (name, arguments) of its calls."""

    def __init__(self, scratch=0):
        self.seen, self.scratch = [], scratch

    def __getattr__(self, name):
        if name.endswith("_scratch_bytes"):
            return lambda *a: self.scratch
        return lambda *a: self.seen.append((name, a)) or 0


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(ops._lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_raw_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    return lib


def _delta_args(B=2, T=2, H=2, D=64):
    rows = _on(0, B * T, H * D, dtype=BF16)
    return rows, rows, rows, _on(0, B * T, H), _on(0, B * T, H), B, T, H


def test_scratch_lives_until_everything_is_launched(library, monkeypatch):
    """Another thread may allocate and launch on the same stream while the native call is running."""
    library.scratch = 1 << 12
    tensors, held = [], []
    empty = torch.empty

    def noted(*args, **kw):
        t = empty(*args, **kw)
        if kw.get("dtype") is torch.uint8:
            tensors.append((weakref.ref(t), t.data_ptr()))
        return t

    monkeypatch.setattr(ops.torch, "empty", noted)
    library.jb200_gated_delta = lambda d, scratch, stream: held.append([ref() is not None and at == scratch for ref, at in tensors]) or 0
    ops.gated_delta_scan(*_delta_args())
    assert held == [[True]]
