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


def _calls():
    """name -> (a call with one of its tensors, the tensors that it may be)"""
    rows, g, x, w = _on(0, 4, 128, dtype=BF16), _on(0, 4, 2), _on(0, 4, 128), _on(0, 128)
    state = _on(0, 2, 2, 64, 64)
    return {
        "scan, q": (lambda t: ops.gated_delta_scan(t, rows, rows, g, g, 2, 2, 2), rows),
        "scan, log_decay": (lambda t: ops.gated_delta_scan(rows, rows, rows, t, g, 2, 2, 2), g),
        "scan, state": (lambda t: ops.gated_delta_scan(rows, rows, rows, g, g, 2, 2, 2, state_in=t), state),
        "norm, y": (lambda t: ops.gated_norm(t, w), x),
        "norm, weight": (lambda t: ops.gated_norm(x, t), w),
        "norm, gate": (lambda t: ops.gated_norm(x, w, t), x),
        "residual, x": (lambda t: ops.residual_norm(t, x, w, w), x),
        "residual, scale": (lambda t: ops.residual_norm(x, x, w, w, scale=t), w),
        "draw, logits": (lambda t: ops.sample_rows(t, _on(0, 4), want_prob=True), x),
        "draw, temperature": (lambda t: ops.sample_rows(x, _on(0, 4), temperature=t, want_prob=True), _on(0, 4)),
        "draw, min_p": (lambda t: ops.sample_rows(x, _on(0, 4), min_p=t, want_prob=True), _on(0, 4)),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_derivatives_are_refused_not_dropped(library, name):
    call, t = _calls()[name]
    call(t)
    assert len(library.seen) == 1
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t.as_subclass(torch.Tensor), torch.ones(t.shape, dtype=t.dtype)).as_subclass(type(t))
        assert torch.autograd.forward_ad.unpack_dual(dual).tangent is not None
        for grad in (True, False):                                # no_grad does not end forward mode
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="tangent"):
                call(dual)
    wanted = t.clone().as_subclass(type(t)).requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        call(wanted)
    with torch.no_grad():
        call(wanted)
    assert len(library.seen) == 2


def test_a_draw_without_its_probability_takes_logits_that_require_a_gradient(library):
    ops.sample_rows(_on(0, 4, 128).requires_grad_(True), _on(0, 4))
    assert [n for n, _ in library.seen] == ["jb200_sample_rows"]


def test_no_tokens_and_no_state_is_an_empty_output(monkeypatch):
    """The library itself, which has no address of an empty output to tell it from none."""
    monkeypatch.setattr(ops, "_raw_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    rows, g = _on(0, 0, 128, dtype=BF16), _on(0, 0, 2)
    for B, T in ((3, 0), (0, 5), (0, 0)):
        o, state = ops.gated_delta_scan(rows, rows, rows, g, g, B, T, 2)
        assert o.shape == (0, 128) and o.dtype is BF16 and state is None


def test_gates_have_row_strides_of_their_own(library):
    rows, both, beta = _on(0, 4, 128, dtype=BF16), _on(0, 4, 4), _on(0, 4, 2)
    seen = []
    library.jb200_gated_delta = lambda d, *a: seen.append((d._obj.ldg, d._obj.ldb)) or 0
    sliced = both[:, :2].as_subclass(type(both))
    ops.gated_delta_scan(rows, rows, rows, sliced, beta, 2, 2, 2)
    ops.gated_delta_scan(rows, rows, rows, beta, sliced, 2, 2, 2)
    ops.gated_delta_scan(rows, rows, rows, sliced, sliced, 2, 2, 2)
    assert seen == [(4, 2), (2, 4), (4, 4)]


@pytest.mark.parametrize("ldb,text", [(3, "row strides"), (-4, "row strides")])
def test_a_stride_of_beta_that_does_not_hold_a_row_is_refused(ldb, text):
    import ctypes

    from jarvis_b200 import _lib
    from tests.test_block_operators_cpu import _delta
    assert _lib.load().jb200_gated_delta(ctypes.byref(_delta(ldb=ldb)), None, None) == _lib.ERR_ARG and text in _lib.last_error()


def _plan(B, T, H, sms=148):
    import ctypes

    from jarvis_b200 import _lib
    out = (ctypes.c_int32 * 2)()
    nbytes = _lib.load().jb200_host_delta_plan(B, T, H, sms, out)
    return out[0], out[1], nbytes


@pytest.mark.parametrize("B,T,H,pieces,chunks", [(1, 16384, 16, 6, 43), (2, 2048, 16, 3, 11), (1, 512, 16, 1, 8), (8, 2048, 16, 1, 32), (4, 2048, 16, 1, 32),
                                                 (1, 64, 16, 1, 1), (3, 777, 16, 1, 13), (0, 100, 16, 1, 0), (2, 0, 16, 1, 0)])
def test_pieces_of_a_sequence(B, T, H, pieces, chunks):
    """Worked out by hand from the rule's costs: (chunks + 1) (waves of 2 n - 3 CTAs a head + waves of n) + 1 + n / 4 against nine tenths of the chunks."""
    assert _plan(B, T, H)[:2] == (pieces, chunks)


@pytest.mark.parametrize("sms", [148, 132, 20])
def test_pieces_hold_a_sequence_and_none_is_empty(sms):
    cut = 0
    for B, H in ((1, 1), (1, 3), (1, 16), (2, 16), (3, 16), (5, 3), (64, 16)):
        for T in (*range(1, 4100, 61), 5000, 8191, 8192, 16384, 65536, 1 << 20, 1 << 30):
            n, chunks, nbytes = _plan(B, T, H, sms)
            whole = -(-T // 64)
            assert n == 1 or (3 <= n <= 32 and B * H * n <= 2 * sms)
            assert (n - 1) * chunks < whole <= n * chunks
            assert nbytes == (0 if n == 1 else (2 * n - 1) * B * H * 64 * 64 * 4)
            cut += n > 1
    assert cut > 100 or sms == 20
    assert _plan(64, 1 << 20, 16, sms)[0] == 1
