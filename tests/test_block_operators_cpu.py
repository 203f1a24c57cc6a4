"""Gated delta rule, norms around a block and draws of rows without a GPU: refusals that need no launch, and scratch sizes."""
import ctypes as C

import pytest
import torch

from jarvis_b200 import _lib, ops

BF16, F32 = torch.bfloat16, torch.float32
A = 4096                     # an address that is never read: every call here is refused first


def _delta(**kw):
    d = _lib.Delta(2, 100, 4, 2, 64, 0, A, A, A, 128, 128, 256, A, A, 4, None, 0.125, None, A, 256, A)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,text", [(dict(B=-1), "bad shape"), (dict(T=-1), "bad shape"), (dict(H=0), "bad shape"), (dict(key_heads=0), "bad shape"),
                                     (dict(key_heads=3), "bad shape"), (dict(key_heads=8), "bad shape"), (dict(head_dim=128), "head_dim"),
                                     (dict(B=2 ** 15, T=2 ** 16), "too many"), (dict(B=2 ** 20, H=2 ** 10), "too many"), (dict(o=None, s_out=None), "neither"),
                                     (dict(q=None), "null"), (dict(beta=None), "null"), (dict(ldq=120), "row strides"), (dict(ldv=248), "row strides"),
                                     (dict(ldg=3), "row strides"), (dict(ldo=0), "row strides"), (dict(k=A + 8), "16-byte"), (dict(s_in=A + 4), "16-byte"),
                                     (dict(ldk=132), "multiples of 8"), (dict(ldo=260), "multiples of 8")])
def test_gated_delta_refuses(kw, text):
    lib = _lib.load()
    assert lib.jb200_gated_delta(C.byref(_delta(**kw)), None, None) == _lib.ERR_ARG
    assert text in _lib.last_error()
    assert lib.jb200_gated_delta(None, None, None) == _lib.ERR_ARG


def test_gated_delta_without_sequences_is_no_call():
    assert _lib.load().jb200_gated_delta(C.byref(_delta(B=0)), None, None) == 0


def test_scratch_is_bounded_by_a_state_for_every_piece():
    """2 n - 1 states a head for n segments, n at most 32, none for short sequences or many heads."""
    lib = _lib.load()
    for B, H in ((1, 1), (1, 16), (2, 16), (5, 3), (64, 16)):
        for T in (0, 1, 23, 64, 128, 1000, 2048, 16384, 1 << 20):
            n = lib.jb200_gated_delta_scratch_bytes(B, T, H)
            assert n % (B * H * 16384) == 0 and n <= 63 * B * H * 16384
            assert T > 128 or n == 0
            assert B * H <= 148 or n == 0
    assert lib.jb200_gated_delta_scratch_bytes(0, 5000, 4) == 0 and lib.jb200_gated_delta_scratch_bytes(1, 5000, 0) == 0


@pytest.mark.parametrize("width,ldy,addr,dtype,text", [(60, 64, A, 0, "multiple of 8"), (0, 64, A, 0, "multiple of 8"), (8200, 8200, A, 0, "at most"),
                                                       (64, 60, A, 0, "row strides"), (64, 68, A, 1, "row strides"), (64, 64, A + 8, 0, "aligned"),
                                                       (64, 64, None, 0, "null"), (64, 64, A, 2, "dtypes")])
def test_norms_refuse(width, ldy, addr, dtype, text):
    lib = _lib.load()
    assert lib.jb200_gated_norm(addr, dtype, ldy, A, None, 0, width, 1e-6, A, 0, 3, width, None) == _lib.ERR_ARG and text in _lib.last_error()
    assert lib.jb200_residual_norm(A, addr, dtype, ldy, A, None, 0, None, A, 1e-6, A, A, 0, 3, width, None) == _lib.ERR_ARG and text in _lib.last_error()


def test_norms_refuse_groups_and_what_is_missing():
    lib = _lib.load()
    for group in (0, 4, 24, 512, 96):
        assert lib.jb200_gated_norm(A, 0, 192, A, None, 0, group, 1e-6, A, 0, 3, 192, None) == _lib.ERR_ARG and "group" in _lib.last_error()
    assert lib.jb200_gated_norm(A, 0, 64, A, A, 56, 64, 1e-6, A, 0, 3, 64, None) == _lib.ERR_ARG and "row strides" in _lib.last_error()
    assert lib.jb200_gated_norm(A, 0, 64, A, A + 8, 64, 64, 1e-6, A, 0, 3, 64, None) == _lib.ERR_ARG and "aligned" in _lib.last_error()
    for x, x_out, w, scale, text in ((None, A, A, None, "null"), (A, None, A, None, "null"), (A, A, None, None, "null"), (A + 4, A, A, None, "aligned"),
                                     (A, A + 4, A, None, "aligned"), (A, A, A, A + 4, "aligned")):
        assert lib.jb200_residual_norm(x, A, 0, 64, A, None, 0, scale, w, 1e-6, x_out, A, 0, 3, 64, None) == _lib.ERR_ARG and text in _lib.last_error()
    assert lib.jb200_gated_norm(A, 0, 64, A, None, 0, 64, 1e-6, A, 0, 0, 64, None) == 0              # no rows


@pytest.mark.parametrize("kw,rows,text", [(dict(V=0), 2, "bad shape"), (dict(ld=90), 2, "bad shape"), (dict(), -1, "bad shape"), (dict(V=2 ** 24 + 1, ld=2 ** 25), 2, "2^24"),
                                          (dict(logits_dtype=2), 2, "dtype"), (dict(logits=None), 2, "null"), (dict(u=None), 2, "null")])
def test_draws_refuse(kw, rows, text):
    lib = _lib.load()
    s = _lib.Sampling(A, 100, 0, 100, A)
    for k, v in kw.items():
        setattr(s, k, v)
    assert lib.jb200_sample_rows(C.byref(s), rows, A, None, None) == _lib.ERR_ARG
    assert text in _lib.last_error()
    assert lib.jb200_sample_rows(C.byref(_lib.Sampling(A, 100, 0, 100, A)), 2, None, None, None) == _lib.ERR_ARG
    assert lib.jb200_sample_rows(None, 2, A, None, None) == _lib.ERR_ARG
    assert lib.jb200_sample_rows(C.byref(_lib.Sampling(A, 100, 0, 100, A)), 0, A, None, None) == 0


def test_host_tensors_raise():
    rows, g, x = torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 2), torch.zeros(4, 128)
    for call in (lambda: ops.gated_delta_scan(rows, rows, rows, g, g, 2, 2, 2), lambda: ops.gated_norm(x, torch.ones(128)),
                 lambda: ops.residual_norm(x, x, torch.ones(128), torch.ones(128)), lambda: ops.sample_rows(x, torch.zeros(4))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="bad shape"):
        ops.gated_delta_scan(rows, rows, rows, g, g, 2, 2, 2, key_heads=3)


class _OnCard(torch.Tensor):
    """A host tensor that says it is on the card `card`."""
    card = 0
    is_cuda = property(lambda self: True)

    def get_device(self):
        return self.card

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))


def _on(card, *shape, dtype=F32):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(_OnCard)
    t.card = card
    return t


def test_launches_on_the_tensors_card(monkeypatch):
    current, seen = [0], []

    class Card:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def __getattr__(self, name):
            if name.endswith("_scratch_bytes"):
                return lambda *a: 0
            return lambda *a: seen.append((name, current[0])) or 0

    monkeypatch.setattr(ops._lib, "load", lambda: Lib())
    monkeypatch.setattr(ops, "_raw_device", lambda: current[0])
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops.torch.cuda, "device", Card)

    def calls(card, other):
        rows, g, x = _on(card, 4, 128, dtype=BF16), _on(card, 4, 2), _on(card, 4, 128)
        return (lambda: ops.gated_delta_scan(rows, rows, rows, g, _on(other, 4, 2), 2, 2, 2), lambda: ops.gated_norm(rows, _on(other, 64), rows, group=64),
                lambda: ops.residual_norm(x, rows, _on(other, 128), _on(card, 128)), lambda: ops.sample_rows(x, _on(other, 4), top_p=_on(card, 4)))

    names = ["jb200_gated_delta", "jb200_gated_norm", "jb200_residual_norm", "jb200_sample_rows"]
    for card in (1, 0):
        for call in calls(card, card):
            call()
        assert seen == [(n, card) for n in names] and current == [0]
        seen.clear()
    for call in calls(0, 1) + calls(1, 0):
        with pytest.raises(RuntimeError, match="tensors on cuda"):
            call()
    assert not seen


def test_tensors_that_require_a_gradient_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_raw_device", lambda: 0)
    rows, g, x, w = _on(0, 4, 128, dtype=BF16), _on(0, 4, 2), _on(0, 4, 128), _on(0, 128)
    w.requires_grad_(True)
    x.requires_grad_(True)
    for call in (lambda: ops.gated_norm(rows, w), lambda: ops.residual_norm(x, rows, _on(0, 128), _on(0, 128)),
                 lambda: ops.gated_delta_scan(rows, rows, rows, g, g, 2, 2, 2, state_in=_on(0, 2, 2, 64, 64).requires_grad_(True))):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
