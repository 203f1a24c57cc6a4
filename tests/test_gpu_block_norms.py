"""Norms around a block with gate and residual scale, against their definitions in 64 bits.

Roundings of f32 on the way to a result: the mean of C squares ((C / 8 + 12) 2^-24 in sums of eight, lanes and vectors, halved by the root), root,
weight, at most 2^-20 for the gate (an exponential of an argument of up to 88, a quotient), scale and sum: E = (C / 16 + 40) 2^-24 + 2^-20 of the
term, 2^-24 of the sum; then the result's own rounding.  The second norm has x' off by that, relative to a row's size.
"""
import pytest
import torch

from jarvis_b200 import _lib, ops

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


def _normal(*shape, seed=0, dtype=F32, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * size).to(dtype)


def _own(dtype):
    return 2.0 ** -8 if dtype is BF16 else 2.0 ** -24


def _norm(y, w, group, eps=EPS):
    y = y.to(F64)
    g = y.view(*y.shape[:-1], y.shape[-1] // group, group)
    return (g / (g.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)).view(y.shape)


def _silu(g):
    g = g.to(F64)
    return g * torch.sigmoid(g)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,C,group", [(1, 64, 64), (1, 8, 8), (37, 1024, 64), (3, 24, 8), (5, 768, 256), (301, 96, 32), (2, 256, 256), (700, 16, 16),
                                       (1, 1024, 1024), (33, 776, 776), (2, 8192, 8192), (700, 1024, 1024), (601, 72, 72), (5, 1032, 1032), (9, 4104, 4104)])
def test_gated_norm(N, C, group, gated, dtype, out_dtype):
    y, w = _normal(N, C, dtype=dtype, size=3.0), 1 + 0.3 * _normal(group, seed=1)
    gate = _normal(N, C, seed=2, dtype=dtype, size=4.0) if gated else None
    want = _norm(y, w, group) * (_silu(gate) if gated else 1.0)
    got = ops.gated_norm(y, w, gate, group=group, eps=EPS, out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == y.shape
    E = (group / 16 + 40) * 2.0 ** -24 + 2.0 ** -20
    assert ((got.to(F64) - want).abs() <= (E + _own(out_dtype) * (1 + E)) * want.abs() + 1e-38).all()


def _check_residual(got, x, y, wa, wb, gate, scale, out_dtype):
    C = x.shape[-1]
    term = _norm(y, wa, C) * (1.0 if gate is None else _silu(gate)) * (1.0 if scale is None else scale.to(F64))
    want = x.to(F64) + term
    E = (C / 16 + 40) * 2.0 ** -24 + 2.0 ** -20
    off = E * term.abs() + 2.0 ** -23 * want.abs() + 1e-38
    assert got[0].dtype == F32 and got[1].dtype == out_dtype
    assert ((got[0].to(F64) - want).abs() <= off).all()
    xn = _norm(want, wb, C)
    rms = (want.square().mean(-1, keepdim=True) + EPS).sqrt()
    moved = off / rms * wb.abs() + off.square().mean(-1, keepdim=True).sqrt() / rms * xn.abs()      # x' moved; the norm with it
    assert ((got[1].to(F64) - xn).abs() <= moved + (E + _own(out_dtype) * (1 + E)) * xn.abs() + 1e-38).all()


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("gated,scaled", [(False, True), (True, True), (True, False), (False, False)])
@pytest.mark.parametrize("N,C", [(1, 1024), (64, 1024), (37, 776), (5, 8), (700, 1024), (593, 72), (3, 8192), (2, 1032), (700, 2048)])
def test_residual_norm(N, C, gated, scaled, dtype, out_dtype):
    x, y = _normal(N, C, size=2.0), _normal(N, C, seed=1, dtype=dtype, size=5.0)
    wa, wb = 1 + 0.3 * _normal(C, seed=2), 1 + 0.3 * _normal(C, seed=3)
    gate = _normal(N, C, seed=4, dtype=dtype, size=4.0) if gated else None
    scale = 0.2 * _normal(C, seed=5) if scaled else None
    before = x.clone()
    got = ops.residual_norm(x, y, wa, wb, gate=gate, scale=scale, eps=EPS, out_dtype=out_dtype)
    assert torch.equal(x, before)
    _check_residual(got, before, y, wa, wb, gate, scale, out_dtype)
    same = ops.residual_norm(x, y, wa, wb, gate=gate, scale=scale, eps=EPS, out_dtype=out_dtype, out=x)
    assert same[0] is x and torch.equal(x, got[0]) and torch.equal(same[1], got[1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N", [1, 50, 900])
def test_strided_rows_and_leading_dimensions(N):
    C = 128
    wide = torch.full((N, 3 * C + 8), float("nan"), device="cuda", dtype=BF16)
    wide[:, :C], wide[:, C:2 * C] = _normal(N, C, dtype=BF16), _normal(N, C, seed=1, dtype=BF16)
    y, gate = wide[:, :C], wide[:, C:2 * C]
    for group in (32, C):
        w = 1 + 0.3 * _normal(group, seed=2)
        assert torch.equal(ops.gated_norm(y, w, gate, group=group), ops.gated_norm(y.contiguous(), w, gate.contiguous(), group=group))
    x, w = _normal(N, C, seed=5), torch.ones(C, device="cuda")
    a, b = ops.residual_norm(x, y, w, w, gate=gate), ops.residual_norm(x, y.contiguous(), w, w, gate=gate.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = ops.gated_norm(wide.view(1, N, -1)[..., :C].contiguous(), w, None)
    assert c.shape == (1, N, C) and torch.equal(c[0], ops.gated_norm(y, w))


def test_extreme_rows():
    """Rows of zeros, gates far out on both sides, rows of every size."""
    N, C = 8, 256
    w = torch.ones(C, device="cuda")
    y = _normal(N, C) * torch.logspace(-15, 15, N, device="cuda")[:, None]
    y[3] = 0
    gate = _normal(N, C, seed=1, size=60.0)
    gate[0, :6] = torch.tensor([1e30, -1e30, 100.0, -100.0, 0.0, -88.0], device="cuda")
    for group in (64, C):
        got = ops.gated_norm(y, w[:group], gate, group=group, out_dtype=F32)
        want = _norm(y, w[:group], group) * _silu(gate)
        E = (group / 16 + 40) * 2.0 ** -24 + 2.0 ** -16        # the gate's exponent of up to 300 is rounded: 300 2^-24
        assert torch.isfinite(got).all() and ((got.to(F64) - want).abs() <= E * want.abs() + 1e-30).all()
    assert not got[3].any()


def test_empty_rows_streams_and_graphs():
    w = torch.ones(64, device="cuda")
    z = torch.empty(0, 64, device="cuda", dtype=BF16)
    assert ops.gated_norm(z, w, z, group=64).shape == (0, 64)
    a, b = ops.residual_norm(torch.empty(0, 64, device="cuda"), z, w, w)
    assert a.shape == (0, 64) and b.shape == (0, 64)
    x, y, g = _normal(30, 64), _normal(30, 64, seed=1, dtype=BF16), _normal(30, 64, seed=2, dtype=BF16)
    want = (ops.gated_norm(y, w, g), *ops.residual_norm(x, y, w, w, gate=g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ops.gated_norm(y, w, g), *ops.residual_norm(x, y, w, w, gate=g))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = (ops.gated_norm(y, w, g), *ops.residual_norm(x, y, w, w, gate=g))
    graph.replay()
    torch.cuda.synchronize()
    for p, q, r in zip(want, got, captured):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_refusals():
    x, y, w = _normal(4, 64), _normal(4, 64, dtype=BF16), torch.ones(64, device="cuda")
    for call, text in ((lambda: ops.gated_norm(y, w, y.float()), "dtype"), (lambda: ops.gated_norm(y, w[:24], group=24), "power of two"),
                       (lambda: ops.gated_norm(y, w, group=32), "do not belong"), (lambda: ops.gated_norm(y, w, y[:3]), "do not belong"),
                       (lambda: ops.gated_norm(y.clone().requires_grad_(), w), "requires a gradient"),
                       (lambda: ops.gated_norm(y.t(), w[:4]), "unit inner stride"), (lambda: ops.gated_norm(y.half(), w), "float32 or bfloat16"),
                       (lambda: ops.gated_norm(_normal(2, 60, dtype=BF16), torch.ones(60, device="cuda")), "multiple of 8"),
                       (lambda: ops.gated_norm(_normal(2, 8200, dtype=BF16), torch.ones(8200, device="cuda")), "at most 8192"),
                       (lambda: ops.residual_norm(x, y[:3], w, w), "one shape"), (lambda: ops.residual_norm(x, y, w[:8], w), "does not fit"),
                       (lambda: ops.residual_norm(x.bfloat16(), y, w, w), "dtype"), (lambda: ops.residual_norm(x, y, w, w, out=x.view(2, 128)), "shape"),
                       (lambda: ops.residual_norm(x, x, w, w, out=x), "overlaps another"),
                       (lambda: ops.residual_norm(x, y, w.clone().requires_grad_(), w), "requires a gradient")):
        with pytest.raises(RuntimeError, match=text):
            call()
