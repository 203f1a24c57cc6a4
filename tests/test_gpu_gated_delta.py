"""The gated delta rule against its recurrence in 64 bits, token by token, in all its forms.

How far results may lie from it:
  state   a token's update takes sums of 64 f32 products (12 2^-24 of the sum of their sizes, as trees of groups), at most six more roundings of u and
          three of the sum: 24 2^-24 of |S_i| + |v_i| for value row i, |k| being 1.  What earlier tokens were off by passes through
          a (I - b k k^T), which does not enlarge it, and roundings are independent: 24 2^-24 (1 + sqrt(T)) of the largest |S_i| + |v_i| there was
  o       rounded to bf16 (2^-8); the addends S q and (q.k) u pass at most three roundings to f16 on the way (2^-11 each, of the addend: with
          A_t = a A_{t-1} + |u| |k|^T they sum to scale A_t |q|), and q meets the state's error
"""
import math

import pytest
import torch

from jarvis_b200 import _lib, ops

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64
D = 64


def _problem(B, T, H, KH, seed=0, carry=True, lean=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * T + B)

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda")

    k = normal(B * T, KH, D) + lean * normal(1, KH, D) * torch.rand(B * T, 1, 1, generator=g, device="cuda")
    q = normal(B * T, KH, D) + 0.5 * k
    v = normal(B * T, H * D)
    log_decay = -0.05 * torch.nn.functional.softplus(3 * normal(B * T, H))
    beta = torch.sigmoid(2 * normal(B * T, H))
    state = normal(B, H, D, D) * 0.5 if carry else None
    return q.to(BF16).view(B * T, KH * D), k.to(BF16).view(B * T, KH * D), v.to(BF16), log_decay, beta, state


def _definition(q, k, v, log_decay, beta, state, B, T, H, KH, lengths=None, scale=0.125, normalize=True):
    """(o, state, what o and the state may be off by)."""
    q, k = (x.to(F64).view(B, T, KH, D).repeat_interleave(H // KH, 2) for x in (q, k))
    if normalize:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    v, a, b = v.to(F64).view(B, T, H, D), log_decay.to(F64).view(B, T, H, 1, 1).exp(), beta.to(F64).view(B, T, H, 1)
    S = torch.zeros(B, H, D, D, dtype=F64, device="cuda") if state is None else state.to(F64)
    A, most = S.abs(), S.norm(dim=-1)
    o, addends, size = (torch.zeros(B, T, H, D, dtype=F64, device="cuda") for _ in range(3))
    for t in range(T):
        on = torch.ones(B, 1, 1, 1, dtype=torch.bool, device="cuda") if lengths is None else (t < lengths).view(B, 1, 1, 1)
        kt, qt, vt = (torch.where(on[..., 0], x[:, t], 0.0) for x in (k, q, v))
        decayed = torch.where(on, a[:, t], 1.0) * S
        u = torch.where(on[..., 0], b[:, t], 0.0) * (vt - (decayed * kt[:, :, None]).sum(-1))
        S = decayed + u[..., None] * kt[:, :, None]
        A = torch.where(on, a[:, t], 1.0) * A + u.abs()[..., None] * kt.abs()[:, :, None]
        most = torch.maximum(most, S.norm(dim=-1) + vt.abs())
        o[:, t] = scale * (S * qt[:, :, None]).sum(-1)
        addends[:, t] = scale * (A * qt.abs()[:, :, None]).sum(-1)
        size[:, t] = scale * most * qt.norm(dim=-1, keepdim=True)
    off = 24 * 2.0 ** -24 * (1 + math.sqrt(T))
    tol = 2.0 ** -8 * o.abs() + 3 * 2.0 ** -11 * addends + off * size + 1e-30
    return o.view(B * T, H * D), S, tol.view(B * T, H * D), (off * most).unsqueeze(-1) + 1e-30


def _check(got, want):
    o, S = got
    wo, wS, tol, off = want
    if o is not None:
        assert o.dtype == BF16 and o.shape == wo.shape
        err = (o.to(F64) - wo).abs()
        assert torch.isfinite(o).all() and (err <= tol).all(), float((err / tol).max())
    if S is not None:
        err = (S.to(F64) - wS).norm(dim=-1, keepdim=True)
        assert torch.isfinite(S).all() and (err <= off).all(), float((err / off).max())


LENGTHS = [1, 2, 3, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 200, 511, 777]


@pytest.mark.parametrize("T", LENGTHS)
def test_lengths(T):
    B, H, KH = 2, 4, 2
    p = _problem(B, T, H, KH)
    _check(ops.gated_delta_scan(*p[:5], B, T, H, key_heads=KH, state_in=p[5], want_state=True), _definition(*p, B, T, H, KH))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("B,T,H,KH", [(1, 1, 1, 1), (1, 5, 3, 1), (1, 300, 1, 1), (1, 1500, 2, 1), (3, 70, 16, 8), (40, 130, 16, 16), (200, 1, 16, 4), (70, 9, 8, 8), (7, 64, 12, 3)])
@pytest.mark.parametrize("carry", [False, True])
def test_batches_and_heads(B, T, H, KH, carry):
    p = _problem(B, T, H, KH, carry=carry)
    _check(ops.gated_delta_scan(*p[:5], B, T, H, key_heads=KH, state_in=p[5], want_state=True), _definition(*p, B, T, H, KH))


@pytest.mark.parametrize("T", [1, 7, 64, 150, 400])
def test_padded_batches(T):
    """Rows behind a length: never read (they hold NaN), output 0, state untouched; lengths of nothing, one and beyond the end."""
    B, H, KH = 7, 2, 2
    q, k, v, g, b, s = _problem(B, T, H, KH)
    lengths = torch.tensor([0, 1, T, T // 2, max(T - 1, 0), T + 5, -3], dtype=torch.int32, device="cuda")
    pad = (torch.arange(T, device="cuda") >= lengths[:, None]).view(B * T)
    want = _definition(q, k, v, g, b, s, B, T, H, KH, lengths)
    for x in (q, k, v, g, b):
        x[pad] = float("nan")
    o, S = ops.gated_delta_scan(q, k, v, g, b, B, T, H, key_heads=KH, lengths=lengths, state_in=s, want_state=True)
    _check((o, S), want)
    assert not o[pad].any()
    assert torch.equal(S[0], s[0]) and torch.equal(S[6], s[6])


@pytest.mark.parametrize("T", [1, 6, 200])
def test_views_of_one_projection(T):
    B, H, KH = 3, 4, 2
    q, k, v, g, b, s = _problem(B, T, H, KH)
    wide = torch.full((B * T, 2 * KH * D + H * D + 24), float("nan"), device="cuda", dtype=BF16)
    wide[:, :KH * D], wide[:, KH * D:2 * KH * D], wide[:, 2 * KH * D:2 * KH * D + H * D] = q, k, v
    gates = torch.cat([g, b, g], 1)
    got = ops.gated_delta_scan(wide[:, :KH * D], wide[:, KH * D:2 * KH * D], wide[:, 2 * KH * D:2 * KH * D + H * D], gates[:, :H], gates[:, H:2 * H], B, T, H,
                               key_heads=KH, state_in=s, want_state=True, out=torch.full((B * T, H * D + 8), 7.0, device="cuda", dtype=BF16)[:, :H * D])
    plain = ops.gated_delta_scan(q, k, v, g, b, B, T, H, key_heads=KH, state_in=s, want_state=True)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


@pytest.mark.parametrize("B,T,H", [(2, 1, 4), (2, 40, 4), (2, 300, 4), (1, 2000, 2)])
def test_in_place_state_and_state_alone(B, T, H):
    p = _problem(B, T, H, H)
    o, S = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)
    none, alone = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True, want_out=False)
    s = p[5].clone()
    o2, S2 = ops.gated_delta_scan(*p[:5], B, T, H, state_in=s, state_out=s)
    o3, nothing = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5])
    assert none is None and nothing is None and S2 is s
    assert torch.equal(o, o2) and torch.equal(o, o3) and torch.equal(S, S2) and torch.equal(S, alone)


@pytest.mark.parametrize("T,cut", [(200, 64), (200, 77), (130, 129), (20, 3)])
def test_state_hands_over(T, cut):
    """A prompt in two calls, the second from the first's state, is the prompt in one."""
    B, H = 2, 3
    q, k, v, g, b, s = _problem(B, T, H, H)
    rows = torch.arange(B * T, device="cuda").view(B, T)
    first, second = rows[:, :cut].reshape(-1), rows[:, cut:].reshape(-1)
    want = _definition(q, k, v, g, b, s, B, T, H, H)
    o1, s1 = ops.gated_delta_scan(*(x[first] for x in (q, k, v, g, b)), B, cut, H, state_in=s, want_state=True)
    o2, s2 = ops.gated_delta_scan(*(x[second] for x in (q, k, v, g, b)), B, T - cut, H, state_in=s1, want_state=True)
    o = torch.empty_like(v)
    o[first], o[second] = o1, o2
    _check((o, s2), want)


@pytest.mark.parametrize("T", [3, 150, 1200])
def test_strong_and_infinite_decays(T):
    """Decays of many e-folds a token, and tokens that forget everything, beside ones that forget nothing."""
    B, H = 1, 2
    q, k, v, g, b, s = _problem(B, T, H, H)
    g[:, 0] = -20.0 * torch.rand(T, device="cuda")
    g[1::5, 1] = -math.inf
    g[2::5, 1] = 0.0
    g[2::7, 1] = -500.0
    b[::3] = 0.0
    b[1::3] = 1.0
    _check(ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True), _definition(q, k, v, g, b, s, B, T, H, H))


@pytest.mark.parametrize("T", [1, 12, 190])
def test_keys_that_are_alike_zero_tiny_or_large(T):
    """Keys that all but coincide (the system of a chunk is as ill-tempered as it gets), rows of zeros, rows of every size."""
    B, H = 2, 2
    for kind in range(3):
        q, k, v, g, b, s = _problem(B, T, H, H, lean=30.0 if kind == 0 else 1.5)
        if kind == 1:
            k[::2] = 0
            q[::3] = 0
        if kind == 2:
            size = torch.logspace(-14, 14, B * T, device="cuda")[:, None]
            k, q = (k.float() * size).to(BF16), (q.float() / size).to(BF16)
        b = b ** 0.1
        _check(ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True), _definition(q, k, v, g, b, s, B, T, H, H))


@pytest.mark.parametrize("T", [1, 10, 170])
@pytest.mark.parametrize("size", [1e-20, 1.0, 1e20])
def test_values_of_any_size(T, size):
    B, H = 1, 3
    q, k, v, g, b, s = _problem(B, T, H, H)
    v, s = (v.float() * size).to(BF16), s * size
    _check(ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True), _definition(q, k, v, g, b, s, B, T, H, H))


@pytest.mark.parametrize("T", [1, 12, 190])
def test_keys_taken_as_they_are(T):
    """normalize=False with keys of norm 0.1 to 1.4 and another scale."""
    B, H = 2, 2
    q, k, v, g, b, s = _problem(B, T, H, H)
    k = (torch.nn.functional.normalize(k.float().view(-1, D), dim=1) * (0.1 + 1.2 * torch.rand(B * T * H, 1, device="cuda"))).to(BF16).view(B * T, H * D)
    got = ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True, normalize=False, scale=0.01)
    wo, wS, tol, off = _definition(q, k, v, g, b, s, B, T, H, H, normalize=False, scale=0.01)
    _check(got, (wo, wS, 2 * tol, 2 * off))          # |k|^2 of up to 1.7 for the 1 of the derivation


def test_one_token_calls_follow_a_prompt():
    B, T, H, KH = 2, 90, 4, 4
    q, k, v, g, b, s = _problem(B, T, H, KH)
    at = torch.arange(B * T, device="cuda").view(B, T)
    want = _definition(q, k, v, g, b, s, B, T, H, KH)
    o = torch.empty_like(v)
    o[at[:, :70].reshape(-1)], S = ops.gated_delta_scan(*(x[at[:, :70].reshape(-1)] for x in (q, k, v, g, b)), B, 70, H, state_in=s, want_state=True)
    for t in range(70, T):
        o[at[:, t]], S = ops.gated_delta_scan(*(x[at[:, t]] for x in (q, k, v, g, b)), B, 1, H, state_in=S, state_out=S)
    _check((o, S), want)


@pytest.mark.parametrize("B,T", [(2, 1), (2, 200), (1, 1500)])
def test_same_bits_every_time_on_any_stream_and_in_a_graph(B, T):
    H = 2
    p = _problem(B, T, H, H)
    o, S = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, S2 = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)
    side.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, S3 = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)
    with torch.cuda.graph(graph2):
        o4, S4 = ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)
    for _ in range(2):
        o3.zero_(), S3.zero_(), o4.zero_(), S4.zero_()
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        for x, y in ((o, o2), (o, o3), (o, o4), (S, S2), (S, S3), (S, S4)):
            assert torch.equal(x, y)


def test_empty_calls():
    z = torch.empty(0, 128, device="cuda", dtype=BF16)
    f = torch.empty(0, 2, device="cuda")
    s = torch.randn(3, 2, D, D, device="cuda")
    o, S = ops.gated_delta_scan(z, z, z, f, f, 3, 0, 2, state_in=s, want_state=True)
    assert o.shape == (0, 128) and torch.equal(S, s)
    o, S = ops.gated_delta_scan(z, z, z, f, f, 3, 0, 2, want_state=True)
    assert not S.any()
    o, S = ops.gated_delta_scan(z, z, z, f, f, 0, 5, 2, want_state=True)
    assert o.shape == (0, 128) and S.shape == (0, 2, D, D)


def test_rows_before_and_behind_are_left_alone():
    B, T, H = 2, 130, 2
    q, k, v, g, b, s = _problem(B, T, H, H)
    buf = torch.full((B * T + 2, H * D), 3.0, device="cuda", dtype=BF16)
    states = torch.full((B + 2, H, D, D), 3.0, device="cuda")
    ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, out=buf[1:-1], state_out=states[1:-1])
    assert (buf[0] == 3).all() and (buf[-1] == 3).all() and (states[0] == 3).all() and (states[-1] == 3).all()


def test_refusals():
    B, T, H = 2, 4, 2
    q, k, v, g, b, s = _problem(B, T, H, H)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        ops.gated_delta_scan(q.clone().requires_grad_(), k, v, g, b, B, T, H)
    with torch.no_grad():
        ops.gated_delta_scan(q.clone().requires_grad_(), k, v, g, b, B, T, H)
    with pytest.raises(RuntimeError, match="overlaps state_in"):
        two = torch.zeros(B * H * D * D + 4, device="cuda")
        ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=two[:-4].view(B, H, D, D), state_out=two[4:].view(B, H, D, D))
    with pytest.raises(RuntimeError, match="overlaps another"):
        ops.gated_delta_scan(q, k, v, g, b, B, T, H, out=v)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        ops.gated_delta_scan(torch.zeros(B * T, H * D + 4, device="cuda", dtype=BF16)[:, :H * D], k, v, g, b, B, T, H)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.gated_delta_scan(torch.zeros(B * T, H * D + 8, device="cuda", dtype=BF16)[:, 4:H * D + 4], k, v, g, b, B, T, H)
    with pytest.raises(RuntimeError, match="expected"):
        ops.gated_delta_scan(q, k, v[:, :64], g, b, B, T, H)
    with pytest.raises(RuntimeError, match="one length"):
        ops.gated_delta_scan(q, k, v, g, b, B, T, H, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="neither"):
        ops.gated_delta_scan(q, k, v, g, b, B, T, H, want_out=False)
    with pytest.raises(RuntimeError, match="state_in must be"):
        ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s[:1])
