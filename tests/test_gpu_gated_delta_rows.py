"""Value rows of the gated delta rule are independent of one another: rows of any sizes side by side, an outlier, an infinity or a NaN in one of them.

Tolerances are those of test_gpu_gated_delta.py, whose bounds go by value row: a row's own largest |S_i| + |v_i|, never another row's.  What the chunks add
to them, f16's floor 2^-40 below a bound of at most 120 |S_i| + 1400 |b v_i| (a norm's, carried over up to four chunks), is 2^-29 of it at each of
three operands: 3 2^-29 of the 24 2^-24 that a token is allowed.

Those bounds know what came before a token.  A chunk of 64 tokens has one power of two a value row, by the largest b v_i of all of them, so that what comes
later in the chunk counts as well (`_of_the_chunk`): with X = max (2 N + 130 |b v_i|) brought into [2^14, 2^15), f16's subnormal step 2^-24 rounds an
element of X and of U by at most 2^-25 / 2^14 X = 2^-39 X.  An error e of every b v_i moves the state's row by at most 64 e (nothing enlarges it), and
so the output by scale |q| 64 e; one of every u_i by at most as much, and one of every element of S by scale |q| 8 e.  Together scale |q| 136 2^-39 X, of which
2 N is covered above.
"""
import math

import pytest
import torch

from jarvis_b200 import _lib, ops
from tests.test_gpu_gated_delta import D, _check, _definition, _problem

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64


def _of_the_chunk(v, b, B, T, H, scale=0.125):
    """What outputs may be off by because of later tokens of their chunk; |q| is 1."""
    bv = (b.to(F64).view(B, T, H, 1) * v.to(F64).view(B, T, H, D)).abs()
    most = torch.cat([c.amax(1, keepdim=True).expand_as(c) for c in bv.split(64, 1)], 1)
    return (136 * 2.0 ** -39 * 130 * scale * most).view(B * T, H * D)


FORMS = [(2, 1), (2, 10), (2, 64), (2, 190), (3, 777), (1, 1500)]            # token by token, a chunk, chunks, segments


def _scan(p, B, T, H, **kw):
    return ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True, **kw)


@pytest.mark.parametrize("B,T", FORMS)
@pytest.mark.parametrize("decades", [6, 24])
def test_value_rows_of_every_size_side_by_side(B, T, decades):
    H = 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=11)
    size = torch.logspace(-decades / 2, decades / 2, D, device="cuda")[torch.randperm(D, generator=torch.Generator().manual_seed(T)).cuda()]
    v, s = (v.float().view(B * T, H, D) * size).to(BF16).view(B * T, H * D), s * size[:, None]
    p = (q, k, v, g, b, s)
    _check(_scan(p, B, T, H), _definition(*p, B, T, H, H))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("B,T", [(2, 10), (2, 190), (1, 1500)])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e12, 1e30])
def test_an_outlier_stays_in_its_value_row(B, T, size):
    """One large element of v in the middle; the other rows keep bounds that know nothing of it, before and behind it, and so does its own before its
    chunk."""
    H = 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=12)
    v[T // 2, 5] = size
    v[T // 3, D + 40] = -size
    p = (q, k, v, g, b, s)
    wo, wS, tol, off = _definition(*p, B, T, H, H)
    _check(_scan(p, B, T, H), (wo, wS, tol + (_of_the_chunk(v, b, B, T, H) if T > 24 else 0.0), off))


@pytest.mark.parametrize("B,T", [(2, 10), (2, 190), (1, 1500)])
def test_tokens_that_write_nothing_may_hold_anything_large(B, T):
    """beta 0 beside values of 1e30: nothing of them is written."""
    H = 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=13)
    v[::3] = (v[::3].float() * 1e30).to(BF16)
    b[::3] = 0.0
    v0 = v.clone()
    v0[::3] = 0.0
    p = (q, k, v, g, b, s)
    _check(_scan(p, B, T, H), _definition(q, k, v0, g, b, s, B, T, H, H))


@pytest.mark.parametrize("B,T", [(2, 10), (2, 190), (1, 1500)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["v", "state"])
def test_infinities_and_nan_stay_in_their_value_row(B, T, bad, where):
    """The other rows: within their bounds, all along.  The row itself: right before the token's chunk (before the token, without chunks), neither
    finite in the state nor in its last output."""
    H, at, row = 2, T // 2, 37
    q, k, v, g, b, s = _problem(B, T, H, H, seed=14)
    want = _definition(q, k, v, g, b, s, B, T, H, H)
    if where == "v":
        v[at, row] = bad                             # sequence 0, head 0
    else:
        s[0, 0, row, 9] = bad
    o, S = _scan((q, k, v, g, b, s), B, T, H)
    wo, wS, tol, off = want
    assert not torch.isfinite(S[0, 0, row]).any() and not torch.isfinite(o[T - 1, row])
    good = 0 if where == "state" else at // 64 * 64 if T > 24 else at
    o[good:T, row] = wo[good:T, row].to(BF16)
    S[0, 0, row] = wS[0, 0, row].float()
    _check((o, S), (wo, wS, tol, off))
    assert _lib.device_status() == 0


def test_rows_do_not_know_of_one_another():
    """The bits of a value row are the same whatever the others hold."""
    B, T, H = 2, 333, 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=15)
    o, S = _scan((q, k, v, g, b, s), B, T, H)
    keep = torch.arange(D, device="cuda") % 3 == 1
    v2 = torch.where(keep.repeat(H), v.float(), v.float() * 1e15 + 3).to(BF16)
    s2 = torch.where(keep[:, None], s, s * 1e-15)
    o2, S2 = _scan((q, k, v2, g, b, s2), B, T, H)
    assert torch.equal(S[:, :, keep], S2[:, :, keep]) and torch.equal(o[:, keep.repeat(H)], o2[:, keep.repeat(H)])


@pytest.mark.parametrize("B,T", FORMS)
def test_keys_and_queries_whose_squares_leave_f32(B, T):
    """Sums of squares from nothing to 2^250: normalised rows are what they are at any size that bf16 holds."""
    H = 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=16)
    size = torch.logspace(-30, 37, B * T, device="cuda")[torch.randperm(B * T, generator=torch.Generator().manual_seed(T)).cuda()][:, None]
    if T == 1:
        size = torch.tensor([[1e37], [1e22]], device="cuda")
    k, q = (k.float() * size).to(BF16), (q.float() * size.flip(0)).to(BF16)
    assert torch.isfinite(k).all() and torch.isfinite(q).all() and (k.float().view(B * T, H, D).square().sum(-1) == math.inf).any()
    p = (q, k, v, g, b, s)
    _check(_scan(p, B, T, H), _definition(*p, B, T, H, H))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("B,T", [(2, 10), (2, 190)])
@pytest.mark.parametrize("size", [1e-25, 1e25, 1e36])
def test_queries_of_any_size_taken_as_they_are(B, T, size):
    H = 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=17)
    k = torch.nn.functional.normalize(k.float().view(-1, D), dim=1).to(BF16).view(B * T, H * D)
    q = (q.float() * size).to(BF16)
    p = (q, k, v, g, b, s)
    wo, wS, tol, off = _definition(*p, B, T, H, H, normalize=False, scale=0.125 / size)
    _check(_scan(p, B, T, H, normalize=False, scale=0.125 / size), (wo, wS, 2 * tol, 2 * off))      # |k|^2 of up to 1 + 2^-7 for the 1 of the derivation


@pytest.mark.parametrize("T,H", [(10, 1), (190, 1), (777, 1), (1500, 1), (777, 128)])       # the last one whole, the two before it in segments
def test_unit_keys_that_bf16_has_rounded_up(T, H):
    """normalize=False, beta 2 and one key throughout, of norm 1 before bf16 rounds half of it up by 2^-8: every token enlarges the state by 1.0078,
    token by token or in chunks alike.  Rows are all along the key, where nothing of their bounds is to spare: one that did not allow for the growth would
    overflow in f16, and nothing would be finite.  Token by token the tolerance holds twice, |k|^2 being 1 + 2^-8 for the 1 of the derivation.  In chunks
    the system of alike keys with beta 2 is ill-conditioned (its inverse is +-2 throughout, sums of 64 that cancel), which the interface states; no
    tolerance is derived for it, and what is asked is that it stays finite."""
    a = 0.12549
    key = torch.tensor([a] * 32 + [math.sqrt(1 / 32 - a * a)] * 32, device="cuda")
    k = key.to(BF16).repeat(H).expand(T, H * D).contiguous()
    assert abs(float(key.norm()) - 1) < 1e-6 and 2 * float(k[0, :D].double().square().sum()) > 2.0076
    v, g, b = torch.zeros(T, H * D, device="cuda", dtype=BF16), torch.zeros(T, H, device="cuda"), torch.full((T, H), 2.0, device="cuda")
    s = (torch.logspace(-3, 3, D, device="cuda")[:, None] * k[0, :D].float()).expand(1, H, D, D).contiguous()
    p = (k, k, v, g, b, s)
    wo, wS, tol, off = _definition(*p, 1, T, H, H, normalize=False, scale=1.0)
    assert float(wS.abs().max()) > 1.007 ** T * 100
    o, S = _scan(p, 1, T, H, normalize=False, scale=1.0)
    assert torch.isfinite(o).all() and torch.isfinite(S).all()
    if T == 10:
        _check((o, S), (wo, wS, 2 * tol, 2 * off))


@pytest.mark.parametrize("B,T", [(2, 10), (2, 190), (1, 1500)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("where", ["q", "k", "log_decay", "beta"])
def test_infinities_and_nan_of_keys_and_gates_stay_in_their_head(B, T, bad, where):
    """The bits of everything else: other heads, other sequences, chunks (tokens, without chunks) before; of a query all but its token's output."""
    H, at = 3, T // 2
    q, k, v, g, b, s = _problem(B, T, H, H, seed=18)
    o, S = _scan((q, k, v, g, b, s), B, T, H)
    if where in "qk":
        (q if where == "q" else k)[at, D + 7] = bad                   # sequence 0, head 1
    else:
        (g if where == "log_decay" else b)[at, 1] = bad
    o2, S2 = _scan((q, k, v, g, b, s), B, T, H)
    same = torch.ones(B * T, H, dtype=torch.bool, device="cuda")
    if where == "q":
        assert not torch.isfinite(o2[at, D:2 * D]).any()
        same[at, 1] = False
    else:
        assert not torch.isfinite(S2[0, 1]).any() and not torch.isfinite(o2[T - 1, D:2 * D]).any()
        same[at // 64 * 64 if T > 24 else at:T, 1] = False
    same = same.repeat_interleave(D, 1)
    assert torch.equal(torch.where(same, o, 0.0), torch.where(same, o2, 0.0))
    others = torch.ones(B, H, dtype=torch.bool, device="cuda")
    others[0, 1] = where == "q"
    assert torch.equal(S[others], S2[others])
    assert _lib.device_status() == 0
