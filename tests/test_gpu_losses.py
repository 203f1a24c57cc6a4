"""Losses of the head without logits, the gradients of head and norm, against their definitions in 64 bits.

How far results may lie from those is bounded element by element from the roundings there are:
  logits   C products in groups of 16, each group's addition to the f32 sum off by at most 2^-23 of a partial sum <= sum |x w|, plus the
           sum inside a group: Z = (C / 16 + 8) 2^-23 max sum |x w|
  losses   a log of a sum whose terms move by a factor exp(+-Z), and the target's logit: 2 Z, plus 2^-22 of the value (f32 logarithm,
           storage); a temperature divides Z and its square multiplies the loss
  dz       e^2Z - 1 < 3 Z of the probability (plus 2^-20 for the exponential and its argument), then f16 relative to 2^-13 of the largest
           factor: 2^-11, and 2^-38 of that factor where f16 is subnormal
  dx, dW   the products of those: |error| <= (2^-11 + 3 Z + 2^-19) sum |dz| |operand|, plus the f32 sum (terms / 16 + 72) 2^-23 of the same
           sum, plus what f16 takes from the other operand, at most 2^-25 of its largest value each, plus the result's own
           rounding, 2^-8 for bf16
where sum |dz| |operand| takes the positive and the negative parts of dz apart (a probability and a target of the same entry cancel only
after the first has been rounded).
"""
import math

import pytest
import torch

from jarvis_b200 import _lib, losses, ops

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _problem(N, V, width, K, seed=0, sharp=2.5):
    g = _gen(seed + 7 * N + V)
    h = torch.randn(N, width, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, width, generator=g, device="cuda") * sharp / math.sqrt(width)).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[1::7] = -100
    ids = torch.randint(0, V, (N, K), generator=g, device="cuda")          # an id may come twice
    logits = torch.randn(N, K, generator=g, device="cuda") * 3
    ids[torch.rand(N, K, generator=g, device="cuda") < 0.2] = -1
    ids[2::9] = -1
    ids[0] = torch.arange(K, device="cuda") % V
    return h, w, t, ids, logits


def _definition(h, w, t, ids, logits, tau, g_ce, g_kd):
    """Rows' losses, dx, dW and the bounds on them.  g_ce, g_kd: the losses' gradients, a value per row."""
    N, width = h.shape
    x, wd = h.to(F64), w.to(F64)
    z = x @ wd.t()
    Z = (width / 16 + 8) * 2.0 ** -23 * float((x.abs() @ wd.abs().t()).max())
    pos, neg = torch.zeros_like(z), torch.zeros_like(z)
    out = dict(Z=Z)
    if t is not None:
        on = t != -100
        lp = torch.log_softmax(z, 1)
        out["ce"] = torch.where(on, -lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
        f = (g_ce.to(F64) * on)[:, None]
        pos += f.abs() * lp.exp()
        neg.scatter_add_(1, t.clamp(min=0)[:, None], f.abs())
        dz = f * lp.exp()
        dz.scatter_add_(1, t.clamp(min=0)[:, None], -f)
    else:
        dz = torch.zeros_like(z)
    if ids is not None:
        kept = ids >= 0
        on = (kept & (logits > -math.inf)).any(1)
        q = torch.softmax(torch.where(kept, logits.to(F64) / tau, -math.inf), 1)
        q = torch.where(kept & on[:, None], q, 0.0)
        full = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
        lp = torch.log_softmax(z / tau, 1)
        out["kd"] = tau * tau * ((torch.special.xlogy(q, q)).sum(1) - (full * lp).sum(1))
        f = (g_kd.to(F64) * on * tau)[:, None]
        pos += f.abs() * lp.exp()
        neg += f.abs() * full
        dz = dz + f * (lp.exp() - full)
    out["dx"], out["dw"] = dz @ wd, dz.t() @ x
    size = pos + neg
    rel = 2.0 ** -11 + 3 * Z + 2.0 ** -19
    factor = max(0.0 if t is None else float((g_ce.abs() * (t != -100)).max()), 0.0 if ids is None else float(g_kd.abs().max()) * tau)
    out["dx_bound"] = (rel + (w.shape[0] / 16 + 72) * 2.0 ** -23) * (size @ wd.abs()) + 2.0 ** -25 * wd.abs().max() * size.sum(1, keepdim=True) + \
        2.0 ** -38 * factor * wd.abs().sum(0)
    out["dw_bound"] = (rel + (N / 16 + 72) * 2.0 ** -23) * (size.t() @ x.abs()) + 2.0 ** -25 * x.abs().max() * size.sum(0)[:, None] + \
        2.0 ** -38 * factor * x.abs().sum(0)
    return out


def _check_rows(got, want, Z, tau=1.0):
    # the divergence also holds q log q, sums of f32 logarithms of at most 10: 2^-20
    assert ((got.to(F64) - want).abs() <= 2 * Z * max(tau, 1.0) + 2.0 ** -22 * want.abs() + tau * tau * 2.0 ** -19).all()


def _check_grad(got, want, bound):
    own = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24
    err = (got.to(F64) - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound * (1 + own) + own * want.abs() + 1e-38).all(), float((err / (bound + own * want.abs() + 1e-38)).max())


SIZES = [(1, 1, 64, 1), (1, 300, 64, 1), (37, 1000, 72, 5), (128, 256, 64, 256), (257, 257, 136, 3), (300, 2049, 256, 16), (64, 250, 128, 100),
         (1000, 777, 776, 33), (2, 50257, 1024, 64), (513, 9001, 2048, 7)]


@pytest.mark.parametrize("mode", ["ce", "kd", "both"])
@pytest.mark.parametrize("N,V,width,K", SIZES)
def test_losses_and_gradients(N, V, width, K, mode):
    h, w, t, ids, logits = _problem(N, V, width, K)
    tau = 2.0 if K % 2 else 1.0
    a, b = 0.3, 0.7
    t, ids = (t if mode != "kd" else None), (ids if mode != "ce" else None)
    n_ce = int((t != -100).sum()) if t is not None else 1
    n_kd = int((ids >= 0).any(1).sum()) if ids is not None else 1
    one = torch.ones(N, device="cuda", dtype=F64)
    want = _definition(h, w, t, ids, logits, tau, one * a / n_ce, one * b / n_kd)
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    rows = []
    if mode == "ce":
        loss = a * losses.linear_cross_entropy(x, wt, t)
        rows = [(losses.linear_cross_entropy(x, wt, t, reduction="none"), "ce", 1.0)]
    elif mode == "kd":
        loss = b * losses.linear_distillation(x, wt, ids, logits, temperature=tau)
        rows = [(losses.linear_distillation(x, wt, ids, logits, temperature=tau, reduction="none"), "kd", tau)]
    else:
        ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=tau)
        loss = a * ce + b * kd
        r = losses.linear_losses(x, wt, t, ids, logits, temperature=tau, reduction="none")
        rows = [(r[0], "ce", 1.0), (r[1], "kd", tau)]
    for got, name, tt in rows:
        assert got.dtype == torch.float32 and got.shape == (N,)
        _check_rows(got, want[name], want["Z"], tt)
    total = sum((a if name == "ce" else b) * want[name].sum() / (n_ce if name == "ce" else n_kd) for _, name, _ in rows)
    assert abs(loss.item() - float(total)) <= 2 * want["Z"] * max(tau, 1) + 2.0 ** -20 * abs(float(total)) + tau * tau * 2.0 ** -19
    dx, dw = torch.autograd.grad(loss, (x, wt))
    assert dx.dtype == dw.dtype == BF16
    _check_grad(dx, want["dx"], want["dx_bound"])
    _check_grad(dw, want["dw"], want["dw_bound"])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N,V", [(9000, 40001), (6500, 60001), (9000, 53300), (20000, 20000)])
def test_pieces_of_the_vocabulary(N, V):
    """More than one piece, one slab of dx and several, a last piece that is short, f32 gradients of f32 arguments."""
    out = (_lib.C.c_int32 * 3)()
    assert _lib.load().jb200_host_head_plan(N, V, 64, 148, out) == 0 and out[1] > 1
    h, w, t, ids, logits = _problem(N, V, 64, 8)
    g = torch.rand(N, generator=_gen(1), device="cuda") - 0.3
    x, wt = h.float().requires_grad_(), w.float().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=1.5, reduction="none")
    dx, dw = torch.autograd.grad((ce * g + kd * g.flip(0)).sum(), (x, wt))
    assert dx.dtype == dw.dtype == torch.float32
    want = _definition(h, w, t, ids, logits, 1.5, g, g.flip(0))
    _check_rows(ce, want["ce"], want["Z"])
    _check_rows(kd, want["kd"], want["Z"], 1.5)
    _check_grad(dx, want["dx"], want["dx_bound"])
    _check_grad(dw, want["dw"], want["dw_bound"])


def test_gradients_against_differences():
    """(L(x + d) - L(x - d)) / 2 = <dL, d> up to the third order: the logits move by at most D = max sum |d w| (rows) and the second
    derivative of log-sum-exp along that is a variance, so the remainder is at most D^3 / 3 of a row's loss."""
    g = _gen(3)
    N, V, width, K = 6, 90, 64, 4
    grid = lambda *s: (torch.randint(-60, 61, s, generator=g, device="cuda") / 64).bfloat16()      # noqa: E731  (and a 64th away: exact)
    h, w = grid(N, width), grid(V, width) / 4
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    ids = torch.randint(0, V, (N, K), generator=g, device="cuda")
    logits = torch.randn(N, K, generator=g, device="cuda")

    def total(x, wt):
        ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=2.0)
        return ce + kd
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(total(x, wt), (x, wt))
    for _ in range(4):
        d = torch.randint(-1, 2, h.shape, generator=g, device="cuda").bfloat16() / 64
        diff = (total(h + d, w).double() - total(h - d, w).double()) / 2
        D = float((d.abs().double() @ w.abs().double().t()).max())
        err = 2 * D ** 3 / 3 + 2.0 ** -19 * 20 + 2.0 ** -7 * float((dx.double() * d.double()).abs().sum())
        assert abs(float(diff) - float((dx.double() * d.double()).sum())) <= err
        e = torch.randint(-1, 2, w.shape, generator=g, device="cuda").bfloat16() / 256
        diff = (total(h, w + e).double() - total(h, w - e).double()) / 2
        D = float((h.abs().double() @ e.abs().double().t()).max())
        err = 2 * D ** 3 / 3 + 2.0 ** -19 * 20 + 2.0 ** -7 * float((dw.double() * e.double()).abs().sum())
        assert abs(float(diff) - float((dw.double() * e.double()).sum())) <= err


def test_rows_that_have_no_part():
    """Rows without target and teacher: loss 0, gradient 0, whatever they hold; entries with a negative id: whatever their logit is."""
    h, w, t, ids, logits = _problem(40, 500, 64, 6)
    t[5:9] = -100
    ids[5:9] = -1
    clean = losses.linear_losses(h, w, t, ids, logits, reduction="none")
    x = h.clone()
    x[5], x[6, 3], x[7, 1], x[8] = math.nan, math.inf, -math.inf, 3e38
    bad = logits.clone()
    bad[ids < 0] = math.nan
    x.requires_grad_()
    wt = w.clone().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, bad, reduction="none")
    assert torch.equal(ce, clean[0]) and torch.equal(kd, clean[1])
    assert (ce[5:9] == 0).all() and (kd[5:9] == 0).all()
    ce, kd = losses.linear_losses(x, wt, t, ids, bad)
    dx, dw = torch.autograd.grad(ce + kd, (x, wt))
    assert torch.isfinite(ce) and torch.isfinite(kd) and torch.isfinite(dw).all()
    assert (dx[5:9] == 0).all() and torch.isfinite(dx).all()
    xc, wc = h.clone().requires_grad_(), w.clone().requires_grad_()
    ce, kd = losses.linear_losses(xc, wc, t, ids, logits)
    want = torch.autograd.grad(ce + kd, (xc, wc))
    assert torch.equal(dw, want[1]) and torch.equal(dx, want[0])


def test_rows_with_one_of_the_two_losses():
    """Logits of a thousand in rows that have a target but no teacher, and the other way round: the loss that a row lacks has no part."""
    h, w, t, ids, logits = _problem(64, 600, 64, 6)
    h = (h * 300).bfloat16()
    t[10:20], ids[30:40] = -100, -1
    ids[10:20, 0], logits[10:20, 0], t[30:40] = 5, 1.0, 7
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits)
    dx, dw = torch.autograd.grad(ce + kd, (x, wt))
    n_ce, n_kd = int((t != -100).sum()), int((ids >= 0).any(1).sum())
    one = torch.ones(64, device="cuda", dtype=F64)
    want = _definition(h, w, t, ids, logits, 1.0, one / n_ce, one / n_kd)
    _check_rows(losses.linear_cross_entropy(h, w, t, reduction="none"), want["ce"], want["Z"])
    _check_grad(dx, want["dx"], want["dx_bound"])
    _check_grad(dw, want["dw"], want["dw_bound"])


def test_gradients_of_tiny_losses():
    """A loss scaled down to the smallest normal numbers: its gradients are the scaled ones."""
    h, w, t, ids, logits = _problem(40, 500, 64, 6)
    x, wt = h.float().requires_grad_(), w.float().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits)
    want = torch.autograd.grad(ce + kd, (x, wt), retain_graph=True)
    got = torch.autograd.grad(ce + kd, (x, wt), grad_outputs=torch.tensor(2.0 ** -100, device="cuda"))
    for a, b in zip(got, want):
        assert torch.equal(a * 2.0 ** 60, b * 2.0 ** -40)


def test_operands_of_any_scale():
    """The f16 copies of the products' operands follow the operands' size: the gradients of scaled rows and weights are the scaled gradients,
    to the bit where the scales are powers of two and the logits the same; large values in rows that take no part change nothing."""
    h, w, t, ids, logits = _problem(60, 700, 128, 6)
    t[1::3], ids[1::3] = -100, -1
    ref = None
    for k in (0, -20, 20, -60, 60):
        x, wt = (h * 2.0 ** k).requires_grad_(), (w * 2.0 ** -k).requires_grad_()
        with torch.no_grad():
            x[1::3] = 3e38
        ce, kd = losses.linear_losses(x, wt, t, ids, logits)
        dx, dw = torch.autograd.grad(ce + kd, (x, wt))
        got = (ce, kd, dx * 2.0 ** k, dw * 2.0 ** -k)
        ref = ref or got
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["weight", "rows", "both"])
@pytest.mark.parametrize("N,V", [(600, 900), (9000, 40001)])
def test_one_row_a_million_times_larger_than_the_others(N, V, which):
    h, w, t, ids, logits = _problem(N, V, 128, 8)
    small = 2.0 ** -20                   # exact in bf16; logits of at most some tens
    if which != "rows":
        w *= small
        w[V - 99] /= small
    if which != "weight":
        h *= small
        h[37] /= small
    one = torch.ones(N, device="cuda", dtype=F64)
    n_ce, n_kd = int((t != -100).sum()), int((ids >= 0).any(1).sum())
    want = _definition(h, w, t, ids, logits, 2.0, one / n_ce, one / n_kd)
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=2.0)
    dx, dw = torch.autograd.grad(ce + kd, (x, wt))
    _check_grad(dx, want["dx"], want["dx_bound"])
    _check_grad(dw, want["dw"], want["dw_bound"])


def test_nothing_to_learn_from():
    h, w, t, ids, logits = _problem(300, 500, 64, 6)
    t[:], ids[:] = -100, -1
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits)
    assert torch.isnan(ce) and torch.isnan(kd)                       # a mean over nothing, as the logits' loss has it
    for g in torch.autograd.grad(ce + kd, (x, wt)):
        assert (g == 0).all()
    ce, kd = losses.linear_losses(h, w, t, ids, logits, reduction="none")
    assert (ce == 0).all() and (kd == 0).all()
    # teachers whose kept logits are all -inf have no probabilities; one finite logit among them has all of it
    ids[0, :3], logits[0] = torch.tensor([4, 9, 4], device="cuda"), -math.inf
    ids[1, :3], logits[1] = torch.tensor([4, 9, 4], device="cuda"), -math.inf
    logits[1, 1] = torch.finfo(torch.float32).min
    kd = losses.linear_distillation(h, w, ids, logits, reduction="none")
    one = losses.linear_cross_entropy(h, w, torch.where(torch.arange(300, device="cuda") == 1, 9, -100), reduction="none")
    assert kd[0] == 0 and (kd[2:] == 0).all()
    assert abs(float(kd[1]) - float(one[1])) <= 2.0 ** -20 * float(one[1])
    # no rows at all
    e = torch.empty(0, 64, dtype=BF16, device="cuda", requires_grad=True)
    wt = w.clone().requires_grad_()
    loss = losses.linear_cross_entropy(e, wt, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert torch.isnan(loss)
    de, dw = torch.autograd.grad(loss, (e, wt))
    assert de.shape == (0, 64) and (dw == 0).all()
    assert losses.linear_distillation(e, w, ids[:0], logits[:0], reduction="none").shape == (0,)


def test_ids_beyond_the_vocabulary_are_nan_and_stay_in_their_row():
    h, w, t, ids, logits = _problem(50, 500, 64, 6)
    good = losses.linear_losses(h, w, t, ids, logits, reduction="none")
    t[3], t[4], ids[10, 2] = 500, -1, 500
    ce, kd = losses.linear_losses(h, w, t, ids, logits, reduction="none")
    assert torch.isnan(ce[3]) and torch.isnan(ce[4]) and torch.isnan(kd[10])
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[3], keep[4] = False, False
    assert torch.equal(ce[keep], good[0][keep])
    keep = torch.arange(50, device="cuda") != 10
    assert torch.equal(kd[keep], good[1][keep])
    assert torch.isnan(losses.linear_cross_entropy(h, w, t)) and torch.isnan(losses.linear_distillation(h, w, ids, logits))
    x = h.clone().requires_grad_()
    dx, = torch.autograd.grad(losses.linear_cross_entropy(x, w, t, reduction="none")[keep].sum(), x)
    assert torch.isnan(dx[3]).all()                                  # its loss was part of the sum
    assert torch.isfinite(dx[5:]).all()


def test_infinite_and_extreme_logits():
    """Logits of -inf leave the softmax; equal and far-apart ones are exact."""
    N, V, width = 33, 700, 64
    h = torch.zeros(N, width, dtype=BF16, device="cuda")
    h[:, 0] = 1.0
    w = torch.zeros(V, width, dtype=BF16, device="cuda")
    w[:, 0] = -math.inf
    w[100:104, 0] = 2.0
    w[500:504, 0] = 2.0
    t = torch.full((N,), 101, device="cuda")
    loss = losses.linear_cross_entropy(h, w, t, reduction="none")
    assert (loss - math.log(8.0)).abs().max() <= 2.0 ** -22 * 3
    w[:, 0] = -3e4
    w[640, 0] = 3e4                                                  # in the last, ragged tile
    # the sum is one exponential, 2^a with |a| <= 1/2: a is off by at most 2^-25, ex2.approx by 2^-22 of its result, so the logarithm
    # of the sum by less than 2^-21
    apart = float(w[640, 0] - w[101, 0].float())
    loss = losses.linear_cross_entropy(h, w, t, reduction="none")
    assert (loss.double() - apart).abs().max() <= 2.0 ** -21 + 2.0 ** -24 * apart
    assert losses.linear_cross_entropy(h, w, torch.full_like(t, 640), reduction="none").abs().max() <= 2.0 ** -21
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(losses.linear_cross_entropy(x, wt, torch.full_like(t, 640)), (x, wt))
    assert (dx == 0).all() and (dw == 0).all()


# (What is rounded is f16 by now: the bound below is f16's, 2^-12 of a target's entry, where the docstring names bf16's 2^-9.)
def test_gradients_of_equal_rows_have_no_common_rounding():
    """1 / rows is no factor of what is rounded to bf16: with flat probabilities a target's entry is -1 + 1 / V, and the gradients of
    2047 rows are as good as those of 2048.  (-1 + 1 / V rounds to -1: 2^-9 of 1 / V for the rest of the row.)"""
    for N in (2047, 2048):
        h = (torch.randint(0, 2, (N, 64), generator=_gen(N), device="cuda") * 2 - 1).bfloat16()
        w = torch.zeros(4096, 64, dtype=BF16, device="cuda")
        t = torch.randint(0, 4096, (N,), generator=_gen(N + 1), device="cuda")
        wt = w.float().requires_grad_()
        dw, = torch.autograd.grad(losses.linear_cross_entropy(h, wt, t), wt)
        z = torch.full((N, 4096), 1 / 4096, dtype=F64, device="cuda")
        z[torch.arange(N, device="cuda"), t] -= 1
        want = z.t() @ h.double() / N
        assert (dw.double() - want).abs().max() <= 2.0 ** -11 / N * 8   # a row's target entry is off by at most 2^-12, at most 8 rows share it


def test_one_gradient_alone():
    h, w, t, ids, logits = _problem(300, 2049, 256, 16)
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(losses.linear_cross_entropy(x, wt, t), (x, wt))
    assert torch.equal(torch.autograd.grad(losses.linear_cross_entropy(x, w, t), x)[0], both[0])
    assert torch.equal(torch.autograd.grad(losses.linear_cross_entropy(h, wt, t), wt)[0], both[1])
    # a loss of the pair that is not used has a gradient of zero
    ce, _ = losses.linear_losses(x, wt, t, ids, logits)
    got = torch.autograd.grad(ce, (x, wt))
    want = _definition(h, w, t, None, None, 1.0, torch.full((300,), 1 / int((t != -100).sum()), device="cuda"), None)
    _check_grad(got[0], want["dx"], want["dx_bound"])
    _check_grad(got[1], want["dw"], want["dw_bound"])


def test_losses_may_be_changed_in_place():
    """`loss /= steps`, `rows *= mask`: the results are nobody else's memory."""
    h, w, t, ids, logits = _problem(30, 300, 64, 5)
    x, wt = h.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(losses.linear_cross_entropy(x, wt, t) / 4, (x, wt))
    loss = losses.linear_cross_entropy(x, wt, t)
    loss /= 4
    for a, b in zip(torch.autograd.grad(loss, (x, wt)), want):
        assert torch.equal(a, b)
    mask = (torch.arange(30, device="cuda") % 3 != 0).float()
    ce, kd = losses.linear_losses(x, wt, t, ids, logits, reduction="none")
    want = torch.autograd.grad((ce * mask + kd).sum(), (x, wt), retain_graph=True)
    ce, kd = losses.linear_losses(x, wt, t, ids, logits, reduction="none")
    ce *= mask
    for a, b in zip(torch.autograd.grad((ce + kd).sum(), (x, wt)), want):
        assert torch.equal(a, b)


def test_shapes_strides_and_types():
    h, w, t, ids, logits = _problem(24, 300, 128, 5)
    want = losses.linear_losses(h, w, t, ids, logits.bfloat16().float(), reduction="none")
    h3 = torch.empty(2, 12, 256, dtype=BF16, device="cuda")[..., ::2].copy_(h.view(2, 12, 128))
    wide = torch.zeros(300, 130, dtype=BF16, device="cuda")
    wide[:, 1:129] = w
    got = losses.linear_losses(h3, wide[:, 1:129], t.view(2, 12), ids.view(2, 12, 5), logits.bfloat16().view(2, 12, 5), reduction="none")
    assert got[0].shape == (2, 12) and torch.equal(got[0].view(-1), want[0]) and torch.equal(got[1].view(-1), want[1])
    got = losses.linear_losses(h.float(), w.float(), t, ids, logits.bfloat16(), reduction="none")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for bad in (dict(h=h.half()), dict(w=w[:, :64]), dict(t=t[:5]), dict(t=t.int()), dict(ids=ids[:, :3]), dict(logits=logits.double()),
                dict(w=w.t()), dict(h=h[:, :60], w=w[:, :60]), dict(w=w[0])):
        a = dict(h=h, w=w, t=t, ids=ids, logits=logits)
        a.update(bad)
        with pytest.raises(RuntimeError):
            losses.linear_losses(a["h"], a["w"], a["t"], a["ids"], a["logits"])
    for x2, w2 in ((h[0], w), (h, w[None]), (h.float(), w), (h, w.float()), (h.t().contiguous().t(), w)):
        with pytest.raises(RuntimeError):
            ops.head_loss(x2, w2, t)
    r = ops.head_loss(h, w, t, want_means=False)
    one = torch.ones((), device="cuda")
    for args in (dict(targets=t, g_ce=one), dict(teacher=ops.teacher_rows(ids, logits, 300), g_kd=one, mean=False),
                 dict(targets=t, g_ce=one, mean=False), dict(targets=t, mean=False)):
        with pytest.raises(RuntimeError):
            ops.head_loss_backward(h, w, r, **args)
    with pytest.raises(RuntimeError, match="vocabulary"):
        ops.head_loss(h, w, teacher=ops.teacher_rows(ids, logits, 301))
    for tau in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="temperature"):
            losses.linear_distillation(h, w, ids, logits, temperature=tau)
    with pytest.raises(RuntimeError, match="1 to 256"):
        losses.linear_distillation(h, w, ids.repeat(1, 52), logits.repeat(1, 52))


def _step(x, w, t, ids, logits):
    ce, kd = losses.linear_losses(x, w, t, ids, logits, temperature=2.0)
    return (ce.detach(), kd.detach(), *torch.autograd.grad(0.5 * ce + 0.5 * kd, (x, w)))


def test_same_bits_every_time_on_any_stream_and_from_graphs():
    sets = [_problem(200, 3001, 128, 9, seed=s) for s in (0, 1)]
    want = [[r.clone() for r in _step(s[0].clone().requires_grad_(), s[1].clone().requires_grad_(), *s[2:])] for s in sets]
    static = [s.clone() for s in sets[0]]
    static[0].requires_grad_(), static[1].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(*static)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want[0]):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):                       # two graphs over the same inputs: each has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*static)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n in (1, 0, 1):
        with torch.no_grad():
            for d, s in zip(static, sets[n]):
                d.copy_(s)
        for (g, _), st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for _, out in graphs:
            for a, b in zip(out, want[n]):
                assert torch.equal(a, b)
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype,dy_dtype", [(torch.float32, BF16), (torch.float32, torch.float32), (BF16, BF16), (BF16, torch.float32)])
@pytest.mark.parametrize("N,width", [(1, 8), (1, 1024), (37, 64), (513, 776), (5000, 1024), (70, 1032), (333, 2048), (90, 4096)])
def test_norm_gradients(N, width, dtype, dy_dtype):
    """f32 sums of a row: C / 32 terms a lane and five joins, 2^-24 each of the sum of magnitudes; dW: N / 8 terms a warp at most, then 300
    parts.  dx = r (w dy - x k): its two parts may cancel, so the bound goes by their sizes."""
    g = _gen(N + width)
    x = (torch.randn(N, width, generator=g, device="cuda") * torch.exp(2 * torch.randn(N, 1, generator=g, device="cuda"))).to(dtype)
    w = torch.randn(width, generator=g, device="cuda")
    dy = torch.randn(N, width, generator=g, device="cuda").to(dy_dtype)
    dx, dw = ops.rmsnorm_backward(x, w, dy, 1e-5)
    assert dx.dtype == dtype and dw.dtype == torch.float32
    xd, wd, gd = x.double(), w.double(), dy.double()
    r = torch.rsqrt(xd.square().mean(1, keepdim=True) + 1e-5)
    k = (wd * gd * xd).mean(1, keepdim=True) * r * r
    rel = (width / 32 + 40) * 2.0 ** -24
    size = r * ((wd * gd).abs() + xd.abs() * (wd * gd * xd).abs().mean(1, keepdim=True) * r * r)
    own = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    want = r * (wd * gd - xd * k)
    assert ((dx.double() - want).abs() <= rel * size + own * want.abs()).all()
    terms = (gd * xd * r).abs().sum(0)
    assert ((dw.double() - (gd * xd * r).sum(0)).abs() <= (rel + (min(N, 64) + N / 2000 + 300) * 2.0 ** -24) * terms).all()
    again = ops.rmsnorm_backward(x, w, dy, 1e-5)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_norm_edges():
    x = torch.zeros(3, 64, device="cuda")
    w, dy = torch.full((64,), 2.0, device="cuda"), torch.ones(3, 64, device="cuda")
    dx, dw = ops.rmsnorm_backward(x, w, dy, 1e-4)
    assert ((dx - 200.0).abs() <= 200 * 2.0 ** -21).all() and (dw == 0).all()        # rsqrt(1e-4) = 100: rsqrt is good to two units in the last place
    dx, dw = ops.rmsnorm_backward(x[:0], w, dy[:0])
    assert dx.shape == (0, 64) and (dw == 0).all()
    for bad in (dict(dy=dy[:, :32]), dict(w=w[:32]), dict(w=w.bfloat16()), dict(x=x.half()), dict(x=x.t().contiguous().t())):
        a = dict(x=x, w=w, dy=dy)
        a.update(bad)
        with pytest.raises(RuntimeError):
            ops.rmsnorm_backward(a["x"], a["w"], a["dy"])


# ------------------------------------------------------------------------------------------------ together
def test_norm_and_head_together():
    """The head's training step: residual stream -> norm -> both losses -> gradients of stream, norm and head, against 64 bits on the
    same rounded hidden rows (the norm's own rounding is the next stage's input)."""
    N, V, width, K = 333, 3001, 256, 12
    _, w, t, ids, logits = _problem(N, V, width, K)
    g = _gen(9)
    x = (torch.randn(N, width, generator=g, device="cuda") * 3).requires_grad_()
    nw = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).requires_grad_()
    wt = w.float().requires_grad_()
    h = losses.rms_norm(x, nw, 1e-6)
    ce, kd = losses.linear_losses(h, wt, t, ids, logits, temperature=2.0)
    dx, dnw, dw = torch.autograd.grad(0.5 * ce + 0.5 * kd, (x, nw, wt))
    n_ce, n_kd = int((t != -100).sum()), int((ids >= 0).any(1).sum())
    one = torch.ones(N, device="cuda", dtype=F64)
    want = _definition(h.detach(), w, t, ids, logits, 2.0, one * 0.5 / n_ce, one * 0.5 / n_kd)
    _check_grad(dw, want["dw"], want["dw_bound"])
    # dh arrives as bf16: its bound passes through the norm's gradient, |r| (w e + |x| mean(w |x| e) r^2)
    xd, wd = x.detach().double(), nw.detach().double()
    r = torch.rsqrt(xd.square().mean(1, keepdim=True) + 1e-6)
    dh, e = want["dx"], want["dx_bound"] * 1.01 + 2.0 ** -8 * want["dx"].abs()
    ref = r * (wd * dh - xd * (wd * dh * xd).mean(1, keepdim=True) * r * r)
    bound = r * (wd.abs() * e + xd.abs() * (wd.abs() * e * xd.abs()).mean(1, keepdim=True) * r * r)
    assert ((dx.double() - ref).abs() <= bound * 1.01 + 1e-30).all()
    assert ((dnw.double() - (dh * xd * r).sum(0)).abs() <= (e * (xd * r).abs()).sum(0) * 1.01).all()


def _model():
    from jarvis_b200 import modules as jm
    torch.manual_seed(5)
    model = jm.Jarvis(vocab_size=301, d_model=128, n_layers=2, n_heads=2, max_seq_len=64).cuda().eval()
    jm.ternary_init_(model, std=0.02, generator=torch.Generator().manual_seed(5))
    return model


def test_model_losses():
    """Jarvis.loss is the loss of its forward (whose logits are rounded to bf16: 2^-8 of a logit, both in the softmax and for the target), and
    Jarvis.head_loss is that loss without the auxiliary terms, with the gradients of norm and head."""
    model = _model()
    g = _gen(6)
    idx = torch.randint(0, 301, (2, 33), generator=g, device="cuda")
    y = torch.randint(0, 301, (2, 33), generator=g, device="cuda")
    y[0, 5:9] = -100
    logits, want = model(idx, targets=y)
    got = model.loss(idx, y)
    top = float(logits.abs().max())
    assert abs(float(got) - float(want)) <= 2 * 2.0 ** -8 * top + 1e-5
    ce = model.head_loss(idx, y)
    aux, reflect = model._aux_terms(ce.device)
    ce.backward()
    ce = ce.detach()
    assert abs(float(ce) - float(got - aux[:, 0].sum() - reflect.sum())) <= 1e-5 * abs(float(got))
    named = {n: p.grad for n, p in model.named_parameters() if p.grad is not None}
    assert set(named) == {"final_norm.weight", "lm_head.weight"}
    assert all(torch.isfinite(v).all() and v.abs().max() > 0 and v.dtype == torch.float32 for v in named.values())
    hidden = model.hidden_rows(idx)
    hd, wd = hidden.double(), model.lm_head.weight.detach().bfloat16().double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(hd @ wd.t(), y.view(-1))
    dref, = torch.autograd.grad(ref, wd)
    assert abs(float(ce) - ref.item()) <= 1e-5 * ref.item()
    assert (named["lm_head.weight"].double() - dref).norm() <= 2.0 ** -8 * dref.norm()      # dz's rounding alone
    # the kernel-by-kernel path has the same
    model.use_chain = False
    assert abs(float(model.head_loss(idx, y).detach()) - float(ce)) <= 1e-3 * float(ce)
    model.use_chain = True
    top_l, top_i = logits.float().topk(9, dim=-1)
    kd = model.head_loss(idx, teacher_ids=top_i, teacher_logits=top_l, temperature=2.0)
    pair = model.head_loss(idx, y, top_i, top_l, temperature=2.0)
    assert torch.equal(pair[1], kd) and torch.equal(pair[0], model.head_loss(idx, y))
    for bad in (dict(), dict(teacher_ids=top_i)):
        with pytest.raises(RuntimeError):
            model.head_loss(idx, **bad)


def test_corpus_evaluation_without_logits():
    from jarvis_b200 import evaluate
    model = _model()
    toks = torch.randint(0, 301, (400,), generator=torch.Generator().manual_seed(3))
    a = evaluate.evaluate_corpus(model, toks, num_windows=3, seq_len=64, seed=1)
    b = evaluate.evaluate_corpus(model, toks, num_windows=3, seq_len=64, seed=1, no_logits=True)
    assert abs(a["mean_loss"] - b["mean_loss"]) <= 2.0 ** -7 * 4 and not b["has_nan_inf"]
    assert evaluate.parse_args(["--no-logits"]).no_logits and not evaluate.parse_args([]).no_logits


def test_first_call_of_a_thread():
    """A thread that has made no CUDA call of its own yet, as autograd's, may begin with any of these calls."""
    import threading
    h, w, t, ids, logits = _problem(40, 500, 64, 6)
    r = ops.head_loss(h, w, t)
    g = torch.ones((), device="cuda")
    want = ops.head_loss_backward(h, w, r, t, g_ce=g)
    torch.cuda.synchronize()
    got = []

    def run(f):
        try:
            got.append(f())
        except Exception as exc:       # reported by the assertion below
            got.append(exc)
    for f in (lambda: ops.head_loss_backward(h, w, r, t, g_ce=g), lambda: ops.head_loss(h, w, t).ce):
        th = threading.Thread(target=run, args=(f,))
        th.start()
        th.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], want[0]) and torch.equal(got[0][1], want[1]) and torch.equal(got[1], r.ce)


def test_weights_beyond_two_to_the_31_elements():
    """Offsets of weight, its gradient and the logits' gradients pass 32 bits: a weight of zeros but for rows near its end.  Logits of the
    zero rows are 0, so their probabilities are one value a row and the definition needs the other rows alone."""
    V, width, N = 1_060_003, 2048, 5
    g = _gen(2)
    w = torch.zeros(V, width, dtype=BF16, device="cuda")
    far = torch.tensor([V - 1, V - 2, V - 300, V - 5000], device="cuda")
    w[far] = (torch.randn(4, width, generator=g, device="cuda") / 30).bfloat16()
    h = torch.randn(N, width, generator=g, device="cuda").bfloat16()
    t = torch.tensor([V - 1, 3, -100, V - 300, V // 2], device="cuda")
    z = h.double() @ w[far].double().t()
    lse = torch.log(z.exp().sum(1) + (V - 4))
    zt = torch.stack([z[0, 0], z[1, 0] * 0, z[2, 0] * 0, z[3, 2], z[4, 0] * 0])
    x, wt = h.clone().requires_grad_(), w.requires_grad_()
    rows = losses.linear_cross_entropy(x, wt, t, reduction="none")
    Z = (width / 16 + 8) * 2.0 ** -23 * float((h.double().abs() @ w.detach()[far].double().abs().t()).max())
    want = torch.where(t >= 0, lse - zt, 0.0)
    assert ((rows.double() - want).abs() <= 2 * Z + 2.0 ** -20 * want.abs()).all()
    dx, dw = torch.autograd.grad(rows.sum(), (x, wt))
    p = (z - lse[:, None]).exp() * (t >= 0)[:, None]
    flat = (-lse).exp() * (t >= 0)
    dz = p.clone()
    dz[0, 0] -= 1
    dz[3, 2] -= 1
    size = p.clone()
    size[0, 0] += 1
    size[3, 2] += 1
    wf, hd = w.detach()[far].double(), h.double()
    _check_grad(dx, dz @ wf, (2.0 ** -11 + 3 * Z + 2.0 ** -18) * (size @ wf.abs()) + 2.0 ** -25 * wf.abs().max() * size.sum(1, keepdim=True))
    rel, floor = 2.0 ** -11 + 3 * Z + 2.0 ** -18, 2.0 ** -25 * hd.abs().max()
    _check_grad(dw[far], dz.t() @ hd, rel * (size.t() @ hd.abs()) + floor * size.sum(0)[:, None])
    for row, n in ((3, 1), (V // 2, 4), (12345, None), (V - 10, None)):
        col = flat.clone()
        if n is not None:
            col[n] -= 1
        big = flat + (0 if n is None else (torch.arange(N, device="cuda") == n))
        _check_grad(dw[row], col @ hd, rel * (big @ hd.abs()) + floor * big.sum())


def test_two_threads_at_once():
    """Calls from two threads on two streams, each over its own rows: the results of calls one after the other."""
    import threading
    sets = [_problem(300 + 100 * i, 4001, 128, 9, seed=i) for i in range(2)]
    want = [_step(s[0].clone().requires_grad_(), s[1].clone().requires_grad_(), *s[2:]) for s in sets]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            x, w = sets[i][0].clone().requires_grad_(), sets[i][1].clone().requires_grad_()
            for _ in range(20):
                got[i] = _step(x, w, *sets[i][2:])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for g, w in zip(got, want):
        assert g is not None and all(torch.equal(a, b) for a, b in zip(g, w))


def test_gradients_are_not_differentiable_and_say_so():
    h, w, t, _, _ = _problem(20, 300, 64, 3)
    x = h.float().requires_grad_()
    g, = torch.autograd.grad(losses.linear_cross_entropy(x, w, t), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    nw = torch.ones(64, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(losses.rms_norm(x, nw).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_a_weight_used_twice_and_rows_that_are_one_row():
    """Gradients of the same tensor from two uses add up; an expanded row's are the sum over its rows."""
    h, w, t, _, _ = _problem(24, 300, 64, 3)
    wt = w.float().requires_grad_()
    both, = torch.autograd.grad(losses.linear_cross_entropy(h[:10], wt, t[:10], reduction="none").sum() +
                                losses.linear_cross_entropy(h[10:], wt, t[10:], reduction="none").sum(), wt)
    one, = torch.autograd.grad(losses.linear_cross_entropy(h, wt, t, reduction="none").sum(), wt)
    want = _definition(h, w, t, None, None, 1.0, torch.ones(24, device="cuda"), None)
    _check_grad(both, want["dw"], 2 * want["dw_bound"])
    _check_grad(one, want["dw"], want["dw_bound"])
    row = h[:1].float().requires_grad_()
    dx, = torch.autograd.grad(losses.linear_cross_entropy(row.expand(24, 64), w, t, reduction="none").sum(), row)
    want = _definition(h[:1].expand(24, 64), w, t, None, None, 1.0, torch.ones(24, device="cuda"), None)
    _check_grad(dx, want["dx"].sum(0, keepdim=True), want["dx_bound"].sum(0, keepdim=True) * 1.01)


# ------------------------------------------------------------------------------------------------ a head that is being trained
def _fresh(model):
    """A model of the same weights that has kept nothing."""
    from jarvis_b200 import modules as jm
    twin = jm.Jarvis(vocab_size=301, d_model=128, n_layers=2, n_heads=2, max_seq_len=64).cuda().eval()
    twin.load_state_dict(model.state_dict())
    twin.final_norm.to(model.final_norm.weight.dtype)
    with torch.no_grad():
        twin.final_norm.weight.copy_(model.final_norm.weight)
    return twin


def _same_as_fresh(model, idx, y):
    twin = _fresh(model)
    for a, b in zip(model(idx, targets=y), twin(idx, targets=y)):
        assert torch.equal(a, b)
    assert torch.equal(model.loss(idx, y), twin.loss(idx, y))
    assert torch.equal(model.step(idx)[0], twin.step(idx)[0])


@pytest.mark.parametrize("norm_dtype", [torch.float32, BF16])
@pytest.mark.parametrize("fused", [True, False])
def test_every_path_reads_the_head_as_it_is_trained(fused, norm_dtype):
    """An update may leave no trace on a tensor (fused optimizers do not count its version up): logits, losses and steps follow it."""
    model = _model()
    model.final_norm.to(norm_dtype)
    g = _gen(6)
    idx, y = (torch.randint(0, 301, (2, 33), generator=g, device="cuda") for _ in range(2))
    params = [model.final_norm.weight, model.lm_head.weight]
    opt = torch.optim.AdamW(params, lr=0.1, fused=fused)
    model(idx, targets=y)                                            # whatever is kept of the weights is there before the first update
    for i in range(3):
        before = model.lm_head.weight.detach().clone()
        model.head_loss(idx, y).backward()
        model(idx)                                                   # ... and made again between backward pass and update
        opt.step()
        opt.zero_grad()
        assert (model.lm_head.weight - before).abs().max() > 0.01
        _same_as_fresh(model, idx, y)
    model.refresh_head()                                             # training is over: copies are kept again
    kept = model._lm_head_weight()
    assert model._lm_head_weight() is kept
    _same_as_fresh(model, idx, y)


def test_every_path_reads_a_head_that_a_captured_step_trains():
    model = _model()
    g = _gen(7)
    idx, y = (torch.randint(0, 301, (2, 33), generator=g, device="cuda") for _ in range(2))
    params = [model.final_norm.weight, model.lm_head.weight]

    def step():
        grads = torch.autograd.grad(model.head_loss(idx, y), params)
        with torch.no_grad():
            for p, d in zip(params, grads):
                p.sub_(0.5 * d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    model(idx, targets=y)
    before = model.lm_head.weight.detach().clone()
    for _ in range(3):
        graph.replay()
        _same_as_fresh(model, idx, y)
    assert (model.lm_head.weight - before).abs().max() > 2.0 ** -8 * before.abs().max()


@pytest.mark.parametrize("how", ["bf16", "f32", "strided", "three axes"])
@pytest.mark.parametrize("op", ["ce", "kd", "norm"])
def test_a_penalty_on_the_gradients_is_refused(op, how):
    """Under create_graph the first gradients are those of any pass; what is formed of them cannot be differentiated with respect to anything
    ahead of the operator, the weight or a factor behind it."""
    _, _, t, ids, logits = _problem(24, 300, 64, 3)
    g = _gen(11)
    theta = torch.randn(24, 128, generator=g, device="cuda", requires_grad=True)
    phi = torch.randn(300 if op != "norm" else 1, 64, generator=g, device="cuda", requires_grad=True)
    s = torch.ones((), device="cuda", requires_grad=True)

    def loss():
        h = theta.tanh()
        if how != "f32":
            h = h.bfloat16()
        h = h[:, ::2] if how == "strided" else h[:, :64].contiguous()
        if how == "three axes":
            h = h.view(2, 12, 64)
        w = phi.sin()
        if op == "norm":
            return s * losses.rms_norm(h, w[0]).float().square().sum()
        if op == "ce":
            return s * losses.linear_cross_entropy(h, w, t.view(h.shape[:-1]))
        return s * losses.linear_distillation(h, w, ids.view(*h.shape[:-1], 3), logits.view(*h.shape[:-1], 3))
    want = torch.autograd.grad(loss(), (theta, phi))
    got = torch.autograd.grad(loss(), (theta, phi), create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for first in got:
        for by in (theta, phi, s):
            with pytest.raises(RuntimeError, match="cannot be differentiated"):
                torch.autograd.grad(first.square().sum(), by, retain_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            first.square().sum().backward(retain_graph=True)
    assert theta.grad is None


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("tau", [0.25, 0.5, 0.9, 1.0, 2.0])
def test_teachers_of_the_types_largest_and_lowest_values(tau, dtype):
    """Probabilities are those of the differences: a row whose entries all hold the type's lowest value has even ones, at any temperature, and an
    entry far above the rest has all."""
    h, w, _, _, _ = _problem(8, 300, 64, 4)
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    ids = torch.arange(8 * 4, device="cuda").view(8, 4)
    logits = torch.tensor([[lo, lo, lo, lo], [lo, lo, 0, lo], [hi, hi, 0, lo], [hi, lo, lo, hi], [0, 0, 0, lo], [hi, hi, hi, hi],
                           [-math.inf, lo, lo, -math.inf], [-math.inf] * 4], device="cuda").to(dtype)
    q = torch.tensor([[1, 1, 1, 1], [0, 0, 1, 0], [1, 1, 0, 0], [1, 0, 0, 1], [1, 1, 1, 0], [1, 1, 1, 1], [0, 1, 1, 0], [0, 0, 0, 0]],
                     device="cuda", dtype=F64)
    # the same probabilities from ordinary values
    plain = torch.where(q > 0, 1.0, -math.inf).float()
    got = losses.linear_distillation(h, w, ids, logits, temperature=tau, reduction="none")
    want = losses.linear_distillation(h, w, ids, plain, temperature=tau, reduction="none")
    assert torch.equal(got, want) and got[7] == 0 and (got[:7] > 0).all()
    q = q / q.sum(1, keepdim=True).clamp(min=1)
    z = h.double() @ w.double().t()
    lp = torch.log_softmax(z / tau, 1).gather(1, ids)
    ref = tau * tau * (torch.special.xlogy(q, q) - q * lp).sum(1)
    Z = (64 / 16 + 8) * 2.0 ** -23 * float((h.double().abs() @ w.double().abs().t()).max())
    _check_rows(got, ref, Z, tau)


@pytest.mark.parametrize("use_chain", [True, False])
def test_training_the_head_leaves_a_carried_state_alone(use_chain):
    """A sequence in progress goes on as if no head_loss had come between."""
    g = _gen(12)
    idx, y = (torch.randint(0, 301, (2, 20), generator=g, device="cuda") for _ in range(2))
    out = []
    for between in (False, True):
        model = _model()
        model.use_chain, model.carry_attention_state = use_chain, True
        model(idx, persist_state=True)
        if between:
            model.head_loss(y, idx)
        out.append(model(y, persist_state=True)[0])
    assert torch.equal(*out)


@pytest.mark.parametrize("N,width", [(37, 1024), (300, 1024), (3, 4096)])
def test_norm_gradients_that_are_not_wanted_are_not_formed(N, width, monkeypatch):
    g = _gen(13)
    x = torch.randn(N, width, generator=g, device="cuda")
    w = torch.randn(width, generator=g, device="cuda")
    dy = torch.randn(N, width, generator=g, device="cuda").bfloat16()
    dx, dw = ops.rmsnorm_backward(x, w, dy)
    none, alone = ops.rmsnorm_backward(x, w, dy, want_dx=False)
    assert none is None and torch.equal(alone, dw)
    seen, inner = [], ops.rmsnorm_backward
    monkeypatch.setattr(ops, "rmsnorm_backward", lambda *a, **k: seen.append(k) or inner(*a, **k))
    for want in (False, True):
        xx = x.clone().requires_grad_(want)
        ww = w.clone().requires_grad_()
        losses.rms_norm(xx, ww).backward(dy)
        assert torch.equal(ww.grad, dw) and (torch.equal(xx.grad, dx) if want else xx.grad is None)
    assert [k["want_dx"] for k in seen] == [False, True]
    xx, ww = x.clone().requires_grad_(), w.clone()
    losses.rms_norm(xx, ww).backward(dy)
    assert torch.equal(xx.grad, dx)


@pytest.mark.parametrize("dtype,dy_dtype", [(torch.float32, BF16), (BF16, torch.float32)])
@pytest.mark.parametrize("N,width", [(1, 4096), (2, 2056), (33, 2056), (64, 4096), (65, 4096), (128, 2048), (129, 2048), (256, 1024), (257, 1024)])
def test_norm_gradients_at_the_limits_of_one_cluster(N, width, dtype, dy_dtype):
    """Rows on one, two and four warps, in one cluster up to 256, 128 and 64 rows and beyond."""
    test_norm_gradients(N, width, dtype, dy_dtype)


@pytest.mark.parametrize("mode", ["ce", "kd", "both"])
def test_rows_of_very_uneven_weights(mode):
    """Rows weighted down to 2^-30 of the heaviest, some not at all: a row's own gradient is as good as if it were alone, and the weight's is off by
    no more than the heaviest rows' share allows."""
    N, V, width = 64, 5000, 128
    h, w, t, ids, logits = _problem(N, V, width, 5)
    t, ids = (t if mode != "kd" else None), (ids if mode != "ce" else None)
    a = 2.0 ** -(torch.arange(N, device="cuda").float() % 31)
    a[5] = 0
    b = a.flip(0) if mode == "both" else a
    x, wt = h.float().requires_grad_(), w.float().requires_grad_()
    if mode == "ce":
        loss = (losses.linear_cross_entropy(x, wt, t, reduction="none") * a).sum()
    elif mode == "kd":
        loss = (losses.linear_distillation(x, wt, ids, logits, temperature=2.0, reduction="none") * b).sum()
    else:
        ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=2.0, reduction="none")
        loss = (ce * a).sum() + (kd * b).sum()
    dx, dw = torch.autograd.grad(loss, (x, wt))
    want = _definition(h, w, t, ids, logits, 2.0, a, b)
    # dx: the last term of its bound goes by the row's own factor instead of the call's
    own = torch.maximum(a if t is not None else 0 * a, 2 * b if ids is not None else 0 * b).double()[:, None]
    call = float(own.max())
    column = w.double().abs().sum(0)
    _check_grad(dx, want["dx"], want["dx_bound"] - 2.0 ** -38 * call * column + 2.0 ** -37 * own * column)
    _check_grad(dw, want["dw"], want["dw_bound"] + 2.0 ** -38 * call * N * h.double().abs().max())


def test_losses_of_very_uneven_weights():
    """Means of both losses, one weighted 2^-30 of the other: the rows that have the light one alone keep their gradient's bits."""
    N, V, width = 64, 5000, 128
    h, w, t, ids, logits = _problem(N, V, width, 5)
    t[:20], ids[20:40] = -100, -1
    t[20:40] = torch.arange(20, device="cuda") * 7
    n_ce, n_kd = int((t != -100).sum()), int((ids >= 0).any(1).sum())
    one = torch.ones(N, device="cuda", dtype=F64)
    column = w.double().abs().sum(0)
    for a, b in ((2.0 ** -30, 1.0), (1.0, 2.0 ** -30)):
        x, wt = h.float().requires_grad_(), w.float().requires_grad_()
        ce, kd = losses.linear_losses(x, wt, t, ids, logits, temperature=2.0)
        dx, dw = torch.autograd.grad(a * ce + b * kd, (x, wt))
        want = _definition(h, w, t, ids, logits, 2.0, one * a / n_ce, one * b / n_kd)
        own = torch.maximum(a / n_ce * (t != -100), 2 * b / n_kd * (ids >= 0).any(1)).double()[:, None]
        call = max(a / n_ce, 2 * b / n_kd)
        _check_grad(dx, want["dx"], want["dx_bound"] - 2.0 ** -38 * call * column + 2.0 ** -37 * own * column)
        _check_grad(dw, want["dw"], want["dw_bound"] + 2.0 ** -38 * call * N * h.double().abs().max())
