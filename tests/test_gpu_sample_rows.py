"""Draws over the whole vocabulary against a plain 64-bit implementation: tokens exactly, probabilities to f32's half step and 2^-40 of the sums.

The uniform numbers lie away from the borders of the running sum by construction: a draw is asked for in the middle of the interval of a token that
has been chosen, so that a token that differs is an error and not a rounding."""
import math

import pytest
import torch

from jarvis_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F64 = torch.float64


def _row(x, temperature, top_k, top_p, min_p):
    """(ids in descending order, weights left, 0 where cut) of one row, on the CPU."""
    x = x.double().cpu().clone()
    x[x.isnan()] = -math.inf
    order = torch.sort(x, descending=True, stable=True).indices
    z = x[order]
    w = torch.where(z == z[0], 1.0, torch.exp((z - z[0]) / max(temperature, 1e-5)))
    if top_k > 0:
        w = torch.where(z >= z[min(top_k, z.numel()) - 1], w, 0.0)
    c = w.cumsum(0)
    left = w > 0
    if 0 < top_p < 1:
        left &= c - w <= top_p * c[-1]
    if min_p > 0:
        left &= w >= min_p
    left[0] = True
    return order, torch.where(left, w, 0.0)


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _check(logits, temperature, top_k, top_p, min_p, seed=0, every=None):
    """Rows with per-row settings (lists); every row's draw is aimed at a token of its own."""
    B, V = logits.shape
    gen = torch.Generator().manual_seed(seed)
    u, want, probs = [], [], []
    for r in range(B):
        order, w = _row(logits[r], _f32(temperature[r]), top_k[r], _f32(top_p[r]), _f32(min_p[r]))
        c = w.cumsum(0)
        wide = torch.nonzero(w > 2.0 ** -20 * c[-1]).flatten()           # u is f32: intervals of at least some of its steps
        at = int(wide[torch.randint(wide.numel(), (1,), generator=gen)]) if every is None else int(wide[min(every, wide.numel() - 1)])
        u.append(float((c[at] - w[at] / 2) / c[-1]))
        want.append(int(order[at]))
        probs.append(float(w[at] / c[-1]))
    dev = logits.device
    args = dict(temperature=torch.tensor(temperature, device=dev), top_k=torch.tensor(top_k, dtype=torch.int32, device=dev),
                top_p=torch.tensor(top_p, device=dev), min_p=torch.tensor(min_p, device=dev))
    token, prob = ops.sample_rows(logits, torch.tensor(u, device=dev), want_prob=True, **args)
    assert token.shape == (B, 1) and token.dtype == torch.int64
    assert token.view(-1).tolist() == want
    probs = torch.tensor(probs, dtype=F64)
    assert ((prob.double().cpu() - probs).abs() <= (2.0 ** -24 + 2.0 ** -40) * probs + 2.0 ** -40).all()
    assert _lib.device_status() == 0


def _logits(B, V, dtype, seed=0, size=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed + V)
    return (torch.randn(B, V, generator=g, device="cuda") * size).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 100, 1023, 4099, 50257])
def test_filters(V, dtype):
    B = 12
    x = _logits(B, V, dtype)
    for n, (t, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.03), (0.9, 50, 1.0, 0.0), (0.9, 1500, 0.8, 0.001), (3.0, 0, 0.999, 0.0),
                                      (20.0, 0, 0.5, 0.0), (0.05, 0, 0.95, 0.0), (1.0, 1, 0.5, 0.5), (1.0, V, 1.0, 1.0), (1e-3, 3, 0.3, 0.2), (1.0, 7, 0.99, 1e-6)]):
        _check(x, [t] * B, [k] * B, [p] * B, [m] * B, seed=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_row_its_own(dtype):
    B, V = 40, 9001
    x = _logits(B, V, dtype)
    g = torch.Generator().manual_seed(3)
    r = torch.rand(4, B, generator=g)
    _check(x, (0.3 + 2 * r[0]).tolist(), [int(a * 3000) if a > 0.4 else 0 for a in r[1]], [float(a) if a > 0.3 else 1.0 for a in r[2]],
           [float(a * 0.1) if a > 0.5 else 0.0 for a in r[3]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties(dtype):
    """Rows of few different values, of one value, and constant up to one token; a cut may fall among equals."""
    V = 6000
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.stack([torch.randint(0, 3, (V,), generator=g, device="cuda").float(), torch.zeros(V, device="cuda"), torch.full((V,), -2.0, device="cuda"),
                     torch.randint(-5, 6, (V,), generator=g, device="cuda").float() / 4, torch.zeros(V, device="cuda")]).to(dtype)
    x[2, 4321] = 1.0
    x[4, ::2] = -0.0                     # equal to 0
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.5, 0, 0.61, 0.0), (1.0, 10, 1.0, 0.0), (1.0, 2500, 0.7, 0.0), (2.0, 0, 1.0, 0.37), (1.0, 0, 0.9, 0.9)]:
        for every in (0, 1, 999, 10 ** 9):
            _check(x, [t] * 5, [k] * 5, [p] * 5, [m] * 5, every=every)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_and_infinite_logits(dtype):
    """-inf, the type's lowest value, NaN and +inf; rows with one token or none left."""
    V = 3001
    x = _logits(8, V, dtype)
    x[0, 5:] = -math.inf
    x[1, 1:] = torch.finfo(dtype).min
    x[2, ::2] = float("nan")
    x[3, 17] = math.inf
    x[3, 99] = math.inf
    x[4] = -math.inf
    x[4, 1234] = -50.0
    x[5] = torch.finfo(dtype).min
    x[6, ::3] = -math.inf
    x[7] = torch.finfo(dtype).max
    n = 8
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 20, 0.95, 0.01), (1.0, 2900, 1.0, 0.0)]:
        for every in (0, 3, 10 ** 9):
            _check(x, [t] * n, [k] * n, [p] * n, [m] * n, every=every)
    nothing = torch.full((3, V), -math.inf, device="cuda", dtype=dtype)
    nothing[1] = float("nan")
    token, prob = ops.sample_rows(nothing, torch.rand(3, device="cuda"), temperature=1.0, top_k=5, top_p=0.9, min_p=0.1, want_prob=True)
    assert not token.any() and not prob.any()


def test_greedy_and_values_for_all_rows():
    x = _logits(9, 777, torch.bfloat16)
    x[:, 700] = x[:, 3] = 20.0
    u = torch.rand(9, device="cuda")
    for t in (0.0, -1.0):
        token, prob = ops.sample_rows(x, u, temperature=t, want_prob=True)
        assert (token == 3).all() and (prob == 1).all()
    a = ops.sample_rows(x, u, temperature=0.8, top_k=40, top_p=0.9, min_p=0.02)
    full = dict(device="cuda", dtype=torch.float32)
    b = ops.sample_rows(x, u, temperature=torch.full((9,), 0.8, **full), top_k=torch.full((9,), 40, device="cuda", dtype=torch.int32),
                        top_p=torch.full((9,), 0.9, **full), min_p=torch.full((9,), 0.02, **full))
    assert torch.equal(a, b)


def test_extreme_numbers():
    """u at both ends and beyond, top_p and min_p outside their ranges, temperatures of every size."""
    V = 500
    x = _logits(1, V, torch.float32).expand(6, V).contiguous()
    order = torch.sort(x[0].double(), descending=True, stable=True).indices
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, -1.0, float("nan"), 2.0], device="cuda")
    token = ops.sample_rows(x, u, temperature=1e4).view(-1)
    assert token.tolist() == [int(order[0]), int(order[-1]), int(order[-1]), int(order[0]), int(order[0]), int(order[-1])]
    assert (ops.sample_rows(x, u, temperature=1.0, min_p=2.0) == order[0]).all()
    assert (ops.sample_rows(x, u, temperature=1e-30) == order[0]).all()
    assert (ops.sample_rows(x, u, temperature=1.0, top_p=1e-9) == order[0]).all()
    for p in (0.0, 1.0, -3.0, 7.0, float("nan"), None):
        assert torch.equal(ops.sample_rows(x, u, temperature=1.0, top_p=p), ops.sample_rows(x, u, temperature=1.0))
    for k in (0, None, -4, V, V + 9, 2 ** 40):
        assert torch.equal(ops.sample_rows(x, u, temperature=1.0, top_k=k), ops.sample_rows(x, u, temperature=1.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_streams_and_graphs(dtype):
    B, V = 5, 1000
    for offset in (0, 1, 3):
        wide = torch.full((B, V + 11), 1e9, device="cuda").to(dtype)
        x = wide[:, offset:offset + V]
        x.copy_(_logits(B, V, dtype))
        u = torch.rand(B, device="cuda")
        args = dict(temperature=0.9, top_k=300, top_p=0.95, min_p=0.001)
        want = ops.sample_rows(x.contiguous(), u, want_prob=True, **args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.sample_rows(x, u, want_prob=True, **args)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = ops.sample_rows(x, u, want_prob=True, **args)
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, got, captured):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_agrees_with_the_sampler_of_top_k_survivors():
    """Where both take a call, they choose the same token (u in the middle of its interval)."""
    B, V = 64, 50257
    x = _logits(B, V, torch.bfloat16)
    u = torch.rand(B, device="cuda")
    a = ops.sample(x, u, temperature=0.7, top_k=50, top_p=0.9, want_prob=True)
    b = ops.sample_rows(x, u, temperature=0.7, top_k=50, top_p=0.9, want_prob=True)
    assert (a[0] != b[0]).sum() <= 1                        # f32 sums there: a border may lie within 1e-6 of u
    same = (a[0] == b[0]).view(-1)
    assert ((a[1] - b[1]).abs()[same] <= 1e-5 * b[1][same]).all()


def test_frequencies():
    """A hundred thousand draws of one row fall as its probabilities say: within five standard deviations each."""
    V, n = 64, 100000
    x = _logits(1, V, torch.float32, size=1.5)
    p = torch.softmax(x[0].double(), 0)
    u = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    token = ops.sample_rows(x.expand(n, V).contiguous(), u, temperature=1.0)
    seen = torch.bincount(token.view(-1), minlength=V).double()
    assert ((seen - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()


def test_no_rows_and_refusals():
    x, u = _logits(4, 100, torch.float32), torch.rand(4, device="cuda")
    assert ops.sample_rows(x[:0], u[:0]).shape == (0, 1)
    for call, text in ((lambda: ops.sample_rows(x[0], u), "B, V"), (lambda: ops.sample_rows(x.half(), u), "float32 or bfloat16"),
                       (lambda: ops.sample_rows(x, u[:3]), "one number per row"), (lambda: ops.sample_rows(x, u.double()), "dtype"),
                       (lambda: ops.sample_rows(x, u, top_k=torch.ones(4, device="cuda")), "dtype"),
                       (lambda: ops.sample_rows(x, u, top_p=torch.ones(3, device="cuda")), "one per row"),
                       (lambda: ops.sample_rows(x.t(), u), "contiguous rows"), (lambda: ops.sample_rows(x.cpu(), u), "CUDA"),
                       (lambda: ops.sample_rows(x[:1].expand(4, 100), u), "overlap")):
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(300, 6007), (2, 50257)])
@pytest.mark.parametrize("few", [1, 1000, 1023, 1024, 1025, 3000])
def test_what_a_filter_leaves_fits_a_list_or_not(few, B, V, dtype):
    """`few` neighbouring tokens, so that one slice has them all, stand out by more than min-p (or top-k) leaves: around the length of its list."""
    x = _logits(B, V, dtype, seed=few, size=0.5) - 20.0
    x[:, 7:7 + few] = (_logits(B, few, dtype, seed=1, size=0.25).float() + 4.0).to(dtype)
    one, rows = [1.0] * 4, [x[:4].contiguous(), x[-4:].contiguous()] if B > 4 else [x]
    for r in rows:
        n = r.shape[0]
        for k, p, m in ((0, 1.0, 0.02), (few, 1.0, 0.0), (few, 0.7, 0.05), (0, 0.9, 0.02), (min(few + 30, V), 1.0, 1e-5)):
            _check(r, one[:n], [k] * n, [p] * n, [m] * n, seed=few)
    # as many rows as make one CTA of each: the same tokens as a few at a time
    u = torch.rand(B, generator=torch.Generator().manual_seed(few)).cuda()
    for kw in (dict(min_p=0.02), dict(top_k=few), dict(top_k=few, top_p=0.7, min_p=0.05)):
        together = ops.sample_rows(x, u, temperature=1.0, **kw)
        apart = torch.cat([ops.sample_rows(x[i:i + 4], u[i:i + 4].contiguous(), temperature=1.0, **kw) for i in range(0, B, 4)])
        assert torch.equal(together, apart)
