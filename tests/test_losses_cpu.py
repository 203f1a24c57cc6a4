"""The head's losses and the norm's gradient without a GPU: refusals that need no launch, and how a backward pass is cut."""
import ctypes as C

import pytest
import torch

from jarvis_b200 import _lib, losses, ops


def _head(**kw):
    h = _lib.Head()
    h.N, h.V, h.C, h.temperature = 4, 100, 64, 1.0
    h.x = h.w = h.targets = h.lse = 4096         # never read: every call here is refused first
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("kw,text", [(dict(C=60), "multiple of 8"), (dict(C=56), "at least 64"), (dict(V=0), "bad shape"), (dict(N=-1), "bad shape"),
                                     (dict(x=None), "null pointer"), (dict(x=4104), "16-byte"), (dict(targets=None), "neither targets nor a teacher"),
                                     (dict(lse=None), "lse is needed"), (dict(teacher=4096, K=0), "1 to 256 entries"),
                                     (dict(teacher=4096, K=257), "1 to 256 entries"), (dict(teacher=4096, K=3), "null pointer"), (dict(teacher=4104, K=3, lse_t=4096), "16-byte"),
                                     (dict(teacher=4096, K=3, lse_t=4096, temperature=0.0), "temperature"),
                                     (dict(teacher=4096, K=3, lse_t=4096, temperature=float("nan")), "temperature"),
                                     (dict(teacher=4096, K=3, lse_t=4096, temperature=4e-39), "temperature"),
                                     (dict(N=2**30, V=2**30), "too many logits")])
def test_head_calls_refuse_bad_arguments(kw, text):
    lib = _lib.load()
    h = _head(**kw)
    assert lib.jb200_head_loss(C.byref(h), 4096, 4096, None, None, None, 4096, None) == _lib.ERR_ARG
    assert text in _lib.last_error()
    assert lib.jb200_head_loss_backward(C.byref(h), 4096, 0, None, 4096, 0, None, 4096, 1, 4096, 1, 4096, None) == _lib.ERR_ARG
    assert text in _lib.last_error()


def test_head_calls_refuse_missing_outputs():
    lib = _lib.load()
    h = _head()
    assert lib.jb200_head_loss(C.byref(h), 4096, None, 4096, None, None, 4096, None) == _lib.ERR_ARG and "counts" in _lib.last_error()
    assert lib.jb200_head_loss(C.byref(h), 4096, None, None, None, None, None, None) == _lib.ERR_ARG and "scratch" in _lib.last_error()
    for dx, dxt, dw, scratch, stride, text in ((4096, 2, 4096, 4096, 0, "dtype"), (4096, 1, 4112, 4096, 0, "32-byte"),
                                               (4112, 1, 4096, 4096, 0, "32-byte"), (4096, 1, 4096, 4100, 0, "256-byte"),
                                               (4096, 1, 4096, 4096, 2, "strides")):
        assert lib.jb200_head_loss_backward(C.byref(h), 4096, stride, None, None, 0, None, dx, dxt, dw, 1, scratch, None) == _lib.ERR_ARG
        assert text in _lib.last_error()
    assert lib.jb200_head_loss_backward(C.byref(h), None, 0, None, None, 0, None, 4096, 1, 4096, 1, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_teacher_rows(4096, 4096, 0, 4, 257, 100, 1.0, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_teacher_rows(4096, 4096, 3, 4, 2, 100, 1.0, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_teacher_rows(4096, 4096, 0, 4, 2, 100, -1.0, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_teacher_rows(4096, 4096, 0, 4, 2, 100, 1.0, 4100, None) == _lib.ERR_ARG
    assert lib.jb200_teacher_rows(None, 4096, 0, 4, 2, 100, 1.0, 4096, None) == _lib.ERR_ARG
    for width, text in ((60, "multiple of 8"), (4104, "at most 4096"), (0, "bad shape")):
        assert lib.jb200_rmsnorm_backward(4096, 0, 4096, 1e-6, 4096, 0, 4, width, 4096, 4096, 4096, None) == _lib.ERR_ARG
        assert text in _lib.last_error()
    assert lib.jb200_rmsnorm_backward(4096, 2, 4096, 1e-6, 4096, 0, 4, 64, 4096, 4096, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_rmsnorm_backward(4100, 0, 4096, 1e-6, 4096, 0, 4, 64, 4096, 4096, 4096, None) == _lib.ERR_ARG
    assert lib.jb200_rmsnorm_backward(4096, 0, 4096, 1e-6, 4096, 0, 4, 64, 4096, None, 4096, None) == _lib.ERR_ARG


def test_cpu_tensors_and_bad_reductions_raise():
    h, w, t = torch.zeros(4, 64), torch.zeros(100, 64), torch.zeros(4, dtype=torch.int64)
    ids, lg = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    for call in (lambda: losses.linear_cross_entropy(h, w, t), lambda: losses.linear_distillation(h, w, ids, lg),
                 lambda: losses.linear_losses(h, w, t, ids, lg), lambda: losses.rms_norm(h, torch.ones(64)),
                 lambda: ops.rmsnorm_backward(h, torch.ones(64), h), lambda: ops.teacher_rows(ids, lg, 100),
                 lambda: ops.head_loss(h.bfloat16(), w.bfloat16(), t)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="reduction"):
        losses.linear_cross_entropy(h, w, t, reduction="median")


@pytest.mark.parametrize("sms", [148, 132, 2])
def test_backward_passes_are_cut_into_pieces_that_cover_the_vocabulary(sms):
    lib = _lib.load()
    out = (C.c_int32 * 3)()
    for N in (1, 37, 255, 2048, 5000, 16384, 300000, 2000000):
        for V in (1, 256, 257, 1000, 32003, 50257, 200000):
            for width in (64, 200, 1024, 2048):
                assert lib.jb200_host_head_plan(N, V, width, sms, out) == 0
                cols, pieces, slabs = out
                assert cols % 256 == 0 and (pieces - 1) * cols < V <= pieces * cols
                assert cols == 256 or N * cols * 2 <= 640 << 20        # the workspace is bounded, down to one tile of columns
                # every slab of the first piece has K-blocks of 64 columns to sum
                assert 1 <= slabs <= 64 and slabs <= (min(V, cols) + 63) // 64
    assert lib.jb200_host_head_plan(0, 5, 64, 148, out) == _lib.ERR_ARG


@pytest.mark.parametrize("n_long,k_long,n_short,k_short,pairs", [(148, 256, 512, 74, 74), (116, 256, 256, 116, 74), (788, 32, 64, 394, 74), (4, 786, 788, 1, 74),
                                                                 (0, 5, 10, 3, 10), (7, 9, 0, 2, 7), (3, 100, 2, 1, 5), (75, 10, 1, 9, 74),
                                                                 (10, 1000, 500, 1, 7), (1, 1, 1, 1, 2), (13, 8, 100, 8, 13)])
def test_every_item_of_the_gradients_products_is_done_once(n_long, k_long, n_short, k_short, pairs):
    lib = _lib.load()
    seen, busiest = [], 0
    for pair in range(pairs):
        i = load = 0
        while (t := lib.jb200_host_head_walk(n_long, k_long, n_short, k_short, pairs, pair, i)) >= 0:
            seen.append(t)
            load += k_long if t < n_long else k_short
            i += 1
        assert t == -1 and lib.jb200_host_head_walk(n_long, k_long, n_short, k_short, pairs, pair, i + 1) == -1
        busiest = max(busiest, load)
    assert sorted(seen) == list(range(n_long + n_short))
    # no pair has more than its even share, rounded up by an item of each kind
    assert busiest <= (n_long * k_long + n_short * k_short) / pairs + k_long + k_short


class _OnCard(torch.Tensor):
    """A host tensor that says it is on the card `card`."""
    card = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.card))

    def get_device(self):
        return self.card

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))


def _on(card, *shape, dtype=torch.float32):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(_OnCard)
    t.card = card
    return t


def test_norm_launches_on_its_tensors_card(monkeypatch):
    current, seen = [0], []

    class Card:
        def __init__(self, device):
            self.index = device.index

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
    for card in (1, 0):
        ops.rmsnorm(_on(card, 4, 64), _on(card, 64))
        ops.rmsnorm_backward(_on(card, 4, 64), _on(card, 64), _on(card, 4, 64))
        assert seen == [("jb200_rmsnorm", card), ("jb200_rmsnorm_backward", card)] and current == [0]
        seen.clear()
    with pytest.raises(RuntimeError, match="cuda:1 and cuda:0"):
        ops.rmsnorm(_on(1, 4, 64), _on(0, 64))
    with pytest.raises(RuntimeError, match="do not belong together"):
        ops.rmsnorm(_on(0, 4, 64), _on(0, 32))
    assert not seen


def test_the_heads_copies_follow_updates_that_leave_no_trace():
    from jarvis_b200 import modules as jm
    torch.manual_seed(1)
    model = jm.Jarvis(vocab_size=301, d_model=128, n_layers=1, n_heads=2, max_seq_len=64).eval()
    w = model.lm_head.weight
    model._lm_head_rows(), model._lm_head_weight()
    opt = torch.optim.AdamW([w], lr=0.1, fused=True)
    for _ in range(2):
        version, w.grad = w._version, torch.randn(301, 128)
        opt.step()
        assert w._version == version                                 # what the test is about
        want = w.detach().bfloat16()
        assert torch.equal(model._lm_head_rows(), want)
        assert torch.equal(model._lm_head_weight()[:301], want) and not model._lm_head_weight()[301:].any()
    opt.zero_grad()
    # an update that neither a loss of this package nor a gradient on the weight announces
    with torch.no_grad():
        w.data.add_(1)
    assert torch.equal(model._lm_head_rows(), w.detach().bfloat16())
    model.refresh_head()
    assert torch.equal(model._lm_head_weight()[:301], w.detach().bfloat16())
    kept = model._lm_head_weight()
    assert model._lm_head_weight() is kept
    # a head in bf16 is its own copy
    model.lm_head.to(torch.bfloat16)
    assert model._lm_head_rows().data_ptr() == model.lm_head.weight.data_ptr()


def test_scratch_is_sized_by_what_is_given():
    """The size goes by the inputs (targets, a teacher), which decide what the statistics hold; the names of the declaration are not those of the
    outputs that may be NULL."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "jarvis_b200.h")).read()
    names = re.search(r"jb200_head_loss_scratch_bytes\(([^)]*)\)", text).group(1).replace("int ", "").split(", ")
    assert names == ["N", "V", "has_targets", "has_teacher"]
    lib = _lib.load()
    for N, V in ((1, 1), (37, 1000), (16384, 50257)):
        ce, kd, both = (lib.jb200_head_loss_scratch_bytes(N, V, *f) for f in ((1, 0), (0, 1), (1, 1)))
        tiles = (V + 255) // 256
        assert (ce, kd, both) == tuple((tiles * k + 3) * N * 4 + 4 for k in (2, 3, 5))


def test_tangents_and_a_teachers_gradient_are_refused():
    """Neither is formed, so neither is dropped without a word."""
    import torch.autograd.forward_ad as fw
    h, w, t = torch.zeros(4, 64), torch.zeros(100, 64), torch.zeros(4, dtype=torch.int64)
    ids, lg = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))         # noqa: E731
        for call in (lambda: losses.linear_cross_entropy(dual(h), w, t), lambda: losses.linear_cross_entropy(h, dual(w), t),
                     lambda: losses.linear_distillation(h, w, ids, dual(lg)), lambda: losses.linear_losses(dual(h), w, t, ids, lg),
                     lambda: losses.rms_norm(dual(h), torch.ones(64)), lambda: losses.rms_norm(h, dual(torch.ones(64)))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="tangent"):
                    call()
    lg.requires_grad_()
    for call in (lambda: losses.linear_distillation(h, w, ids, lg), lambda: losses.linear_losses(h, w, t, ids, lg)):
        with pytest.raises(RuntimeError, match="teacher_logits: no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):      # nothing to lose here
            call()


def test_the_heads_calls_launch_on_their_tensors_card(monkeypatch):
    current, seen = [0], []

    class Card:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return lambda *a: 64
            return lambda *a: seen.append((name, current[0])) or 0

    real = {n: getattr(torch, n) for n in ("empty", "empty_like")}
    monkeypatch.setattr(ops._lib, "load", lambda: Lib())
    monkeypatch.setattr(ops, "_raw_device", lambda: current[0])
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops.torch.cuda, "device", Card)
    monkeypatch.setattr(ops.torch, "empty", lambda s, dtype=None, device=None: _on(device.index, s if isinstance(s, tuple) else (s,), dtype=dtype))
    monkeypatch.setattr(ops.torch, "empty_like", lambda t, dtype=None: real["empty_like"](t, dtype=dtype).as_subclass(_OnCard))

    def rows(card):
        bf, i64 = torch.bfloat16, torch.int64
        return _on(card, 4, 64, dtype=bf), _on(card, 100, 64, dtype=bf), _on(card, 4, dtype=i64), _on(card, 4, 3, dtype=i64), _on(card, 4, 3), _on(card, 1)
    for card in (1, 0):
        x, w, t, ids, lg, g = rows(card)
        teacher = ops.teacher_rows(ids, lg, 100)
        r = ops.head_loss(x, w, t, teacher)
        ops.head_loss_backward(x, w, r, t, teacher, g_ce=g, g_kd=g)
        assert seen == [(n, card) for n in ("jb200_teacher_rows", "jb200_head_loss", "jb200_head_loss_backward")] and current == [0]
        seen.clear()
    x, w, t, ids, lg, g = rows(0)
    _, w1, t1, _, lg1, g1 = rows(1)
    for call in (lambda: ops.teacher_rows(ids, lg1, 100), lambda: ops.head_loss(x, w1, t), lambda: ops.head_loss(x, w, t1),
                 lambda: ops.head_loss_backward(x, w, r, t, teacher, g_ce=g1, g_kd=g)):
        with pytest.raises(RuntimeError, match="cuda:0 and cuda:1"):
            call()
    assert not seen
