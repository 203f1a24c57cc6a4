"""Losses of the language-model head straight from its hidden rows, and the norm in front of it, with gradients.

    loss = linear_cross_entropy(hidden, weight, targets)                      F.cross_entropy(hidden @ weight.T, targets)
    loss = linear_distillation(hidden, weight, teacher_ids, teacher_logits, temperature=2.0)
    ce, kd = linear_losses(hidden, weight, targets, teacher_ids, teacher_logits, temperature=2.0)       both, the products once
    y = rms_norm(x, weight)

The reference forms lm_head's logits and takes F.cross_entropy of them (jarvis_engine/jarvis_model.py:535-540); at 16,384 rows and its
vocabulary those are 1.6 GB in bf16.  Here they are not stored, in neither direction; a backward pass holds their gradients, in f16 and at
most 640 MiB at a time (beyond some 6,600 rows of that vocabulary less than all of them).

These are torch.autograd functions over the calls in `ops` (which have a forward and a backward call each, for programs without
autograd).  Gradients formed under create_graph raise when they are differentiated, and tensors with a forward-mode tangent are refused.
A captured training step takes its gradients with torch.autograd.grad, or backward() when no graph from outside the capture holds the
same parameters' accumulators; the operators themselves launch on the current stream and synchronise with nothing.

Numerics: hidden rows and weight enter the products as bf16 (an f32 argument is rounded to it, as under autocast), sums and softmax are
f32, the gradient of the logits is rounded to f16 for the products it enters (2^-12 of a value down to 2^-27 of the row's factor in the
loss, whatever the other rows' are; values below 2^-38 of it are lost), rows and weight enter those exactly within 2^32 of their
largest value (in the weight's gradient: of a row's value times its factor), gradients are returned in their argument's dtype from f32
sums.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import ops


def _bf16(t: torch.Tensor, what: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: expected a CUDA tensor (this path has no CPU fallback)")
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"{what}: expected float32 or bfloat16, got {t.dtype}")
    return (t if t.dtype is torch.bfloat16 else t.to(torch.bfloat16)).contiguous()


def _trains(weight: torch.Tensor):
    """Marks a weight that is about to get a gradient: updates may leave no trace on it, so nobody keeps a copy (modules._in_training)."""
    if weight.requires_grad:
        weight._jb_trained = True


def _no_tangents(what: str, *tensors):
    """Dual tensors do not require gradients: their tangents would go missing where nothing else does."""
    if getattr(forward_ad, "_current_level", 0) < 0:       # outside every dual_level there are none
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what}: a tensor carries a tangent, and there is no forward-mode derivative")


def _rows(t: torch.Tensor, lead, dtypes, what: str, columns: int | None = None) -> torch.Tensor:
    """`t` of shape (*lead) or (*lead, columns) as contiguous rows."""
    if t.dtype not in dtypes:
        raise RuntimeError(f"{what}: expected {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    shape = tuple(lead) if columns is None else (*lead, columns)
    if tuple(t.shape) != shape:
        raise RuntimeError(f"{what}: expected shape {shape}, got {tuple(t.shape)}")
    return t.reshape(-1) if columns is None else t.reshape(-1, columns).contiguous()


def _forward(hidden, weight, targets, ids, logits, temperature, mean):
    """The operators' common forward pass -> (bf16 rows, bf16 weight, targets, teacher, result, leading shape)."""
    x, w = _bf16(hidden, "hidden"), _bf16(weight, "weight")
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise RuntimeError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} must be (..., C) and (V, C)")
    lead = x.shape[:-1]
    if x.dim() != 2:
        x = x.view(-1, w.shape[1])
    teacher = None
    if targets is not None:
        targets = _rows(targets, lead, (torch.int64,), "targets").contiguous()
    if ids is not None:
        if ids.dim() < 1 or ids.shape[-1] < 1:
            raise RuntimeError(f"teacher_ids: expected (..., K) with at least one entry a row, got {tuple(ids.shape)}")
        ids = _rows(ids, lead, (torch.int64,), "teacher_ids", ids.shape[-1])
        logits = _rows(logits, lead, (torch.float32, torch.bfloat16), "teacher_logits", ids.shape[1])
        teacher = ops.teacher_rows(ids, logits, w.shape[0], temperature)
    return x, w, targets, teacher, ops.head_loss(x, w, targets, teacher, want_rows=not mean, want_means=mean), lead


def _results(r, lead):
    """(cross entropy, distillation), None where not asked for."""
    if r.info[2]:
        return r.mean_ce, r.mean_kd
    if len(lead) == 1:
        return r.ce, r.kd
    return (None if r.ce is None else r.ce.view(lead)), (None if r.kd is None else r.kd.view(lead))


class _FirstOnly(torch.autograd.Function):
    """A gradient formed under create_graph: part of the graph of all it was formed from, so that whoever differentiates it meets the error
    (without the node it would be a constant, and a penalty on gradients lose this operator's term without a word)."""

    @staticmethod
    def forward(ctx, gradient, what, *formed_from):
        ctx.what = what
        return gradient.view_as(gradient)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"the gradients of {ctx.what} cannot be differentiated: there is no second derivative")


def _first_only(gradients, what, formed_from):
    formed_from = [t for t in formed_from if t is not None]
    return tuple(g if g is None else _FirstOnly.apply(g, what, *formed_from) for g in gradients)


def _origin(t: torch.Tensor, saved: torch.Tensor):
    """What leads to `t`'s graph where `saved`, the form of it that is kept for the backward pass, does not: `t` itself when it is a leaf,
    which the graph holds anyway, else an empty tensor made from it, which keeps none of its memory."""
    if saved is t or not t.requires_grad:
        return None
    if t.is_leaf:
        return t
    with torch.enable_grad():
        return t[..., :0].clone()


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ids, logits, temperature, mean):
        x, w, targets, teacher, r, lead = _forward(hidden, weight, targets, ids, logits, temperature, mean)
        ctx.origins = None if x is hidden and w is weight else (_origin(hidden, x), _origin(weight, w))
        ctx.save_for_backward(x, w, targets, r.buf, None if teacher is None else teacher.buf)
        ctx.info = (hidden.shape, hidden.dtype, weight.dtype, mean, None if teacher is None else (teacher.K, teacher.vocab, teacher.temperature))
        return _results(r, lead)

    @staticmethod
    def backward(ctx, g_ce, g_kd):
        saved = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return _head_backward(ctx, saved, g_ce, g_kd)
        with torch.no_grad():
            got = _head_backward(ctx, saved, g_ce, g_kd)
        return _first_only(got, "the head's losses", (*saved[:2], *(ctx.origins or ()), g_ce, g_kd))


def _head_backward(ctx, saved, g_ce, g_kd):
    x, w, targets, buf, teacher = saved
    shape, dx_dtype, dw_dtype, mean, info = ctx.info
    N = x.shape[0]
    if teacher is not None:
        teacher = ops.TeacherRows(teacher, N, *info)
    if not mean:
        g_ce, g_kd = (None if g is None else g.reshape(-1).contiguous() for g in (g_ce, g_kd))
    want_dx, want_dw = ctx.needs_input_grad[:2]
    dx, dw = ops.head_loss_backward(x, w, ops.HeadLoss(N, buf, (targets is not None, teacher is not None, mean)), targets, teacher, g_ce=g_ce,
                                    g_kd=g_kd, mean=mean, dx_dtype=dx_dtype, dw_dtype=dw_dtype, want_dx=want_dx, want_dw=want_dw)
    if want_dx and len(shape) != 2:
        dx = dx.view(shape)
    return dx, dw, None, None, None, None, None


def _head_loss(hidden, weight, targets, ids, logits, temperature, reduction):
    if reduction not in ("mean", "none"):
        raise RuntimeError(f"reduction must be 'mean' or 'none', got {reduction!r}")
    _no_tangents("the head's losses", hidden, weight, logits)
    if logits is not None and logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("teacher_logits: no gradient is formed for them; pass them detached")
    mean = reduction == "mean"
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        _trains(weight)
        return _HeadLoss.apply(hidden, weight, targets, ids, logits, temperature, mean)
    r, lead = _forward(hidden, weight, targets, ids, logits, temperature, mean)[4:]
    return _results(r, lead)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, reduction: str = "mean") -> torch.Tensor:
    """-log softmax(hidden @ weight.T)[targets], differentiable in hidden (..., C) and weight (V, C), bf16, or f32 and rounded to bf16
    for the products.  targets: int64 (...); -100 marks a row without one (loss 0, no part in any gradient), another value outside
    [0, V) makes its row NaN.  reduction: "mean" over the rows with a target (NaN when there is none) -> f32 scalar; "none" -> f32
    (...).  C: a multiple of 8, at least 64.  The gradient of a logit is rounded to f16 relative to its row's factor in the whole
    loss: 2^-12 of itself, nothing of what is below 2^-38 of that factor."""
    return _head_loss(hidden, weight, targets, None, None, 1.0, reduction)[0]


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                        temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """t^2 KL(softmax(teacher_logits / t) over the row's entries || softmax(hidden @ weight.T / t)), t the temperature, differentiable in
    hidden and weight (their types and roundings: linear_cross_entropy).  teacher_ids: int64 (..., K), teacher_logits: f32 or bf16 (..., K),
    K <= 256, in any order; a negative id is no entry, a row without entries has no part (loss 0), an id beyond the vocabulary makes its
    row NaN.  No gradient is formed for teacher_logits: ones that require one are refused.  "mean": over the rows with entries.  A difference of f32 logarithms: off by up to
    t^2 2^-19."""
    return _head_loss(hidden, weight, None, teacher_ids, teacher_logits, temperature, reduction)[1]


def linear_losses(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, teacher_ids: torch.Tensor,
                  teacher_logits: torch.Tensor, *, temperature: float = 1.0, reduction: str = "mean"):
    """(linear_cross_entropy, linear_distillation) of the same rows: one pass forward, one pass backward whatever their weights are."""
    return _head_loss(hidden, weight, targets, teacher_ids, teacher_logits, temperature, reduction)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, out_dtype):
        rows, w = x.contiguous(), weight.float().contiguous()
        ctx.save_for_backward(rows, w)
        ctx.eps, ctx.weight_dtype, ctx.origins = eps, weight.dtype, None if rows is x and w is weight else (_origin(x, rows), _origin(weight, w))
        return ops.rmsnorm(rows, w, eps, out_dtype)

    @staticmethod
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return _norm_backward(ctx, saved, dy)
        with torch.no_grad():
            got = _norm_backward(ctx, saved, dy)
        return _first_only(got, "rms_norm", (*saved, *(ctx.origins or ()), dy))


def _norm_backward(ctx, saved, dy):
    x, w = saved
    want_dx, want_dw = ctx.needs_input_grad[:2]
    dx, dw = ops.rmsnorm_backward(x, w, dy.contiguous(), ctx.eps, want_dx=want_dx)
    if not want_dw:
        return dx, None, None, None
    return dx, dw if ctx.weight_dtype is torch.float32 else dw.to(ctx.weight_dtype), None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, out_dtype=torch.bfloat16) -> torch.Tensor:
    """RMSNorm.forward (jarvis_engine/jarvis_model.py:25-26) over the last axis, differentiable in x (f32 or bf16) and weight."""
    if weight.dim() != 1 or x.dim() < 1 or weight.shape[0] != x.shape[-1]:
        raise RuntimeError(f"rms_norm: weight {tuple(weight.shape)} does not fit rows of {tuple(x.shape)}")
    _no_tangents("rms_norm", x, weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        _trains(weight)
        return _RMSNorm.apply(x, weight, eps, out_dtype)
    return ops.rmsnorm(x.contiguous(), weight.float().contiguous(), eps, out_dtype)
