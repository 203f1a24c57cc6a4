"""The head's operators as cases that can be timed and compared: the losses of the language-model head straight from
hidden rows and weight (the N x V logits are never an input or an output), with their gradients, and the RMS norm in front
of the head with its backward pass.

With `own` false, `run` computes each operator from elementary torch operations in 32 bits; with `own` true it makes the
calls a user makes of the framework.  Sizes: d_model 1024 and vocabulary 50257 are the model's own; the others are generic.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
VOCAB, C = 50257, 1024
ROWS_MAX = 16384          # 8 sequences of 2048 tokens, the benchmark's batch
IGNORE = -100
EPS = 1e-6


def listed():
    return [
        # scoring, forward only: one token as it arrives; one window of the corpus evaluation; a batch of documents
        dict(name="score_1", kind="score", N=1, V=VOCAB, C=C),
        dict(name="score_256", kind="score", N=256, V=VOCAB, C=C),
        dict(name="score_16384", kind="score", N=16384, V=VOCAB, C=C),
        # cross entropy with both gradients: a short odd sample; one sequence; the benchmark's batch; another model's ragged sizes
        dict(name="train_37", kind="train", N=37, V=VOCAB, C=C),
        dict(name="train_2048", kind="train", N=2048, V=VOCAB, C=C),
        dict(name="train_16384", kind="train", N=16384, V=VOCAB, C=C),
        dict(name="train_1023_v32003", kind="train", N=1023, V=32003, C=776),
        # distillation from a teacher's top logits with both gradients: a window, and a batch with a softened teacher
        dict(name="distill_256_k16", kind="distill", N=256, V=VOCAB, C=C, K=16, tau=1.0),
        dict(name="distill_8192_k64", kind="distill", N=8192, V=VOCAB, C=C, K=64, tau=2.0),
        # the usual recipe: half cross entropy, half distillation, of the same rows
        dict(name="both_4096_k32", kind="both", N=4096, V=VOCAB, C=C, K=32, tau=2.0),
        # the norm in front of the head, forward and backward: the f32 residual stream of a batch; bf16 rows of an odd width
        dict(name="norm_16384_f32", kind="norm", N=16384, C=C, dtype="f32"),
        dict(name="norm_513_bf16", kind="norm", N=513, C=776, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "train", "train", "distill", "distill", "both", "norm"])
    if kind == "norm":
        return dict(kind=kind, N=_log_int(rng, 1, ROWS_MAX), C=8 * _log_int(rng, 8, 256), dtype=rng.choice(["f32", "bf16"]))
    v = rng.choice([VOCAB, _log_int(rng, 500, 65536)])
    c = rng.choice([C, 8 * _log_int(rng, 8, 256)])
    most = min(ROWS_MAX, ROWS_MAX * VOCAB * C // (v * c))
    case = dict(kind=kind, N=_log_int(rng, 1, most), V=v, C=c)
    if kind in ("distill", "both"):
        case.update(K=_log_int(rng, 1, 128), tau=rng.choice([1.0, 1.5, 2.0, 4.0]))
    return case


# ----------------------------------------------------------------------------------------------
# what a program holds before the call
# ----------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """Hidden rows of unit mean square, a head whose logits have a standard deviation of 2.5, and, in nine rows of ten, a
    hidden row that leans towards its target, so that the probabilities are those of a trained model and not flat."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    N = case["N"]
    if case["kind"] == "norm":
        dt = torch.float32 if case["dtype"] == "f32" else BF16
        scale = torch.exp(normal(N, 1))                       # a residual stream's rows differ in size
        return dict(x=(normal(N, case["C"]) * scale).to(dt), weight=1.0 + 0.2 * normal(case["C"]),
                    dy=(normal(N, case["C"]) / N).to(BF16))
    V, width = case["V"], case["C"]
    w = (normal(V, width) * (2.5 / math.sqrt(width))).to(BF16)
    # token ids follow the logarithm: half of them below the square root of the vocabulary, as words do
    target = torch.exp(uniform(N) * math.log(V)).long().clamp_(max=V) - 1
    h = normal(N, width) + (uniform(N, 1) < 0.9) * w[target].float()
    h = (h * torch.rsqrt(h.square().mean(1, keepdim=True))).to(BF16)
    inp = dict(h=h, w=w)
    if case["kind"] != "distill":
        padding = uniform(N) < 0.05                           # the ends of padded sequences have no target
        padding[0] = False
        inp["targets"] = torch.where(padding, torch.full_like(target, IGNORE), target)
    if case["kind"] in ("distill", "both"):
        # a teacher's top K, distinct ids: the target first, then others at a stride of the row's own; the logits descend.  Some rows keep
        # fewer (id -1), a few have none
        K = min(case["K"], V)
        step = 1 + (uniform(N, 1) * max(1, V // K - 1)).long()
        ids = (target[:, None] + step * torch.arange(K, device="cuda")) % V
        logits = 12.0 - 1.5 * torch.log1p(torch.arange(K, device="cuda").float()) * (1.0 + uniform(N, 1)) + 0.05 * normal(N, K)
        kept = (K // 2 + 1 + (uniform(N, 1) * K).long()).clamp_(max=K)
        kept[uniform(N, 1) < 0.03] = 0
        kept[0] = K
        inp["ids"] = torch.where(torch.arange(K, device="cuda") < kept, ids, torch.full_like(ids, -1))
        inp["logits"] = logits.sort(1, descending=True).values
    return inp


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    for name in ("h", "w", "x", "weight"):
        if name in state and case["kind"] != "score":
            state[name].requires_grad_(True)
    return state


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from jarvis_b200 import losses
    kind, case = s["case"]["kind"], s["case"]
    if kind == "score":
        with torch.no_grad():
            return {"rows": losses.linear_cross_entropy(s["h"], s["w"], s["targets"], reduction="none")}
    if kind == "norm":
        y = losses.rms_norm(s["x"], s["weight"], EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if kind == "train":
        loss = losses.linear_cross_entropy(s["h"], s["w"], s["targets"])
    elif kind == "distill":
        loss = losses.linear_distillation(s["h"], s["w"], s["ids"], s["logits"], temperature=case["tau"])
    else:
        ce, kd = losses.linear_losses(s["h"], s["w"], s["targets"], s["ids"], s["logits"], temperature=case["tau"])
        loss = 0.5 * ce + 0.5 * kd
    dh, dw = torch.autograd.grad(loss, (s["h"], s["w"]))
    return {"loss": loss.detach(), "dh": dh, "dw": dw}


@torch.no_grad()
def _run_plain(s):
    kind, case = s["case"]["kind"], s["case"]
    if kind == "norm":
        x, weight, dy = s["x"].float(), s["weight"], s["dy"].float()
        r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
        xh = x * r
        y = xh * weight
        g = dy * weight
        dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
        return {"y": y.to(BF16), "dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0)}

    h, w = s["h"].float(), s["w"].float()
    z = h @ w.t()
    rows = torch.arange(z.shape[0], device=z.device)
    dz, loss = None, 0.0
    if kind in ("score", "train", "both"):
        has = s["targets"] != IGNORE
        t = torch.where(has, s["targets"], torch.zeros_like(s["targets"]))
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        row = torch.where(has, (top + torch.log(total)).squeeze(1) - z[rows, t], torch.zeros_like(top[:, 0]))
        if kind == "score":
            return {"rows": row}
        part = 0.5 if kind == "both" else 1.0
        count = has.sum()
        loss = loss + part * row.sum() / count
        dz = e / total
        dz[rows, t] -= 1.0
        dz *= (part * has / count)[:, None]
    if kind in ("distill", "both"):
        tau = case["tau"]
        kept = s["ids"] >= 0
        some = kept.any(1)
        ids = torch.where(kept, s["ids"], torch.zeros_like(s["ids"]))
        tl = torch.where(kept, s["logits"] / tau, torch.full_like(s["logits"], -1e30))
        q = torch.where(kept, torch.exp(tl - tl.amax(1, keepdim=True)), torch.zeros_like(tl))
        q = q / q.sum(1, keepdim=True).clamp_min(1e-30)
        log_q = torch.log(torch.where(q > 0, q, torch.ones_like(q)))
        zt = z / tau
        top = zt.amax(1, keepdim=True)
        e = torch.exp(zt - top)
        total = e.sum(1, keepdim=True)
        row = (q * (log_q - zt.gather(1, ids) + top + torch.log(total))).sum(1) * tau ** 2
        part = 0.5 if kind == "both" else 1.0
        count = some.sum()
        loss = loss + part * row.sum() / count
        scale = (part * tau * some / count)[:, None]
        soft = (e / total) * scale
        soft.scatter_add_(1, ids, -q * scale)
        dz = soft if dz is None else dz + soft
    return {"loss": loss, "dh": (dz @ w).to(BF16), "dw": (dz.t() @ h).to(BF16)}


# ----------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    f64 = torch.float64
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x, weight, dy = (s[k].to(f64) for k in ("x", "weight", "dy"))
        ms = (x ** 2).sum(1) / case["C"] + EPS
        y = x * weight / ms.sqrt()[:, None]
        along = (dy * weight * x).sum(1) / (case["C"] * ms)
        dx = (dy * weight - along[:, None] * x) / ms.sqrt()[:, None]
        dw = torch.einsum("nc,nc,n->c", dy, x, ms.rsqrt())
        return {"y": y, "dx": dx, "dw": dw}

    N, V = case["N"], case["V"]
    h, w = s["h"].to(f64), s["w"].to(f64)
    ce = kd = 0.0
    n_ce = n_kd = 0
    half = 0.5 if kind == "both" else 1.0
    if kind != "distill":
        n_ce = int((s["targets"] >= 0).sum())
    if kind in ("distill", "both"):
        n_kd = int((s["ids"][:, 0] >= 0).sum())
    rows, dh, dw = [], [], torch.zeros_like(w)
    for a in range(0, N, 1024):
        b = min(N, a + 1024)
        z = torch.einsum("nc,vc->nv", h[a:b], w)
        g = torch.zeros_like(z)
        if kind != "distill":
            t = s["targets"][a:b]
            on = torch.nonzero(t >= 0).squeeze(1)
            logp = torch.log_softmax(z[on], 1)
            nll = -logp[torch.arange(on.numel(), device=z.device), t[on]]
            if kind == "score":
                r = torch.zeros(b - a, dtype=f64, device=z.device)
                r[on] = nll
                rows.append(r)
                continue
            ce = ce + nll.sum()
            p = logp.exp()
            p[torch.arange(on.numel(), device=z.device), t[on]] -= 1.0
            g[on] += half * p / n_ce
        if kind in ("distill", "both"):
            tau = case["tau"]
            ids = s["ids"][a:b]
            q = torch.softmax(torch.where(ids < 0, -math.inf, s["logits"][a:b].to(f64) / tau), 1)
            q = torch.where(ids < 0, torch.zeros_like(q), q)          # rows without any entry: 0 / 0 before, nothing now
            full = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
            logp = torch.log_softmax(z / tau, 1)
            kd = kd + tau * tau * (torch.special.xlogy(q, q).sum() - (full * logp).sum())
            on = (ids[:, 0] >= 0).to(f64)[:, None]
            g += half * tau / n_kd * (logp.exp() * on - full)
        dh.append(g @ w)
        dw += g.t() @ h[a:b]
    if kind == "score":
        return {"rows": torch.cat(rows)}
    loss = half * ((ce / n_ce if n_ce else 0.0) + (kd / n_kd if n_kd else 0.0))
    return {"loss": loss, "dh": torch.cat(dh), "dw": dw}


def work(case):
    """Each input read once, each output written once; a training pass has three products of the same size."""
    N, kind = case["N"], case["kind"]
    if kind == "norm":
        n, size = N * case["C"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * (2 * size + 2 + 2) + 8 * case["C"], "flops": 12 * n}
    V, width = case["V"], case["C"]
    product = 2 * N * V * width
    if kind == "score":
        return {"bytes": 2 * (N + V) * width + 12 * N, "flops": product}
    teacher = 12 * N * case["K"] if "K" in case else 0
    targets = 8 * N if kind != "distill" else 0
    return {"bytes": 4 * (N + V) * width + teacher + targets, "flops": 3 * product}
