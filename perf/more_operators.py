"""Operators of a served layer with a gated delta rule as cases that can be timed and compared: the rule itself over whole prompts and for
single tokens, the norms behind it and around the residual stream with gate and scale, and the draw of the next token from the whole
vocabulary with every sequence's own temperature, top-k, top-p and min-p.

With `own` false, `run` computes each operator from elementary torch operations in 32 bits (64 for sums of log decays and for what decides a
draw); with `own` true it makes the calls a user makes of the framework.  Sizes: 16 heads of 64, d_model 1024 and vocabulary 50257 are the
model's own, B x T those of its benchmark; the others are generic.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
VOCAB, C, HEADS, D = 50257, 1024, 16, 64
ROWS_MAX = 16384          # 8 sequences of 2048 tokens, the benchmark's batch
EPS = 1e-6
CHUNK = 64                # tokens that the plain form of the delta rule takes at a time


def listed():
    return [
        # the delta rule, one token a step: a single conversation, 256 ragged sequences
        dict(name="delta_step_1", kind="delta", B=1, T=1, H=HEADS, KH=HEADS, carry=True, ragged=False),
        dict(name="delta_step_256", kind="delta", B=256, T=1, H=HEADS, KH=HEADS, carry=True, ragged=False),
        # prompts of their own lengths continued from a carried state, two value heads to a key head
        dict(name="delta_3x777", kind="delta", B=3, T=777, H=HEADS, KH=HEADS // 2, carry=True, ragged=True),
        # batch prefill at the size the benchmark quotes; one long document
        dict(name="delta_8x2048", kind="delta", B=8, T=2048, H=HEADS, KH=HEADS, carry=False, ragged=False),
        dict(name="delta_1x16384", kind="delta", B=1, T=16384, H=HEADS, KH=HEADS, carry=False, ragged=False),
        # the norm of every head behind it with its gate, for the batch
        dict(name="headnorm_16384", kind="headnorm", N=16384, C=C, group=D),
        # norm of a block's output, scaled into the residual stream, and the next block's norm: the batch, a decode batch, an odd width
        dict(name="resid_16384", kind="resid", N=16384, C=C, gate=False),
        dict(name="resid_64", kind="resid", N=64, C=C, gate=False),
        dict(name="resid_1023_gate", kind="resid", N=1023, C=776, gate=True),
        # the next token: one conversation with a nucleus of the whole vocabulary, 64 serving slots with settings of their own,
        # 256 sequences of f32 logits with min-p alone
        dict(name="sample_1", kind="sample", N=1, V=VOCAB, dtype="bf16", how="top_p"),
        dict(name="sample_64", kind="sample", N=64, V=VOCAB, dtype="bf16", how="mixed"),
        dict(name="sample_256_f32", kind="sample", N=256, V=VOCAB, dtype="f32", how="min_p"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "step", "headnorm", "resid", "sample", "sample"])
    if kind in ("delta", "step"):
        KH = rng.choice([1, 2, 3, 4, 8, 16])
        H = KH * rng.choice([h for h in (1, 2, 4) if KH * h <= HEADS])
        T = 1 if kind == "step" else _log_int(rng, 2, 8192)
        most = ROWS_MAX * HEADS // (T * H) if T > 1 else 256
        return dict(kind="delta", B=_log_int(rng, 1, max(1, min(most, 256))), T=T, H=H, KH=KH, carry=rng.random() < 0.5, ragged=T > 1 and rng.random() < 0.5)
    if kind == "headnorm":
        group = rng.choice([32, 64, 128])
        return dict(kind=kind, N=_log_int(rng, 1, ROWS_MAX), C=group * rng.randint(1, C // group), group=group)
    if kind == "resid":
        return dict(kind=kind, N=_log_int(rng, 1, ROWS_MAX), C=8 * rng.randint(8, C // 8), gate=rng.random() < 0.5)
    return dict(kind=kind, N=_log_int(rng, 1, 256), V=rng.choice([VOCAB, _log_int(rng, 500, VOCAB)]), dtype=rng.choice(["bf16", "f32"]),
                how=rng.choice(["top_p", "min_p", "plain", "mixed"]))


# ----------------------------------------------------------------------------------------------
# what a program holds before the call
# ----------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s, kind = dict(case=case), case["kind"]
    if kind == "delta":
        B, T, H, KH = case["B"], case["T"], case["H"], case["KH"]
        # keys of one head lean towards a common direction, as those of a trained layer do, so that they overwrite one another
        k = normal(B * T, KH, D) + 1.5 * normal(1, KH, D) * uniform(B * T, 1, 1)
        q = normal(B * T, KH, D) + 0.5 * k
        s["q"], s["k"], s["v"] = q.to(BF16).view(B * T, KH * D), k.to(BF16).view(B * T, KH * D), normal(B * T, H * D).to(BF16)
        # per-head decays as in the model, 0.90 to 0.999 a token, moved by every token
        rate = torch.log(0.90 + 0.099 * uniform(1, H))
        s["log_decay"] = rate * torch.nn.functional.softplus(2.0 * normal(B * T, H))
        s["beta"] = torch.sigmoid(normal(B * T, H))
        s["state"] = normal(B, H, D, D) * 0.5 if case["carry"] else None
        s["lengths"] = None
        if case["ragged"]:
            lengths = (uniform(B) * T).int() + 1
            lengths[0] = T
            s["lengths"] = lengths.clamp(max=T).to(torch.int32)
    elif kind == "headnorm":
        N, width, group = case["N"], case["C"], case["group"]
        s["y"] = (normal(N, width) * torch.exp(0.5 * normal(N, 1))).to(BF16)
        s["gate"] = (1.5 * normal(N, width)).to(BF16)
        s["weight"] = 1.0 + 0.2 * normal(group)
    elif kind == "resid":
        N, width = case["N"], case["C"]
        s["x"] = normal(N, width) * torch.exp(0.5 * normal(N, 1))             # a residual stream's rows differ in size
        s["y"] = (normal(N, width) * torch.exp(normal(N, 1))).to(BF16)
        s["gate"] = (1.5 * normal(N, width)).to(BF16) if case["gate"] else None
        s["w_after"], s["w_before"] = 1.0 + 0.2 * normal(width), 1.0 + 0.2 * normal(width)
        s["scale"] = 0.1 + 0.05 * normal(width)                               # a residual scale that training grows from a small one
    else:
        N, V = case["N"], case["V"]
        logits = 2.0 * normal(N, V)
        # a trained model's rows: some forty tokens stand out, in half of the rows one by far
        likely = (uniform(N, 40) * V).long()
        logits.scatter_add_(1, likely, 6.0 + 2.0 * normal(N, 40) + (uniform(N, 1) < 0.5) * (torch.arange(40, device="cuda") == 0) * 6.0)
        s["logits"] = logits.to(BF16) if case["dtype"] == "bf16" else logits
        s["u"] = uniform(N)
        one = torch.ones(N, device="cuda")
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.7 + 0.5 * uniform(N), torch.zeros(N, dtype=torch.int32, device="cuda"), one, 0 * one
        if case["how"] == "top_p":
            s["top_p"] = 0.85 + 0.13 * uniform(N)
        elif case["how"] == "min_p":
            s["min_p"] = 0.02 + 0.08 * uniform(N)
        elif case["how"] == "mixed":
            s["temperature"] = torch.where(uniform(N) < 0.15, 0 * one, s["temperature"])                       # some slots are greedy
            s["top_k"] = torch.where(uniform(N) < 0.5, (1 + 2000 * uniform(N) ** 3).int(), s["top_k"]).to(torch.int32)
            s["top_p"] = torch.where(uniform(N) < 0.5, 0.8 + 0.19 * uniform(N), one)
            s["min_p"] = torch.where(uniform(N) < 0.3, 0.1 * uniform(N), 0 * one)
    return s


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from jarvis_b200 import ops
    case = s["case"]
    kind = case["kind"]
    if kind == "delta":
        o, state = ops.gated_delta_scan(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], case["B"], case["T"], case["H"], key_heads=case["KH"],
                                        lengths=s["lengths"], state_in=s["state"], want_state=True)
        return {"o": o, "state": state}
    if kind == "headnorm":
        return {"y": ops.gated_norm(s["y"], s["weight"], s["gate"], group=case["group"], eps=EPS)}
    if kind == "resid":
        x, xn = ops.residual_norm(s["x"], s["y"], s["w_after"], s["w_before"], gate=s["gate"], scale=s["scale"], eps=EPS)
        return {"x": x, "xn": xn}
    token, prob = ops.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                  want_prob=True)
    return {"token": token, "prob": prob}


@torch.no_grad()
def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "delta":
        return _plain_delta(s)
    if kind == "headnorm":
        N, width = s["y"].shape
        group = s["case"]["group"]
        y = s["y"].float().view(N, width // group, group)
        y = y * torch.rsqrt(y.square().mean(2, keepdim=True) + EPS) * s["weight"]
        g = s["gate"].float()
        return {"y": (y.view(N, width) * g / (1.0 + torch.exp(-g))).to(BF16)}
    if kind == "resid":
        y = s["y"].float()
        y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + EPS) * s["w_after"]
        if s["gate"] is not None:
            g = s["gate"].float()
            y = y * g / (1.0 + torch.exp(-g))
        x = s["x"] + s["scale"] * y
        return {"x": x, "xn": (x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * s["w_before"]).to(BF16)}
    return _plain_sample(s)


def _plain_delta(s):
    """S_t = a_t S_{t-1} (I - b_t k k^T) + b_t v k^T and o_t = S_t q / sqrt(D), 64 tokens at a time: with G the running sum of log a in
    the chunk, u = (I + A)^-1 b (v - e^G S k) for A_ij = b_i e^(G_i - G_j) k_i.k_j below the diagonal.  The chunks follow one another."""
    case = s["case"]
    B, T, H, KH = case["B"], case["T"], case["H"], case["KH"]
    n = -(-T // CHUNK)
    if T == 1:
        return _plain_step(s, B, H, KH)

    def chunks(x, heads):                                  # (B T, heads w) -> (n, B, H, 64, w), zero behind the end
        x = x.float().view(B, T, heads, -1)
        if heads != H:
            x = x.repeat_interleave(H // heads, 2)
        if s["lengths"] is not None:
            x = torch.where((torch.arange(T, device=x.device) < s["lengths"][:, None])[:, :, None, None], x, torch.zeros_like(x))
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * CHUNK - T))
        return x.view(B, n, CHUNK, H, -1).permute(1, 0, 3, 2, 4)

    q, k, v = chunks(s["q"], KH), chunks(s["k"], KH), chunks(s["v"], H)
    q = q * (torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS) / math.sqrt(D))
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS)
    beta = chunks(s["beta"], H)
    G = chunks(s["log_decay"], H).double().cumsum(-2)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp(torch.where(lower, G - G.transpose(-1, -2), torch.full_like(G[..., :1], -math.inf))).float()
    A = (beta * decay * (k @ k.transpose(-1, -2))).tril(-1)
    P = decay * (q @ k.transpose(-1, -2))
    # (I + A)^-1 by doubling: the inverses of diagonal blocks of 1, 2, 4, ... 32 give those of twice the size
    at = torch.arange(CHUNK, device=q.device)
    inv = torch.eye(CHUNK, device=q.device).expand_as(A)
    for level in range(6):
        half = (at[:, None] >> level + 1 == at >> level + 1) & (at[:, None] >> level != at >> level)
        inv = inv - inv @ (A * half) @ inv
    first, last = torch.exp(G).float(), torch.exp(G[..., -1:, :] - G).float()
    whole = torch.exp(G[..., -1:, :]).float()
    S = s["state"] if s["state"] is not None else torch.zeros(B, H, D, D, device=q.device)
    o = torch.empty_like(v)
    for c in range(n):
        u = inv[c] @ (beta[c] * (v[c] - first[c] * (k[c] @ S.transpose(-1, -2))))
        o[c] = first[c] * (q[c] @ S.transpose(-1, -2)) + P[c] @ u
        S = whole[c] * S + u.transpose(-1, -2) @ (last[c] * k[c])
    o = o.permute(1, 0, 3, 2, 4).reshape(B, n * CHUNK, H * D)[:, :T]
    if s["lengths"] is not None:
        o = torch.where((torch.arange(T, device=o.device) < s["lengths"][:, None])[:, :, None], o, torch.zeros_like(o))
    return {"o": o.reshape(B * T, H * D).to(BF16), "state": S}


def _plain_step(s, B, H, KH):
    q, k = (s[x].float().view(B, KH, D).repeat_interleave(H // KH, 1) for x in ("q", "k"))
    q = q * (torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS) / math.sqrt(D))
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS)
    v, beta = s["v"].float().view(B, H, D), s["beta"].unsqueeze(-1)
    S = torch.zeros(B, H, D, D, device=q.device) if s["state"] is None else s["state"] * torch.exp(s["log_decay"])[:, :, None, None]
    u = beta * (v - (S * k[:, :, None, :]).sum(-1))
    S = S + u[..., None] * k[:, :, None, :]
    return {"o": (S * q[:, :, None, :]).sum(-1).view(B, H * D).to(BF16), "state": S}


def _plain_sample(s):
    """Order of the logits, ties by the lower id; every filter is a cut of that order; the draw is the inverse of the running sum."""
    x, ids = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
    N, V = x.shape
    greedy = s["temperature"] <= 0
    t = s["temperature"].double().clamp_min(1e-5)[:, None]
    w = torch.exp((x - x[:, :1]) / t)
    k = torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], V)).clamp(max=V).long()
    w = torch.where(x >= x.gather(1, k[:, None] - 1), w, torch.zeros_like(w))
    c = w.cumsum(1)
    p = torch.where((s["top_p"] > 0) & (s["top_p"] < 1), s["top_p"].double(), torch.full_like(t[:, 0], 2.0))[:, None]
    kept = (c - w <= p * c[:, -1:]) & (w >= s["min_p"].double()[:, None]) & (w > 0)
    kept[:, 0] = True
    w = torch.where(kept, w, torch.zeros_like(w))
    c = w.cumsum(1)
    at = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1).minimum(kept.sum(1) - 1)
    at = torch.where(greedy, torch.zeros_like(at), at)[:, None]
    prob = torch.where(greedy[:, None], torch.ones_like(t), w.gather(1, at) / c[:, -1:])
    return {"token": ids.gather(1, at), "prob": prob.float()[:, 0]}


# ----------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    f64 = torch.float64
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "delta":
        B, T, H, KH = case["B"], case["T"], case["H"], case["KH"]
        q, k = (s[x].to(f64).view(B, T, KH, D).repeat_interleave(H // KH, 2) for x in ("q", "k"))
        q = q / (q.square().sum(-1, keepdim=True) + EPS).sqrt() / D ** 0.5
        k = k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()
        v = s["v"].to(f64).view(B, T, H, D)
        a, b = s["log_decay"].to(f64).view(B, T, H, 1, 1).exp(), s["beta"].to(f64).view(B, T, H, 1)
        on = torch.ones(B, T, 1, 1, dtype=torch.bool, device=q.device)
        if s["lengths"] is not None:
            on = (torch.arange(T, device=q.device) < s["lengths"][:, None]).view(B, T, 1, 1)
        S = torch.zeros(B, H, D, D, dtype=f64, device=q.device) if s["state"] is None else s["state"].to(f64)
        o = torch.zeros(B, T, H, D, dtype=f64, device=q.device)
        for t in range(T):
            decayed = a[:, t] * S
            u = b[:, t] * (v[:, t] - torch.einsum("bhvk,bhk->bhv", decayed, k[:, t]))
            new = torch.baddbmm(decayed.view(B * H, D, D), u.reshape(B * H, D, 1), k[:, t].reshape(B * H, 1, D)).view(B, H, D, D)
            S = torch.where(on[:, t].unsqueeze(-1), new, S)
            o[:, t] = torch.einsum("bhvk,bhk->bhv", S, q[:, t]) * on[:, t]
        return {"o": o.view(B * T, H * D), "state": S}
    if kind == "headnorm":
        N, width, group = case["N"], case["C"], case["group"]
        y, g = s["y"].to(f64).view(N, -1, group), s["gate"].to(f64)
        y = y / (torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / group + EPS).sqrt()
        return {"y": (y * s["weight"].to(f64)).view(N, width) * g * torch.sigmoid(g)}
    if kind == "resid":
        width = case["C"]
        y, x = s["y"].to(f64), s["x"].to(f64)
        y = y / (torch.linalg.vector_norm(y, dim=1, keepdim=True) ** 2 / width + EPS).sqrt() * s["w_after"].to(f64)
        if case["gate"]:
            g = s["gate"].to(f64)
            y = y * g * torch.sigmoid(g)
        x = torch.addcmul(x, s["scale"].to(f64), y)
        return {"x": x, "xn": x / (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / width + EPS).sqrt() * s["w_before"].to(f64)}
    # row by row: softmax over what each filter leaves, token by token in descending order
    tokens, probs = [], []
    for r in range(case["N"]):
        x = s["logits"][r].to(f64)
        t, k, p, m = (s[name][r].item() for name in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(x, descending=True, stable=True)
        if t <= 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        z = x[order] / max(t, 1e-5)
        if k > 0:
            z = torch.where(z < z[min(k, z.numel()) - 1], -math.inf, z)
        q = torch.softmax(z, 0)
        if 0 < p < 1:
            gone = q.cumsum(0) > p
            gone = torch.cat([torch.zeros_like(gone[:1]), gone[:-1]])
            z = torch.where(gone, -math.inf, z)
        z = torch.where(q < m * q[0], -math.inf, z)
        q = torch.softmax(z, 0)
        at = int(torch.searchsorted(q.cumsum(0), s["u"][r].to(f64), right=True).clamp(max=int((q > 0).sum()) - 1))
        tokens.append(int(order[at]))
        probs.append(q[at])
    return {"token": torch.tensor(tokens, device="cuda").view(-1, 1), "prob": torch.stack([torch.as_tensor(x, dtype=f64, device="cuda") for x in probs])}


def work(case):
    """Each input read once, each output written once; the delta rule's operations are those of its recurrence, token by token."""
    kind = case["kind"]
    if kind == "delta":
        rows, H, states = case["B"] * case["T"], case["H"], case["B"] * case["H"] * D * D
        return {"bytes": rows * (2 * D * (2 * case["KH"] + 2 * H) + 8 * H) + 4 * states * (2 if case["carry"] else 1), "flops": 7 * rows * H * D * D}
    if kind == "headnorm":
        n = case["N"] * case["C"]
        return {"bytes": 6 * n + 4 * case["group"], "flops": 10 * n}
    if kind == "resid":
        n = case["N"] * case["C"]
        return {"bytes": n * (4 + 2 + 4 + 2 + (2 if case["gate"] else 0)) + 12 * case["C"], "flops": 14 * n}
    n = case["N"] * case["V"]
    return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 32 * case["N"], "flops": 4 * n}
