"""The operators of a served layer in the order in which a model calls them: scan over padded prompts, norm of the heads with their gate, norm into
the residual stream, draw of the next token, then single tokens by the carried state, eager and as a replayed graph.  Every operator is held
against its 64-bit definition on what it was given, with the tolerances of its own tests."""
import pytest
import torch

from jarvis_b200 import _lib, ops, serving
from tests import test_gpu_block_norms as norms
from tests import test_gpu_gated_delta as delta
from tests import test_gpu_sample_rows as draws
from tests.test_gpu_serving import _tiny_model

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
H, KH, D, V = 4, 2, 64, 5003
C, COLS = H * D, (2 * KH + 2 * H) * D


def _weights():
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return dict(proj=(normal(C, COLS) / 16).to(BF16), gates=(normal(C, 2 * H) / 16).to(BF16), out=(normal(C, C) / 16).to(BF16), head=(normal(V, C) / 4).to(BF16),
                head_norm=1 + 0.2 * normal(D), after=1 + 0.2 * normal(C), before=1 + 0.2 * normal(C), scale=0.3 + 0.1 * normal(C))


def _layer(w, x, xn, B, T, state, lengths=None, check=False):
    """x (B T, C) is updated in place -> xn of the next block; the state in place."""
    p = xn @ w["proj"]
    q, k, v, z = p[:, :KH * D], p[:, KH * D:2 * KH * D], p[:, 2 * KH * D:2 * KH * D + C], p[:, 2 * KH * D + C:]
    g = (xn @ w["gates"]).float()
    log_decay, beta = -0.1 * torch.nn.functional.softplus(g[:, :H]), torch.sigmoid(g[:, H:]).contiguous()
    before = state.clone() if check else None
    o, _ = ops.gated_delta_scan(q, k, v, log_decay, beta, B, T, H, key_heads=KH, lengths=lengths, state_in=state, state_out=state)
    n = ops.gated_norm(o, w["head_norm"], z, group=D)
    y = n @ w["out"]
    x_was = x.clone() if check else None
    _, xn = ops.residual_norm(x, y, w["after"], w["before"], scale=w["scale"], out=x)
    if check:
        delta._check((o, state), delta._definition(q.contiguous(), k.contiguous(), v.contiguous(), log_decay, beta, before, B, T, H, KH, lengths))
        want = norms._norm(o, w["head_norm"], D) * norms._silu(z)
        E = (D / 16 + 40) * 2.0 ** -24 + 2.0 ** -20
        assert ((n.to(F64) - want).abs() <= (E + 2.0 ** -8 * (1 + E)) * want.abs() + 1e-38).all()
        norms._check_residual((x, xn), x_was, y, w["after"], w["before"], None, w["scale"], BF16)
    return xn


def test_prompts_then_single_tokens():
    w, B, T, steps = _weights(), 3, 150, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    lengths = torch.tensor([150, 77, 1], dtype=torch.int32, device="cuda")
    x = torch.randn(B * T, C, generator=g, device="cuda")
    state = torch.zeros(B, H, D, D, device="cuda")
    table = torch.randn(V, C, generator=g, device="cuda")
    xn = _layer(w, x, x.to(BF16), B, T, state, lengths, check=True)
    last = xn.view(B, T, C)[torch.arange(B, device="cuda"), lengths.long() - 1]
    logits = last @ w["head"].t()
    settings = dict(temperature=[0.8, 0.0, 1.2], top_k=[0, 5, 300], top_p=[0.9, 1.0, 0.8], min_p=[0.0, 0.0, 0.02])
    draws._check(logits, **settings)
    args = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else F32, device="cuda") for n, v in settings.items()}
    u = torch.rand(steps + 1, B, generator=g, device="cuda")
    token = ops.sample_rows(logits, u[0], **args)

    def step(token, u, state, check=False):
        x = table[token.view(-1)]
        logits = _layer(w, x, x.to(BF16), B, 1, state, check=check) @ w["head"].t()
        if check:
            draws._check(logits, **settings)
        return ops.sample_rows(logits, u, **args)

    # eager, every operator checked
    eager, s, t = [], state.clone(), token
    for i in range(steps):
        t = step(t, u[1 + i], s, check=True)
        eager.append(t.view(-1).tolist())
    # the same steps as one graph, replayed: the same bits
    s2, t2, u2 = state.clone(), token.clone(), torch.empty(B, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        u2.copy_(u[1])
        step(t2, u2, s2.clone())
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t2.copy_(step(t2, u2, s2))
    replayed = []
    for i in range(steps):
        u2.copy_(u[1 + i])
        graph.replay()
        replayed.append(t2.view(-1).tolist())
    assert replayed == eager and torch.equal(s2, s)
    assert _lib.device_status() == 0


def test_two_calls_at_once_do_not_share_anything():
    """Prompts in segments (scratch of their own) and draws by clusters, on two streams at the same time: the bits of calls alone."""
    problems = [delta._problem(1, 2500, 4, 4, seed=s) for s in (1, 2)]
    rows = [draws._logits(5, 50257, BF16, seed=s) for s in (1, 2)]
    u = torch.rand(5, device="cuda")

    def work(i):
        q, k, v, g, b, s = problems[i]
        o, state = ops.gated_delta_scan(q, k, v, g, b, 1, 2500, 4, state_in=s, want_state=True)
        return o, state, ops.sample_rows(rows[i], u, temperature=0.9, top_p=0.95)

    alone = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        both = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                both.append(work(i))
        torch.cuda.synchronize()
        for got, want in zip(both, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("B,T,H,KH,lengths", [(2, 2048, 16, 4, [2048, 700]), (1, 1100, 16, 16, [1]), (3, 2100, 2, 1, [0, 2100, 65])])
def test_segments_of_padded_batches_and_shared_heads(B, T, H, KH, lengths):
    """Long prompts are cut into segments: sequences that end in an early one, none at all, shared key heads."""
    assert _lib.load().jb200_gated_delta_scratch_bytes(B, T, H) > 0
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q, k, v, g, b, s = delta._problem(B, T, H, KH, seed=9)
    for t in (q, k, v, g, b):                                     # rows behind a sequence are not read
        t.view(B, T, -1)[torch.arange(T, device="cuda") >= lengths.view(B, 1)] = float("nan")
    got = ops.gated_delta_scan(q, k, v, g, b, B, T, H, key_heads=KH, lengths=lengths, state_in=s, want_state=True)
    delta._check(got, delta._definition(q, k, v, g, b, s, B, T, H, KH, lengths))


def test_requests_with_settings_of_their_own():
    model, _ = _tiny_model()
    kw = dict(max_batch_size=3, max_position=128, temperature=0.9, top_k=20, top_p=0.9, seed=11)
    runs = []
    for use_graph in (False, True):
        sched = serving.build_scheduler(model, per_request=True, use_cuda_graph=use_graph, record=True, **kw)
        for i, own in enumerate((None, {"temperature": 0.0}, {"top_k": 1}, {"top_k": 0, "min_p": 0.05}, {"temperature": 1.5, "top_k": 3, "top_p": None})):
            sched.add_request(serving.Request(i, [5, 6, 7 + i], max_new_tokens=4 + i, sampling=own))
        sched.run()
        runs.append([r.generated_tokens for r in sorted(sched.completed, key=lambda r: r.req_id)])
        assert [len(t) for t in runs[-1]] == [4, 5, 6, 7, 8]
        # requests 0 to 2 sit in slots 0 to 2; 1 draws at temperature 0 and 2 from one token
        for i in (1, 2):
            for rec, token in zip(sched.engine.record, runs[-1][i]):
                logits = rec["logits"][i]
                assert int(rec["tokens"][i]) == token and logits[token] == logits.max()
    assert runs[0] == runs[1]


def test_an_engine_with_a_nucleus_of_the_whole_vocabulary():
    model, _ = _tiny_model()
    for kw in (dict(top_k=0, top_p=0.95), dict(top_k=None, top_p=None, min_p=0.1), dict(top_k=2000)):
        outs = []
        for _ in range(2):
            sched = serving.build_scheduler(model, max_batch_size=2, max_position=128, temperature=0.9, seed=3, use_cuda_graph=False, record=True, **kw)
            for i in range(3):
                sched.add_request(serving.Request(i, [5, 6, 7 + i], max_new_tokens=6))
            sched.run()
            outs.append([r.generated_tokens for r in sorted(sched.completed, key=lambda r: r.req_id)])
        assert outs[0] == outs[1] and all(len(t) == 6 for t in outs[0])
        if kw.get("min_p"):
            for rec in sched.engine.record:
                w = ((rec["logits"] - rec["logits"].amax(dim=1, keepdim=True)) / 0.9).exp()
                assert (w.gather(1, rec["tokens"]) >= 0.1 * (1 - 2.0 ** -18)).all()


def test_rows_further_apart_than_32_bits_count():
    """Views with 2^20 elements from row to row, 2500 rows: the bits of contiguous copies."""
    B, T, H, far = 1, 2500, 2, 1 << 20
    buf = torch.zeros(B * T, far, dtype=BF16, device="cuda")
    q, k, v, g, b, s = delta._problem(B, T, H, H, seed=4)
    wide = [buf[:, i * 128:(i + 1) * 128] for i in range(3)]
    for view, t in zip(wide, (q, k, v)):
        view.copy_(t)
    out = torch.empty(B * T, far, dtype=BF16, device="cuda")[:, 64:192]
    with pytest.raises(RuntimeError, match="overlaps"):          # other columns of an argument's buffer count as the argument
        ops.gated_delta_scan(*wide, g, b, B, T, H, out=buf[:, 512:640])
    near = ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True)
    got = ops.gated_delta_scan(*wide, g, b, B, T, H, state_in=s, want_state=True, out=out)
    assert torch.equal(got[0], near[0]) and torch.equal(got[1], near[1])
    w = 1 + 0.2 * torch.randn(64, generator=torch.Generator().manual_seed(1)).cuda()
    assert torch.equal(ops.gated_norm(wide[0], w, wide[1], group=64), ops.gated_norm(q, w, k, group=64))
    w2, x = w.repeat(2), torch.randn(B * T, 128, generator=torch.Generator().manual_seed(2)).cuda()
    for a, b_ in zip(ops.residual_norm(x, wide[0], w2, w2, gate=wide[1]), ops.residual_norm(x, q, w2, w2, gate=k)):
        assert torch.equal(a, b_)
    rows = buf[:, 1:1004]                                        # not aligned either
    rows.copy_(draws._logits(B * T, 1003, BF16, seed=6))
    u = torch.rand(B * T, device="cuda")
    for kw in (dict(top_p=0.9), dict(top_k=20, min_p=0.05), dict(temperature=0.0)):
        assert torch.equal(ops.sample_rows(rows, u, **kw), ops.sample_rows(rows.contiguous(), u, **kw))
    # a vocabulary of 2^24, the largest
    logits = draws._logits(1, 1 << 24, BF16, seed=8)
    draws._check(logits, [1.0], [0], [0.9], [0.0])
    draws._check(logits, [0.7], [3000], [1.0], [0.0])
