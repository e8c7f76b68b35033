"""The embedding, the residual norm and the experts' products together with the operators beside them, as
a model's training step and as a decoding loop use them; captured, replayed and on several streams
(GPU)."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_embedding import _check as check_table
from test_gpu_grouped import _check as check_experts
from test_gpu_residual_norm import LANE_TERMS, U, _close, _formula, _half

pytestmark = pytest.mark.gpu
PACKAGE = Path(__file__).resolve().parents[1] / "warpstate-ai_amd"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-5
D, HIDDEN, EXPERTS, VOCAB = 128, 192, 5, 300


def _model(dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    leaf = lambda *s, std, mean=0.0: (mean + std * torch.randn(s, generator=g)).to(dtype).cuda().requires_grad_(True)
    return {"table": leaf(VOCAB, D, std=1.0), "proj": leaf(D, D, std=0.1),
            "norm1": leaf(D, std=0.1, mean=1.0), "norm2": leaf(D, std=0.1, mean=1.0),
            "up": leaf(EXPERTS, 2 * HIDDEN, D, std=0.1), "down": leaf(EXPERTS, D, HIDDEN, std=0.1)}


def _route(tokens):
    """(order, place of each row in it, offsets) of rows sent to expert token mod EXPERTS; the last
    expert but one gets none. Nothing here waits for the device."""
    expert = tokens % EXPERTS
    expert = torch.where(expert == EXPERTS - 2, 0, expert)
    ranked, order = torch.sort(expert, stable=True)
    offsets = torch.searchsorted(ranked, torch.arange(EXPERTS + 1, device=tokens.device))
    return order, torch.argsort(order), offsets


def _forward(m, tokens, keep=None):
    from ops.activation_execution import bf16_swiglu
    from ops.embedding_execution import embedding
    from ops.fp8_execution import fp8_linear
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm

    order, place, offsets = _route(tokens)
    h = embedding(tokens, m["table"], 0.5)
    p = fp8_linear(h, m["proj"])
    y1, s1 = add_rmsnorm(p, h, m["norm1"], EPS)
    rows = y1[order]
    packed = grouped_mm(rows, m["up"], offsets)
    act = bf16_swiglu(packed)
    z = grouped_mm(act, m["down"], offsets)
    moved = z[place]
    y2, s2 = add_rmsnorm(moved, s1, m["norm2"], EPS)
    if keep is not None:
        keep.update(order=order, place=place, offsets=offsets, h=h, p=p, y1=y1, s1=s1, rows=rows, packed=packed,
                    act=act, z=z, moved=moved, y2=y2, s2=s2)
    return y2, s2


def _loss(m, tokens, targets):
    from ops.token_scores import linear_token_scores

    y2, s2 = _forward(m, tokens)
    logprob, entropy = linear_token_scores(y2, m["table"], targets)
    return -logprob.mean() - 0.01 * entropy.mean() + 1e-3 * s2.float().square().mean()


def _tokens(rows, seed):
    g = torch.Generator().manual_seed(seed)
    tokens = ((VOCAB + 1.0) ** torch.rand(rows, generator=g)).long().sub_(1).clamp_(0, VOCAB - 1)
    return tokens.cuda(), torch.randint(0, VOCAB, (rows,), generator=g).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 67, 700])
def test_training_step(rows, dtype):
    """Every new operator's results and gradients, from the operands and upstream gradients that
    reached it; the tied table gets both of its gradients."""
    from ops.token_scores import linear_token_scores

    m, (tokens, targets) = _model(dtype), _tokens(rows, 3)
    k = {}
    y2, s2 = _forward(m, tokens, k)
    for t in k.values():
        if t.requires_grad:
            t.retain_grad()
    logprob, entropy = linear_token_scores(y2, m["table"], targets)
    loss = -logprob.mean() - 0.01 * entropy.mean() + 1e-3 * s2.float().square().mean()
    loss.backward()

    dh = k["h"].grad
    table = m["table"].detach().clone().requires_grad_(True)
    from ops.embedding_execution import embedding
    d, = torch.autograd.grad(embedding(tokens, table, 0.5), [table], dh)
    check_table(d, tokens.cpu(), dh, VOCAB, 0.5)
    table2 = m["table"].detach().clone().requires_grad_(True)
    lp, en = linear_token_scores(y2.detach(), table2, targets)
    head, = torch.autograd.grad(-lp.mean() - 0.01 * en.mean(), [table2])
    assert torch.equal(m["table"].grad, head + d) or torch.equal(m["table"].grad, d + head)

    for x, out, stream, weight, dy, ds in (("p", "y1", "s1", "norm1", "y1", "s1"),
                                           ("moved", "y2", "s2", "norm2", "y2", "s2")):
        s, w = k[stream].detach(), m[weight].detach().float()
        y, want, want_w, near, near_w = _formula(s, w, k[dy].grad, k[ds].grad)
        _close(k[out].detach(), y, y.abs() * (_half(BF16) + LANE_TERMS * U))
        _close(k[x].grad, want, want.abs() * _half(BF16) + near)
        _close(m[weight].grad, want_w, near_w * U * (rows + 520 + LANE_TERMS) + want_w.abs() * _half(dtype))
    for x, weight, out in (("rows", "up", "packed"), ("act", "down", "z")):
        check_experts(k[x].detach(), m[weight].detach(), k[out].grad, k["offsets"].cpu(), k[out].detach(), k[x].grad,
                      m[weight].grad)
    assert not m["up"].grad[EXPERTS - 2].any()


def _grads(m, tokens, targets):
    leaves = list(m.values())
    loss = _loss(m, tokens, targets)
    return [loss.detach(), *torch.autograd.grad(loss, leaves)]


def test_training_step_in_a_graph():
    """A captured step replayed with other tokens, other experts' counts and eager work between."""
    m = _model()
    tokens, targets = _tokens(200, 1)
    _grads(m, tokens, targets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(m, tokens, targets)
    for seed in (1, 2, 3, 4):
        a, b = _tokens(200, seed)
        if seed == 3:
            a.fill_(7)  # one token, one expert
        tokens.copy_(a)
        targets.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        want = _grads(m, a, b)
        assert all(torch.equal(x, y) for x, y in zip(kept, want)), seed


def test_decoding_loop_in_a_graph():
    """Greedy decoding through the embedding, the 8-bit norms and projection, the experts and the tied
    head: one captured step replayed follows the eager one."""
    from ops import fp8_execution as fp8
    from ops import fused_execution as fx
    from ops.activation_execution import bf16_swiglu
    from ops.embedding_execution import embedding
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize
    from ops.token_scores import token_scores

    m = {k: v.detach() for k, v in _model(BF16).items()}
    q, scale = fp8.quantize_weight(m["proj"])[:2]
    head = m["table"].T

    def step(ids):
        order, place, offsets = _route(ids)
        h = embedding(ids, m["table"], 0.5)
        p = fp8.fp8_mm(*rmsnorm_quantize(h, m["norm1"], EPS)[:2], q, scale)
        a, a_scale, s1 = rmsnorm_quantize(p, m["norm1"], EPS, residual=h)
        p2 = fp8.fp8_mm(a, a_scale, q, scale)
        y, s2 = add_rmsnorm(p2, s1, m["norm2"], EPS)
        z = grouped_mm(bf16_swiglu(grouped_mm(y[order], m["up"], offsets)), m["down"], offsets)[place]
        y, _ = add_rmsnorm(z, s2, m["norm2"], EPS)
        return token_scores(fx.mm(y, head), ids, 3)

    ids = torch.tensor([1, 2, 3, 250], device="cuda")
    step(ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ids)
    eager = ids.clone()
    for _ in range(6):
        ids.copy_(eager)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        want = step(eager)
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
        eager = want.top_ids[:, 0].contiguous()


def test_two_streams_at_once():
    """Steps on two streams that run at the same time give the bits of steps one after the other."""
    jobs = [(_model(seed=s), *_tokens(500 + 100 * s, s)) for s in (1, 2)]
    want = [_grads(*job) for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, job in zip(streams, jobs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_grads(*job))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_replayed_in_turn():
    """Two captured steps of one process keep apart."""
    jobs = [(_model(seed=s), *_tokens(150 * s, s)) for s in (1, 2)]
    want = [_grads(*job) for job in jobs]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for job in jobs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_grads(*job))
    for i in (0, 1, 1, 0, 1):
        for t in outs[i]:
            t.zero_()
        graphs[i].replay()
        graphs[1 - i].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_accumulation_joins_the_heads_gradient():
    """A tied table's FP32 gradient buffer: the head's, accumulated by the cross-entropy's backward, then
    the embedding's, in place."""
    from ops import fused_execution as fx
    from ops.embedding_execution import embedding_accumulate_

    g = torch.Generator().manual_seed(2)
    hidden = torch.randn((160, D), generator=g).to(BF16).cuda()
    table = (0.1 * torch.randn((VOCAB, D), generator=g)).to(BF16).cuda()
    tokens, targets = _tokens(160, 8)
    state = fx.CrossEntropyState(160, VOCAB, hidden.device)
    fx.linear_cross_entropy_forward(hidden, table, targets, state)
    buffer = torch.zeros((VOCAB, D), device="cuda")
    one = torch.ones((), device="cuda")
    dy = fx.linear_cross_entropy_backward(hidden, table, targets, state, one, weight_grad=buffer)
    head = buffer.clone()
    embedding_accumulate_(buffer, tokens, dy, 0.5)
    check_table(buffer, tokens.cpu(), dy, VOCAB, 0.5, base=head)


SCRIPT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from ops.embedding_execution import embedding
from ops.grouped_execution import grouped_mm
from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

def make_step(rows, d, n, experts):
    x = torch.randn((rows, d), device="cuda").bfloat16().requires_grad_(True)
    r = torch.randn((rows, d), device="cuda").requires_grad_(True)
    w = torch.ones(d, device="cuda", requires_grad=True)
    table = torch.randn((500, d), device="cuda").requires_grad_(True)
    tokens = torch.randint(0, 500, (rows,), device="cuda")
    up = torch.randn((experts, n, d), device="cuda").bfloat16().requires_grad_(True)
    offsets = torch.linspace(0, rows, experts + 1, device="cuda").long()
    def step():
        y, s = add_rmsnorm(x, r, w)
        e = embedding(tokens, table)
        z = grouped_mm(y + e, up, offsets)
        q, scale, _ = rmsnorm_quantize(x, w, residual=r)
        grads = torch.autograd.grad([z, s], [x, r, w, table, up], [torch.ones_like(z), torch.ones_like(s)])
        return [z, s, q.view(torch.uint8), scale.view(torch.uint8), *grads]
    return step

make_step(100, 64, 64, 2)()
torch.cuda.synchronize()
for shape in ((8000, 1280, 2048, 4), (3000, 512, 640, 8), (40, 2048, 256, 3), (2000, 72, 136, 3)):
    step = make_step(*shape)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    want = step()
    for _ in range(2):
        for t in out:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), shape
    print(shape, "ok", flush=True)
"""


def test_capture_at_sizes_that_have_not_run():
    """A kernel's first launch may fall into a capture; in a process of its own."""
    run = subprocess.run([sys.executable, "-c", SCRIPT, str(PACKAGE)], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stdout + run.stderr[-2000:]
    assert run.stdout.count("ok") == 4
