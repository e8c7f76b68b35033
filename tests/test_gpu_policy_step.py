"""The 8-bit projections and the token scores together, as a policy's training step and as a
decoding loop use them, each piece against 64-bit arithmetic from what it was given."""
import numpy as np
import pytest
import torch

from fp8_reference import BLOCK, dequantize, quantize, values
from test_gpu_fp8 import _check
from test_gpu_token_scores import U, _bounds, _near, _reference

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E8M0 = torch.float8_e8m0fnu


@pytest.mark.parametrize("master", [True, False])
def test_policy_step(master):
    """Two 8-bit projections around a nonlinearity, the head's scores and a policy loss with an
    entropy bonus: every gradient on the way, from the gradient that reached its operator."""
    from ops import fp8_execution as fp8
    from ops import token_scores as ts

    rows, d, hidden, vocab = 200, 136, 264, 517
    g = torch.Generator().manual_seed(5)
    dtype = F32 if master else BF16
    leaf = lambda *s, std: (torch.randn(s, generator=g) * std).to(dtype).cuda().requires_grad_(True)
    w_in, w_out, head = leaf(hidden, d, std=0.1), leaf(d, hidden, std=0.1), leaf(vocab, d, std=0.2)
    x = torch.randn((rows, d), generator=g).to(BF16).cuda().requires_grad_(True)
    tokens = torch.randint(0, vocab, (rows,), generator=g).cuda()
    tokens[::17] = -100
    advantage = torch.randn(rows, generator=g).cuda()

    y = fp8.fp8_linear(x, w_in)
    act = torch.tanh(y)
    z = fp8.fp8_linear(act, w_out)
    logprob, entropy = ts.linear_token_scores(z, head, tokens)
    for t in (y, act, z, logprob, entropy):
        t.retain_grad()
    loss = -(advantage * logprob).mean() - 0.01 * entropy.mean()
    loss.backward()

    # The products, from their own operands and upstream gradients.
    for out, src, weight in ((y, x, w_in), (z, act, w_out)):
        w_q, w_s, wt_q, wt_s = fp8.quantize_weight(weight)
        _check(out.detach(), *fp8.quantize_rows(src), w_q, w_s)
        _check(src.grad, *fp8.quantize_rows(out.grad), wt_q, wt_s)
        fdy, fx = values(out.grad), values(src)
        if master:
            size = np.abs(fdy).T @ np.abs(fx)
            assert np.all(np.abs(values(weight.grad) - fdy.T @ fx) <= (rows + 2) * 2.0 ** -23 * size + 1e-38)
        else:
            _check(weight.grad, *fp8.quantize_columns(out.grad), *fp8.quantize_columns(src))
    # The scores and the head's gradients.
    fz, fh = z.detach().double().cpu(), head.detach().to(BF16).double().cpu()
    up_g, up_h = logprob.grad, entropy.grad
    want_lp, want_e, logp, dl = _reference(fz @ fh.T, tokens, 1.0, up_g, up_h)
    extra = 2 * (d + 2) * U * float((fz.abs() @ fh.abs().T).max())
    score_tol, entropy_tol, rel = _bounds(fz @ fh.T, 1.0, extra)
    _near(logprob.detach(), want_lp, score_tol)
    _near(entropy.detach(), want_e, entropy_tol)
    p = logp.exp()
    size = p * (up_g.abs().cpu()[:, None] + up_h.abs().cpu()[:, None] * (logp.abs() + want_e[:, None]))
    err = size * (rel + score_tol + 16 * U) + p * up_h.abs().cpu()[:, None] * (score_tol + entropy_tol)
    err = err + (dl.abs() + err) * 2.0 ** -8
    for got, want, bound, final in ((z.grad, dl @ fh, err @ fh.abs(), 2.0 ** -8),
                                    (head.grad, dl.T @ fz, err.T @ fz.abs(), torch.finfo(dtype).eps / 2)):
        bound = bound + (vocab + rows) * U * (dl.abs().max() * fz.abs().max().clamp_min(1) + bound)
        bound = bound + (want.abs() + bound) * final + 1e-30
        assert bool(((got.double().cpu() - want).abs() <= bound).all())


def test_decoding_loop_in_a_graph():
    """Three sequences decoded greedily through one 8-bit projection and the head: rows
    quantized, the product, the logits, the likeliest token, its embedding; one captured step
    replayed follows the eager one, and its scores are those of its logits."""
    from ops import fp8_execution as fp8
    from ops import fused_execution as fx
    from ops import token_scores as ts

    vocab, d = 1000, 128
    g = torch.Generator().manual_seed(9)
    embed = torch.randn((vocab, d), generator=g).to(BF16).cuda()
    q, scale = fp8.quantize_weight(torch.randn((d, d), generator=g).cuda() * 0.2)[:2]
    token = torch.tensor([1, 2, 3], device="cuda")

    def step(ids):
        h = fp8.fp8_mm(*fp8.quantize_rows(embed[ids]), q, scale)
        logits = fx.mm(h, embed.T)
        return logits, ts.token_scores(logits, ids, 4)

    step(token)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    ids = token.clone()
    with torch.cuda.graph(graph):
        logits, scores = step(ids)
    eager = token.clone()
    for _ in range(6):
        ids.copy_(eager)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (logits, *scores)]
        want_logits, want = step(eager)
        for a, b in zip(kept, (want_logits, *want)):
            assert torch.equal(a, b)
        ref_lp, ref_e, logp, _ = _reference(kept[0], eager, 1.0)
        score_tol, entropy_tol, _rel = _bounds(kept[0].cpu(), 1.0)
        _near(kept[1], ref_lp, score_tol)
        _near(kept[2], ref_e, entropy_tol)
        first = kept[0].float().max(-1)
        assert torch.equal(kept[0].float().gather(1, kept[4][:, :1])[:, 0], first[0])
        eager = want.top_ids[:, 0].contiguous()


def test_quantized_reference_is_what_the_product_reads():
    """The quantizer's values agree with the 64-bit restatement at a projection's size."""
    from ops import fp8_execution as fp8

    w = torch.randn((264, 400), generator=torch.Generator().manual_seed(1)).cuda()
    q, scale, qt, scale_t = fp8.quantize_weight(w)
    want_q, want_scale = quantize(values(w), E8M0, BLOCK)
    assert np.array_equal(dequantize(values(q), values(scale)), dequantize(want_q, want_scale))
    assert np.array_equal(dequantize(values(qt), values(scale_t)).T, dequantize(want_q, want_scale))


def _training_step(master, seed=5):
    """(inputs, step): forward and every gradient of a projection and the head's scores, from
    leaves made within the step."""
    from ops import fp8_execution as fp8
    from ops import token_scores as ts

    rows, d, hidden, vocab = 300, 136, 264, 1037
    g = torch.Generator().manual_seed(seed)
    dtype = F32 if master else BF16
    make = lambda t, *s: torch.randn(s, generator=g).to(t).cuda()
    inputs = [make(BF16, rows, d), make(dtype, hidden, d), make(dtype, vocab, hidden),
              torch.randint(0, vocab, (rows,), generator=g).cuda(), make(F32, rows)]

    def step():
        x, w, head = (t.detach().requires_grad_(True) for t in inputs[:3])
        tokens, up = inputs[3:]
        logprob, entropy = ts.linear_token_scores(fp8.fp8_linear(x, w), head, tokens, 0.8, 128)
        return (logprob, entropy, *torch.autograd.grad([logprob, entropy], [x, w, head], [up, -up]))

    return inputs, step


@pytest.mark.parametrize("master", [True, False])
def test_training_step_in_a_captured_graph(master):
    """Three chunks of rows, both kinds of weight: each replay is the eager step on its inputs,
    with eager work between the replays."""
    inputs, step = _training_step(master)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        g = torch.Generator().manual_seed(50 + seed)
        inputs[0].copy_(torch.randn(inputs[0].shape, generator=g))
        inputs[4].copy_(torch.randn(inputs[4].shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_two_steps_on_two_streams():
    """Steps that overlap share no workspace: each gives what it gives alone."""
    steps = [_training_step(True, 5)[1], _training_step(False, 6)[1]]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(5):
        for i, (stream, step) in enumerate(zip(streams, steps)):
            with torch.cuda.stream(stream):
                got[i].append(step())
    torch.cuda.synchronize()
    for results, alone in zip(got, want):
        for result in results:
            for a, b in zip(result, alone):
                assert torch.equal(a, b)
