"""Token scores at the edges of what their documentation allows: tokens without a score under
masked losses, the smallest and largest temperatures, more rows than one launch takes,
chunks past 32 bits (GPU)."""
import pytest
import torch

from test_gpu_token_scores import BF16, F32, _logits

pytestmark = pytest.mark.gpu


def _scores():
    from ops import token_scores

    return token_scores


@pytest.mark.parametrize("rows,vocab", [(6, 300), (6, 9001)])
def test_rows_outside_the_loss_pass_no_gradient(rows, vocab):
    """A row whose two upstream gradients are zero gets zeros whatever its token: padding rows
    marked by an id outside the vocabulary, under a masked loss. With an entropy gradient only,
    such a row gets the entropy's; with one on its log probability, NaN."""
    ts = _scores()
    tokens = torch.tensor([3, vocab, -1, -100, -7, vocab + 5]).cuda()
    up = torch.tensor([0.5, 0.0, 0.0, 0.0, 0.0, 1.0]).cuda()
    eup = torch.tensor([0.0, 0.0, 0.0, 0.0, 2.0, 0.0]).cuda()
    safe = tokens.clamp(0, vocab - 1)

    def check(score, leaves, row_of):
        got = torch.autograd.grad(score(tokens), leaves, [up, eup])
        want = torch.autograd.grad(score(safe), leaves, [up * (tokens == safe), eup])
        rows_got, rows_want = got[row_of], want[row_of]
        assert bool(torch.isnan(rows_got[5]).all())
        assert not bool(torch.isnan(rows_got[:5]).any())
        assert not bool(rows_got[1:4].any()) and bool(rows_got[4].any())
        assert torch.equal(rows_got[:5], rows_want[:5])
        return got, want

    x = _logits(rows, vocab, F32, 3).cuda().requires_grad_(True)
    check(lambda t: ts.token_scores(x, t)[:2], [x], 0)
    hidden = _logits(rows, 24, BF16, 4, std=1.0).cuda().requires_grad_(True)
    weight = _logits(vocab, 24, BF16, 5, std=0.5).cuda().requires_grad_(True)
    check(lambda t: ts.linear_token_scores(hidden, weight, t), [hidden, weight], 0)
    # Without the row that has none, the head weight's gradient is whole.
    up[5] = 0.0
    got = torch.autograd.grad(ts.linear_token_scores(hidden, weight, tokens), [weight], [up, eup])
    want = torch.autograd.grad(ts.linear_token_scores(hidden, weight, safe), [weight],
                               [up * (tokens == safe), eup])
    assert not bool(torch.isnan(got[0]).any()) and torch.equal(got[0], want[0])


@pytest.mark.parametrize("temperature", [1e-38, 4.5e-39])
def test_smallest_temperatures(temperature):
    """All probability on the largest logits, in a row of equal ones on each alike."""
    ts = _scores()
    x = torch.tensor([[1.0, 2.0, 2.0, -1.0], [5.0, 5.0, 5.0, 5.0]]).cuda()
    got = ts.token_scores(x, torch.tensor([1, 0]).cuda(), 2, temperature)
    want = torch.tensor([2.0, 4.0]).log()
    assert torch.allclose(got.logprob.cpu(), -want, rtol=2.0 ** -20) and torch.allclose(got.entropy.cpu(), want, rtol=2.0 ** -20)
    assert got.top_ids.tolist() == [[1, 2], [0, 1]]


def test_largest_temperature():
    """Every finite logit counts alike."""
    ts = _scores()
    x = _logits(3, 300, F32, 1)
    x[1, ::3] = -float("inf")
    got = ts.token_scores(x.cuda(), torch.tensor([0, 1, 2]).cuda(), 2, 8.5e37)
    want = torch.tensor([300.0, 200.0, 300.0]).log()
    assert torch.allclose(got.logprob.cpu(), -want, rtol=2.0 ** -20) and torch.allclose(got.entropy.cpu(), want, rtol=2.0 ** -20)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("temperature", [4e-39, 3.0e-39, 8.6e37, 1e45, 1e300])
def test_temperatures_beyond_fp32_are_refused(temperature, native, monkeypatch):
    """log2 e over such a temperature overflows, or its inverse is no normal number."""
    from ops import _hip

    ts = _scores()
    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    x, tokens = torch.zeros((2, 16), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="temperature"):
        ts.token_scores(x, tokens, 0, temperature)
    with pytest.raises(ValueError, match="temperature"):
        ts.linear_token_scores(x, torch.zeros((4, 16), device="cuda"), tokens, temperature)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_rows_than_one_launch_takes(dtype):
    """2^24 workgroups of 256 threads are 2^32 threads, which no launch has: the rows beyond are
    scored, and their gradients written, as on their own."""
    ts = _scores()
    rows, vocab = 2 ** 24 + 3000, 3
    x = torch.empty((rows, vocab), dtype=dtype, device="cuda").normal_().requires_grad_(True)
    tokens = torch.arange(rows, device="cuda") % vocab
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    got = ts.token_scores(x, tokens, 2)
    dx, = torch.autograd.grad([got.logprob, got.entropy], [x], [g, h])
    for part in (slice(0, 5000), slice(2 ** 24 - 1500, 2 ** 24 + 1500), slice(rows - 2000, rows)):
        own = x.detach()[part].clone().requires_grad_(True)
        alone = ts.token_scores(own, tokens[part], 2)
        want, = torch.autograd.grad([alone.logprob, alone.entropy], [own], [g[part], h[part]])
        for a, b in zip(got, alone):
            assert torch.equal(a[part], b)
        assert torch.equal(dx[part], want) and bool(want.any())


def test_chunks_past_32_bits_are_refused_before_the_forward():
    """With gradients; without them, chunk_rows is not used."""
    ts = _scores()
    rows, vocab = 70000, 32768
    hidden = torch.ones((rows, 8), device="cuda", dtype=BF16)
    weight = torch.zeros((vocab, 8), device="cuda", dtype=BF16)
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="chunk_rows times the vocabulary"):
        ts.linear_token_scores(hidden.requires_grad_(True), weight, tokens, 1.0, rows)
    logprob, _ = ts.linear_token_scores(hidden.detach(), weight, tokens, 1.0, rows)
    assert torch.allclose(logprob, torch.full_like(logprob, -15 * 0.6931472))
    logprob, _ = ts.linear_token_scores(hidden, weight, tokens, 1.0, 65000)
    dh, = torch.autograd.grad(logprob.sum(), [hidden])
    assert not bool(dh.any())
