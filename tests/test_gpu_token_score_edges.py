"""Token scores at the edges of what their documentation allows: tokens without a score under
masked losses, the smallest temperatures (GPU)."""
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
