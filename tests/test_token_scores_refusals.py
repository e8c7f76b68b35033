"""What the token-score entry points refuse, before any launch (CPU)."""
import pytest
import torch

from ops import _hip
from ops import token_scores as ts

P = 1 << 20  # never dereferenced: every call below fails validation first


def test_scores_need_the_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ts.token_scores(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ts.linear_token_scores(torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("inf"), float("nan"), 1e-39])
def test_temperature(temperature):
    with pytest.raises(ValueError, match="temperature"):
        ts._inverse(temperature)


def test_tokens():
    device = torch.device("cpu")
    assert ts._check_tokens(torch.zeros(3, dtype=torch.int64), 3, device).shape == (3,)
    for bad in (torch.zeros(3), torch.zeros(4, dtype=torch.int64), torch.zeros((3, 1), dtype=torch.int64)):
        with pytest.raises(ValueError, match="int64 vector"):
            ts._check_tokens(bad, 3, device)


def _forward(**over):
    a = dict(x=P, ld=100, f32=0, t=P, rows=2, vocab=100, inv=1.0, k=3, ws=None, lse=P, lp=P, en=P, tl=P, ti=P)
    a.update(over)
    _hip.call("ws_token_scores", *a.values(), None)


@pytest.mark.parametrize("over,match", [
    (dict(x=None), "null operand"), (dict(t=None), "null operand"), (dict(rows=0), "at least one row"),
    (dict(vocab=524289, ld=524289), "524288"), (dict(ld=99), "leading dimension"), (dict(f32=2), "type"),
    (dict(inv=0.0), "temperature"), (dict(inv=float("nan")), "temperature"), (dict(k=65), "top_k"),
    (dict(vocab=2, k=3), "top_k"), (dict(k=-1), "top_k"), (dict(lse=None), "null output"),
    (dict(ti=None), "null output"), (dict(vocab=9000, ld=9000), "workspace"),
    (dict(vocab=9000, ld=9000, ws=P + 8), "workspace"), (dict(rows=1 << 30, vocab=9000, ld=9000), "too many")])
def test_forward_arguments(over, match):
    with pytest.raises(RuntimeError, match=match):
        _forward(**over)


def test_backward_arguments():
    def call(lse=P, out=P, ld_out=100):
        _hip.call("ws_token_scores_backward", P, 100, 0, P, 2, 100, 1.0, lse, P, P, P, out, ld_out, None)

    for over, match in ((dict(lse=None), "null"), (dict(out=None), "null"), (dict(ld_out=99), "leading")):
        with pytest.raises(RuntimeError, match=match):
            call(**over)


def _head(**over):
    a = dict(h=P, ldh=64, w=P, ldw=64, t=P, rows=4, vocab=50, d=64, inv=1.0, ws=P, lse=P, lp=P, en=P)
    a.update(over)
    _hip.call("ws_linear_token_scores", *a.values(), None)


@pytest.mark.parametrize("over,match", [
    (dict(h=None), "null operand"), (dict(vocab=0), "invalid"), (dict(ldh=63), "leading"),
    (dict(d=60), "16-byte"), (dict(h=P + 2), "16-byte"), (dict(ldw=68), "16-byte"),
    (dict(inv=-1.0), "temperature"), (dict(ws=None), "null output")])
def test_head_arguments(over, match):
    with pytest.raises(RuntimeError, match=match):
        _head(**over)


def _head_backward(**over):
    a = dict(h=P, ldh=64, w=P, ldw=64, wt=None, t=P, lse=P, en=P, g=P, e=P, rows=4, vocab=50, d=64, inv=1.0,
             ws=P, chunk=4, dh=P, ldd=64, dw=P, lddw=64, bf=0)
    a.update(over)
    _hip.call("ws_linear_token_scores_backward", *a.values(), None)


@pytest.mark.parametrize("over,match", [
    (dict(ws=P + 16), "256-byte"), (dict(chunk=0), "chunk_rows"), (dict(dh=None, dw=None), "null"),
    (dict(ldd=63), "dhidden leading"), (dict(lddw=63), "dweight leading"), (dict(lse=None), "null"),
    (dict(ldd=4_200_000), "row stride"), (dict(bf=1, chunk=3), "one chunk"), (dict(bf=1, lddw=72), "one chunk"),
    (dict(rows=1 << 20, chunk=1 << 20, vocab=32768), "chunk_rows")])
def test_head_backward_arguments(over, match):
    with pytest.raises(RuntimeError, match=match):
        _head_backward(**over)


def test_workspace_queries():
    q = _hip.query
    assert q("ws_token_scores_workspace_bytes", 1000, 8192, 5) == 0  # a part per row
    assert q("ws_token_scores_workspace_bytes", 1000, 8193, 5) == 1000 * 2 * (16 + 40)
    assert q("ws_token_scores_workspace_bytes", 1, 32768, 8) == 16 * (16 + 64)  # parts of 2048
    assert q("ws_linear_token_scores_workspace_floats", 16384, 1000, 512) == 16384 * (3 * 8 + 1)  # parts of 128
    assert q("ws_linear_token_scores_workspace_floats", 10, 1000, 512) == 10 * (3 * 16 + 1)  # parts of 64
    # Coefficients, one chunk of logit gradients padded to whole 64-column pieces.
    assert q("ws_linear_token_scores_backward_workspace_bytes", 4096, 10883, 2048, 4096) >= \
        4096 * 16 + 4096 * 10944 * 2
