"""What the residual norm and the embedding refuse, in Python and at the C entry points (CPU)."""
import pytest
import torch

from ops import _hip

BF16, F32 = torch.bfloat16, torch.float32
GPU = 1 << 20  # a pointer that is never read: every call below fails its checks first


def test_cpu_tensors_are_refused():
    from ops.embedding_execution import embedding, embedding_accumulate_
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    x, w = torch.zeros((2, 8), dtype=BF16), torch.ones(8)
    t = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: add_rmsnorm(x, x, w), lambda: rmsnorm_quantize(x, w),
                 lambda: embedding(t, x), lambda: embedding_accumulate_(x.float(), t, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("change,match", [
    (dict(rows=-1), "shape"), (dict(d=0), "shape"), (dict(d=8193), "8192"), (dict(x=None), "null"),
    (dict(residual=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(out=None), "null"), (dict(ldx=7), "overlap"),
    (dict(ldr=7), "overlap"), (dict(rows=2 ** 30 + 1), "shape")])
def test_add_rmsnorm_arguments(change, match):
    a = dict(x=GPU, ldx=8, residual=GPU, ldr=8, w=GPU, rows=4, d=8, y=GPU, out=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_add_rmsnorm", a["x"], a["ldx"], a["residual"], a["ldr"], 0, a["w"], 1e-5, a["rows"],
                  a["d"], a["y"], a["out"], None)


@pytest.mark.parametrize("change,match", [
    (dict(d=8193), "8192"), (dict(scale_type=2), "scale type"), (dict(q=None), "null"),
    (dict(out=None), "null"), (dict(residual=None), "null"), (dict(ldq=24), "16-byte"),
    (dict(q=GPU + 8), "16-byte"), (dict(ldq=0), "16-byte"), (dict(ld_scale=1, d=129, ldx=130, ldr=130, ldq=144),
                                                             "overlap"),
    (dict(scale_type=1, ld_scale=3), "overlap")])
def test_rmsnorm_quantize_arguments(change, match):
    a = dict(x=GPU, ldx=8, residual=GPU, ldr=8, w=GPU, rows=4, d=8, scale_type=0, q=GPU, ldq=16,
             scale=GPU, ld_scale=4, out=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_rmsnorm_quantize", a["x"], a["ldx"], a["residual"], a["ldr"], 0, a["w"], 1e-5,
                  a["rows"], a["d"], a["scale_type"], a["q"], a["ldq"], a["scale"], a["ld_scale"],
                  a["out"], None)


@pytest.mark.parametrize("change,match", [
    (dict(rows=0), "shape"), (dict(d=8193), "8192"), (dict(s=None), "null"), (dict(dy=None), "null"),
    (dict(partial=None, rows=40), "null"), (dict(dresidual=GPU), "BF16 stream"), (dict(ld_dy=7), "overlap"),
    (dict(ds=GPU, ld_ds=7), "overlap")])
def test_add_rmsnorm_backward_arguments(change, match):
    a = dict(s=GPU, w=GPU, dy=GPU, ld_dy=8, ds=None, ld_ds=0, rows=4, d=8, dx=GPU,
             dresidual=None, dw=GPU, partial=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_add_rmsnorm_backward", a["s"], 0, a["w"], 1e-5, a["dy"], a["ld_dy"], a["ds"],
                  a["ld_ds"], a["rows"], a["d"], a["dx"], a["dresidual"], a["dw"], a["partial"], None)


def test_partial_floats_of_bad_sizes():
    assert _hip.query("ws_grouped_workspace_floats", 0, 2, 16, 2048, 0) == 0
    assert _hip.query("ws_grouped_workspace_floats", 100, 2, 16, 2048, 2) == 0
    assert _hip.query("ws_grouped_workspace_floats", 100, 2, 13, 2048, 0) % (100 * 16) == 0
    assert _hip.query("ws_grouped_workspace_floats", 100, 2, 13, 2048, 0) > 0
    assert _hip.query("ws_add_rmsnorm_backward_partial_floats", 0, 8) == 0
    assert _hip.query("ws_add_rmsnorm_backward_partial_floats", 4, 8193) == 0
    assert _hip.query("ws_embedding_backward_workspace_bytes", -1, 8, 8) == 0
    assert _hip.query("ws_embedding_backward_workspace_bytes", 8, 2 ** 22 + 1, 8) == 0


@pytest.mark.parametrize("change,match", [
    (dict(rows=-1), "shape"), (dict(vocab=0), "shape"), (dict(d=0), "shape"), (dict(table=None), "null"),
    (dict(tokens=None), "null"), (dict(y=None), "null"), (dict(ld=7), "overlap"),
    (dict(rows=2 ** 24 + 1), "shape"), (dict(vocab=2 ** 22 + 1), "shape"),
    (dict(d=2 ** 20 + 1, ld=2 ** 20 + 1), "shape")])
def test_embedding_arguments(change, match):
    a = dict(table=GPU, ld=8, tokens=GPU, rows=4, vocab=10, d=8, y=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_embedding", a["table"], a["ld"], 0, a["tokens"], a["rows"], a["vocab"], a["d"], 1.0,
                  a["y"], 0, None)


@pytest.mark.parametrize("change,match", [
    (dict(rows=-1), "shape"), (dict(vocab=0), "shape"), (dict(mode=3), "mode"), (dict(mode=-1), "mode"),
    (dict(dy=None), "null"), (dict(tokens=None), "null"), (dict(out=None), "null"),
    (dict(work=None, rows=65), "null"), (dict(work=GPU + 4), "aligned"), (dict(ld_dy=7), "overlap"),
    (dict(ld=7), "overlap"), (dict(d=2 ** 20 + 1, ld=2 ** 20 + 1, ld_dy=2 ** 20 + 1), "shape")])
def test_embedding_backward_arguments(change, match):
    a = dict(dy=GPU, ld_dy=8, tokens=GPU, rows=4, vocab=10, d=8, out=GPU, ld=8, mode=0, work=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_embedding_backward", a["dy"], a["ld_dy"], 0, a["tokens"], a["rows"], a["vocab"],
                  a["d"], 1.0, a["out"], a["ld"], a["mode"], a["work"], None)


@pytest.mark.parametrize("change,match", [
    (dict(form=2), "form"), (dict(groups=0), "groups"), (dict(groups=16385), "groups"), (dict(rows=-1), "shape"),
    (dict(form=1, n=12), "multiple of 8"), (dict(k=12), "multiple of 8"), (dict(n=0), "shape"), (dict(x=None), "null"),
    (dict(n=17), "overlap"), (dict(form=1, k=17), "overlap"), (dict(w=None), "null"), (dict(offsets=None), "null"), (dict(y=None), "null"), (dict(x=GPU + 8), "aligned"),
    (dict(ldx=20), "aligned"), (dict(ldx=8), "overlap"), (dict(ldw=8), "overlap"), (dict(ldy=8), "overlap"),
    (dict(stride=12), "aligned"), (dict(stride=-8), "aligned"), (dict(ldy=4200000), "stride"),
    (dict(rows=2 ** 30, n=2 ** 20, ldy=2 ** 20), "tiles"), (dict(rows=2 ** 30 + 1), "shape"),
    (dict(rows=4, ldx=8), "overlap"), (dict(rows=4, ldw=8), "overlap"), (dict(rows=4, x=GPU + 1), "aligned"),
    (dict(rows=4, w=GPU + 1), "aligned"), (dict(rows=4, stride=-8), "aligned"),
    (dict(work=GPU + 4), "aligned"), (dict(rows=100, k=2048, ldx=2048, ldw=2048), "null")])
def test_grouped_mm_arguments(change, match):
    a = dict(x=GPU, ldx=16, w=GPU, ldw=16, stride=256, form=0, offsets=GPU, groups=2, rows=40, n=16, k=16, y=GPU,
             ldy=16, work=None) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_grouped_mm", a["x"], a["ldx"], a["w"], a["ldw"], a["stride"], a["form"], a["offsets"],
                  a["groups"], a["rows"], a["n"], a["k"], a["y"], a["ldy"], a["work"], None)


@pytest.mark.parametrize("change,match", [
    (dict(groups=0), "groups"), (dict(rows=-1), "shape"), (dict(k=12), "multiple of 8"), (dict(dy=None), "null"),
    (dict(n=17), "overlap"),
    (dict(x=None), "null"), (dict(offsets=None), "null"), (dict(dw=None), "null"), (dict(dw=GPU + 8), "aligned"),
    (dict(dy=GPU + 2), "aligned"), (dict(ldx=8), "overlap"), (dict(k=2200000, ldx=2200000), "stride"),
    (dict(groups=16384, n=4096, k=4096, ld_dy=4096, ldx=4096), "tiles")])
def test_grouped_weight_grad_arguments(change, match):
    a = dict(dy=GPU, ld_dy=16, x=GPU, ldx=16, offsets=GPU, groups=2, rows=4, n=16, k=16, dw=GPU) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_grouped_weight_grad", a["dy"], a["ld_dy"], a["x"], a["ldx"], a["offsets"], a["groups"],
                  a["rows"], a["n"], a["k"], a["dw"], 1, None)


def test_grouped_tile_of_bad_sizes():
    assert _hip.query("ws_grouped_tile", 0, 1, 8, 8, 0) == -1
    assert _hip.query("ws_grouped_tile", 8, 0, 8, 8, 0) == -1
    assert _hip.query("ws_grouped_tile", 8, 1, 0, 8, 0) == -1
    assert _hip.query("ws_grouped_tile", 8, 1, 8, 8, 3) == -1


@pytest.mark.parametrize("change,match", [
    (dict(groups=-1), "sizes"), (dict(rows_in=-1), "sizes"), (dict(cols_out=2 ** 31), "sizes"),
    (dict(groups=2 ** 25), "sizes"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(ld_out=4), "overlap"),
    (dict(group_out=20), "overlap"), (dict(out_f32=1), "type")])
def test_copy_rows_arguments(change, match):
    a = dict(x=GPU, in_f32=0, group_in=40, ld_in=8, rows_in=5, cols_in=8, out=GPU, out_f32=0, group_out=30, ld_out=6,
             rows_out=5, cols_out=6, groups=2) | change
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_copy_rows", a["x"], a["in_f32"], a["group_in"], a["ld_in"], a["rows_in"], a["cols_in"], a["out"],
                  a["out_f32"], a["group_out"], a["ld_out"], a["rows_out"], a["cols_out"], a["groups"], None)
