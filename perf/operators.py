"""Performance cases of the 8-bit products and of the token scores, with their plain forms.

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges. A case is a
dict with a ``kind`` and its sizes:

* ``quantize``: a BF16 activation to e4m3 in blocks of 128 along its rows and, from the same
  read, along its columns (what a training step keeps of it), or (``weight``) an FP32 master
  weight in blocks of 128 x 128 with its transpose.
* ``mm``: the product of two e4m3 matrices with a scale per block of 128, from operands that
  are there already: the second in blocks of 128 x 128 (a projection or its input gradient)
  or, with ``by_rows``, of 1 x 128 as the first (a weight gradient).
* ``linear``: a projection as inference runs it: BF16 rows quantized, then the product with
  the weight that was quantized when the model was loaded.
* ``train``: a projection's training step, its operands and the gradient quantized in it: Y
  and dX in 8 bits, and dW: of a BF16 weight in 8 bits too, of an FP32 master (``master``) as
  the FP32 sums of the BF16 operands' products.
* ``logits``: log probability of a given token, entropy and the ``top_k`` likeliest tokens of
  each row of logits; with ``grad`` also the gradient of the logits.
* ``head``: log probability and entropy from the hidden state and the head weight; with
  ``grad`` also the gradients of both.

Model widths run from 512 to 2048 (the default configuration's 1280, the layer benchmark's
2048), projections up to 11264 wide (the layer benchmark's packed up/gate projection), tokens
per call from one (a decoding step) to 16384 (the layer benchmark), vocabularies up to 32768.
"""

from __future__ import annotations

import os
import sys

import torch

_package = os.path.abspath("warpstate-ai_amd")
if _package not in sys.path:
    sys.path.insert(0, _package)

#: False: ``run`` computes the plain form. True: it calls the framework.
own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 128
E4M3_MAX = 448.0
IGNORED = -100


def listed():
    return [
        # Quantization of an FFN activation of the benchmarked layer, both directions at once.
        {"name": "quantize_16384x5632", "kind": "quantize", "rows": 16384, "k": 5632,
         "weight": False, "scales": "e8m0"},
        # The default configuration's packed up/gate master weight, once per optimizer step.
        {"name": "quantize_weight_8960x1280", "kind": "quantize", "rows": 8960, "k": 1280,
         "weight": True, "scales": "float32"},
        # The reference's measured input projection on 8-bit operands.
        {"name": "mm_8192x10240x2048", "kind": "mm", "rows": 8192, "n": 10240, "k": 2048,
         "scales": "e8m0", "by_rows": False},
        # The same kind of product under FP32 scales, as published 8-bit checkpoints hold
        # them, on a ragged last batch at the default width.
        {"name": "mm_f32_scales_1999x8960x1280", "kind": "mm", "rows": 1999, "n": 8960,
         "k": 1280, "scales": "float32", "by_rows": False},
        # One token through the down projection of the benchmarked layer: a decoding step.
        {"name": "linear_1x2048x5632", "kind": "linear", "rows": 1, "n": 2048, "k": 5632,
         "scales": "e8m0"},
        # A batch of 48 decoding sequences through the up/gate projection.
        {"name": "linear_48x11264x2048", "kind": "linear", "rows": 48, "n": 11264, "k": 2048,
         "scales": "e8m0"},
        # The benchmarked layer's up/gate projection, forward and backward.
        {"name": "train_16384x11264x2048", "kind": "train", "rows": 16384, "n": 11264,
         "k": 2048, "scales": "e8m0", "master": False},
        # One decoding step's logits with the likeliest eight tokens: the smallest call.
        {"name": "logits_1x32768_top8", "kind": "logits", "rows": 1, "vocab": 32768,
         "dtype": "bf16", "top_k": 8, "temperature": 1.0, "masked": False, "grad": False},
        # Scores of a scored prompt batch under a vocabulary mask, at a sampling temperature.
        {"name": "logits_4096x32768_top20", "kind": "logits", "rows": 4096, "vocab": 32768,
         "dtype": "bf16", "top_k": 20, "temperature": 0.7, "masked": True, "grad": False},
        # FP32 logits of a ragged vocabulary, with the gradient of a policy loss.
        {"name": "logits_1000x10883_grad", "kind": "logits", "rows": 1000, "vocab": 10883,
         "dtype": "float32", "top_k": 0, "temperature": 1.0, "masked": False, "grad": True},
        # A reference model's scores of 8 sequences of 1000 tokens: no gradient.
        {"name": "head_8000", "kind": "head", "rows": 8000, "d": 1280, "vocab": 32768,
         "temperature": 1.0, "grad": False},
        # The policy's scores of the benchmarked batch, with gradients: the largest call.
        {"name": "head_16384_grad", "kind": "head", "rows": 16384, "d": 2048, "vocab": 32768,
         "temperature": 1.0, "grad": True},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _width(rng, low, high):
    """A feature width: a multiple of 64, now and then of 8 only, now and then any."""
    kind = rng.random()
    step = 1 if kind < 0.12 else 8 if kind < 0.3 else 64
    return max(low, _log(rng, low, high) // step * step)


def draw(rng):
    kind = rng.choice(["quantize", "mm", "mm", "linear", "linear", "train", "logits", "logits",
                       "logits", "head", "head"])
    case = {"kind": kind}
    if kind == "logits":
        case.update(rows=_log(rng, 1, 4096), vocab=_log(rng, 1000, 32768),
                    dtype=rng.choice(["bf16", "float32"]), top_k=rng.choice([0, 1, 5, 8, 20, 64]),
                    temperature=rng.choice([1.0, 0.7, 1.3]), masked=rng.random() < 0.4,
                    grad=rng.random() < 0.4)
        return case
    if kind == "head":
        vocab = _log(rng, 4096, 32768)
        case.update(rows=_log(rng, 1, 16384), d=_width(rng, 512, 2048) // 8 * 8,
                    vocab=vocab // 128 * 128 if rng.random() < 0.6 else vocab,
                    temperature=rng.choice([1.0, 1.0, 0.8]), grad=rng.random() < 0.5)
        return case
    case["scales"] = rng.choice(["e8m0", "e8m0", "float32"])
    case["k"] = _width(rng, 512, 2048)
    if kind == "quantize":
        case["weight"] = rng.random() < 0.4
        case["rows"] = _log(rng, 512, 11264) if case["weight"] else _log(rng, 128, 16384)
        return case
    case["n"] = _width(rng, 512, 11264)
    case["rows"] = _log(rng, 1, 128) if kind == "linear" else _log(rng, 128, 16384)
    if kind == "mm":
        case["by_rows"] = rng.random() < 0.33
        if rng.random() < 0.4:
            case["rows"] = _log(rng, 1, 128)
    elif kind == "train":
        case["master"] = rng.random() < 0.4
    return case


# --- inputs --------------------------------------------------------------------------------

class _Draw:
    """Normal draws on the GPU from one seeded generator, FP32 rounded to the wanted type."""

    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)

    def __call__(self, *shape, std=1.0, dtype=BF16):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=F32)
        return t.mul_(std).to(dtype)


def _inputs(case, seed):
    """Unit-variance activations with a few features ten times as large (what makes a scale
    per block of 128 worth having), N(0, 0.02) weights, gradients of 1e-2; logits of a trained
    model's spread; tokens with some rows ignored."""
    kind, draws = case["kind"], _Draw(seed)
    if kind in ("logits", "head"):
        rows, vocab = case["rows"], case["vocab"]
        tokens = torch.randint(0, vocab, (rows,), generator=draws.gen, device="cuda")
        ignored = torch.rand((rows,), generator=draws.gen, device="cuda") < 0.05
        t = {"tokens": tokens.masked_fill_(ignored, IGNORED)}
        if kind == "logits":
            logits = draws(rows, vocab, std=2.5, dtype=F32)
            if case["masked"]:
                banned = torch.rand((rows, vocab), generator=draws.gen, device="cuda") < 0.3
                logits.masked_fill_(banned, -float("inf"))
                # A grammar allows the tokens that it goes on to score.
                index = tokens.clamp_min(0)[:, None]
                logits.scatter_(1, index, draws(rows, 1, std=2.5, dtype=F32))
            t["logits"] = logits.to(BF16 if case["dtype"] == "bf16" else F32)
        else:
            d = case["d"]
            t["hidden"] = draws(rows, d)
            t["weight"] = draws(vocab, d, std=0.04)
        if case["grad"]:
            t["dlogprob"] = draws(rows, std=1.0 / rows, dtype=F32)
            t["dentropy"] = draws(rows, std=0.01 / rows, dtype=F32)
        return t
    rows, k = case["rows"], case["k"]
    if kind == "quantize" and case["weight"]:
        return {"x": draws(rows, k, std=0.02, dtype=F32)}
    loud = torch.rand((k,), generator=draws.gen, device="cuda") < 0.005
    x = draws(rows, k, dtype=F32).mul_(torch.where(loud, 10.0, 1.0)).to(BF16)
    if kind == "quantize":
        return {"x": x}
    bf16 = kind == "train" and not case["master"] or kind == "mm" and case["by_rows"]
    t = {"x": x, "weight": draws(case["n"], k, std=0.02, dtype=BF16 if bf16 else F32)}
    if kind == "train":
        t["grad"] = draws(rows, case["n"], std=1e-2)
    return t


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    kind = case["kind"]
    if kind == "mm":
        state["a"], state["a_scale"] = _quantize(state.pop("x"), case["scales"], 1)
        state["b"], state["b_scale"] = _quantize(state.pop("weight"), case["scales"],
                                                 1 if case["by_rows"] else BLOCK)
    elif kind == "linear":
        state["b"], state["b_scale"] = _quantize(state.pop("weight"), case["scales"], BLOCK)
    elif kind == "train":
        state["x"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    elif kind in ("logits", "head") and case["grad"]:
        for name in ("logits",) if kind == "logits" else ("hidden", "weight"):
            state[name].requires_grad_(True)
    return state


# --- plain forms ---------------------------------------------------------------------------

def _blocks(x, rows_per_block):
    """x [M, K] zero-padded to whole blocks, as [M blocks, rows, K blocks, 128]."""
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -m % rows_per_block))
    return x.view(-1, rows_per_block, x.shape[1] // BLOCK, BLOCK)


def _quantize(x, scales, rows_per_block):
    """(e4m3 x / scale, scale) with one scale per rows_per_block x 128 block: the smallest
    power of two that brings the block's largest magnitude to at most 448, or that magnitude
    over 448 in FP32."""
    m, k = x.shape
    wide = _blocks(x.detach().float(), rows_per_block)
    amax = wide.abs().amax((1, 3))
    if scales == "e8m0":
        mantissa, exponent = torch.frexp(amax)
        code = (exponent - 9 + (mantissa > 0.875) + 127).clamp_(1, 254)
        scale = code.to(torch.uint8).view(E8M0)
        inverse = ((254 - code) << 23).to(torch.int32).view(F32)
    else:
        amax = amax.clamp_min(2.0 ** -100)
        scale, inverse = amax / E4M3_MAX, E4M3_MAX / amax
    q = (wide * inverse[:, None, :, None]).view(-1, wide.shape[2] * BLOCK)[:m, :k].to(E4M3)
    return q, scale


def _power(scale):
    """FP32 value of e8m0 scales (or FP32 scales themselves)."""
    if scale.dtype == F32:
        return scale
    return (scale.view(torch.uint8).to(torch.int32) << 23).view(F32)


def _dequantize(q, scale):
    m, k = q.shape
    rows_per_block = 1 if scale.shape[0] == m else BLOCK
    wide = _blocks(q.float(), rows_per_block)
    wide = wide * _power(scale)[:, None, :, None]
    return wide.view(-1, wide.shape[2] * BLOCK)[:m, :k]


def _plain_scores(logits, tokens, temperature):
    """(logprob, entropy, logits - lse, softmax) of FP32 logits."""
    scaled = logits * (1.0 / temperature)
    top = scaled.amax(-1, keepdim=True)
    lse = top + (scaled - top).exp_().sum(-1, keepdim=True).log_()
    logp = scaled.sub_(lse)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    valid = tokens != IGNORED
    logprob = torch.where(valid, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    return logprob, entropy, logp, p


def _plain_dlogits(tokens, temperature, entropy, logp, p, dlogprob, dentropy):
    """Gradient of sum(dlogprob logprob + dentropy entropy) with respect to the logits."""
    g = torch.where(tokens != IGNORED, dlogprob, 0.0)[:, None]
    inner = torch.where(p > 0, p * (g + dentropy[:, None] * (logp + entropy[:, None])), 0.0)
    grad = inner.neg_()
    grad.scatter_add_(1, tokens.clamp_min(0)[:, None], g)
    return grad.mul_(1.0 / temperature)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        x = state["x"]
        if case["weight"]:
            q, scale = _quantize(x, case["scales"], BLOCK)
            return {"q": q, "scale": scale, "qt": q.T.contiguous(),
                    "scale_t": scale.T.contiguous()}
        q, scale = _quantize(x, case["scales"], 1)
        qt, scale_t = _quantize(x.T, case["scales"], 1)
        return {"q": q, "scale": scale, "qt": qt, "scale_t": scale_t}
    if kind == "mm":
        a, b = _dequantize(state["a"], state["a_scale"]), _dequantize(state["b"], state["b_scale"])
        return {"out": (a @ b.T).to(BF16)}
    if kind == "linear":
        a = _dequantize(*_quantize(state["x"], case["scales"], 1))
        return {"y": (a @ _dequantize(state["b"], state["b_scale"]).T).to(BF16)}
    if kind == "train":
        x, weight, grad = state["x"].detach(), state["weight"].detach(), state["grad"]
        scales = case["scales"]
        w = _dequantize(*_quantize(weight, scales, BLOCK))
        y = (_dequantize(*_quantize(x, scales, 1)) @ w.T).to(BF16)
        dx = (_dequantize(*_quantize(grad, scales, 1)) @ w).to(BF16)
        if case["master"]:
            dweight = grad.float().T @ x.float()
        else:
            dweight = (_dequantize(*_quantize(grad.T, scales, 1))
                       @ _dequantize(*_quantize(x.T, scales, 1)).T).to(BF16)
        return {"y": y, "dx": dx, "dweight": dweight}
    tokens, temperature = state["tokens"], case["temperature"]
    if kind == "logits":
        logits = state["logits"].detach()
        logprob, entropy, logp, p = _plain_scores(logits.float(), tokens, temperature)
        out = {"logprob": logprob, "entropy": entropy}
        if case["top_k"]:
            # A stable sort: equal logits in the order of their ids.
            ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :case["top_k"]]
            ids = ids.contiguous()
            out.update(top_logprobs=logp.gather(1, ids), top_ids=ids)
        if case["grad"]:
            out["dlogits"] = _plain_dlogits(tokens, temperature, entropy, logp, p,
                                            state["dlogprob"], state["dentropy"]).to(logits.dtype)
        return out
    hidden, weight = state["hidden"].detach().float(), state["weight"].detach().float()
    logprob, entropy, logp, p = _plain_scores(hidden @ weight.T, tokens, temperature)
    out = {"logprob": logprob, "entropy": entropy}
    if case["grad"]:
        dlogits = _plain_dlogits(tokens, temperature, entropy, logp, p, state["dlogprob"],
                                 state["dentropy"])
        out.update(dhidden=(dlogits @ weight).to(BF16), dweight=(dlogits.T @ hidden).to(BF16))
    return out


# --- the framework's calls -----------------------------------------------------------------

def _own(state):
    case = state["case"]
    kind = case["kind"]
    if kind in ("quantize", "mm", "linear", "train"):
        from ops import fp8_execution as fp8

        scale_dtype = E8M0 if case["scales"] == "e8m0" else F32
        if kind == "quantize":
            if case["weight"]:
                q, scale, qt, scale_t = fp8.quantize_weight(state["x"], scale_dtype)
            else:
                q, scale, qt, scale_t = fp8.quantize_rows_and_columns(state["x"], scale_dtype)
            return {"q": q, "scale": scale, "qt": qt, "scale_t": scale_t}
        if kind == "mm":
            return {"out": fp8.fp8_mm(state["a"], state["a_scale"], state["b"], state["b_scale"])}
        if kind == "linear":
            q, scale = fp8.quantize_rows(state["x"], scale_dtype)
            return {"y": fp8.fp8_mm(q, scale, state["b"], state["b_scale"])}
        y = fp8.fp8_linear(state["x"], state["weight"], scale_dtype)
        dx, dweight = torch.autograd.grad(y, [state["x"], state["weight"]], state["grad"])
        return {"y": y, "dx": dx, "dweight": dweight}
    from ops import token_scores as scores

    if kind == "logits":
        leaves = [state["logits"]]
        got = scores.token_scores(state["logits"], state["tokens"], case["top_k"],
                                  case["temperature"])
        out = {"logprob": got.logprob, "entropy": got.entropy}
        if case["top_k"]:
            out.update(top_logprobs=got.top_logprobs, top_ids=got.top_ids)
        names = ("dlogits",)
    else:
        leaves = [state["hidden"], state["weight"]]
        logprob, entropy = scores.linear_token_scores(state["hidden"], state["weight"],
                                                      state["tokens"], case["temperature"])
        out = {"logprob": logprob, "entropy": entropy}
        names = ("dhidden", "dweight")
    if case["grad"]:
        grads = torch.autograd.grad([out["logprob"], out["entropy"]], leaves,
                                    [state["dlogprob"], state["dentropy"]])
        out.update(zip(names, grads))
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read and each output written once; the products' multiplications."""
    kind = case["kind"]
    if kind in ("logits", "head"):
        rows, vocab, grad = case["rows"], case["vocab"], case["grad"]
        row_bytes = 8 + 8 + (8 if grad else 0)
        if kind == "logits":
            size = 2 if case["dtype"] == "bf16" else 4
            return {"bytes": rows * (vocab * size * (2 if grad else 1) + row_bytes
                                     + 12 * case["top_k"]), "flops": 0}
        d = case["d"]
        copies = 2 if grad else 1
        return {"bytes": 2 * (rows + vocab) * d * copies + rows * row_bytes,
                "flops": 2 * rows * vocab * d * (3 if grad else 1)}
    rows, k = case["rows"], case["k"]
    scale = 1 if case["scales"] == "e8m0" else 4
    if kind == "quantize":
        blocks = (rows / BLOCK * k / BLOCK if case["weight"] else rows * k / BLOCK)
        return {"bytes": rows * k * ((4 if case["weight"] else 2) + 2) + 2 * scale * blocks,
                "flops": 0}
    n = case["n"]
    if kind == "train":
        return {"bytes": 2 * (2 * rows * k + 2 * rows * n) + (8 if case["master"] else 4) * n * k,
                "flops": 6 * rows * n * k}
    a = 2 if kind == "linear" else 1
    return {"bytes": rows * k * a + n * k + 2 * rows * n, "flops": 2 * rows * n * k}


# --- the same values in 64 bits -------------------------------------------------------------

def _exact_e4m3(x):
    """The e4m3 value nearest to x (ties to the even one), |x| <= 448: steps of an eighth of
    the value's power of two, of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_quantized(x, scales, rows_per_block):
    """(e4m3 values, scale, their product) of x in 64 bits."""
    x = x.to(F64)
    m, k = x.shape
    mb, kb = -(-m // rows_per_block), -(-k // BLOCK)
    padded = torch.zeros((mb * rows_per_block, kb * BLOCK), dtype=F64, device=x.device)
    padded[:m, :k] = x
    tiles = padded.reshape(mb, rows_per_block, kb, BLOCK)
    largest = tiles.abs().amax(3).amax(1).clamp_min(2.0 ** -100)
    scale = largest / E4M3_MAX
    if scales == "e8m0":
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    wide = scale[:, None, :, None]
    q = _exact_e4m3(tiles / wide)
    crop = lambda t: t.reshape(mb * rows_per_block, kb * BLOCK)[:m, :k]  # noqa: E731
    return crop(q), scale, crop(q * wide)


def _exact_scores(logits, case, t):
    tokens, temperature = t["tokens"], case["temperature"]
    logp = torch.log_softmax(logits / temperature, -1)
    p = logp.exp()
    surprise = torch.where(p > 0, logp, torch.zeros_like(logp))
    entropy = -(p * surprise).sum(-1)
    valid = tokens != IGNORED
    index = tokens.clamp_min(0)[:, None]
    out = {"logprob": logp.gather(1, index)[:, 0] * valid, "entropy": entropy}
    if not case["grad"]:
        return out, logp, None
    g = t["dlogprob"].to(F64) * valid
    grad = torch.zeros_like(p).scatter_(1, index, g[:, None]) - g[:, None] * p
    grad -= t["dentropy"].to(F64)[:, None] * p * (surprise + entropy[:, None])
    return out, logp, grad / temperature


def exact(case, seed):
    """The outputs of ``run`` in 64-bit arithmetic from the same inputs."""
    kind = case["kind"]
    t = _inputs(case, seed)
    if kind == "logits":
        logits = t["logits"].to(F64)
        out, logp, grad = _exact_scores(logits, case, t)
        if case["top_k"]:
            out.update(top_logprobs=torch.topk(logp, case["top_k"], dim=-1)[0], top_ids=None)
        if case["grad"]:
            out["dlogits"] = grad
        return out
    if kind == "head":
        hidden, weight = t["hidden"].to(F64), t["weight"].to(F64)
        out, _logp, grad = _exact_scores(hidden @ weight.T, case, t)
        if case["grad"]:
            out.update(dhidden=grad @ weight, dweight=grad.T @ hidden)
        return out
    scales, x = case["scales"], t["x"]
    if kind == "quantize":
        if case["weight"]:
            q, scale, _value = _exact_quantized(x, scales, BLOCK)
            return {"q": q, "scale": scale, "qt": q.T.contiguous(),
                    "scale_t": scale.T.contiguous()}
        q, scale, _value = _exact_quantized(x, scales, 1)
        qt, scale_t, _value = _exact_quantized(x.T, scales, 1)
        return {"q": q, "scale": scale, "qt": qt, "scale_t": scale_t}
    if kind == "mm":
        rows_of_b = 1 if case["by_rows"] else BLOCK
        return {"out": _exact_quantized(x, scales, 1)[2]
                @ _exact_quantized(t["weight"], scales, rows_of_b)[2].T}
    w = _exact_quantized(t["weight"], scales, BLOCK)[2]
    y = _exact_quantized(x, scales, 1)[2] @ w.T
    if kind == "linear":
        return {"y": y}
    grad = t["grad"]
    dx = _exact_quantized(grad, scales, 1)[2] @ w
    if case["master"]:
        return {"y": y, "dx": dx, "dweight": grad.to(F64).T @ x.to(F64)}
    return {"y": y, "dx": dx, "dweight": _exact_quantized(grad.T, scales, 1)[2]
            @ _exact_quantized(x.T, scales, 1)[2].T}
