"""Performance cases of the residual norm, the embedding and the experts' products.

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges. A case is a
dict with a ``kind`` and its sizes:

* ``norm_quantize``: a projection's output added to the residual stream, the RMSNorm of the sum
  and its 8-bit form with a scale per block of 128: what a decoding step or a prompt hands to
  the next 8-bit projection.
* ``norm_train``: the same addition and norm with a BF16 result, and the gradients of both
  inputs and of the norm's weight. The residual stream is BF16 or FP32 (``stream``).
* ``lookup``: rows of an embedding table by token, scaled.
* ``embed_train``: the lookup and the table's gradient. Tokens follow Zipf's law, as text does.
* ``experts``: the products of rows sorted by expert with their expert's weight; the counts of
  rows are those of a router that prefers some experts. With ``train`` also the gradients of
  the rows and of the weights.

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
BLOCK, E4M3_MAX = 128, 448.0
EPS = 1e-5
IGNORED = -100


# --- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # One token between two projections of a decoding step: the smallest call.
        {"name": "norm_quantize_1x2048", "kind": "norm_quantize", "rows": 1, "d": 2048,
         "stream": "bf16", "scales": "e8m0"},
        # A prompt of one long sequence at the default width, scales as checkpoints hold them.
        {"name": "norm_quantize_5001x1280", "kind": "norm_quantize", "rows": 5001, "d": 1280,
         "stream": "float32", "scales": "float32"},
        # The benchmarked layer's batch, forward and backward.
        {"name": "norm_train_16384x2048", "kind": "norm_train", "rows": 16384, "d": 2048,
         "stream": "bf16"},
        # A ragged last batch on an FP32 residual stream at the default width.
        {"name": "norm_train_1999x1280_f32", "kind": "norm_train", "rows": 1999, "d": 1280,
         "stream": "float32"},
        # The tokens of 48 decoding sequences.
        {"name": "lookup_48x2048", "kind": "lookup", "rows": 48, "vocab": 32768, "d": 2048,
         "dtype": "bf16", "scale": 1.0},
        # The benchmarked batch against an FP32 master table, with its gradient.
        {"name": "embed_train_16384x2048", "kind": "embed_train", "rows": 16384, "vocab": 32768,
         "d": 2048, "dtype": "float32", "scale": 1.0},
        # A microbatch on a ragged vocabulary, BF16 table, rows scaled by the square root of d.
        {"name": "embed_train_2000x1280", "kind": "embed_train", "rows": 2000, "vocab": 10883,
         "d": 1280, "dtype": "bf16", "scale": 35.777},
        # A decoding step of 16 sequences with two experts each: few rows for each weight.
        {"name": "experts_32_of_8x5632x2048", "kind": "experts", "rows": 32, "experts": 8,
         "n": 5632, "k": 2048, "dtype": "bf16", "train": False},
        # A prompt over many experts, the down projection at the default width.
        {"name": "experts_6000_of_32x1280x896", "kind": "experts", "rows": 6000, "experts": 32,
         "n": 1280, "k": 896, "dtype": "bf16", "train": False},
        # Training of many small experts, some without rows.
        {"name": "experts_4096_of_64x512x1280_train", "kind": "experts", "rows": 4096,
         "experts": 64, "n": 512, "k": 1280, "dtype": "bf16", "train": True},
        # The benchmarked batch through eight experts of the benchmarked up/gate width, FP32
        # masters: the largest call.
        {"name": "experts_16384_of_8x11264x2048_train", "kind": "experts", "rows": 16384,
         "experts": 8, "n": 11264, "k": 2048, "dtype": "float32", "train": True},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _width(rng, low, high):
    """A feature width: a multiple of 64, now and then of 8 only, now and then any."""
    kind = rng.random()
    step = 1 if kind < 0.1 else 8 if kind < 0.25 else 64
    return max(low, _log(rng, low, high) // step * step)


def draw(rng):
    kind = rng.choice(["norm_quantize", "norm_train", "norm_train", "lookup", "embed_train",
                       "embed_train", "experts", "experts", "experts"])
    if kind.startswith("norm"):
        case = {"kind": kind, "rows": _log(rng, 1, 16384), "d": _width(rng, 512, 2048),
                "stream": rng.choice(["bf16", "bf16", "float32"])}
        if kind == "norm_quantize":
            case["scales"] = rng.choice(["e8m0", "e8m0", "float32"])
        return case
    if kind in ("lookup", "embed_train"):
        return {"kind": kind, "rows": _log(rng, 1, 16384), "vocab": _log(rng, 1000, 32768),
                "d": _width(rng, 512, 2048), "dtype": rng.choice(["bf16", "float32"]),
                "scale": rng.choice([1.0, 1.0, 0.125, 35.777])}
    train = rng.random() < 0.5
    k = _width(rng, 512, 2048)
    n = _width(rng, 512, 11264)
    most = max(1, 8 * 11264 * 2048 // (n * k))
    return {"kind": kind, "rows": _log(rng, 64 if train else 1, 16384),
            "experts": _log(rng, 2, min(64, max(2, most))), "n": n, "k": k,
            "dtype": rng.choice(["bf16", "float32"]) if train else "bf16", "train": train}


# --- inputs --------------------------------------------------------------------------------

class _Draw:
    """Normal draws on the GPU from one seeded generator, FP32 rounded to the wanted type."""

    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)

    def __call__(self, *shape, std=1.0, dtype=BF16):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=F32)
        return t.mul_(std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda", dtype=F32)


def _type(name):
    return BF16 if name == "bf16" else F32


def prepare(case, seed):
    """Unit-variance rows beside a residual stream that has grown to a few times that and holds
    a few loud features; N(0, 0.02) weights; gradients of 1e-2; a norm weight around 1."""
    kind, draws, rows = case["kind"], _Draw(seed), case["rows"]
    state = {"case": case}
    if kind.startswith("norm"):
        d, stream = case["d"], _type(case["stream"])
        loud = torch.where(draws.uniform(d) < 0.005, 20.0, 3.0)
        state["x"] = draws(rows, d)
        state["residual"] = draws(rows, d, dtype=F32).mul_(loud).to(stream)
        state["weight"] = draws(d, std=0.1, dtype=F32).add_(1.0)
        if kind == "norm_train":
            state["dy"] = draws(rows, d, std=1e-2)
            state["dstream"] = draws(rows, d, std=1e-2, dtype=stream)
            for name in ("x", "residual", "weight"):
                state[name].requires_grad_(True)
        return state
    if kind in ("lookup", "embed_train"):
        vocab, d = case["vocab"], case["d"]
        # Rank v is drawn with a probability of about 1 / v; a fixed permutation of the ranks.
        rank = torch.exp(draws.uniform(rows).double() * torch.log(torch.tensor(vocab + 1.0)).item())
        rank = (rank.long() - 1).clamp_(0, vocab - 1)
        state["tokens"] = torch.randperm(vocab, generator=draws.gen, device="cuda")[rank]
        state["table"] = draws(vocab, d, std=0.02, dtype=_type(case["dtype"]))
        if kind == "embed_train":
            state["dy"] = draws(rows, d, std=1e-2)
            state["table"].requires_grad_(True)
        return state
    n, k, experts = case["n"], case["k"], case["experts"]
    liking = draws(experts, std=0.5, dtype=F32).softmax(0)
    chosen = torch.multinomial(liking, rows, replacement=True, generator=draws.gen)
    counts = torch.bincount(chosen, minlength=experts)
    state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    state["most"] = int(counts.max())
    state["x"] = draws(rows, k)
    state["weight"] = draws(experts, n, k, std=0.02, dtype=_type(case["dtype"]))
    if case["train"]:
        state["dy"] = draws(rows, n, std=1e-2)
        state["x"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


# --- plain forms ---------------------------------------------------------------------------

def _quantize(x, scales):
    """(e4m3 x / scale, scale) of FP32 x with one scale per block of 128 along its rows: the
    smallest power of two that brings the block's largest magnitude to at most 448, or that
    magnitude over 448."""
    m, k = x.shape
    wide = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(m, -1, BLOCK)
    amax = wide.abs().amax(2)
    if scales == "e8m0":
        mantissa, exponent = torch.frexp(amax)
        code = (exponent - 9 + (mantissa > 0.875) + 127).clamp_(1, 254)
        scale = code.to(torch.uint8).view(E8M0)
        inverse = ((254 - code) << 23).to(torch.int32).view(F32)
    else:
        amax = amax.clamp_min(2.0 ** -100)
        scale, inverse = amax / E4M3_MAX, E4M3_MAX / amax
    return (wide * inverse[:, :, None]).view(m, -1)[:, :k].to(E4M3), scale


def _plain_norm(state):
    case = state["case"]
    residual, weight = state["residual"].detach(), state["weight"].detach()
    stream = (state["x"].detach().float() + residual.float()).to(residual.dtype)
    s = stream.float()
    rstd = (s.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = s * rstd * weight
    if case["kind"] == "norm_quantize":
        q, scale = _quantize(y, case["scales"])
        return {"q": q, "scale": scale, "stream": stream}
    dy, dstream = state["dy"].float(), state["dstream"].float()
    g = dy * weight
    d = dstream + rstd * (g - s * rstd.square() * (g * s).mean(1, keepdim=True))
    return {"y": y.to(BF16), "stream": stream, "dx": d.to(BF16), "dresidual": d.to(residual.dtype),
            "dweight": (dy * s * rstd).sum(0)}


def _plain_embedding(state):
    case, tokens, table = state["case"], state["tokens"], state["table"].detach()
    out = {"y": (table[tokens].float() * case["scale"]).to(BF16)}
    if case["kind"] == "embed_train":
        sums = torch.zeros(table.shape, dtype=F32, device=table.device)
        sums.index_add_(0, tokens, state["dy"].float())
        out["dtable"] = sums.mul_(case["scale"]).to(table.dtype)
    return out


def _padded(t, index, valid):
    """Rows of t by expert, [experts, most, width] FP32, zeros past an expert's last."""
    return torch.where(valid[:, :, None], t[index.clamp_max(t.shape[0] - 1)].float(), 0.0)


def _plain_experts(state):
    """Every expert's rows padded to the largest count, so that each product is one batch."""
    case, offsets, x = state["case"], state["offsets"], state["x"].detach()
    weight = state["weight"].detach().to(BF16).float()
    place = torch.arange(state["most"], device=x.device)
    index = offsets[:-1, None] + place
    valid = index < offsets[1:, None]
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offsets, row, right=True) - 1
    back = expert * state["most"] + row - offsets[expert]
    wide = _padded(x, index, valid)
    y = torch.bmm(wide, weight.transpose(1, 2)).flatten(0, 1)[back].to(BF16)
    if not case["train"]:
        return {"y": y}
    grad = _padded(state["dy"], index, valid)
    dx = torch.bmm(grad, weight).flatten(0, 1)[back].to(BF16)
    dweight = torch.bmm(grad.transpose(1, 2), wide).to(state["weight"].dtype)
    return {"y": y, "dx": dx, "dweight": dweight}


def _plain(state):
    kind = state["case"]["kind"]
    if kind.startswith("norm"):
        return _plain_norm(state)
    return _plain_experts(state) if kind == "experts" else _plain_embedding(state)


# --- the framework's calls -----------------------------------------------------------------

def _own(state):
    case = state["case"]
    kind = case["kind"]
    if kind.startswith("norm"):
        from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

        x, residual, weight = state["x"], state["residual"], state["weight"]
        if kind == "norm_quantize":
            q, scale, stream = rmsnorm_quantize(x, weight, EPS, residual=residual,
                                                scale_dtype=_scale_type(case))
            return {"q": q, "scale": scale, "stream": stream}
        y, stream = add_rmsnorm(x, residual, weight, EPS)
        dx, dresidual, dweight = torch.autograd.grad([y, stream], [x, residual, weight],
                                                     [state["dy"], state["dstream"]])
        return {"y": y, "stream": stream, "dx": dx, "dresidual": dresidual, "dweight": dweight}
    if kind in ("lookup", "embed_train"):
        from ops.embedding_execution import embedding

        y = embedding(state["tokens"], state["table"], case["scale"])
        if kind == "lookup":
            return {"y": y}
        return {"y": y, "dtable": torch.autograd.grad(y, state["table"], state["dy"])[0]}
    from ops.grouped_execution import grouped_mm

    y = grouped_mm(state["x"], state["weight"], state["offsets"])
    if not case["train"]:
        return {"y": y}
    dx, dweight = torch.autograd.grad(y, [state["x"], state["weight"]], state["dy"])
    return {"y": y, "dx": dx, "dweight": dweight}


def _scale_type(case):
    return E8M0 if case["scales"] == "e8m0" else F32


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read and each output written once; the products' multiplications."""
    kind, rows = case["kind"], case["rows"]
    if kind.startswith("norm"):
        d, stream = case["d"], 2 if case["stream"] == "bf16" else 4
        if kind == "norm_quantize":
            scale = 1 if case["scales"] == "e8m0" else 4
            return {"bytes": rows * (d * (2 + stream + stream + 1) + scale * d / BLOCK) + 4 * d,
                    "flops": 0}
        # In: x, the stream, both upstream gradients. Out: y, the stream and one gradient for
        # both inputs, in two types where they differ.
        out = 2 if stream == 2 else 6
        return {"bytes": rows * d * (4 + 2 * stream + 2 + stream + out) + 8 * d, "flops": 0}
    if kind in ("lookup", "embed_train"):
        d, size = case["d"], 2 if case["dtype"] == "bf16" else 4
        lookup = rows * (8 + d * (size + 2))
        if kind == "lookup":
            return {"bytes": lookup, "flops": 0}
        return {"bytes": lookup + rows * 2 * d + case["vocab"] * d * size, "flops": 0}
    n, k, size = case["n"], case["k"], 2 if case["dtype"] == "bf16" else 4
    weights = min(rows, case["experts"]) * n * k * size
    if not case["train"]:
        return {"bytes": 2 * rows * (n + k) + weights, "flops": 2 * rows * n * k}
    return {"bytes": 4 * rows * (n + k) + weights + case["experts"] * n * k * size,
            "flops": 6 * rows * n * k}


# --- the same values in 64 bits -------------------------------------------------------------

def _exact_e4m3(x):
    """The e4m3 value nearest to x (ties to the even one), |x| <= 448: steps of an eighth of
    the value's power of two, of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("norm"):
        x, residual, weight = (state[n].detach().to(F64) for n in ("x", "residual", "weight"))
        # The stream is an output: its rounding is part of what the norm is taken of.
        stream = (x + residual).to(state["residual"].dtype)
        s = stream.to(F64)
        root = torch.sqrt((s * s).sum(1) / case["d"] + EPS)[:, None]
        z = s / root
        y = z * weight
        if kind == "norm_quantize":
            m, k = y.shape
            wide = torch.zeros((m, -(-k // BLOCK) * BLOCK), dtype=F64, device=y.device)
            wide[:, :k] = y
            wide = wide.reshape(m, -1, BLOCK)
            top = wide.abs().amax(2)
            if case["scales"] == "e8m0":
                scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp_min(-126))
            else:
                scale = top.clamp_min(2.0 ** -100) / E4M3_MAX
            q = _exact_e4m3(wide / scale[:, :, None]).reshape(m, -1)[:, :k]
            return {"q": q, "scale": scale, "stream": x + residual}
        dy, dstream = state["dy"].to(F64), state["dstream"].to(F64)
        along = (dy * y).sum(1, keepdim=True) / case["d"]
        d = dstream + (dy * weight - z * along) / root
        return {"y": y, "stream": x + residual, "dx": d, "dresidual": d,
                "dweight": (dy * z).sum(0)}
    if kind in ("lookup", "embed_train"):
        tokens, table = state["tokens"], state["table"].detach()
        out = {"y": table.index_select(0, tokens).to(F64) * case["scale"]}
        if kind == "embed_train":
            sums = torch.zeros(table.shape, dtype=F64, device=table.device)
            out["dtable"] = sums.index_add_(0, tokens, state["dy"].to(F64) * case["scale"])
        return out
    bounds = state["offsets"].tolist()
    x, weight = state["x"].detach(), state["weight"].detach()
    parts = [(lo, hi, weight[e].to(BF16).to(F64))
             for e, (lo, hi) in enumerate(zip(bounds, bounds[1:]))]
    out = {"y": torch.cat([x[lo:hi].to(F64) @ w.T for lo, hi, w in parts])}
    if case["train"]:
        dy = state["dy"]
        out["dx"] = torch.cat([dy[lo:hi].to(F64) @ w for lo, hi, w in parts])
        out["dweight"] = torch.stack([dy[lo:hi].to(F64).T @ x[lo:hi].to(F64)
                                      for lo, hi, w in parts])
    return out
