"""Timed cases of the training operators beside the pair stack: LayerNorm with
its gradients, and the global norm of a set of gradients with clipping.

A case names an operator (``op``), a form of it and its sizes:

* ``op = "layer_norm"``: rows of ``d`` values, ``rows`` of them.  ``mode`` is
  ``infer`` (the output alone) or ``train`` (the output, and the gradients of
  the rows, the weight and the bias for a given output gradient).  ``dtype`` is
  the rows' type, ``params`` the weight's and bias' (``none``: no affine).
  ``gap`` > 0 makes the rows a slice of rows that much wider.
* ``op = "grads"``: a set of gradients, either the parameters of ``layers``
  pair-stack layers of ``c`` channels (58 tensors a layer, each starting on 16
  bytes as the framework's backward passes leave them), or ``count`` tensors of
  uneven sizes that hold ``total`` values, one right behind the other as in a
  communication bucket.  ``form`` is ``norm`` (the global norm), ``clip`` (in
  place) or ``master`` (clipped into fp32, the gradients of fp32 master
  weights).  ``p`` is the norm's order.  ``over`` says whether the norm is above
  the limit.

Rows are N(0, 1) around a mean of their own, as activations are; LayerNorm
weights are near 1.  Gradients are small and of uneven scale from tensor to
tensor.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "genie-tk_amd"))

own = False

DEVICE = "cuda"
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


def _ln(rows, d, mode, dtype, params=None, gap=0, name=None):
    case = {"op": "layer_norm", "mode": mode, "dtype": dtype, "params": params or dtype,
            "rows": rows, "d": d, "gap": gap}
    return case if name is None else {"name": name, **case}


def _grads(form, dtype, layers=0, c=128, count=0, total=0, p=2.0, over=True, name=None):
    case = {"op": "grads", "form": form, "dtype": dtype, "layers": layers, "c": c, "count": count,
            "total": total, "p": p, "over": over}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one token's row in a sampling loop: the call itself
        _ln(1, 1024, "infer", "bf16", name="ln_token_bf16_d1024"),
        # a pair tensor of 301 residues with 100 channels (no round size), rows cut from wider ones
        _ln(301 * 301, 100, "infer", "fp32", gap=28, name="ln_rows_fp32_n301_d100"),
        # a training step on a short chain in the modules' default type
        _ln(64 * 64, 128, "train", "fp32", name="ln_train_fp32_n64_d128"),
        # the crop most folding programs train at, bf16 with fp32 parameters
        _ln(512 * 512, 128, "train", "bf16", params="fp32", name="ln_train_bf16_n512_d128"),
        # the longest pair tensor: memory bandwidth
        _ln(1024 * 1024, 128, "train", "bf16", name="ln_train_bf16_n1024_d128"),
        # sequence activations of a wide trunk
        _ln(4096, 4096, "train", "bf16", name="ln_train_bf16_r4096_d4096"),
        # a width of no round size
        _ln(10007, 1023, "train", "fp32", name="ln_train_fp32_r10007_d1023"),
        # the gradients of one layer: the call itself
        _grads("norm", "fp32", layers=1, name="norm_fp32_layer"),
        # an eight-layer net, clipped into the gradients of its fp32 master weights
        _grads("master", "bf16", layers=8, name="master_bf16_8_layers"),
        # a 24-layer net whose norm is below the limit, as in most steps: nothing changes
        _grads("clip", "fp32", layers=24, over=False, name="clip_fp32_24_layers"),
        # a large model's gradients: few tensors, memory bandwidth
        _grads("norm", "bf16", count=37, total=400_000_001, name="norm_bf16_400m"),
        _grads("master", "fp32", count=61, total=150_000_001, name="master_fp32_150m"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(("bf16", "fp32"))
    if rng.random() < 0.55:
        d = _log_int(rng, 8, 16384)
        if rng.random() < 0.4:
            d = (d + 63) // 64 * 64
        most = 120_000_000 // SIZE[dtype]
        rows = _log_int(rng, 1, max(2, min(1 << 20, most // d)))
        params = rng.choice((dtype, dtype, "fp32", "none"))
        gap = rng.randint(1, 64) if rng.random() < 0.25 else 0
        return _ln(rows, d, rng.choice(("infer", "train", "train")), dtype, params, gap)
    p = rng.choice((2.0, 2.0, 2.0, 1.0, math.inf))
    form = rng.choice(("norm", "clip", "master"))
    over = form == "master" or rng.random() < 0.3
    if rng.random() < 0.5:
        return _grads(form, dtype, layers=_log_int(rng, 1, 32), c=rng.choice((64, 128)), p=p, over=over)
    count = _log_int(rng, 1, 300)
    return _grads(form, dtype, count=count, total=_log_int(rng, 64 * count, 100_000_000), p=p, over=over)


# ---------------------------------------------------------------------------
# The gradients' sizes
# ---------------------------------------------------------------------------
def _layer_sizes(c):
    """Parameters of one pair-stack layer: two multiplicative updates, two
    attentions (full width), the transition."""
    square = c * c
    update = [c, c] + [square, c] * 5 + [c, c] + [square, c]
    attention = [c, c, 4 * c, square, square, square, square, c, square, c]
    transition = [c, c, 4 * square, 4 * c, 4 * square, c]
    return update * 2 + attention * 2 + transition


def _sizes(case):
    if case["layers"]:
        return _layer_sizes(case["c"]) * case["layers"]
    rng = random.Random(case["count"] * 1000003 + case["total"])
    shares = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(case["count"])]
    scale = (case["total"] - case["count"]) / sum(shares)
    sizes = [1 + int(s * scale) for s in shares]
    sizes[-1] += case["total"] - sum(sizes)
    return sizes


def _places(case):
    """Where each gradient starts in the flat buffer, and the buffer's size."""
    step = 16 // SIZE[case["dtype"]] if case["layers"] else 1
    places, at = [], 0
    for n in _sizes(case):
        places.append(at)
        at += (n + step - 1) // step * step
    return places, at


# ---------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen, dtype=torch.float32)

    if case["op"] == "layer_norm":
        rows, d = case["rows"], case["d"]
        wide = normal(rows, d + case["gap"])
        wide += normal(rows, 1)
        x = wide.to(dtype)[:, case["gap"] // 2:case["gap"] // 2 + d]
        state = {"case": case, "x": x, "weight": None, "bias": None}
        if case["params"] != "none":
            kind = DTYPES[case["params"]]
            state["weight"] = (1 + 0.2 * normal(d)).to(kind)
            state["bias"] = (0.2 * normal(d)).to(kind)
        if case["mode"] == "train":
            state["dy"] = normal(rows, d).to(dtype)
            state["leaves"] = [t for t in (x, state["weight"], state["bias"]) if t is not None]
            for t in state["leaves"]:
                t.requires_grad_(True)
        return state

    # uneven scales from tensor to tensor; the limit is set beside the norm
    sizes, (places, room) = _sizes(case), _places(case)
    flat = torch.zeros(room, device=DEVICE, dtype=dtype)
    grads = [flat[at:at + n] for n, at in zip(sizes, places)]
    for k, g in enumerate(grads):
        g.copy_(normal(g.numel()).mul_(10.0 ** (-3 - (k * 7 % 5) / 4)))
    if case["p"] == 1.0:
        norm = flat.double().abs().sum()
    elif case["p"] == math.inf:
        norm = flat.abs().max()
    else:
        norm = flat.double().square().sum().sqrt()
    state = {"case": case, "flat": flat, "grads": grads, "sizes": sizes,
             "max_norm": float(norm) * (0.1 if case["over"] else 10.0)}
    if case["form"] == "clip":
        state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
        for p, g in zip(state["params"], grads):
            p.grad = g
    if case["form"] == "master":
        state["master"] = torch.zeros(room, device=DEVICE)
        state["outs"] = [state["master"][at:at + n] for n, at in zip(sizes, places)]
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_norm(x, weight, bias):
    xf = x.float()
    d = xf - xf.mean(-1, keepdim=True)
    rstd = (d.square().mean(-1, keepdim=True) + EPS).rsqrt()
    h = d * rstd
    y = h
    if weight is not None:
        y = h * weight.float() + bias.float()
    return y.to(x.dtype), h, rstd


def _plain_norm_grads(x, dy, weight, h, rstd):
    dyf = dy.float()
    g = dyf if weight is None else dyf * weight.float()
    dx = (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)) * rstd
    out = {"dx": dx.to(x.dtype)}
    if weight is not None:
        out["dweight"] = (dyf * h).sum(0).to(weight.dtype)
        out["dbias"] = dyf.sum(0).to(weight.dtype)
    return out


def _plain_global_norm(every, p):
    if p == math.inf:
        return every.abs().max().float()
    if p == 1.0:
        return every.float().abs().sum(dtype=torch.float64).float()
    return every.float().square().sum(dtype=torch.float64).sqrt().float()


def _plain_run(state):
    case = state["case"]
    with torch.no_grad():
        if case["op"] == "layer_norm":
            x, w = state["x"], state["weight"]
            y, h, rstd = _plain_norm(x, w, state["bias"])
            if case["mode"] == "infer":
                return y
            return {"y": y, **_plain_norm_grads(x, state["dy"], w, h, rstd)}
        grads = [q.grad for q in state["params"]] if case["form"] == "clip" else state["grads"]
        every = torch.cat(grads)
        norm = _plain_global_norm(every, case["p"])
        if case["form"] == "norm":
            return norm
        coef = (state["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
        if case["form"] == "master":
            torch._foreach_copy_(state["outs"], grads)
            torch._foreach_mul_(state["outs"], coef)
            return {"norm": norm, "grads": state["master"]}
        if case["dtype"] == "fp32":
            torch._foreach_mul_(grads, coef)
        else:  # the product in 32 bits
            clipped = (every.float() * coef).to(every.dtype)
            torch._foreach_copy_(grads, torch.split(clipped, state["sizes"]))
        return {"norm": norm, "grads": state["flat"]}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_run(state):
    from genie_tk.gradients import clip_grad_norm_, clip_grads, grad_norm
    from genie_tk.primitives import layer_norm

    case = state["case"]
    if case["op"] == "layer_norm":
        if case["mode"] == "infer":
            with torch.no_grad():
                return layer_norm(state["x"], state["weight"], state["bias"], EPS)
        y = layer_norm(state["x"], state["weight"], state["bias"], EPS)
        got = torch.autograd.grad(y, state["leaves"], state["dy"])
        return {"y": y, **dict(zip(("dx", "dweight", "dbias"), got))}
    if case["form"] == "norm":
        return grad_norm(state["grads"], case["p"])
    if case["form"] == "clip":
        norm = clip_grad_norm_(state["params"], state["max_norm"], case["p"])
        return {"norm": norm, "grads": state["flat"]}
    norm, _ = clip_grads(state["grads"], state["max_norm"], case["p"], out=state["outs"])
    return {"norm": norm, "grads": state["master"]}


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ---------------------------------------------------------------------------
# Floors and exact values
# ---------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "layer_norm":
        n = case["rows"] * case["d"]
        params = 0 if case["params"] == "none" else 2 * case["d"] * SIZE[case["params"]]
        if case["mode"] == "infer":
            return {"bytes": 2 * n * e + params, "flops": 8 * n}
        return {"bytes": 4 * n * e + 2 * params, "flops": 21 * n}
    n = sum(_sizes(case))
    written = 0
    if case["form"] == "master":
        written = 4 * n
    elif case["form"] == "clip" and case["over"]:
        written = e * n
    return {"bytes": n * e + written, "flops": 2 * n + (n if written else 0)}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            x = state["x"].detach().to(torch.float64)
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            std = torch.sqrt(var + EPS)
            x = x.sub_(mean).div_(std)  # normalised
            scale = None if state["weight"] is None else state["weight"].detach().to(torch.float64)
            shift = None if scale is None else state["bias"].detach().to(torch.float64)
            y = x.clone() if scale is None else torch.addcmul(shift, x, scale)
            if case["mode"] == "infer":
                return y
            up = state["dy"].to(torch.float64)
            out = {"y": y}
            if scale is not None:
                out["dweight"] = (up * x).sum(dim=0)
                out["dbias"] = up.sum(dim=0)
                up = up * scale
            along = (up * x).sum(dim=1, keepdim=True) / case["d"]
            up = up.sub_(up.sum(dim=1, keepdim=True) / case["d"])
            out["dx"] = up.sub_(x.mul_(along)).div_(std)
            return out
        wide = state["flat"].to(torch.float64)
        norm = torch.linalg.vector_norm(wide, ord=case["p"])
        if case["form"] == "norm":
            return norm
        return {"norm": norm, "grads": wide * min(1.0, state["max_norm"] / (float(norm) + 1e-6))}
