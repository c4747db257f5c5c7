"""Timed cases of two more training operators around the pair stack: dropout whose
mask comes from a counter-based generator and is never stored, and group norm
with an activation over channels-last tensors.

A case names an operator (``op``), a form of it and its sizes:

* ``op = "dropout"``: ``x`` is ``[b, n, m, c]``.  ``shared`` says along which
  dimension one mask is shared: ``row`` (-3), ``col`` (-2) or ``none``.
  ``residual`` is the type of the tensor that the result is added to, or
  ``none``.  ``device_seed``: the seed lies on the GPU, as in a captured step.
* ``op = "group_norm"``: ``x`` is ``[b, n, m, c]`` in ``groups`` groups, ``act`` its
  activation.  ``params`` is the weight's and bias' type (``none``: no affine).
  ``live`` < 1 masks rows and columns past that share of the plane, as a padded
  batch has them (each sample ends elsewhere).

``mode`` is ``infer`` (the output alone) or ``train`` (the output and the
gradients for a given output gradient); ``dtype`` is the type of ``x``.

The dropout mask.  ``x`` is seen as ``[outer, shared, inner]``.  Value ``r`` of
``inner`` under ``outer`` index ``o`` has 16 bits of its own: half ``r % 2`` (low
first) of word ``r % 8 // 2`` of Philox4x32-10 (Salmon et al., "Parallel random
numbers: as easy as 1, 2, 3", 2011) at counter ``o * ceil(inner / 8) + r // 8``
(low 64 bits) and ``offset`` (high 64 bits) under the key ``seed``.  It is kept
where they are at least ``t = round(65536 p)``, and scaled by
``65536 / (65536 - t)``.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "genie-tk_amd"))

own = False

DEVICE = "cuda"
EPS = 1e-5
OFFSET = 5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
SHARED = {"row": -3, "col": -2, "none": None}
MOST = 1024 * 1024 * 120  # values of a drawn case, somewhat below the largest listed one


def _drop(shared, dtype, residual, n, c, b=1, m=None, mode="train", p=0.25, device_seed=False, name=None):
    case = {"op": "dropout", "mode": mode, "shared": shared, "dtype": dtype, "residual": residual, "b": b, "n": n,
            "m": m or n, "c": c, "p": p, "device_seed": device_seed}
    return case if name is None else {"name": name, **case}


def _norm(dtype, b, n, c, groups, act, m=None, mode="train", params="fp32", live=1.0, name=None):
    case = {"op": "group_norm", "mode": mode, "dtype": dtype, "params": params, "b": b, "n": n, "m": m or n, "c": c,
            "groups": groups, "act": act, "live": live}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # a short chain's update added to its pair tensor: the call itself
        _drop("row", "bf16", "bf16", 64, 128, name="drop_row_bf16_n64_c128"),
        # the crop most folding programs train at
        _drop("row", "bf16", "bf16", 512, 128, name="drop_row_bf16_n512_c128"),
        # the ending node's update of a chain and a width of no round size
        _drop("col", "fp32", "fp32", 301, 100, name="drop_col_fp32_n301_c100"),
        # bf16 updates into an fp32 residual stream, a batch of two, the seed of a captured step
        _drop("col", "bf16", "fp32", 384, 128, b=2, device_seed=True, name="drop_col_mixed_b2_n384_c128"),
        # a mask of its own for each value: the transition's hidden activation
        _drop("none", "bf16", "none", 384, 512, p=0.1, name="drop_full_bf16_n384_c512"),
        # one token's channels: the call itself
        _norm("bf16", 1, 1, 1024, 16, "none", mode="infer", name="gn_token_bf16_c1024"),
        # a sequence's tokens, each normalised by itself, a group a head
        _norm("bf16", 4096, 1, 512, 8, "silu", name="gn_tokens_bf16_r4096_c512"),
        # feature maps of a batch, ten channels a group
        _norm("fp32", 16, 16, 320, 32, "silu", name="gn_maps_fp32_b16_n16_c320"),
        # larger maps: many samples, each of which one compute unit can nearly hold
        _norm("bf16", 8, 64, 256, 32, "silu", name="gn_maps_bf16_b8_n64_c256"),
        # a padded pair plane of no round size
        _norm("fp32", 1, 301, 100, 20, "gelu", mode="infer", live=0.9, name="gn_plane_fp32_n301_c100"),
        # the training crop, padded
        _norm("bf16", 1, 512, 128, 32, "silu", live=0.8, name="gn_plane_bf16_n512_c128"),
        # the longest pair tensor: memory bandwidth
        _norm("bf16", 1, 1024, 128, 8, "gelu", params="bf16", name="gn_plane_bf16_n1024_c128"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    dtype = rng.choice(("bf16", "fp32"))
    most = MOST // (1 if dtype == "bf16" else 2)
    mode = rng.choice(("infer", "train", "train"))
    b = _log_int(rng, 1, 16)
    n = _log_int(rng, 4, 1024)
    m = n if rng.random() < 0.7 else _log_int(rng, 4, 1024)
    if rng.random() < 0.5:
        c = _log_int(rng, 3, 1024)
        if rng.random() < 0.5:
            c = (c + 15) // 16 * 16
        residual = rng.choice((dtype, dtype, "fp32", "none"))
        n = max(1, min(n, most // (2 * b * m * c)))
        return _drop(rng.choice(("row", "row", "col", "none")), dtype, residual, n, c, b=b, m=m, mode=mode,
                     p=rng.choice((0.1, 0.15, 0.25, 0.5)), device_seed=rng.random() < 0.3)
    width = _log_int(rng, 1, 64)  # channels a group
    if rng.random() < 0.6:
        width = 1 << width.bit_length() - 1
    groups = _log_int(rng, 1, max(1, 1024 // width))
    c = width * groups
    if rng.random() < 0.2:  # tokens
        b, n, m = _log_int(rng, 1, 8192), 1, 1
    n = max(1, min(n, most // (b * m * c)))
    if n * m * width == 1:  # a group of one value has no spread
        n = m = 2
        b = max(1, min(b, most // (4 * c)))
    return _norm(dtype, b, n, c, groups, rng.choice(("none", "silu", "silu", "gelu")), m=m, mode=mode,
                 params=rng.choice((dtype, "fp32", "none")),
                 live=rng.uniform(0.5, 0.95) if n > 4 and m > 4 and rng.random() < 0.5 else 1.0)


# ---------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    b, n, m, c = (case[k] for k in ("b", "n", "m", "c"))

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen, dtype=torch.float32)

    state = {"case": case, "residual": None}
    x = normal(b, n, m, c)
    if case["op"] == "dropout":
        state["x"] = x.to(dtype)
        if case["residual"] != "none":
            state["residual"] = (2.0 * normal(b, n, m, c)).to(DTYPES[case["residual"]])
        state["seed"] = seed * 0x9E3779B97F4A7C15 % (1 << 62) + 1
        if case["device_seed"]:
            state["seed"] = torch.tensor([state["seed"]], device=DEVICE)
        leaves = [state["x"], state["residual"]]
        out = torch.promote_types(dtype, dtype if leaves[1] is None else leaves[1].dtype)
    else:
        # channels differ in mean and spread, as a layer's outputs do
        x *= torch.exp(0.5 * normal(c))
        x += normal(c)
        state["x"] = x.to(dtype)
        state["weight"] = state["bias"] = state["mask"] = None
        if case["params"] != "none":
            kind = DTYPES[case["params"]]
            state["weight"] = (1 + 0.2 * normal(c)).to(kind)
            state["bias"] = (0.2 * normal(c)).to(kind)
        if case["live"] < 1:
            # sample k ends a little before sample k - 1
            mask = torch.zeros(b, n, m, device=DEVICE)
            for k in range(b):
                share = case["live"] * (1 - 0.3 * k / b)
                mask[k, :max(1, int(n * share)), :max(1, int(m * share))] = 1
            state["mask"] = mask
        leaves = [state["x"], state["weight"], state["bias"]]
        out = dtype
    del x
    if case["mode"] == "train":
        state["dy"] = normal(b, n, m, c).to(out)
        state["leaves"] = [t for t in leaves if t is not None]
        for t in state["leaves"]:
            t.requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
_LOW = 0xFFFFFFFF


def _geometry(case):
    """(outer, shared, inner) of the mask."""
    b, n, m, c = (case[k] for k in ("b", "n", "m", "c"))
    if case["shared"] == "row":
        return b, n, m * c
    if case["shared"] == "col":
        return b * n, m, c
    return 1, 1, b * n * m * c


def _plain_keep(case, seed):
    """The mask, in 64-bit integers: products wrap, their halves are as unsigned ones."""
    outer, _, inner = _geometry(case)
    blocks = (inner + 7) // 8
    at = torch.arange(outer * blocks, device=DEVICE)
    c0, c1 = at & _LOW, at >> 32
    c2, c3 = torch.full_like(at, OFFSET), torch.zeros_like(at)
    if not isinstance(seed, torch.Tensor):
        seed = torch.tensor([seed], device=DEVICE)
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):
        p0, p1 = c0 * _M0, c2 * _M1
        c0, c1, c2, c3 = p1 >> 32 & _LOW ^ c1 ^ k0, p1 & _LOW, p0 >> 32 & _LOW ^ c3 ^ k1, p0 & _LOW
        k0, k1 = k0 + _W0 & _LOW, k1 + _W1 & _LOW
    halves = [h for w in (c0, c1, c2, c3) for h in (w & 0xFFFF, w >> 16)]
    bits = torch.stack(halves, -1).view(outer, blocks * 8)[:, :inner]
    return (bits >= round(65536 * case["p"])).view(outer, 1, inner)


def _scale(case):
    return 65536 / (65536 - round(65536 * case["p"]))


def _plain_dropout(state):
    case, x = state["case"], state["x"]
    keep = _plain_keep(case, state["seed"])
    view, scale = _geometry(case), _scale(case)

    def drop(t):
        return torch.where(keep, t.float().view(view) * scale, 0.0).view(x.shape)

    y, residual = drop(x), state["residual"]
    kind = x.dtype
    if residual is not None:
        kind = torch.promote_types(x.dtype, residual.dtype)
        y = y + residual.float()
    y = y.to(kind)
    if case["mode"] == "infer":
        return y
    out = {"y": y, "dx": drop(state["dy"]).to(x.dtype)}
    if residual is not None:
        out["dresidual"] = state["dy"].to(residual.dtype)
    return out


def _plain_norm(state):
    case = state["case"]
    b, c, groups = case["b"], case["c"], case["groups"]
    x, weight, bias, mask = (state[k] for k in ("x", "weight", "bias", "mask"))
    split = (b, -1, groups, c // groups)
    xf = x.float().view(split)
    if mask is None:
        live, count = None, xf.shape[1] * xf.shape[3]
    else:
        live = (mask != 0).view(b, -1, 1, 1)
        count = live.sum((1, 2, 3), keepdim=True) * xf.shape[3]

    def only(t):  # the counted values
        return t if live is None else torch.where(live, t, 0.0)

    def mean(t):
        return t.sum((1, 3), keepdim=True) / count

    d = only(xf)
    d = only(d - mean(d))
    rstd = (mean(d.square()) + EPS).rsqrt()
    h = d * rstd
    z = h
    if weight is not None:
        wf = weight.float().view(groups, -1)
        z = h * wf + bias.float().view(groups, -1)
    act = case["act"]
    if act == "none":
        y = z
    elif act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        y = z * sig
    else:
        phi = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        y = z * phi
    y = only(y).to(x.dtype).view(x.shape)
    if case["mode"] == "infer":
        return y
    dz = only(state["dy"].float().view(split))
    if act == "silu":
        dz = dz * (sig * (1 + z * (1 - sig)))
    elif act == "gelu":
        dz = dz * (phi + z * torch.exp(-0.5 * z.square()) * (1 / math.sqrt(2 * math.pi)))
    g = dz if weight is None else dz * wf
    dx = only((g - mean(g) - h * mean(g * h)) * rstd)
    out = {"y": y, "dx": dx.to(x.dtype).view(x.shape)}
    if weight is not None:
        out["dweight"] = (dz * h).sum((0, 1)).view(c).to(weight.dtype)
        out["dbias"] = dz.sum((0, 1)).view(c).to(weight.dtype)
    return out


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_run(state):
    from genie_tk.primitives import dropout, group_norm

    case = state["case"]
    with torch.set_grad_enabled(case["mode"] == "train"):
        if case["op"] == "dropout":
            y = dropout(state["x"], case["p"], state["seed"], OFFSET, SHARED[case["shared"]], state["residual"])
            names = ("dx", "dresidual")
        else:
            y = group_norm(state["x"], case["groups"], state["weight"], state["bias"], EPS,
                           None if case["act"] == "none" else case["act"], state["mask"])
            names = ("dx", "dweight", "dbias")
        if case["mode"] == "infer":
            return y
        return {"y": y, **dict(zip(names, torch.autograd.grad(y, state["leaves"], state["dy"])))}


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return _plain_dropout(state) if state["case"]["op"] == "dropout" else _plain_norm(state)


# ---------------------------------------------------------------------------
# Floors and exact values
# ---------------------------------------------------------------------------
def work(case):
    n = case["b"] * case["n"] * case["m"] * case["c"]
    e = SIZE[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "dropout":
        res = 0 if case["residual"] == "none" else SIZE[case["residual"]]
        out = max(e, res)
        outer, _, inner = _geometry(case)
        mask = 15 * outer * inner  # some 120 operations for eight values' bits
        return {"bytes": n * (e + res + out) + (n * (out + e) if train else 0),
                "flops": (2 if train else 1) * (3 * n + mask)}
    params = 0 if case["params"] == "none" else 2 * case["c"] * SIZE[case["params"]]
    mask = n // case["c"] * 4 if case["live"] < 1 else 0
    act = {"none": 0, "silu": 5, "gelu": 20}[case["act"]]
    if train:
        return {"bytes": 4 * n * e + 2 * mask + 3 * params, "flops": n * (27 + 3 * act)}
    return {"bytes": 2 * n * e + mask + params, "flops": n * (10 + act)}


def _exact_bits(outer, blocks, seed):
    """Philox4x32-10 with products of 16-bit limbs, [outer * blocks, 8] halves."""
    at = torch.arange(outer * blocks, device=DEVICE)

    def times(word, factor):  # (high, low) 32 bits
        a0, a1, f0, f1 = word % 65536, word // 65536, factor % 65536, factor // 65536
        cross = a1 * f0 + (a0 * f0) // 65536
        other = a0 * f1 + cross % 65536
        return a1 * f1 + cross // 65536 + other // 65536, other % 65536 * 65536 + (a0 * f0) % 65536

    word = [at % (1 << 32), at // (1 << 32), torch.full_like(at, OFFSET), torch.zeros_like(at)]
    key = [seed % (1 << 32), seed // (1 << 32)]
    for _ in range(10):
        high0, low0 = times(word[0], 0xD2511F53)
        high1, low1 = times(word[2], 0xCD9E8D57)
        word = [high1.bitwise_xor(word[1]).bitwise_xor(key[0]), low1,
                high0.bitwise_xor(word[3]).bitwise_xor(key[1]), low0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    return torch.cat([w.unsqueeze(1) // d % 65536 for w in word for d in (1, 65536)], dim=1)


def _exact_dropout(state):
    case = state["case"]
    b, n, m, c = state["x"].shape
    # the mask as a tensor that broadcasts over x
    shape = {"row": (b, 1, m, c), "col": (b, n, 1, c), "none": (b, n, m, c)}[case["shared"]]
    outer = {"row": b, "col": b * n, "none": 1}[case["shared"]]
    inner = math.prod(shape) // outer
    drawn = _exact_bits(outer, -(-inner // 8), int(state["seed"])).reshape(outer, -1)
    limit = round(case["p"] * 65536)
    factor = (drawn[:, :inner].reshape(shape) >= limit).to(torch.float64)
    del drawn
    factor.div_(1 - limit / 65536)
    y = state["x"].detach().to(torch.float64).mul_(factor)
    if state["residual"] is not None:
        y.add_(state["residual"].detach())
    if case["mode"] == "infer":
        return y
    out = {"y": y, "dx": factor * state["dy"]}
    if state["residual"] is not None:
        out["dresidual"] = state["dy"].to(torch.float64)
    return out


def _exact_norm(state):
    case = state["case"]
    b, c, groups = case["b"], case["c"], case["groups"]
    train = case["mode"] == "train"

    def rows(t):  # a row of values for each sample and group
        return t.reshape(b, -1, groups, c // groups).transpose(1, 2).reshape(b * groups, -1)

    def back(t):
        return t.reshape(b, groups, -1, c // groups).transpose(1, 2).reshape(state["x"].shape)

    def channel(t):  # a parameter for each value of those rows, as a view that broadcasts
        return t.detach().to(torch.float64).reshape(1, groups, 1, c // groups)

    x = rows(state["x"].detach().to(torch.float64))
    on = torch.ones((), dtype=torch.float64, device=DEVICE)
    if state["mask"] is not None:
        on = rows((state["mask"] != 0).to(torch.float64).unsqueeze(-1).expand(state["x"].shape))
    total = (on.expand_as(x)).sum(1, keepdim=True)
    x = (x - (x * on).sum(1, keepdim=True) / total) * on
    std = ((x * x).sum(1, keepdim=True) / total + EPS).sqrt()
    x = x / std
    wide = (b, groups, -1, c // groups)
    scale = None if state["weight"] is None else channel(state["weight"])
    z = x if scale is None else (x.view(wide) * scale + channel(state["bias"])).view_as(x)
    slope = None
    if case["act"] == "silu":
        gate = torch.sigmoid(z)
        slope = gate + z * gate * torch.sigmoid(-z) if train else None
        z = z * gate
    elif case["act"] == "gelu":
        below = torch.special.erfc(-z / math.sqrt(2)) / 2
        slope = below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi) if train else None
        z = z * below
    y = back(z * on)
    if not train:
        return y
    up = rows(state["dy"].to(torch.float64)) * on
    if slope is not None:
        up = up * slope
    out = {"y": y}
    if scale is not None:
        out["dweight"] = (up * x).view(wide).sum((0, 2)).reshape(c)
        out["dbias"] = up.view(wide).sum((0, 2)).reshape(c)
        up = (up.view(wide) * scale).view_as(x)
    along = (up * x).sum(1, keepdim=True) / total
    out["dx"] = back((up - up.sum(1, keepdim=True) / total - x * along) / std * on)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_dropout(state) if case["op"] == "dropout" else _exact_norm(state)
