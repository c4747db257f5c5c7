"""64-bit statements of the training operators beside the pair stack: LayerNorm
with its gradients, group norm with an activation and its gradients, dropout with a
counter-based generator, the global norm of a set of gradients and clipping by it.
The reference leaves all of them to torch (torch.nn.LayerNorm, nn.GroupNorm,
nn.Dropout, torch.nn.utils.clip_grad_norm_)."""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
from scipy.special import erfc, expit


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(y, h, rstd) over the last axis."""
    x = np.asarray(x, dtype=np.float64)
    d = x - x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    h = d * rstd
    y = h if weight is None else h * np.asarray(weight, dtype=np.float64)
    return (y if bias is None else y + np.asarray(bias, dtype=np.float64)), h, rstd


def layer_norm_grads(x, dy, weight=None, eps: float = 1e-5):
    """(dx, dweight, dbias) for rows x [R, D] and the output's gradient dy."""
    _, h, rstd = layer_norm(x, None, None, eps)
    dy = np.asarray(dy, dtype=np.float64)
    g = dy if weight is None else dy * np.asarray(weight, dtype=np.float64)
    dx = rstd * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def activation(z, act):
    """(act(z), act'(z)) of None, "silu" and "gelu"."""
    if act is None:
        return z, np.ones_like(z)
    if act == "silu":
        s = expit(z)
        return z * s, s + z * s * expit(-z)
    below = 0.5 * erfc(-z / np.sqrt(2.0))
    return z * below, below + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act=None, mask=None):
    """(y, h, z, rstd, live) of x [B, P, C] with mask [B, P]: h and z are 0 where the
    mask is, rstd is [B, 1, C] (each channel's group's), live [B, P, 1]."""
    x = np.asarray(x, dtype=np.float64)
    B, P, C = x.shape
    live = np.ones((B, P, 1), dtype=bool) if mask is None else (np.asarray(mask) != 0)[:, :, None]
    x = np.where(live, x, 0.0)
    h, rstd = np.zeros_like(x), np.zeros((B, 1, C))
    for b in range(B):
        for g in range(groups):
            at = slice(g * C // groups, (g + 1) * C // groups)
            v = x[b, live[b, :, 0], at]
            if v.size == 0:
                continue
            d = v - v.mean()
            rstd[b, 0, at] = 1.0 / np.sqrt((d * d).mean() + eps)
            h[b, live[b, :, 0], at] = d * rstd[b, 0, at]
    z = h if weight is None else h * np.asarray(weight, dtype=np.float64)
    if bias is not None:
        z = z + np.asarray(bias, dtype=np.float64)
    return np.where(live, activation(z, act)[0], 0.0), h, z, rstd, live


def group_norm_grads(x, dy, groups: int, weight=None, bias=None, eps: float = 1e-5, act=None, mask=None):
    """(dx, dweight, dbias, dz) for the output's gradient dy."""
    _, h, z, rstd, live = group_norm(x, groups, weight, bias, eps, act, mask)
    dz = np.where(live, np.asarray(dy, dtype=np.float64), 0.0) * activation(z, act)[1]
    g = dz if weight is None else dz * np.asarray(weight, dtype=np.float64)
    dx = np.zeros_like(h)
    for b in range(h.shape[0]):
        for k in range(groups):
            at = (b, live[b, :, 0], slice(k * h.shape[2] // groups, (k + 1) * h.shape[2] // groups))
            if g[at].size:
                dx[at] = rstd[b, :, at[2]] * (g[at] - g[at].mean() - h[at] * (g[at] * h[at]).mean())
    return dx, (dz * h).sum((0, 1)), dz.sum((0, 1)), dz


def philox(counter, offset: int, key: int):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) at the 128-bit counters
    (counter, offset): 4 words each, in Python's integers."""
    low = 0xFFFFFFFF
    out = []
    for n in counter:
        c = [n & low, n >> 32 & low, offset & low, offset >> 32 & low]
        k = [key & low, key >> 32 & low]
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [q >> 32 ^ c[1] ^ k[0], q & low, p >> 32 ^ c[3] ^ k[1], p & low]
            k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
        out.append(c)
    return out


def dropout_keep(outer: int, inner: int, p: float, seed: int, offset: int = 0) -> np.ndarray:
    """[outer, inner]: which values are kept."""
    blocks = -(-inner // 8)
    words = philox(range(outer * blocks), offset, seed)
    bits = np.array([[w >> s & 0xFFFF for w in c for s in (0, 16)] for c in words], dtype=np.int64)
    return bits.reshape(outer, blocks * 8)[:, :inner] >= round(65536 * p)


def dropout(x, p: float, seed: int, offset: int = 0, shared_dim=None, residual=None):
    x = np.asarray(x, dtype=np.float64)
    shape, outer = list(x.shape), 1
    if shared_dim is not None:
        shape[shared_dim] = 1
        outer = int(np.prod(x.shape[:shared_dim % x.ndim]))
    keep = dropout_keep(outer, int(np.prod(shape)) // outer if outer else 0, p, seed, offset).reshape(shape)
    t = round(65536 * p)
    y = np.where(keep, x * (65536 / (65536 - t) if t < 65536 else 0.0), 0.0)
    return y if residual is None else y + np.asarray(residual, dtype=np.float64)


def global_norm(tensors: Sequence[np.ndarray], p: float = 2.0) -> float:
    flat = np.concatenate([np.abs(np.asarray(t, dtype=np.float64)).ravel() for t in tensors] or [np.zeros(1)])
    if flat.size == 0:
        return 0.0
    if p == np.inf:
        return float(flat.max())
    return float((flat ** p).sum() ** (1.0 / p))


def clip_factor(norm: float, max_norm: float) -> float:
    k = max_norm / (norm + 1e-6)
    return 1.0 if k > 1.0 else k


def clip(tensors: Sequence[np.ndarray], max_norm: float, p: float = 2.0, norm: Optional[float] = None):
    k = clip_factor(global_norm(tensors, p) if norm is None else norm, max_norm)
    return [np.asarray(t, dtype=np.float64) * k for t in tensors]
