"""64-bit statements of the training operators beside the pair stack: LayerNorm
with its gradients, the global norm of a set of gradients and clipping by it.
The reference leaves all of them to torch (torch.nn.LayerNorm,
torch.nn.utils.clip_grad_norm_)."""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np


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
