"""Linear layer with AlphaFold-style initialisers, gated multi-head attention
and LayerNorm.

API and semantics of ``src/genie_tk/primitives.py`` in the reference:
``_init_weights`` (:17-40), ``Linear`` (:43-62), ``Attention`` (:65-178).
``LayerNorm`` and ``layer_norm`` are additions: torch's LayerNorm with the
forward and the backward pass on the HIP kernels.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from genie_tk import _dispatch, _ext


def _init_weights(linear: nn.Linear, init: str = "default", std: float = 0.02) -> None:
    """In-place initialisation of an ``nn.Linear``.

    default: kaiming-uniform(a=sqrt(5)) weight, U(+-1/sqrt(fan_in)) bias (the
    nn.Linear default); final: zeros; gating: zero weight, unit bias;
    normal: N(0, std^2) weight, zero bias.
    """
    w, b = linear.weight, linear.bias
    if init == "default":
        nn.init.kaiming_uniform_(w, a=math.sqrt(5))
        if b is not None:
            fan_in = w.shape[1]
            bound = 1.0 / math.sqrt(fan_in) if fan_in > 0 else 0.0
            nn.init.uniform_(b, -bound, bound)
    elif init == "final":
        nn.init.zeros_(w)
        if b is not None:
            nn.init.zeros_(b)
    elif init == "gating":
        nn.init.zeros_(w)
        if b is not None:
            nn.init.ones_(b)
    elif init == "normal":
        nn.init.normal_(w, std=std)
        if b is not None:
            nn.init.zeros_(b)


class _DenseMatmul(torch.autograd.Function):
    """a @ b over equal leading (batch) dims, every operand made contiguous
    first, in the forward and in the backward (dA = G B^T, dB = A^T G).

    torch.matmul over batches on a transposed or permuted view makes a strided
    batched product, and so does its autograd backward by itself; in bfloat16
    that form has faulted gfx950 devices.  The products here are the same ones
    on contiguous copies."""

    @staticmethod
    def forward(ctx, a: Tensor, b: Tensor) -> Tensor:
        a, b = a.contiguous(), b.contiguous()
        ctx.save_for_backward(a, b)
        return torch.matmul(a, b)

    @staticmethod
    def backward(ctx, g: Tensor):
        a, b = ctx.saved_tensors
        g = g.contiguous()
        ga = gb = None
        if ctx.needs_input_grad[0]:
            ga = torch.matmul(g, b.transpose(-1, -2).contiguous())
        if ctx.needs_input_grad[1]:
            gb = torch.matmul(a.transpose(-1, -2).contiguous(), g)
        return ga, gb


def dense_matmul(a: Tensor, b: Tensor) -> Tensor:
    """``torch.matmul(a, b)`` for operands of equal leading dims, computed on
    contiguous operands in the forward and the backward."""
    assert a.shape[:-2] == b.shape[:-2], (a.shape, b.shape)
    return _DenseMatmul.apply(a, b)


class Linear(nn.Linear):
    """``nn.Linear`` whose parameters are initialised by ``_init_weights(init)``."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 init: str = "default"):
        super().__init__(in_features, out_features, bias=bias)
        _init_weights(self, init)


class Attention(nn.Module):
    """Gated multi-head attention with additive score biases.

    ``c_hidden`` is the total width over heads (head_dim = c_hidden / no_heads).
    forward: q, k, v projections without bias; scores = q k^T / sqrt(head_dim)
    plus every tensor in ``biases`` (added in list order); softmax over keys;
    o = attn v; o *= sigmoid(linear_g(q_x)) when gating; linear_o(o).
    """

    def __init__(self, c_q: int, c_k: int, c_v: int, c_hidden: int, no_heads: int,
                 gating: bool = True):
        super().__init__()
        assert c_hidden % no_heads == 0
        self.c_q, self.c_k, self.c_v = c_q, c_k, c_v
        self.c_hidden = c_hidden
        self.no_heads = no_heads
        self.gating = gating
        self.head_dim = c_hidden // no_heads
        self.linear_q = Linear(c_q, c_hidden, bias=False)
        self.linear_k = Linear(c_k, c_hidden, bias=False)
        self.linear_v = Linear(c_v, c_hidden, bias=False)
        self.linear_o = Linear(c_hidden, c_q, init="final")
        if gating:
            self.linear_g = Linear(c_q, c_hidden, init="gating")
        self.sigmoid = nn.Sigmoid()
        self.softmax = nn.Softmax(dim=-1)

    def _heads(self, t: Tensor) -> Tensor:
        # [*, L, H*D] -> [*, H, L, D]
        return t.unflatten(-1, (self.no_heads, self.head_dim)).transpose(-2, -3)

    def forward(self, q_x: Tensor, k_x: Tensor, v_x: Tensor,
                biases: Optional[List[Tensor]] = None) -> Tensor:
        q = self._heads(self.linear_q(q_x))
        k = self._heads(self.linear_k(k_x))
        v = self._heads(self.linear_v(v_x))
        scores = dense_matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(self.head_dim))
        for extra in biases or ():
            scores = scores + extra
        o = dense_matmul(self.softmax(scores), v)           # [*, H, Q, D]
        o = o.transpose(-2, -3).flatten(-2)                 # [*, Q, H*D]
        if self.gating:
            o = o * self.sigmoid(self.linear_g(q_x))
        return self.linear_o(o)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5) -> Tensor:
    """LayerNorm over the last dimension of ``x`` with optional ``weight`` and
    ``bias`` ([D]), differentiable once.

    Kernel path (bf16 or fp32 GPU tensor, parameters in bf16 or fp32, also
    mixed): ``genie_tk._C.layer_norm``, whose autograd node is the C++ one of
    ``layer_norm_forward`` and ``layer_norm_backward``.  The output and dL/dx
    have the type of ``x``, the parameters' gradients their own; statistics and
    sums are fp32.  Rows that lie one stride apart (a slice of wider rows, a
    repeated row) are read as they are.  Other tensors, and those with a
    forward-mode tangent, run torch's LayerNorm.  Under autocast GPU tensors
    narrower than fp32 are taken to fp32 first, as torch's LayerNorm takes them,
    and so is the output."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        x, weight, bias = (t.float() if t is not None and t.is_floating_point() and t.dtype != torch.float64 else t
                           for t in (x, weight, bias))
    params = [p for p in (weight, bias) if p is not None]
    if x.is_cuda:
        if _ext.C is None or not torch.cuda.is_available():
            _ext.missing("layer_norm")
        elif (x.dim() >= 1 and 1 <= x.shape[-1] <= 1 << 24 and x.dtype in _dispatch.SUPPORTED_DTYPES
              and all(p.dtype in _dispatch.SUPPORTED_DTYPES for p in params)):
            y = _ext.C.layer_norm(x, weight, bias, eps, False)
            if y is not None:
                return y
    wide = x.dtype
    for p in params:
        wide = torch.promote_types(wide, p.dtype)
    if any(p.dtype != x.dtype for p in params):  # in the widest of the types, rounded once
        weight, bias = (None if p is None else p.to(wide) for p in (weight, bias))
        return F.layer_norm(x.to(wide), x.shape[-1:], weight, bias, eps).to(x.dtype)
    return F.layer_norm(x, x.shape[-1:], weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same constructor arguments, parameters and state_dict)
    on ``layer_norm``; ``use_fused_kernel=False`` selects torch's."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None, use_fused_kernel: bool = True):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        self._fused_requested = use_fused_kernel

    def forward(self, x: Tensor) -> Tensor:
        shape = self.normalized_shape
        if not self._fused_requested or not shape or tuple(x.shape[-len(shape):]) != tuple(shape):
            return super().forward(x)  # torch's, or its error for the shape
        if len(shape) == 1:
            return layer_norm(x, self.weight, self.bias, self.eps)
        # several dimensions are one: each row is contiguous in the flat view
        flat = [None if p is None else p.flatten() for p in (self.weight, self.bias)]
        return layer_norm(x.flatten(-len(shape)), *flat, self.eps).reshape(x.shape)
