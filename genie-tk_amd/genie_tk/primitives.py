"""Linear layer with AlphaFold-style initialisers, gated multi-head attention,
LayerNorm, group norm and dropout.

API and semantics of ``src/genie_tk/primitives.py`` in the reference:
``_init_weights`` (:17-40), ``Linear`` (:43-62), ``Attention`` (:65-178).
``LayerNorm`` and ``layer_norm`` are additions: torch's LayerNorm with the
forward and the backward pass on the HIP kernels.  So are ``GroupNorm`` and
``group_norm`` (channels last, with an activation and a mask) and ``dropout``
(the mask of a counter-based generator, never stored).
"""
from __future__ import annotations

import math
import operator
from typing import List, Optional, Union

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


def _autocast_fp32(x: Tensor, *params: Optional[Tensor]) -> List[Optional[Tensor]]:
    """What torch's autocast makes of a norm's arguments on the GPU."""
    if not (x.is_cuda and torch.is_autocast_enabled("cuda")):
        return [x, *params]
    return [t.float() if t is not None and t.is_floating_point() and t.dtype != torch.float64 else t
            for t in (x, *params)]


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
    x, weight, bias = _autocast_fp32(x, weight, bias)
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


# the codes of genie_tk._C's group norm
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}
_GROUP_NORM_CHANNELS = 1 << 24  # what its kernels take


def _group_norm_pytorch(x: Tensor, num_groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                        activation: Optional[str], mask: Optional[Tensor]) -> Tensor:
    """In the widest of the types and at least fp32, rounded once."""
    wide = torch.promote_types(x.dtype, torch.float32)
    for p in (weight, bias):
        if p is not None:
            wide = torch.promote_types(wide, p.dtype)
    B, C = x.shape[0], x.shape[-1]
    P = math.prod(x.shape[1:-1])  # also where another size is 0
    xf = x.to(wide).reshape(B, P, num_groups, C // num_groups)
    if mask is None:
        live, count = None, max(P * xf.shape[3], 1)
    else:
        live = (mask != 0).reshape(B, P, 1, 1)
        count = (live.sum((1, 2, 3), keepdim=True) * xf.shape[3]).clamp(min=1)

    def only(v: Tensor) -> Tensor:
        return v if live is None else torch.where(live, v, v.new_zeros(()))

    def mean(v: Tensor) -> Tensor:
        return (v.sum((1, 3), keepdim=True, dtype=torch.float64) / count).to(wide)

    # the mean is rounded by its own size; what is left of it, by the values' spread
    d = only(xf)
    d = only(d - mean(d))
    d = only(d - mean(d))
    y = d * torch.rsqrt(mean(d.square()) + eps)
    if weight is not None:
        y = y * weight.to(wide).view(num_groups, -1)
    if bias is not None:
        y = y + bias.to(wide).view(num_groups, -1)
    if activation is not None:
        y = F.silu(y) if activation == "silu" else F.gelu(y)
    return only(y).to(x.dtype).reshape(x.shape)


def group_norm(x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None, mask: Optional[Tensor] = None) -> Tensor:
    """Group norm of channels-last ``x`` ([B, ..., C]) with optional ``weight`` and
    ``bias`` ([C]) and an ``activation`` behind it (None, "silu" or "gelu", the exact
    one), differentiable once.

    A sample's group of C / ``num_groups`` channels is normalised over all of the
    sample's positions; [B, C] normalises each row's groups by themselves, and
    ``num_groups`` = C each channel (instance norm).  With a ``mask`` (broadcast to
    x's shape without its channels; no gradient) only positions where it is not 0
    count: elsewhere the output and dL/dx are 0, whatever x and dL/dy hold there.  A
    sample without any is all 0.

    Kernel path (bf16 or fp32 GPU tensor of up to 2^24 channels, parameters in bf16 or
    fp32, also mixed): ``genie_tk._C.group_norm``.  The output and dL/dx have the type
    of ``x``, the parameters' gradients their own; sums and statistics are held in fp32
    or more.  Positions that lie one stride apart (a slice of wider channels) are read
    as they are.  Other tensors, and those with a forward-mode tangent, run the same formula
    in PyTorch.  Under autocast GPU tensors narrower than fp32 are taken to fp32
    first, as torch's group norm takes them, and so is the output."""
    if x.dim() < 2:
        raise ValueError(f"group_norm: x must be [B, ..., C], got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"group_norm: {C} channels in {num_groups} groups")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"group_norm: activation must be None, 'silu' or 'gelu', got {activation!r}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and p.shape != (C,):
            raise ValueError(f"group_norm: {name} must be [{C}], got {tuple(p.shape)}")
    if mask is not None:
        mask = mask.detach().expand(x.shape[:-1])
    x, weight, bias = _autocast_fp32(x, weight, bias)
    if x.is_cuda:
        if _ext.C is None or not torch.cuda.is_available():
            _ext.missing("group_norm")
        elif (x.dtype in _dispatch.SUPPORTED_DTYPES and C <= _GROUP_NORM_CHANNELS
              and all(p is None or p.dtype in _dispatch.SUPPORTED_DTYPES for p in (weight, bias))):
            y = _ext.C.group_norm(x, num_groups, weight, bias, eps, _ACTIVATIONS[activation], mask, False)
            if y is not None:
                return y
    return _group_norm_pytorch(x, num_groups, weight, bias, eps, activation, mask)


class GroupNorm(nn.GroupNorm):
    """``nn.GroupNorm`` (same parameters and state_dict) over channels-last tensors
    on ``group_norm``, with its ``activation`` and ``forward(x, mask=None)``;
    ``use_fused_kernel=False`` selects the PyTorch path."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 device=None, dtype=None, activation: Optional[str] = None, use_fused_kernel: bool = True):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        if activation not in _ACTIVATIONS:
            raise ValueError(f"GroupNorm: activation must be None, 'silu' or 'gelu', got {activation!r}")
        self.activation = activation
        self._fused_requested = use_fused_kernel

    def extra_repr(self) -> str:
        return super().extra_repr() + f", activation={self.activation!r}"

    def forward(self, x: Tensor, mask: Optional[Tensor] = None) -> Tensor:
        if x.dim() < 2 or x.shape[-1] != self.num_channels:
            raise ValueError(f"GroupNorm: x must be [B, ..., {self.num_channels}], got {tuple(x.shape)}")
        if self._fused_requested:
            return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation, mask)
        if mask is not None:
            mask = mask.detach().expand(x.shape[:-1])
        x, weight, bias = _autocast_fp32(x, self.weight, self.bias)
        return _group_norm_pytorch(x, self.num_groups, weight, bias, self.eps, self.activation, mask)


_U32 = 0xFFFFFFFF
_U64 = 0xFFFFFFFFFFFFFFFF


def _signed(value: int) -> int:
    """The int64 with the low 64 bits of ``value``."""
    value = operator.index(value) & _U64
    return value - (1 << 64) if value >> 63 else value


def dropout_mask(shape, p: float, seed: Union[int, Tensor], offset: int = 0, shared_dim: Optional[int] = None,
                 device=None) -> Tensor:
    """The mask that ``dropout`` applies to an x of ``shape``: True where a value is
    kept, of size 1 along ``shared_dim``.  In PyTorch, on any device.

    x is seen as [outer, shared, inner].  Value r of outer index o has 16 bits of
    its own, half r % 2 (low first) of word r % 8 // 2 of Philox4x32-10 (J. Salmon,
    M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC
    2011) at counter o * ceil(inner / 8) + r // 8 (low 64 bits) and ``offset`` (high
    64 bits) under the key ``seed``; it is kept where they are at least
    round(65536 p)."""
    shape = list(shape)
    outer, inner = 1, math.prod(shape)
    if shared_dim is not None:
        dim = range(len(shape))[shared_dim]
        outer, inner = math.prod(shape[:dim]), math.prod(shape[dim + 1:])
        shape[dim] = 1
    if isinstance(seed, Tensor):
        device = seed.device if device is None else device
        key = seed.detach().reshape(1).to(device)
    else:
        # a fill, which a captured graph may hold
        key = torch.full((1,), _signed(seed), dtype=torch.int64, device=device)
    blocks = (inner + 7) // 8
    c0 = torch.arange(outer * blocks, device=device)
    c1 = c0 >> 32
    c0 = c0 & _U32
    offset = operator.index(offset)
    c2, c3 = torch.full_like(c0, offset & _U32), torch.full_like(c0, offset >> 32 & _U32)
    k0, k1 = key & _U32, key >> 32 & _U32
    for _ in range(10):  # products wrap at 64 bits, whose halves are those of unsigned ones
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & _U32) ^ c1 ^ k0, p1 & _U32, (p0 >> 32 & _U32) ^ c3 ^ k1, p0 & _U32
        k0, k1 = k0 + 0x9E3779B9 & _U32, k1 + 0xBB67AE85 & _U32
    bits = torch.stack([h for w in (c0, c1, c2, c3) for h in (w & 0xFFFF, w >> 16)], -1)
    keep = bits.view(outer, blocks * 8)[:, :inner] >= round(65536 * p)
    return keep.reshape(shape)


def dropout(x: Tensor, p: float, seed: Union[int, Tensor], offset: int = 0, shared_dim: Optional[int] = None,
            residual: Optional[Tensor] = None) -> Tensor:
    """``residual + dropout(x)`` (without ``residual``: ``dropout(x)``), the mask drawn
    from a counter-based generator and never stored: the backward pass draws it
    again.  ``dropout_mask`` is the mask.

    ``seed`` (64 bits) and ``offset`` (64 bits: the layer, the place in it) choose the
    mask; equal ones give equal masks on every device and in every type.  A ``seed``
    tensor (one int64 value on x's device) is read when the kernel runs, so that a
    captured graph draws another mask when the tensor has changed; it must not change
    between a forward pass and its backward.  With ``shared_dim`` one mask holds for
    all indices of that dimension.  Each value is dropped with probability t / 65536,
    t = round(65536 p), and what is kept is scaled by 65536 / (65536 - t).  Dropped
    values count for nothing, also where they are not finite.  The result has the
    wider of the types of x and residual and is rounded once.

    Kernel path (bf16 and fp32 GPU tensors): ``genie_tk._C.dropout``, differentiable
    any number of times.  Other tensors, and those with a forward-mode tangent, run
    the same formula in PyTorch, where the product is rounded to fp32 before the sum:
    the kernel has one fused multiply-add, so a sum in the middle between two results
    may go to the other one.  Whether a module is training is the caller's to ask."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    if shared_dim is not None and not -x.dim() <= shared_dim < x.dim():
        raise IndexError(f"dropout: shared_dim {shared_dim} of {x.dim()} dimensions")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"dropout: residual {tuple(residual.shape)} for x {tuple(x.shape)}")
    drawn = isinstance(seed, Tensor)
    if drawn and (seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device):
        raise ValueError("dropout: a seed tensor is one int64 value on x's device")
    kind = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
    if x.is_cuda:
        if _ext.C is None or not torch.cuda.is_available():
            _ext.missing("dropout")
        elif (x.dtype in _dispatch.SUPPORTED_DTYPES
              and (residual is None or residual.dtype in _dispatch.SUPPORTED_DTYPES)):
            wide = None if residual is None else residual.to(kind)
            key = 0 if drawn else operator.index(seed) & _U64
            y = _ext.C.dropout(x, p, key, operator.index(offset) & _U64, shared_dim, wide, seed if drawn else None,
                               False)
            if y is not None:
                return y
    wide = torch.promote_types(kind, torch.float32)
    t = round(65536 * p)
    keep = dropout_mask(x.shape, p, seed, offset, shared_dim, x.device)
    scaled = x.to(wide) * (65536 / (65536 - t) if t < 65536 else 0.0)
    y = torch.where(keep, scaled, scaled.new_zeros(()))
    return (y if residual is None else y + residual.to(wide)).to(kind)
