"""The global norm of a set of gradients, and clipping by it.

What a training loop does between the backward pass and the optimizer, with
the names and arithmetic of ``torch.nn.utils``: the reference has no training
loop (its users take torch's).  Kernel path (bf16 or fp32 GPU tensors, norms of
order 1, 2 and inf): ``genie_tk._C.grad_norm``, ``grad_clip`` and
``grad_clip_with_norm``; the squares and sums are 64-bit there, the norm is an
fp32 value on the GPU, and nothing waits for the host.  Other tensors and
orders run the same formulas in PyTorch.  All tensors of a call are on one
device.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from genie_tk import _dispatch, _ext

_EPS = 1e-6  # torch.nn.utils' addend of the norm


def _kernels(like: Tensor, norm_type: float):
    """The extension, where the kernels have this norm and ``like`` is on a GPU
    (whether every tensor is one for them is for the extension to see)."""
    if not like.is_cuda or norm_type not in (1.0, 2.0, math.inf):
        return None
    if _ext.C is None:
        _ext.missing("gradients")
    return _ext.C


def _check(tensors: Sequence[Tensor], what: str) -> None:
    device = tensors[0].device
    for t in tensors:
        if t.layout != torch.strided:
            raise ValueError(f"{what}: sparse gradients are not supported")
        if t.is_complex() or not t.is_floating_point():
            raise ValueError(f"{what}: gradients must be real floating-point tensors, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{what}: gradients on {device} and {t.device}")


def _check_max_norm(max_norm: float, what: str) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be >= 0, got {max_norm}")
    return max_norm


def _norm_dtype(tensors: Sequence[Tensor]) -> torch.dtype:
    return torch.float64 if any(t.dtype == torch.float64 for t in tensors) else torch.float32


def _norm_pytorch(tensors: Sequence[Tensor], p: float) -> Tensor:
    wide = [t.detach().double().flatten() for t in tensors if t.numel()]
    if not wide:
        return tensors[0].new_zeros((), dtype=_norm_dtype(tensors))
    each = torch.stack([torch.linalg.vector_norm(w, p) for w in wide])
    return torch.linalg.vector_norm(each, p).to(_norm_dtype(tensors))


def _share_memory(a: Tensor, b: Tensor) -> bool:
    """Whether two strided tensors share a byte: whether the distance of their
    addresses is a sum of c_s s over the distinct strides s (1 for the bytes of a
    value), each c_s in a range that the sizes give.  Searched from the largest
    stride down, which leaves few c_s to try where strides nest; past 2^16 tries
    the answer is yes."""
    axes: Dict[int, List[int]] = {}
    for t, sign in ((a, 1), (b, -1)):
        size = t.element_size()
        for n, stride in [(n, s * size) for n, s in zip(t.shape, t.stride()) if s] + [(size, 1)]:
            bounds = axes.setdefault(stride, [0, 0])
            bounds[sign > 0] += sign * (n - 1)
    order = sorted(axes.items(), reverse=True)
    low, high = [0], [0]  # of the sum from each axis on
    for stride, (lo, hi) in reversed(order):
        low.insert(0, low[0] + lo * stride)
        high.insert(0, high[0] + hi * stride)
    tries = 1 << 16

    def reach(k: int, to: int) -> bool:
        nonlocal tries
        if not low[k] <= to <= high[k]:
            return False
        if k == len(order):
            return True
        stride, (lo, hi) = order[k]
        for c in range(max(lo, -((high[k + 1] - to) // stride)), min(hi, (to - low[k + 1]) // stride) + 1):
            tries -= 1
            if tries < 0 or reach(k + 1, to - c * stride):
                return True
        return False

    return reach(0, b.data_ptr() - a.data_ptr())


def _check_apart(tensors: Sequence[Tensor], outs: Sequence[Tensor]) -> None:
    """Raises RuntimeError where a tensor of ``outs``, which are written, shares
    memory with another one or with another one's gradient, or is expanded, as
    the kernels' calls do: before anything is written."""
    pieces = []  # (begin, end, tensor, index, written)
    for i, (t, o) in enumerate(zip(tensors, outs)):
        for v, written in ((o, True),) if t is o else ((o, True), (t, False)):
            if written and any(s == 0 and n > 1 for n, s in zip(v.shape, v.stride())):
                raise RuntimeError("a tensor that is written is expanded: several of its values are one")
            if v.numel() and v.device.type != "meta":
                end = 1 + sum((n - 1) * s for n, s in zip(v.shape, v.stride()))
                pieces.append((v.data_ptr(), v.data_ptr() + end * v.element_size(), v, i, written))
    pieces.sort(key=lambda p: p[0])
    reaching: list = []
    for p in pieces:
        reaching = [q for q in reaching if q[1] > p[0]]
        for q in reaching:
            if q[3] != p[3] and (q[4] or p[4]) and _share_memory(q[2], p[2]):
                raise RuntimeError("a tensor that is written overlaps another (or is given twice)")
        reaching.append(p)


def _clip_pytorch(tensors: Sequence[Tensor], outs: Sequence[Tensor], max_norm: float, norm: Tensor) -> None:
    _check_apart(tensors, outs)
    coef = (max_norm / (norm.double() + _EPS)).clamp(max=1.0)
    with torch.no_grad():
        for t, o in zip(tensors, outs):
            # the product in 32 bits at least, then rounded to the output's type
            wide = t.double() if t.dtype == torch.float64 else t.float()
            o.copy_(wide * coef.to(wide.dtype))


def grad_norm(tensors: Iterable[Tensor], norm_type: float = 2.0) -> Tensor:
    """``(sum |g|^p)^(1/p)`` over every value of ``tensors``, ``p = norm_type``
    (the largest |g| for ``inf``): a scalar on their device, fp32 (fp64 where one
    of them is).  No tensors give 0."""
    tensors = list(tensors)
    norm_type = float(norm_type)
    if not tensors:
        return torch.zeros(())
    C = _kernels(tensors[0], norm_type)
    norm = None if C is None else C.grad_norm(tensors, norm_type, False)
    if norm is not None:
        return norm
    _check(tensors, "grad_norm")
    return _norm_pytorch(tensors, norm_type)


def clip_grads(grads: Iterable[Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[Tensor]] = None) -> Tuple[Tensor, List[Tensor]]:
    """``(norm, clipped)``: every gradient times ``min(1, max_norm / (norm +
    1e-6))``.  ``grads`` are left as they are; the products, formed in fp32, are
    rounded to ``out``, tensors of the same shapes in bf16 or fp32 (fp32 ones hold
    the gradients of fp32 master weights), or to new ones like ``grads``."""
    grads = list(grads)
    norm_type, max_norm = float(norm_type), _check_max_norm(max_norm, "clip_grads")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"clip_grads: {len(out)} outputs for {len(grads)} gradients")
    if not grads:
        return torch.zeros(()), []
    outs = [torch.empty_like(g) for g in grads] if out is None else list(out)
    C = _kernels(grads[0], norm_type)
    norm = None if C is None else C.grad_clip(grads, outs, max_norm, norm_type, False)
    if norm is not None:
        return norm, outs
    _check(grads, "clip_grads")
    _check(outs, "clip_grads")
    for g, o in zip(grads, outs):
        if g.shape != o.shape or g.device != o.device:
            raise ValueError(f"clip_grads: an output is {tuple(o.shape)} on {o.device} for a gradient "
                             f"{tuple(g.shape)} on {g.device}")
    norm = _norm_pytorch(grads, norm_type)
    _clip_pytorch(grads, outs, max_norm, norm)
    return norm, outs


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> Tensor:
    """Clips the gradients of ``parameters`` in place by their global norm and
    returns the norm (fp32, before the clipping), as
    ``torch.nn.utils.clip_grad_norm_``.  Parameters without a gradient are
    passed over.  ``error_if_nonfinite`` looks at the norm on the host first (it
    waits for the GPU) and raises RuntimeError with the gradients untouched.
    ``foreach`` is accepted for torch's signature and changes nothing: the kernels
    take all gradients in one launch."""
    max_norm, norm_type = _check_max_norm(max_norm, "clip_grad_norm_"), float(norm_type)
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    if parameters and not error_if_nonfinite:
        C = _kernels(parameters[0], norm_type)
        norm = None if C is None else C.grad_clip_parameters(parameters, max_norm, norm_type)
        if norm is not None:
            return norm
    grads = _grads_of(parameters)
    if not grads:
        return torch.zeros(())
    norm = grad_norm(grads, norm_type)
    if error_if_nonfinite and not math.isfinite(float(norm)):
        raise RuntimeError(f"clip_grad_norm_: the gradients' norm of order {norm_type} is {float(norm)}")
    _clip_with_norm(grads, max_norm, norm)
    return norm


def clip_grads_with_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float,
                          total_norm: Tensor, foreach: Optional[bool] = None) -> None:
    """Clips the gradients of ``parameters`` in place by a given norm: one over
    the shards of several processes, say, joined from their ``grad_norm``.
    ``foreach`` as in ``clip_grad_norm_``."""
    max_norm = _check_max_norm(max_norm, "clip_grads_with_norm_")
    grads = _grads_of(parameters)
    if not grads:
        return
    _check(grads, "clip_grads_with_norm_")
    if total_norm.numel() != 1:
        raise ValueError("clip_grads_with_norm_: total_norm must be one value")
    _clip_with_norm(grads, max_norm, total_norm.detach().to(device=grads[0].device, dtype=_norm_dtype(grads)))


def _clip_with_norm(grads: Sequence[Tensor], max_norm: float, total_norm: Tensor) -> None:
    if all(g.is_cuda and g.dtype in _dispatch.SUPPORTED_DTYPES for g in grads):
        C = _kernels(grads[0], 2.0)
        if C is not None:
            C.grad_clip_with_norm(grads, None, max_norm, total_norm)
            return
    _clip_pytorch(grads, grads, max_norm, total_norm)


def _grads_of(parameters: Union[Tensor, Iterable[Tensor]]) -> List[Tensor]:
    if isinstance(parameters, Tensor):
        parameters = (parameters,)
    return [p.grad for p in parameters if p.grad is not None]
