"""Group norm with an activation, channels last (genie_tk.primitives.group_norm /
GroupNorm, genie_tk._C.group_norm_forward / group_norm_backward, gtk_group_norm_*):
the oracle, the PyTorch path and the refusals on the CPU, the kernels against the
64-bit oracle on the GPU.

Tolerances.  u = 2^-24, half_t = finfo(t).eps / 2 of the output's type.  Statistics
are sums of x and x^2 in 64 bits, at most CHAIN additions one behind the other:
* the mean is kept to 48 bits, d = x - mean is off by its two roundings; with M the
  group's largest |x| the variance is off by CHAIN 2^-53 M^2 and r by half of that
  times r^2, h = d r (rounded, as r and r w are) by eh = 8 u |h| + 4 u^2 M r +
  CHAIN 2^-53 M^2 r^2 |h|;
* z = h w + b by ez = |w| eh + 2 u (|h w| + |b|);
* silu: e^-z has the rounding of its argument, |z| u, and an ulp or two for the
  exponential, the sum and the quotient: (|z| + 8) u of the result.  gelu: e^(-z^2/2)
  by z^2 u, and the polynomial, the quotient and the products: (z^2 + 16) u of it.  In
  bf16 its polynomial has fewer terms and is 3.5e-5 of its value off (2^-14 allowed,
  a 64th of the result's rounding).
  Their slopes are at most 1.13, the slopes' own at most 0.5 and 0.8;
* fp32 sums of the backward pass: at most CHAIN additions one behind the other.
Each result is rounded once to its own type."""
import ctypes
import os

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from genie_tk import _ext
from genie_tk.primitives import GroupNorm, dropout, group_norm
from oracle import train_ops

U = 2.0 ** -24
EPS = 1e-5
CHAIN = 600
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().double().cpu().numpy()


def values(shape, seed, dtype, device="cpu", mean=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen) * 1.5 + mean * torch.randn(shape[-1], generator=gen)
    return x.to(dtype).to(device)


def params(C, seed, dtype, device="cpu"):
    gen = torch.Generator().manual_seed(1000 + seed)
    w = 1 + 0.3 * torch.randn(C, generator=gen)
    b = 0.5 * torch.randn(C, generator=gen)
    return w.to(dtype).to(device), b.to(dtype).to(device)


def bounds(x, dy, G, w, b, act, mask, eps=EPS, narrow=False):
    """Allowed |errors| of y, dx, dweight, dbias before the last rounding."""
    _, h, z, r, live = train_ops.group_norm(x, G, w, b, eps, act, mask)
    B, P, C = x.shape
    wa = 1.0 if w is None else np.abs(w)
    ba = 0.0 if b is None else np.abs(b)

    def grouped(t, f):  # f over a sample's group, for each of its channels
        t = np.where(live, t, 0.0).reshape(B, P, G, C // G)
        return np.repeat(f(t, (1, 3)), C // G, axis=1).reshape(B, 1, C)

    M = grouped(np.abs(np.where(live, x, 0.0)), lambda t, a: t.max(a))
    eh = 8 * U * np.abs(h) + 4 * U * U * M * r + CHAIN * 2.0 ** -53 * (M * r) ** 2 * np.abs(h)
    ez = wa * eh + 2 * U * (np.abs(h) * wa + ba)
    a, s = train_ops.activation(z, act)
    own = {None: 0.0 * z, "silu": np.abs(z) + 8, "gelu": z * z + 16}[act] * U
    if narrow and act == "gelu":
        own = own + 2.0 ** -14
    ey = np.abs(s) * ez + ez * ez + own * np.abs(a)
    bend = {None: 0.0, "silu": 0.5, "gelu": 0.8}[act]
    # the slope is a sum of two terms, each off by its own share
    gate = {None: 0.0 * z, "silu": np.abs(s) + np.abs(z) * np.exp(-np.abs(z)), "gelu": np.abs(s) + np.abs(z) *
            np.exp(-0.5 * z * z)}[act]
    es = bend * ez + 2 * own * gate
    dyl = np.where(live, np.nan_to_num(dy), 0.0)
    dz = dyl * s
    edz = np.abs(dyl) * es + 2 * U * np.abs(dz)
    g = dz * (1.0 if w is None else w)
    eg = wa * edz + 2 * U * np.abs(g)
    count = np.maximum(live.sum(1, keepdims=True) * (C // G), 1)
    mean = lambda t: grouped(t, lambda v, ax: v.sum(ax)) / count  # noqa: E731
    ec1 = mean(eg) + CHAIN * U * mean(np.abs(g))
    ec2 = mean(eg * np.abs(h) + np.abs(g) * eh) + CHAIN * U * mean(np.abs(g * h))
    c1, c2 = np.abs(mean(g)), np.abs(mean(g * h))
    er = 2 * U + CHAIN * 2.0 ** -53 * (M * r) ** 2
    edx = r * (eg + ec1 + np.abs(h) * ec2 + eh * c2 + (er + 4 * U) * (np.abs(g) + c1 + np.abs(h) * c2))
    ew = (edz * np.abs(h) + np.abs(dz) * eh).sum((0, 1)) + CHAIN * U * np.abs(dz * h).sum((0, 1))
    eb = edz.sum((0, 1)) + CHAIN * U * np.abs(dz).sum((0, 1))
    return ey, edx, ew, eb


def check(got, ref, err, what):
    dtype = got.dtype
    got = np64(got).reshape(ref.shape)
    assert np.isfinite(got).all(), f"{what}: non-finite"
    excess = np.abs(got - ref) - (half(dtype) * np.abs(ref) + (1 + half(dtype)) * err + 1e-36)
    assert (excess <= 0).all(), (f"{what}: {int((excess > 0).sum())} of {excess.size} out of tolerance, worst by "
                                 f"{excess.max():.3e}, error {np.abs(got - ref).max():.3e}")


def check_all(x, dy, G, w, b, act, mask, y, dx=None, dw=None, db=None, eps=EPS):
    B, C = x.shape[0], x.shape[-1]
    xn, dn = np64(x).reshape(B, -1, C), np64(dy).reshape(B, -1, C)
    wn, bn = (None if t is None else np64(t) for t in (w, b))
    mn = None if mask is None else np64(mask).reshape(B, -1)
    if mn is not None:  # what is masked may be anything
        xn, dn = (np.where(mn[:, :, None] != 0, t, 0.0) for t in (xn, dn))
    ey, edx, ew, eb = bounds(xn, dn, G, wn, bn, act, mn, eps, x.dtype == torch.bfloat16)
    check(y, train_ops.group_norm(xn, G, wn, bn, eps, act, mn)[0], ey, "y")
    dxr, dwr, dbr, _ = train_ops.group_norm_grads(xn, dn, G, wn, bn, eps, act, mn)
    for got, ref, err, what in ((dx, dxr, edx, "dx"), (dw, dwr, ew, "dweight"), (db, dbr, eb, "dbias")):
        if got is not None:
            check(got, ref, err, what)


def run(x, G, w, b, dy, act=None, mask=None, eps=EPS):
    """The public path: y and the gradients of x, w, b."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = group_norm(leaves[0], G, leaves[1], leaves[2], eps, act, mask)
    got = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    return (y, *(None if t is None else next(got) for t in leaves))


def some_mask(lead, seed, device="cpu", empty=False):
    """[B, ...]: random positions, the first sample without any if `empty`."""
    gen = torch.Generator().manual_seed(seed)
    m = (torch.rand(*lead, generator=gen) < 0.7).float()
    m.view(lead[0], -1)[:, -1] = 1
    if empty:
        m[0] = 0
    return m.to(device)


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_oracle_matches_autograd_in_64_bits(act):
    x, dy = values((2, 5, 12), 0, torch.float64), values((2, 5, 12), 1, torch.float64)
    w, b = params(12, 2, torch.float64)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = F.group_norm(x.transpose(1, 2), 4, w, b, EPS).transpose(1, 2)
    y = y if act is None else F.silu(y) if act == "silu" else F.gelu(y)
    got = torch.autograd.grad(y, leaves, dy)
    args = (np64(x), np64(dy), 4, np64(w), np64(b), EPS, act)
    np.testing.assert_allclose(np64(y), train_ops.group_norm(args[0], 4, *args[3:])[0], rtol=0, atol=1e-12)
    for g, r in zip(got, train_ops.group_norm_grads(*args)):
        np.testing.assert_allclose(np64(g), r, rtol=0, atol=1e-12)


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_oracle_gradient_against_differences(act):
    x, dy, v = (np64(values((2, 7, 6), k, torch.float64)) for k in range(3))
    w, b = (np64(t) for t in params(6, 0, torch.float64))
    mask = np64(some_mask((2, 7), 3))
    f = lambda t, ww, bb: (train_ops.group_norm(t, 2, ww, bb, EPS, act, mask)[0] * dy).sum()  # noqa: E731
    dx, dw, db, _ = train_ops.group_norm_grads(x, dy, 2, w, b, EPS, act, mask)
    t = 1e-5
    for lo, hi, g in ((f(x - t * v, w, b), f(x + t * v, w, b), (dx * v).sum()),
                      (f(x, w - t * v[0, 0], b), f(x, w + t * v[0, 0], b), (dw * v[0, 0]).sum()),
                      (f(x, w, b - t * v[0, 0]), f(x, w, b + t * v[0, 0]), (db * v[0, 0]).sum())):
        assert abs((hi - lo) / (2 * t) - g) < 1e-6


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("dt,pdt", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16"), ("fp32", None)])
def test_pytorch_path(dt, pdt, act, masked):
    x, dy = values((3, 4, 5, 12), 0, DT[dt]), values((3, 4, 5, 12), 1, DT[dt])
    w, b = (None, None) if pdt is None else params(12, 2, DT[pdt])
    mask = some_mask((3, 4, 5), 3, empty=True) if masked else None
    y, dx, dw, db = run(x, 3, w, b, dy, act, mask)
    assert y.dtype == dx.dtype == x.dtype and y.shape == x.shape
    # torch's functions and its order of the sums: looser than the kernels
    mn = None if mask is None else np64(mask).reshape(3, -1)
    wn, bn = (None if t is None else np64(t) for t in (w, b))
    args = (3, wn, bn, EPS, act, mn)
    xn, dn = np64(x).reshape(3, 20, 12), np64(dy).reshape(3, 20, 12)
    refs = [train_ops.group_norm(xn, *args)[0], *train_ops.group_norm_grads(xn, dn, *args)[:3]]
    for got, ref in zip((y, dx, dw, db), refs):
        if got is not None:
            np.testing.assert_allclose(np64(got).reshape(ref.shape), ref, rtol=2 * half(got.dtype) + 1e-5, atol=1e-4)
    if masked:
        assert not y[mask == 0].any() and not dx[mask == 0].any() and not y[0].any()


def test_pytorch_path_keeps_64_bits():
    x = values((2, 9, 8), 0, torch.float64)
    w, b = params(8, 1, torch.float32)
    ref = train_ops.group_norm(np64(x), 2, np64(w), np64(b), EPS, "gelu")[0]
    np.testing.assert_allclose(np64(group_norm(x, 2, w, b, EPS, "gelu")), ref, rtol=0, atol=1e-12)


def test_masked_places_may_hold_anything():
    x, dy = values((2, 6, 8), 0, torch.float32), values((2, 6, 8), 1, torch.float32)
    w, b = params(8, 2, torch.float32)
    mask = some_mask((2, 6), 3)
    one = run(x, 2, w, b, dy, "silu", mask)
    for v in (float("nan"), float("inf"), torch.finfo(torch.float32).min):
        x2, dy2 = (torch.where(mask.unsqueeze(-1) != 0, t, v) for t in (x, dy))
        assert all(torch.equal(p, q) for p, q in zip(one, run(x2, 2, w, b, dy2, "silu", mask)))
    # any value but 0 counts, of any type, and masks broadcast
    assert torch.equal(one[0], group_norm(x, 2, w, b, EPS, "silu", mask * 0.25))
    assert torch.equal(one[0], group_norm(x, 2, w, b, EPS, "silu", mask.bool()))
    row = some_mask((1, 6), 4)
    assert torch.equal(group_norm(x, 2, w, b, EPS, "silu", row), group_norm(x, 2, w, b, EPS, "silu", row.expand(2, 6)))


def test_module():
    m = GroupNorm(4, 12, activation="silu")
    t = torch.nn.GroupNorm(4, 12)
    t.load_state_dict(m.state_dict())
    assert isinstance(m, torch.nn.GroupNorm) and "activation='silu'" in repr(m)
    x = values((2, 5, 6, 12), 0, torch.float32)
    ref = F.silu(t(x.movedim(-1, 1))).movedim(1, -1)
    torch.testing.assert_close(m(x), ref, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(GroupNorm(12, 12, affine=False)(x), torch.nn.InstanceNorm2d(12)(x.movedim(-1, 1)).movedim(1, -1),
                               rtol=1e-5, atol=1e-5)
    assert torch.equal(m(x), GroupNorm(4, 12, activation="silu", use_fused_kernel=False)(x))
    mask = some_mask((2, 5, 6), 1)
    assert torch.equal(m(x, mask), group_norm(x, 4, m.weight, m.bias, m.eps, "silu", mask))


def test_refusals():
    x = torch.ones(2, 3, 12)
    for groups in (0, -1, 5, 24):
        with pytest.raises(ValueError, match="groups"):
            group_norm(x, groups)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 3, activation="relu")
    with pytest.raises(ValueError, match="activation"):
        GroupNorm(3, 12, activation="tanh")
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, 3, torch.ones(6))
    with pytest.raises(ValueError, match="bias"):
        group_norm(x, 3, None, torch.ones(12, 1))
    with pytest.raises(ValueError, match="x must be"):
        group_norm(torch.ones(12), 3)
    for bad in (torch.ones(2, 4), torch.ones(2, 3, 12)):
        with pytest.raises(RuntimeError):
            group_norm(x, 3, mask=bad)
    with pytest.raises(ValueError, match="x must be"):
        GroupNorm(3, 12)(torch.ones(2, 12, 3))
    if _ext.C is not None:
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            _ext.C.group_norm(x, 3)


LIB = os.path.join(os.path.dirname(os.path.abspath(_ext.__file__)), "libgenie_tk_hip.so")
i64, sz, vp, fp, ci = ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float, ctypes.c_int


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    L = ctypes.CDLL(LIB)
    L.gtk_last_error.restype = ctypes.c_char_p
    for name in ("gtk_group_norm_workspace_size", "gtk_group_norm_backward_workspace_size"):
        getattr(L, name).restype = sz
        getattr(L, name).argtypes = [i64, i64, i64, i64, ci]
    L.gtk_group_norm_forward.argtypes = [vp, i64, vp, vp, vp, vp, vp, ci, i64, i64, i64, i64, fp, ci, ci, vp, sz, vp]
    L.gtk_group_norm_backward.argtypes = [vp, i64, vp, vp, i64, vp, vp, vp, ci, vp, vp, vp, i64, i64, i64, i64, ci, ci,
                                          vp, sz, vp]
    return L


BAD_SHAPES = [(-1, 4, 8, 2, 0), (2, 0, 8, 2, 0), (2, -1, 8, 2, 0), (2, 4, 0, 1, 0), (2, 4, 8, 3, 0), (2, 4, 8, 0, 0),
              (2, 4, 8, 16, 0), (2, 4, 8, 2, 2), (2, 4, (1 << 24) + 2, 2, 0), (1, 1 << 46, 8, 2, 0),
              (1 << 40, 1 << 20, 8, 2, 0)]


def test_c_refusals(lib):
    q = 4096  # never dereferenced: every call below is refused on the host, or has nothing to do
    big = 1 << 40
    fwd = lambda s=(2, 4, 8, 2, 0), x=q, y=q, st=q, xs=8, pdt=0, act=0, n=big, ws=q: lib.gtk_group_norm_forward(  # noqa: E731
        x, xs, None, y, st, None, None, pdt, *s[:4], EPS, act, s[4], ws, n, None)
    bwd = lambda s=(2, 4, 8, 2, 0), x=q, dy=q, st=q, xs=8, ds=8, pdt=0, act=0, n=big, dx=q, dw=q, ws=q: (  # noqa: E731
        lib.gtk_group_norm_backward(x, xs, None, dy, ds, st, None, None, pdt, dx, dw, None, *s[:4], act, s[4], ws, n,
                                    None))
    assert [fwd(s) for s in BAD_SHAPES] == [1] * len(BAD_SHAPES)
    assert [bwd(s) for s in BAD_SHAPES] == [1] * len(BAD_SHAPES)
    for name in ("gtk_group_norm_workspace_size", "gtk_group_norm_backward_workspace_size"):
        assert [getattr(lib, name)(*s) for s in BAD_SHAPES] == [0] * len(BAD_SHAPES)
    assert [fwd(x=None), fwd(y=None), fwd(st=None), fwd(xs=-8), fwd(pdt=2), fwd(act=3), fwd(act=-1)] == [1] * 7
    assert [bwd(x=None), bwd(dy=None), bwd(st=None), bwd(xs=-8), bwd(ds=-1), bwd(pdt=2), bwd(act=3)] == [1] * 7
    assert b"null pointer" in (fwd(x=None), lib.gtk_last_error())[1]
    assert fwd((0, 4, 8, 2, 0), x=None, y=None) == 0 and bwd(dx=None, dw=None) == 0
    assert bwd((0, 4, 8, 2, 0), x=None, dy=None, st=None, dw=None) == 0
    for s in ((1, 1 << 18, 128, 32, 1), (2, 100, 64, 4, 0), (1, 1 << 20, 128, 8, 0)):
        for call, name in ((fwd, "gtk_group_norm_workspace_size"), (bwd, "gtk_group_norm_backward_workspace_size")):
            need = getattr(lib, name)(*s)
            if need:
                assert call(s, n=need - 1) == 3 and call(s, ws=None) == 3 and b"workspace" in lib.gtk_last_error()


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
# [B, P, C], groups: widths of a group from one channel to all, vectors that a group
# does not fill or that end inside one, planes from one position on
SHAPES = [((1, 1, 1024), 16), ((5, 1, 512), 8), ((3, 1, 7), 1), ((2, 3, 1), 1), ((2, 2, 3), 3), ((4, 5, 6), 2),
          ((2, 40, 12), 4), ((3, 64, 16), 16), ((2, 301, 20), 4), ((1, 1000, 32), 32), ((2, 256, 320), 32),
          ((1, 500, 128), 32), ((2, 777, 100), 20), ((1, 900, 1023), 33), ((3, 33, 1030), 2), ((2, 130, 2048), 32),
          ((1, 21, 8), 8), ((2, 1111, 24), 3), ((70, 16, 64), 8), ((1, 5003, 64), 1), ((2, 3001, 40), 5),
          ((1, 9001, 100), 20), ((1, 4097, 9), 3), ((300, 7, 96), 6), ((1, 600, 5000), 5), ((2, 130, 12288), 64),
          ((1, 70, 9002), 2), ((1, 3, 20000), 1), ((40, 1, 16384), 16)]


@gpu
@pytest.mark.parametrize("dt,act", [("fp32", "silu"), ("bf16", "gelu"), ("bf16", None), ("fp32", "gelu")])
@pytest.mark.parametrize("shape,G", SHAPES, ids=str)
def test_shapes(shape, G, dt, act):
    x, dy = values(shape, 0, DT[dt], "cuda"), values(shape, 1, DT[dt], "cuda")
    w, b = params(shape[-1], 2, DT[dt], "cuda")
    for mask in (None, some_mask(shape[:2], 3, "cuda", empty=shape[0] > 1)):
        print("group_norm", shape, G, dt, act, mask is not None, flush=True)
        check_all(x, dy, G, w, b, act, mask, *run(x, G, w, b, dy, act, mask))


@gpu
@pytest.mark.parametrize("shape,G", [((1, 128, 128, 128), 32), ((1, 101, 99, 100), 5), ((2, 90, 90, 64), 8),
                                     ((16, 16, 16, 320), 32), ((4096, 1, 1, 512), 8), ((1, 1, 40000, 8), 2),
                                     ((2, 50, 50, 513), 27), ((1, 64, 64, 1024), 8)], ids=str)
@pytest.mark.parametrize("dt,pdt", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "bf16"),
                                    ("bf16", None)])
def test_planes(shape, G, dt, pdt):
    x, dy = values(shape, 0, DT[dt], "cuda"), values(shape, 1, DT[dt], "cuda")
    w, b = (None, None) if pdt is None else params(shape[-1], 2, DT[pdt], "cuda")
    for act, mask in (("silu", None), (None, some_mask(shape[:-1], 3, "cuda"))):
        print("group_norm", shape, G, dt, pdt, act, flush=True)
        y, dx, dw, db = run(x, G, w, b, dy, act, mask)
        assert y.dtype == dx.dtype == x.dtype and (w is None or dw.dtype == db.dtype == w.dtype)
        check_all(x, dy, G, w, b, act, mask, y, dx, dw, db)


@gpu
def test_parameters_of_two_types_and_one_alone():
    x, dy = values((2, 200, 96), 0, torch.bfloat16, "cuda"), values((2, 200, 96), 1, torch.bfloat16, "cuda")
    w, b = params(96, 2, torch.bfloat16, "cuda")
    for ww, bb in ((w, b.float()), (w.float(), b), (w, None), (None, b), (None, b.float())):
        y, dx, dw, db = run(x, 12, ww, bb, dy, "silu")
        assert (dw is None or dw.dtype == ww.dtype) and (db is None or db.dtype == bb.dtype)
        check_all(x, dy, 12, ww, bb, "silu", None, y, dx, dw, db)


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("P,C", [(60, 24), (4000, 64), (3000, 100)])
def test_strides(P, C, dt):
    w, b = params(C, 2, DT[dt], "cuda")
    wide = values((2, P, C + 11), 0, DT[dt], "cuda")
    four = values((4, P // 4, 3 * C), 3, DT[dt], "cuda").view(4, P // 4, 3, C)
    cases = [wide[..., 3:3 + C], wide[:, ::2, 5:5 + C], wide[:1, :1, 1:1 + C].expand(2, 33, C), four[:, :, 1],
             four.transpose(0, 1), values((2, C, 50), 4, DT[dt], "cuda").transpose(1, 2)]
    for k, x in enumerate(cases):
        print("stride case", k, tuple(x.shape), x.stride(), flush=True)
        dy = torch.randn(x.shape, device="cuda").to(DT[dt])
        mask = some_mask(x.shape[:-1], 5, "cuda")
        check_all(x, dy, C // 4, w, b, "silu", mask, *run(x, C // 4, w, b, dy, "silu", mask))
        for up in (dy.transpose(0, 1).contiguous().transpose(0, 1), dy[..., :1].expand(x.shape),
                   dy[:1].expand(x.shape)):
            check_all(x, up, C // 4, w, b, None, None, *run(x, C // 4, w, b, up))


@gpu
@pytest.mark.parametrize("shape,G", [((3, 40, 24), 4), ((2, 3000, 64), 8)], ids=str)
def test_each_gradient_alone(shape, G):
    x, dy = values(shape, 0, torch.float32, "cuda"), values(shape, 1, torch.float32, "cuda")
    w, b = params(shape[-1], 2, torch.float32, "cuda")
    _, *every = run(x, G, w, b, dy, "gelu")
    for keep in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        leaves = [t.clone().requires_grad_(k in keep) for k, t in enumerate((x, w, b))]
        y = group_norm(*leaves[:1], G, *leaves[1:], EPS, "gelu")
        for k, g in zip(keep, torch.autograd.grad(y, [leaves[k] for k in keep], dy)):
            assert torch.equal(g, every[k]), (keep, k)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = group_norm(*leaves[:1], G, *leaves[1:], EPS, "gelu")
    for k in (2, 0, 1):
        g, = torch.autograd.grad(y, leaves[k], dy, retain_graph=True)
        assert torch.equal(g, every[k]), k
    C = _ext.require()
    y, stats = C.group_norm_forward(x, G, w, b, EPS, 2)
    assert C.group_norm_backward(x, dy, stats, G, w, b, 2, None, False, False, False) == [None, None, None]
    # a bias alone
    y = group_norm(x, G, None, leaves[2])
    assert torch.autograd.grad(y, leaves[2], dy)[0].shape == b.shape


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("P", [30, 5000])
def test_values_at_the_edges(P, dt):
    C, G = 32, 4
    x, dy = values((8, P, C), 0, DT[dt], "cuda"), values((8, P, C), 1, DT[dt], "cuda")
    w, b = params(C, 2, DT[dt], "cuda")
    x[0] = 3.25                       # no variance
    x[1] = 0
    x[2] = x[2] * 1e-4                # a variance below eps
    x[3] = x[3] + 4096                # far from zero
    x[4] = x[4] * 1e15
    dy[5] = 0
    dy[6] = dy[6] * 1e10
    for act in (None, "silu", "gelu"):
        y, dx, dw, db = run(x, G, w, b, dy, act)
        check_all(x, dy, G, w, b, act, None, y, dx, dw, db)
    # a value that is not finite spoils its sample's group and the sums of its channels, nothing else
    y, dx, dw, db = run(x, G, w, b, dy, "silu")
    x[7, 3, 9], x[5, P - 1, 31] = float("nan"), float("inf")
    y2, dx2, dw2, db2 = run(x, G, w, b, dy, "silu")
    spoilt = torch.zeros(8, G, dtype=torch.bool, device="cuda")
    spoilt[7, 1] = spoilt[5, 3] = True
    spoilt = spoilt.repeat_interleave(C // G, 1).unsqueeze(1).expand(8, P, C)
    for one, two in ((y, y2), (dx, dx2)):
        assert torch.equal(one[~spoilt], two[~spoilt]) and two[spoilt].isnan().all()
    cols = spoilt.any(0).any(0)
    assert torch.equal(dw[~cols], dw2[~cols]) and dw2[cols].isnan().all()


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("P", [30, 5000])
def test_large_arguments_of_the_activations(P, dt):
    """z from -1e3 to 1e3: the exponentials overflow and underflow."""
    C = 16
    x, dy = values((2, P, C), 0, DT[dt], "cuda"), values((2, P, C), 1, DT[dt], "cuda")
    w, b = params(C, 2, torch.float32, "cuda")
    w = w * torch.logspace(-1, 2.5, C, device="cuda")
    for act in ("silu", "gelu"):
        check_all(x, dy, 4, w, b, act, None, *run(x, 4, w, b, dy, act))


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,G", [((3, 50, 24), 4), ((2, 6000, 64), 8), ((2, 3001, 20), 4)], ids=str)
def test_masked_places_may_hold_anything_on_the_gpu(shape, G, dt):
    x, dy = values(shape, 0, DT[dt], "cuda"), values(shape, 1, DT[dt], "cuda")
    w, b = params(shape[-1], 2, torch.float32, "cuda")
    mask = some_mask(shape[:-1], 3, "cuda", empty=True)
    one = run(x, G, w, b, dy, "silu", mask)
    check_all(x, dy, G, w, b, "silu", mask, *one)
    assert not one[0][mask == 0].any() and not one[1][mask == 0].any()
    for v in (float("nan"), float("inf"), torch.finfo(DT[dt]).min):
        x2, dy2 = (torch.where(mask.unsqueeze(-1) != 0, t, v).to(DT[dt]) for t in (x, dy))
        assert all(torch.equal(p, q) for p, q in zip(one, run(x2, G, w, b, dy2, "silu", mask)))
    assert torch.equal(one[0], group_norm(x, G, w, b, EPS, "silu", mask.bool()))
    # a mask of ones is no mask
    full = run(x, G, w, b, dy, "silu", torch.ones_like(mask))
    assert all(torch.equal(p, q) for p, q in zip(full, run(x, G, w, b, dy, "silu")))
    # the type's lowest value where it counts: a mean and a variance that 32 bits may not hold
    x[1, 0, 0] = torch.finfo(DT[dt]).min
    y, dx, dw, db = run(x, G, w, b, dy, None, None)
    assert all(torch.isfinite(t).all() for t in (y, dx, dw, db))


@gpu
def test_no_samples_and_no_positions():
    w, b = params(16, 0, torch.float32, "cuda")
    for shape in ((0, 5, 16), (0, 16), (3, 0, 16), (2, 4, 0, 16)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        y, dx, dw, db = run(x, 4, w, b, torch.empty_like(x), "silu")
        assert y.shape == dx.shape == x.shape
        assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


@gpu
def test_gradient_against_differences():
    """Central differences of sum(y dy) of the fp32 kernels along a direction v: with
    t = 2^-6 the third-order term is below t^2 of the size of the sums of |terms|
    (times 16: three derivatives of the activation and of the division), and each
    loss is off by the error of y, over 2 t."""
    shape, G = (2, 400, 24), 4
    x, dy, v = (values(shape, k, torch.float32, "cuda", 0.0) for k in range(3))
    w, b = params(24, 2, torch.float32, "cuda")
    mask = some_mask(shape[:2], 3, "cuda")
    _, dx, dw, db = run(x, G, w, b, dy, "silu", mask)
    t = 2.0 ** -6
    loss = lambda a, ww, bb: float((group_norm(a, G, ww, bb, EPS, "silu", mask).double() * dy.double()).sum())  # noqa: E731
    size = float((dy.double().abs() * w.double().abs()).sum())
    vw, vb = torch.randn_like(w), torch.randn_like(b)
    for lo, hi, g in ((loss(x - t * v, w, b), loss(x + t * v, w, b), dx.double() * v.double()),
                      (loss(x, w - t * vw, b), loss(x, w + t * vw, b), dw.double() * vw.double()),
                      (loss(x, w, b - t * vb), loss(x, w, b + t * vb), db.double() * vb.double())):
        assert abs((hi - lo) / (2 * t) - float(g.sum())) < t * t * 16 * size


@gpu
@pytest.mark.parametrize("shape,G", [((4, 64, 64), 8), ((1, 256, 256, 128), 32)], ids=str)
def test_same_bits_on_every_call_and_stream(shape, G):
    x, dy = values(shape, 0, torch.bfloat16, "cuda"), values(shape, 1, torch.bfloat16, "cuda")
    w, b = params(shape[-1], 2, torch.float32, "cuda")
    first = run(x, G, w, b, dy, "silu")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            out.append(run(x, G, w, b, dy, "silu"))
    torch.cuda.synchronize()
    for got in out:
        assert all(torch.equal(p, q) for p, q in zip(first, got))


@gpu
def test_autocast_tangents_and_second_derivatives():
    x, dy = values((2, 30, 24), 0, torch.bfloat16, "cuda"), values((2, 30, 24), 1, torch.float32, "cuda")
    w, b = params(24, 2, torch.float32, "cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = group_norm(x, 4, w, b)
    assert y.dtype == torch.float32
    assert torch.equal(y, group_norm(x.float(), 4, w, b))
    xf = x.float().requires_grad_(True)
    g, = torch.autograd.grad(group_norm(xf, 4, w, b, EPS, "silu"), xf, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        out = ad.unpack_dual(group_norm(ad.make_dual(xf.detach(), dy), 4, w, b, EPS, "silu"))
        with pytest.raises(NotImplementedError):
            _ext.C.group_norm(ad.make_dual(xf.detach(), dy), 4)
    t = 2.0 ** -8
    num = (group_norm(xf.double() + t * dy, 4, w, b, EPS, "silu") - group_norm(xf.double() - t * dy, 4, w, b, EPS, "silu")) / (2 * t)
    assert (out.tangent - num).abs().max() < 64 * t * t


@gpu
def test_refusals_on_the_gpu():
    C = _ext.require()
    x = values((2, 6, 24), 0, torch.float32, "cuda")
    y, stats = C.group_norm_forward(x, 4)
    for call, match in ((lambda: C.group_norm(x, 5), "groups"), (lambda: C.group_norm(x, 4, activation=3), "activation"),
                        (lambda: C.group_norm(x.double(), 4), "float32 or bfloat16"),
                        (lambda: C.group_norm(x, 4, weight=torch.ones(24)), "weight is on"),
                        (lambda: C.group_norm(x, 4, mask=torch.ones(2, 6)), "mask is on"),
                        (lambda: C.group_norm(x, 4, mask=torch.ones(2, 5, device="cuda")), "mask must be"),
                        (lambda: C.group_norm_backward(x, y[:1], stats, 4), "dy must match"),
                        (lambda: C.group_norm_backward(x, y, stats[:1], 4), "stats are"),
                        (lambda: C.group_norm_backward(x, y, stats, 8), "stats are")):
        with pytest.raises(RuntimeError, match=match):
            call()
    assert group_norm(x.double(), 4).dtype == torch.float64  # the PyTorch path


@gpu
def test_more_than_2_to_the_31_values():
    """[1, P, 64] with 2^31 + 64 * 999 values, a pattern of period 4096 positions and
    a tail of ones: its statistics are known."""
    P, C, G = (1 << 25) + 999, 64, 4
    x = torch.ones(1, P, C, dtype=torch.bfloat16, device="cuda")
    period = values((4096, C), 0, torch.bfloat16, "cuda")
    x[0, :1 << 25].view(1 << 13, 4096, C).copy_(period)
    n64 = np64(period).reshape(4096, G, C // G)
    y = group_norm(x, G, activation="silu")
    total = P * (C // G)
    mean = ((n64.sum((0, 2)) * (1 << 13)) + 999 * (C // G)) / total
    var = (((n64 - mean[None, :, None]) ** 2).sum((0, 2)) * (1 << 13) + 999 * (C // G) * (1 - mean) ** 2) / total
    r = 1 / np.sqrt(var + EPS)
    for at in (0, 1 << 24, (1 << 25) - 4096):
        z = (n64 - mean[None, :, None]) * r[None, :, None]
        ref = train_ops.activation(z, "silu")[0].reshape(4096, C)
        check(y[0, at:at + 4096], ref, 64 * U * (1 + np.abs(ref)), at)
    ref = np.repeat(train_ops.activation((1 - mean) * r, "silu")[0], C // G)[None, :].repeat(999, 0)
    check(y[0, 1 << 25:], ref, 64 * U * (1 + np.abs(ref)), "tail")


@gpu
@pytest.mark.parametrize("shape,G", [((4, 64, 64), 8), ((1, 128, 128, 64), 8)], ids=str)
def test_captured_step_and_a_run_of_the_operators(shape, G):
    """Norm, activation, dropout and residual of a block, forward and backward, as a
    training step has them: captured once, replayed with other inputs and seeds, and
    equal to the eager step each time; two graphs share nothing."""
    C = shape[-1]
    x = values(shape, 0, torch.bfloat16, "cuda").requires_grad_(True)
    w, b = (t.requires_grad_(True) for t in params(C, 2, torch.float32, "cuda"))
    dy = values(shape, 1, torch.bfloat16, "cuda")
    mask = some_mask(shape[:-1], 3, "cuda")
    seed = torch.tensor([40], device="cuda")

    def step():
        h = group_norm(x, G, w, b, EPS, "silu", mask)
        y = dropout(h, 0.25, seed, 2, None, x)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    def eager(k):
        with torch.no_grad():
            x.copy_(values(shape, 10 + k, torch.bfloat16))
        seed.fill_(40 + k)
        return [t.clone() for t in step()]

    refs = [eager(k) for k in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for k in (0, 1, 2, 3, 1):
        with torch.no_grad():
            x.copy_(values(shape, 10 + k, torch.bfloat16))
        seed.fill_(40 + k)
        for graph, got in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, refs[k])), k
        values((1000,), 3, torch.float32, "cuda").square().sum().item()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_64_bit_mask_counts_what_is_not_zero(device):
    """1e-300 is 0 in fp32."""
    x = values((3, 40, 24), 61, torch.float32, device)
    mask = some_mask((3, 40), 62, device).double()
    w, b = params(24, 63, torch.float32, device)
    y = group_norm(x, 4, w, b, EPS, "silu", mask * 1e-300)
    assert torch.equal(y, group_norm(x, 4, w, b, EPS, "silu", mask))
    assert y.count_nonzero() > 0


@gpu
@pytest.mark.parametrize("shape,G", [((2, 3, 10007), 10007), ((2, 700, 10007), 10007), ((1, 5, 20014), 10007),
                                     ((2, 65, 4099), 1), ((1, 300, 8198), 2)], ids=str)
def test_prime_numbers_of_groups_and_of_channels(shape, G):
    x, dy = values(shape, 71, torch.bfloat16, "cuda"), values(shape, 72, torch.bfloat16, "cuda", 0.0)
    w, b = params(shape[-1], 73, torch.float32, "cuda")
    y, *grads = run(x, G, w, b, dy, "silu")
    check_all(x, dy, G, w, b, "silu", None, y, *grads)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,G", [((3, 5, 4096), 4096), ((2, 900, 4096), 16), ((2, 700, 512), 512),
                                     ((1, 1200, 4096), 4096), ((2, 16, 2048), 2048), ((2, 700, 4095), 819)], ids=str)
def test_most_shared_memory(shape, G, dt):
    """Slices as wide as a block's threads span, groups of one channel: up to 128 KB."""
    x, dy = values(shape, 81, DT[dt], "cuda"), values(shape, 82, DT[dt], "cuda", 0.0)
    w, b = params(shape[-1], 83, torch.float32, "cuda")
    y, *grads = run(x, G, w, b, dy, "silu")
    check_all(x, dy, G, w, b, "silu", None, y, *grads)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,G", [((1, 1, 4096), 16), ((1, 5003, 64), 4), ((3, 300, 96), 8), ((1, 3, 20000), 1)], ids=str)
def test_gelu_is_as_exact_for_bf16_inputs(shape, G, dt):
    """bounds() without its allowance for a shorter polynomial.  One position a
    channel: dbias is one value of dL/dz, with the slope's error and no sum's."""
    x, dy = values(shape, 91, DT[dt], "cuda"), values(shape, 92, DT[dt], "cuda", 0.0)
    w, b = params(shape[-1], 93, torch.float32, "cuda")
    y, dx, dw, db = run(x, G, w, b, dy, "gelu")
    arg = (np64(x), np64(dy), G, np64(w), np64(b))
    ey, edx, ew, eb = bounds(*arg, "gelu", None)
    check(y, train_ops.group_norm(arg[0], *arg[2:], EPS, "gelu")[0], ey, "y")
    dxr, dwr, dbr, dz = train_ops.group_norm_grads(*arg, EPS, "gelu")
    if shape[1] == 1:  # without the sum's share
        eb = eb - CHAIN * U * np.abs(dz).sum((0, 1))
    for got, ref, err, what in ((dx, dxr, edx, "dx"), (dw, dwr, ew, "dweight"), (db, dbr, eb, "dbias")):
        check(got, ref, err, what)


def plain_reference(x, dy, G, w, b, mask=None, narrow=False):
    """(y, dx, dweight, dbias) without an activation in 64 bits, on x's device, and
    their bounds: those of the module's first lines, but that the statistics are joined
    from sums around values of the group itself.  With M the group's largest |x| and
    s = 1 / r its spread, the mean is then off by CHAIN 2^-53 M and the variance by
    CHAIN 2^-53 (s^2 + s M), so h by eh = 8 u |h| + k (1 + |h|), k = (4 u^2 + CHAIN
    2^-53) M r: of the first order in M, not of the second.  narrow: sums of 32 bits
    over x - m1, m1 the mean in 32 bits (off by CHAIN u M, which leaves CHAIN u^2 M in
    the differences' rounding), and again over what is left: k = CHAIN u (1 + u M r)."""
    B, C = x.shape[0], x.shape[-1]
    split = (B, -1, G, C // G)
    xd, dyd = x.double().reshape(split), dy.double().reshape(split)
    live = torch.ones_like(xd[..., :1, :1], dtype=torch.bool) if mask is None else (mask != 0).reshape(B, -1, 1, 1)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    only = lambda t: torch.where(live, t, zero)  # noqa: E731
    xd, dyd = only(xd), only(dyd)
    count = (live.sum(1, keepdim=True) * (C // G)).clamp(min=1)
    mean = lambda t: t.sum((1, 3), keepdim=True) / count  # noqa: E731
    d = only(xd - mean(xd))
    d = only(d - mean(d))
    r = (mean(d * d) + EPS).rsqrt()
    h = d * r
    wd, bd = w.double().view(G, -1), b.double().view(G, -1)
    M = xd.abs().amax((1, 3), keepdim=True)
    k = CHAIN * U * (1 + U * M * r) if narrow else (4 * U * U + CHAIN * 2.0 ** -53) * M * r
    eh = only(8 * U * h.abs() + k * (1 + h.abs()))
    y = only(h * wd + bd)
    ey = wd.abs() * eh + 2 * U * (h.abs() * wd.abs() + bd.abs())
    g = dyd * wd
    eg = 2 * U * g.abs()
    c1, c2 = mean(g), mean(g * h)
    ec1 = mean(eg) + CHAIN * U * mean(g.abs())
    ec2 = mean(eg * h.abs() + g.abs() * eh) + CHAIN * U * mean((g * h).abs())
    er = 2 * U + k
    dx = only(r * (g - c1 - h * c2))
    edx = r * (eg + ec1 + h.abs() * ec2 + eh * c2.abs() + (er + 4 * U) * (g.abs() + c1.abs() + h.abs() * c2.abs()))
    dw, db = (dyd * h).sum((0, 1)), dyd.sum((0, 1))
    ew = (dyd.abs() * eh).sum((0, 1)) + CHAIN * U * (dyd * h).abs().sum((0, 1))
    eb = CHAIN * U * dyd.abs().sum((0, 1))
    return (y, dx, dw, db), (ey, edx, ew, eb)


def check_plain(got, refs, errs, what):
    for name, t, ref, err in zip(("y", "dx", "dweight", "dbias"), got, refs, errs):
        t64 = t.detach().double().reshape(ref.shape)
        excess = (t64 - ref).abs() - (half(t.dtype) * ref.abs() + (1 + half(t.dtype)) * err + 1e-36)
        assert bool((excess <= 0).all()), (what, name, int((excess > 0).sum()), excess.numel(), excess.max().item())


@gpu
@pytest.mark.parametrize("shape,G", [((3, 60, 24), 4), ((2, 6000, 64), 8), ((2, 3001, 20), 4), ((70, 1, 512), 8),
                                     ((1, 33, 4101), 1), ((2, 3, 5), 5)], ids=str)
def test_values_far_from_zero(shape, G):
    """The statistics do not lose what the values' distance from zero takes of the
    squares, whatever part is masked, the first positions among it."""
    C = shape[-1]
    w, b = params(C, 102, torch.float32, "cuda")
    dy = values(shape, 101, torch.float32, "cuda", 0.0)
    late = some_mask(shape[:2], 103, "cuda")
    late[:, :shape[1] // 3] = 0
    for mean, spread in ((1e5, 0.01), (1e6, 0.1), (1e6, 1.0), (-1e3, 1e-3), (9.5e4, 0.0), (8.4e5, 0.0), (0.0, 1.0)):
        x = (mean + spread * values(shape, 100, torch.float64, mean=0.0)).float().cuda()
        for mask in (None, late):
            case = (shape, G, mean, spread, mask is not None)
            print("far from zero", *case, flush=True)
            if mask is None:
                seen = x
            else:
                seen = torch.where(mask.unsqueeze(-1) != 0, x, float("nan"))
            check_plain(run(seen, G, w, b, dy, None, mask), *plain_reference(x, dy, G, w, b, mask), case)
    # a constant in bf16, and one value far from the others in the first place
    x = torch.full(shape, 94720.0, dtype=torch.bfloat16, device="cuda")
    check_plain(run(x, G, w, b, dy.bfloat16()), *plain_reference(x, dy.bfloat16(), G, w, b), "constant")
    x = values(shape, 100, torch.float32, "cuda")
    x[:, 0] = 1e4
    check_plain(run(x, G, w, b, dy), *plain_reference(x, dy, G, w, b), "first")


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,G", [((20000, 40, 40), 8), ((9000, 100, 24), 3), ((30001, 12, 33), 11)], ids=str)
def test_many_small_samples(shape, G, dt):
    """Teams of a few threads with up to 16 vectors each, also of eight groups' channels."""
    x, dy = values(shape, 105, DT[dt], "cuda"), values(shape, 106, DT[dt], "cuda", 0.0)
    w, b = params(shape[-1], 107, torch.float32, "cuda")
    for mask in (None, some_mask(shape[:2], 108, "cuda", empty=True)):
        got = run(x, G, w, b, dy, None, mask)
        check_plain(got, *plain_reference(x, dy, G, w, b, mask), (shape, G, dt, mask is not None))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("far", [10.0, 100.0, 1e4])
def test_pytorch_path_far_from_zero(far, masked):
    """A mean that is rounded to fp32 once is off by u of itself; what is left of it in
    x - mean is taken off there."""
    shape = (1, 20000, 8)
    x, dy = values(shape, 110, torch.float32, mean=0.0) + far, values(shape, 111, torch.float32, mean=0.0)
    w, b = params(8, 112, torch.float32)
    mask = None
    if masked:
        mask = some_mask(shape[:2], 113)
        mask[:, :500] = 0
    check_plain(run(x, 2, w, b, dy, None, mask), *plain_reference(x, dy, 2, w, b, mask, True), far)


@gpu
def test_autocast_without_the_kernels():
    """use_fused_kernel=False changes the path, not the type."""
    x = values((2, 30, 24), 121, torch.bfloat16, "cuda")
    mask = some_mask((2, 30), 122, "cuda")
    for dtype in (torch.float32, torch.bfloat16):
        m = GroupNorm(4, 24, activation="silu", device="cuda", dtype=dtype)
        u = GroupNorm(4, 24, activation="silu", device="cuda", dtype=dtype, use_fused_kernel=False)
        u.load_state_dict(m.state_dict())
        for live in (None, mask):
            with torch.autocast("cuda", dtype=torch.bfloat16):
                one, two = m(x, live), u(x, live)
            assert one.dtype == two.dtype == torch.float32
            torch.testing.assert_close(one, two, rtol=1e-5, atol=1e-5)
            assert u(x, live).dtype == torch.bfloat16


def test_plans_of_many_groups_are_found_at_once(lib):
    """Each call plans anew: no walk over all of 2^24 numbers of groups."""
    import time
    for name in ("gtk_group_norm_workspace_size", "gtk_group_norm_backward_workspace_size"):
        for groups in (16777213, 1 << 24, 10007, 3):  # prime, a power of two, prime
            size = getattr(lib, name)
            size(2, 3, groups, groups, 1)
            times = []
            for _ in range(5):
                t = time.perf_counter()
                size(2, 3, groups, groups, 1)
                times.append(time.perf_counter() - t)
            assert min(times) < 2e-3, (name, groups, times)


@gpu
def test_more_channels_than_the_kernels_take():
    """They run the PyTorch path, as layer_norm's do."""
    C = (1 << 24) + 2
    x = values((1, 2, C), 131, torch.bfloat16, "cuda", 0.0).requires_grad_(True)
    y = group_norm(x, 3, activation="silu")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.no_grad():
        xf = x.double().view(2, 3, -1)
        d = xf - xf.mean((0, 2), keepdim=True)
        ref = F.silu(d * (d.square().mean((0, 2), keepdim=True) + EPS).rsqrt()).view(1, 2, C)
    assert y.dtype == dx.dtype == torch.bfloat16 and torch.isfinite(dx).all()
    assert ((y.double() - ref).abs() <= half(y.dtype) * ref.abs() + 1e-5 * (1 + ref.abs())).all()


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("P", [30, 5000])
def test_activations_of_the_largest_arguments(P, dt):
    """gelu(inf) = inf, as silu's and torch's; and the slope of a finite z is finite."""
    C = 16
    x, dy = values((2, P, C), 141, DT[dt], "cuda"), values((2, P, C), 142, DT[dt], "cuda")
    w, b = params(C, 143, torch.float32, "cuda")
    far = b.clone()
    far[3] = float("inf")
    for act in ("silu", "gelu"):
        y = group_norm(x, 4, w, far, EPS, act)
        rest = torch.arange(C, device="cuda") != 3
        assert (y[..., 3] == float("inf")).all()
        assert torch.equal(y[..., rest], group_norm(x, 4, w, b, EPS, act)[..., rest])
    for value in (3e38, -3e38):
        far[3] = value
        for act in ("silu", "gelu"):
            y, dx, dw, db = run(x, 4, w, far, dy, act)
            slope = 1.0 if value > 0 else 0.0
            assert torch.equal(y[..., 3], torch.full_like(y[..., 3], max(value, 0.0)))
            assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
            ref = slope * np64(dy)[..., 3].sum()
            assert abs(db[3].item() - ref) <= (half(torch.float32) + CHAIN * U) * np.abs(np64(dy)[..., 3]).sum()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape,G", [((2, 400, 24), 4), ((1, 6000, 16), 2)], ids=str)
def test_gradients_against_differences_along_themselves(shape, G, act, device):
    """Along the signs of a gradient nothing cancels: the derivative is sum |g|, and
    what differences leave open is a small part of it.  With D(t) the central difference
    at step t, off by c t^2 + O(t^4), (4 D(t / 2) - D(t)) / 3 is off by O(t^4), below
    |D(t) - D(t / 2)|; the losses' roundings (y is off by 16 u (1 + |y|) or less) add their sum over t."""
    x, dy = values(shape, 151, torch.float32, device, 0.0), values(shape, 152, torch.float32, device, 0.0)
    w, b = params(shape[-1], 153, torch.float32, device)
    mask = some_mask(shape[:2], 154, device)
    y, *grads = run(x, G, w, b, dy, act, mask)
    y = y.detach()
    loss = lambda *a: float((group_norm(a[0], G, *a[1:], EPS, act, mask).double() * dy.double()).sum())  # noqa: E731
    round_off = 16 * U * float((dy.double().abs() * (1 + y.double().abs())).sum())
    t = 2.0 ** -5
    for k, g in enumerate(grads):
        def central(step):
            at = [[s * step * g.sign() if j == k else 0.0 for j in range(3)] for s in (1, -1)]
            hi, lo = (loss(*(p + d for p, d in zip((x, w, b), ds))) for ds in at)
            return (hi - lo) / (2 * step)
        whole, halved = central(t), central(t / 2)
        size = float(g.double().abs().sum())
        allowed = abs(whole - halved) + 2 * round_off / t + CHAIN * U * size
        assert allowed < 0.03 * size, (k, allowed, size)
        assert abs((4 * halved - whole) / 3 - size) <= allowed, (k, whole, halved, size)


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape,G,dt", [((1, 17000 * 32 + 5, 128), 32, "bf16"), ((2, 8300 * 32 + 7, 128), 8, "bf16"),
                                        ((1, 16500 * 81 + 80, 24), 4, "fp32"), ((3, 5600 * 34 + 33, 60), 12, "fp32")], ids=str)
def test_second_launches_with_chunks_of_their_own(shape, G, dt, masked):
    """Long samples: the launch that applies has more chunks than the one that sums, at
    512 threads and 256 CUs from 16384 steps of 512 / (vectors of a row) positions on."""
    x = torch.empty(shape, device="cuda")
    x.normal_(generator=torch.Generator("cuda").manual_seed(161)).mul_(1.5).add_(0.5)
    dy = torch.empty(shape, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(162))
    x, dy = x.to(DT[dt]), dy.to(DT[dt])
    w, b = params(shape[-1], 163, torch.float32, "cuda")
    mask = None
    if masked:
        mask = (torch.rand(shape[:2], device="cuda", generator=torch.Generator("cuda").manual_seed(164)) < 0.8).float()
        mask[:, shape[1] * 9 // 10:] = 0
        mask[0, :70000] = 0
    got = run(x, G, w, b, dy, None, mask)
    check_plain(got, *plain_reference(x, dy, G, w, b, mask), (shape, dt, masked))
    again = run(x, G, w, b, dy, None, mask)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@gpu
def test_gradients_of_more_than_2_to_the_31_values():
    """[1, P, 64] with 2^31 + 64 * 999 values: x and dL/dy have a period of 4096 positions
    and a tail of ones and zeros, so one period gives every sum."""
    P, C, G, many = (1 << 25) + 999, 64, 4, 1 << 13
    period, up = (values((4096, C), k, torch.bfloat16, "cuda", m) for k, m in ((171, 1.0), (172, 0.0)))
    w, b = params(C, 173, torch.float32, "cuda")
    x = torch.ones(1, P, C, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(1, P, C, dtype=torch.bfloat16, device="cuda")
    for t, one in ((x, period), (dy, up)):
        t[0, :1 << 25].view(many, 4096, C).copy_(one)
    _, dx, dw, db = run(x, G, w, b, dy)
    n, d, wn = np64(period), np64(up), np64(w)
    cg, total = C // G, P * (C // G)
    spread = lambda t: np.repeat(t, cg)  # noqa: E731
    grouped = lambda t: t.reshape(-1, G, cg).sum((0, 2))  # noqa: E731
    mean = (grouped(n) * many + 999 * cg) / total
    var = (grouped((n - spread(mean)) ** 2) * many + 999 * cg * (1 - mean) ** 2) / total
    r = spread(1 / np.sqrt(var + EPS))
    h, tail = (n - spread(mean)) * r, (1 - spread(mean)) * r
    g = d * wn
    c1, c2 = spread(grouped(g) * many / total), spread(grouped(g * h) * many / total)
    # a thread adds some 2^25 / 64 / 256 positions up, one behind the other
    chain = 2048 + CHAIN
    ec1 = spread(grouped(np.abs(g)) * many / total) * chain * U
    ec2 = spread(grouped(np.abs(g * h)) * many / total) * chain * U
    for at in (0, 1 << 24, (1 << 25) - 4096):
        ref = r * (g - c1 - h * c2)
        err = r * (ec1 + np.abs(h) * ec2 + 32 * U * (np.abs(g) + np.abs(c1) + np.abs(h * c2)))
        check(dx[0, at:at + 4096], ref, err, ("dx", at))
    ref = np.broadcast_to(r * (-c1 - tail * c2), (999, C))
    check(dx[0, 1 << 25:], ref, r * (ec1 + np.abs(tail) * ec2 + 32 * U * (np.abs(c1) + np.abs(tail * c2))), "the tail")
    check(dw, (d * h).sum(0) * many, (chain + 16) * U * np.abs(d * h).sum(0) * many, "dweight")
    check(db, d.sum(0) * many, chain * U * np.abs(d).sum(0) * many, "dbias")
