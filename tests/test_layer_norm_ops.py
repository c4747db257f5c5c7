"""LayerNorm as training uses it (genie_tk.primitives.layer_norm / LayerNorm,
genie_tk._C.layer_norm_forward / layer_norm_backward, gtk_layer_norm_*): the
oracle, the PyTorch path and the refusals on the CPU, the kernels against the
64-bit oracle on the GPU.

Tolerances.  u = 2^-24 (fp32), half_t = finfo(t).eps / 2 of the output's type.
A row's sums are chains of at most D / 64 additions a lane and 16 between lanes
and waves, so `adds` = D / 64 + 16 and, with M the row's largest |x|, r = rstd:
* the mean is off by adds u M, d = x - mean by that and u |d|, and the relative
  error of r is half that of the variance: h is off by 2 adds u (M r + |h|);
* dx = r (g - c1 - h c2): with G the row's largest |g| (|c1|, |c2| <= G as the
  mean |h| is at most 1) it is off by 4 adds u r G (1 + |h|) (1 + M r);
* a column sum over R rows is a chain of at most R / 16 + 64 additions of terms
  that are off as h is.
Each result is rounded once to its own type."""
import ctypes
import os

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from genie_tk import _ext
from genie_tk.primitives import LayerNorm, layer_norm
from oracle import train_ops

U = 2.0 ** -24
EPS = 1e-5
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().double().cpu().numpy()


def bounds(x, dy, w, eps=EPS):
    """(|error| allowed of h, dx, dweight, dbias) before the last rounding."""
    D, R = x.shape[-1], x.shape[0]
    adds = D / 64 + 16
    _, h, r = train_ops.layer_norm(x, None, None, eps)
    M = np.abs(x).max(-1, keepdims=True)
    eh = 2 * adds * U * (M * r + np.abs(h))
    g = np.abs(dy if w is None else dy * w)
    edx = 4 * adds * U * r * g.max(-1, keepdims=True) * (1 + np.abs(h)) * (1 + M * r)
    chain = R / 16 + 64
    ew = (np.abs(dy) * eh).sum(0) + chain * U * np.abs(dy * h).sum(0)
    eb = chain * U * np.abs(dy).sum(0)
    return eh, edx, ew, eb


def check(got, ref, err, what):
    dtype = got.dtype
    got = np64(got)
    assert got.shape == ref.shape, what
    assert np.isfinite(got).all(), f"{what}: non-finite"
    excess = np.abs(got - ref) - (half(dtype) * np.abs(ref) + (1 + half(dtype)) * err + 1e-37)
    assert (excess <= 0).all(), (f"{what}: {int((excess > 0).sum())} of {excess.size} out of tolerance, worst by "
                                 f"{excess.max():.3e}, error {np.abs(got - ref).max():.3e}")


def rows(R, D, seed, dtype, device="cpu", mean=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(R, D, generator=gen) * 1.5 + mean * torch.randn(R, 1, generator=gen)
    return x.to(dtype).to(device)


def params(D, seed, dtype, device="cpu"):
    gen = torch.Generator().manual_seed(1000 + seed)
    w = 1 + 0.3 * torch.randn(D, generator=gen)
    b = 0.5 * torch.randn(D, generator=gen)
    return w.to(dtype).to(device), b.to(dtype).to(device)


def check_all(x, dy, w, b, y, dx, dw, db, eps=EPS):
    xn, dn = np64(x).reshape(-1, x.shape[-1]), np64(dy).reshape(-1, x.shape[-1])
    wn = None if w is None else np64(w)
    bn = None if b is None else np64(b)
    eh, edx, ew, eb = bounds(xn, dn, wn, eps)
    yr, h, _ = train_ops.layer_norm(xn, wn, bn, eps)
    wa = 1.0 if wn is None else np.abs(wn)
    ey = eh * wa + 2 * U * (np.abs(h) * wa + (0 if bn is None else np.abs(bn)))
    dxr, dwr, dbr = train_ops.layer_norm_grads(xn, dn, wn, eps)
    if y is not None:
        check(y.reshape(xn.shape), yr, ey, "y")
    if dx is not None:
        check(dx.reshape(xn.shape), dxr, edx, "dx")
    if dw is not None:
        check(dw, dwr, ew, "dweight")
    if db is not None:
        check(db, dbr, eb, "dbias")


# ---------------------------------------------------------------------------
# CPU: the oracle, the PyTorch path, the refusals
# ---------------------------------------------------------------------------
def test_oracle_matches_autograd_in_64_bits():
    x, dy = rows(7, 13, 0, torch.float64), rows(7, 13, 1, torch.float64)
    w, b = params(13, 2, torch.float64)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = F.layer_norm(x, (13,), w, b, EPS)
    got = torch.autograd.grad(y, leaves, dy)
    ref = train_ops.layer_norm_grads(np64(x), np64(dy), np64(w))
    np.testing.assert_allclose(np64(y), train_ops.layer_norm(np64(x), np64(w), np64(b))[0], rtol=0, atol=1e-13)
    for g, r in zip(got, ref):
        np.testing.assert_allclose(np64(g), r, rtol=0, atol=1e-12)


def test_oracle_gradient_against_differences():
    x, dy, v = (np64(rows(3, 9, k, torch.float64)) for k in range(3))
    w = np64(params(9, 0, torch.float64)[0])
    loss = lambda t: (train_ops.layer_norm(t, w)[0] * dy).sum()  # noqa: E731
    t = 1e-5
    num = (loss(x + t * v) - loss(x - t * v)) / (2 * t)
    assert abs(num - (train_ops.layer_norm_grads(x, dy, w)[0] * v).sum()) < 1e-7


@pytest.mark.parametrize("pdt", ["fp32", "bf16", None])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_pytorch_path(dt, pdt):
    x = rows(6, 24, 0, DT[dt])
    w, b = (None, None) if pdt is None else params(24, 1, DT[pdt])
    y = layer_norm(x, w, b)
    ref = train_ops.layer_norm(np64(x), *(None if p is None else np64(p) for p in (w, b)))[0]
    assert y.dtype == x.dtype
    np.testing.assert_allclose(np64(y), ref, rtol=half(DT[dt]), atol=1e-5)


def test_pytorch_path_keeps_64_bits():
    x = rows(5, 33, 0, torch.float64)
    w, b = params(33, 1, torch.float32)
    ref = train_ops.layer_norm(np64(x), np64(w), np64(b))[0]
    np.testing.assert_allclose(np64(layer_norm(x, w, b)), ref, rtol=0, atol=1e-13)


def test_module_is_a_drop_in():
    a, b = torch.nn.LayerNorm((3, 8), eps=1e-4), LayerNorm((3, 8), eps=1e-4)
    b.load_state_dict(a.state_dict())
    x = rows(10, 24, 0, torch.float32).view(10, 3, 8)
    torch.testing.assert_close(a(x), b(x))
    assert sorted(LayerNorm(4, bias=False).state_dict()) == ["weight"]
    assert not LayerNorm(4, elementwise_affine=False).state_dict()
    torch.testing.assert_close(LayerNorm(24, use_fused_kernel=False)(x.flatten(1)), LayerNorm(24)(x.flatten(1)))
    with pytest.raises(RuntimeError):
        LayerNorm(5)(x)
    with pytest.raises(RuntimeError):
        layer_norm(x, torch.ones(7))


LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genie-tk_amd", "genie_tk",
                   "libgenie_tk_hip.so")
i64, sz, vp, fp, ci = ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float, ctypes.c_int


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    L = ctypes.CDLL(LIB)
    L.gtk_last_error.restype = ctypes.c_char_p
    L.gtk_layer_norm_forward.argtypes = [vp, i64, vp, vp, vp, ci, i64, i64, fp, ci, vp]
    L.gtk_layer_norm_backward.argtypes = [vp, i64, vp, i64, vp, ci, vp, vp, vp, i64, i64, fp, ci, vp, sz, vp]
    L.gtk_layer_norm_backward_workspace_size.restype = sz
    L.gtk_layer_norm_backward_workspace_size.argtypes = [i64, i64, ci]
    return L


def test_c_refusals(lib):
    p = 4096  # never dereferenced: every call below is refused on the host
    fwd = lambda x=p, xs=8, y=p, pdt=0, r=4, d=8, dt=0: lib.gtk_layer_norm_forward(  # noqa: E731
        x, xs, y, None, None, pdt, r, d, EPS, dt, None)
    assert [fwd(r=-1), fwd(d=0), fwd(d=(1 << 24) + 1), fwd(dt=2), fwd(pdt=7), fwd(xs=-8), fwd(x=None), fwd(y=None),
            fwd(r=(1 << 40) + 1)] == [1] * 9
    assert b"null pointer" in (fwd(x=None), lib.gtk_last_error())[1]
    assert fwd(r=0, x=None, y=None) == 0
    need = lib.gtk_layer_norm_backward_workspace_size(4, 8, 0)
    assert need > 0
    bwd = lambda x=p, dy=p, ds=8, dx=p, r=4, d=8, dt=0, ws=p, n=need: lib.gtk_layer_norm_backward(  # noqa: E731
        x, 8, dy, ds, None, 0, dx, None, None, r, d, EPS, dt, ws, n, None)
    assert [bwd(x=None), bwd(dy=None), bwd(ds=-1), bwd(d=0), bwd(dt=3), bwd(ws=None)] == [1] * 6
    assert bwd(n=need - 1) == 3
    assert bwd(dx=None) == 0 and bwd(r=0) == 0  # nothing to write
    assert [lib.gtk_layer_norm_backward_workspace_size(*a) for a in ((-1, 8, 0), (4, 0, 0), (4, 8, 2))] == [0] * 3


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def run(x, w, b, dy, eps=EPS):
    """The public path: y and the gradients of x, w, b."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    got = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    return (y, *(None if t is None else next(got) for t in leaves))


WIDTHS = [1, 2, 3, 5, 7, 8, 9, 16, 31, 33, 64, 77, 100, 128, 129, 256, 320, 511, 512, 520, 1000, 1024, 1027, 2048,
          2049, 4096, 5001, 8192, 8200, 16384, 16391]


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(D, dt):
    for R in (1, 37) if D > 600 else (1, 3, 301):
        print(f"layer_norm R={R} D={D} {dt}", flush=True)
        x, dy = rows(R, D, 0, DT[dt], "cuda"), rows(R, D, 1, DT[dt], "cuda")
        w, b = params(D, 2, DT[dt], "cuda")
        check_all(x, dy, w, b, *run(x, w, b, dy))


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("R,D", [(2, 40000), (3, 65537), (1, 300001)])
def test_very_wide_rows(R, D, dt):
    x, dy = rows(R, D, 0, DT[dt], "cuda"), rows(R, D, 1, DT[dt], "cuda")
    w, b = params(D, 2, DT[dt], "cuda")
    check_all(x, dy, w, b, *run(x, w, b, dy))


@gpu
@pytest.mark.parametrize("R,D", [(4097, 128), (20011, 64), (9001, 100), (2500, 1024), (5003, 24), (70001, 8),
                                 (100003, 3), (1031, 4096)])
@pytest.mark.parametrize("dt,pdt", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "bf16"),
                                    ("bf16", None)])
def test_many_rows(R, D, dt, pdt):
    x, dy = rows(R, D, 0, DT[dt], "cuda"), rows(R, D, 1, DT[dt], "cuda")
    w, b = (None, None) if pdt is None else params(D, 2, DT[pdt], "cuda")
    y, dx, dw, db = run(x, w, b, dy)
    assert y.dtype == dx.dtype == x.dtype and (w is None or dw.dtype == db.dtype == w.dtype)
    check_all(x, dy, w, b, y, dx, dw, db)


@gpu
def test_parameters_of_two_types_and_one_alone():
    x, dy = rows(200, 96, 0, torch.bfloat16, "cuda"), rows(200, 96, 1, torch.bfloat16, "cuda")
    w, b = params(96, 2, torch.bfloat16, "cuda")
    for ww, bb in ((w, b.float()), (w.float(), b), (w, None), (None, b), (None, b.float())):
        y, dx, dw, db = run(x, ww, bb, dy)
        assert (dw is None or dw.dtype == ww.dtype) and (db is None or db.dtype == bb.dtype)
        check_all(x, dy, ww, bb, y, dx, dw, db)


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [100, 128, 513])
def test_strides(D, dt):
    w, b = params(D, 2, DT[dt], "cuda")
    wide = rows(60, D + 11, 0, DT[dt], "cuda")
    four = rows(60, D * 3, 3, DT[dt], "cuda").view(4, 15, 3, D)
    cases = [wide[:, 3:3 + D], wide[::2, 5:5 + D], wide[:1, 1:1 + D].expand(33, D), four[:, :, 1],
             four.transpose(0, 1), rows(D, 50, 4, DT[dt], "cuda").t(), four[:, ::2]]
    for k, x in enumerate(cases):
        print("stride case", k, tuple(x.shape), x.stride(), flush=True)
        dy = torch.randn(x.shape, device="cuda").to(DT[dt])
        check_all(x, dy, w, b, *run(x, w, b, dy))
        # the output gradient at other strides, a broadcast one among them
        for up in (dy.transpose(0, 1).contiguous().transpose(0, 1), dy[..., :1].expand(x.shape),
                   dy[:1].expand(x.shape)):
            check_all(x, up, w, b, *run(x, w, b, up))


@gpu
def test_each_gradient_alone():
    x, dy = rows(90, 72, 0, torch.float32, "cuda"), rows(90, 72, 1, torch.float32, "cuda")
    w, b = params(72, 2, torch.float32, "cuda")
    _, *every = run(x, w, b, dy)
    for keep in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        leaves = [t.clone().requires_grad_(k in keep) for k, t in enumerate((x, w, b))]
        y = layer_norm(*leaves)
        for k, g in zip(keep, torch.autograd.grad(y, [leaves[k] for k in keep], dy)):
            assert torch.equal(g, every[k]), (keep, k)
    # all three differentiable, one asked for
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    for k in (2, 0, 1):
        g, = torch.autograd.grad(y, leaves[k], dy, retain_graph=True)
        assert torch.equal(g, every[k]), k
    C = _ext.require()
    assert C.layer_norm_backward(x, dy, w, EPS, False, False, False) == [None, None, None]


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_values_at_the_edges(dt):
    D = 128
    x, dy = rows(12, D, 0, DT[dt], "cuda"), rows(12, D, 1, DT[dt], "cuda")
    w, b = params(D, 2, DT[dt], "cuda")
    x[0] = 3.25                       # no variance
    x[1] = 0
    x[2] = x[2] * 1e-4                # a variance below eps
    x[3] = x[3] + 4096                # far from zero
    x[4] = x[4] * 1e15
    dy[5] = 0
    dy[6] = dy[6] * 1e10
    y, dx, dw, db = run(x, w, b, dy)
    check_all(x, dy, w, b, y, dx, dw, db)
    # a row that is not finite spoils itself and the sums, nothing else
    x[7, 5], x[8, 100], x[9, 0] = float("nan"), float("inf"), float("-inf")
    y2, dx2, dw2, db2 = run(x, w, b, dy)
    keep = [0, 1, 2, 3, 4, 5, 6, 10, 11]
    assert torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep]) and torch.equal(db2, db)
    assert y2[[7, 8, 9]].isnan().all() and dx2[[7, 8, 9]].isnan().all() and dw2.isnan().all()


@gpu
def test_no_rows():
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        w, b = params(16, 0, torch.float32, "cuda")
        y, dx, dw, db = run(x, w, b, torch.empty_like(x))
        assert y.shape == dx.shape == x.shape
        assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


@gpu
def test_gradient_against_differences():
    """Central differences of sum(y dy) of the fp32 kernels along a direction v.
    With t = 2^-6 the third-order term is below t^2 = 2.4e-4 of the size of the
    sums of |terms|, and each loss is off by the error of y, over 2 t."""
    R, D = 16, 200
    x, dy, v = (rows(R, D, k, torch.float32, "cuda", 0.0) for k in range(3))
    w, b = params(D, 2, torch.float32, "cuda")
    _, dx, dw, _ = run(x, w, b, dy)
    t = 2.0 ** -6
    loss = lambda a, ww: float((layer_norm(a, ww, b).double() * dy.double()).sum())  # noqa: E731
    size = float((dy.double().abs() * w.double().abs()).sum())
    num = (loss(x + t * v, w) - loss(x - t * v, w)) / (2 * t)
    assert abs(num - float((dx.double() * v.double()).sum())) < t * t * 4 * size
    vw = torch.randn_like(w)
    num = (loss(x, w + t * vw) - loss(x, w - t * vw)) / (2 * t)
    err = 2 * (D / 64 + 16) * U * 8 * size / (2 * t)
    assert abs(num - float((dw.double() * vw.double()).sum())) < err


@gpu
def test_same_bits_on_every_call_and_stream():
    x, dy = rows(5000, 384, 0, torch.bfloat16, "cuda"), rows(5000, 384, 1, torch.bfloat16, "cuda")
    w, b = params(384, 2, torch.float32, "cuda")
    first = run(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


@gpu
def test_captured_and_replayed():
    C = _ext.require()
    x, dy = rows(700, 128, 0, torch.bfloat16, "cuda"), rows(700, 128, 1, torch.bfloat16, "cuda")
    w, b = params(128, 2, torch.float32, "cuda")
    step = lambda: (C.layer_norm_forward(x, w, b), *C.layer_norm_backward(x, dy, w))  # noqa: E731
    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append(g)
        outs.append(out)
    for k in range(4):
        x.copy_(rows(700, 128, 10 + k, torch.bfloat16, "cuda"))
        ref = step()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, c in zip(out, ref):
                assert torch.equal(a, c), k


@gpu
def test_captured_through_autograd():
    """The public path captured, as torch asks for it: warmed up on a side
    stream, with no eager graph of the leaves alive."""
    x = rows(700, 128, 0, torch.float32, "cuda").requires_grad_(True)
    w, b = (t.requires_grad_(True) for t in params(128, 2, torch.float32, "cuda"))
    dy = rows(700, 128, 1, torch.float32, "cuda")

    def step():
        y = layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(rows(700, 128, 30 + k, torch.float32, "cuda"))
        ref = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, ref):
            assert torch.equal(a, c), k


@gpu
def test_offsets_past_32_bits():
    R, D = (1 << 24) + 9, 128  # 2^31 + 1152 values
    x = torch.empty(R, D, device="cuda", dtype=torch.bfloat16)
    dy = torch.empty_like(x)
    block = rows(4096, D, 0, torch.bfloat16, "cuda")
    for a in range(0, R, 4096):
        x[a:a + 4096] = block[:min(4096, R - a)]
    dy.zero_()
    at = torch.tensor([0, 4095, 8388608, R - 9, R - 2, R - 1], device="cuda")
    dy[at] = rows(6, D, 1, torch.bfloat16, "cuda")
    w, b = params(D, 2, torch.float32, "cuda")
    y, dx, dw, db = run(x, w, b, dy)
    check_all(x[at], dy[at], w, b, y[at], dx[at], None, None)
    # every other row's gradient is zero: the sums are those of the six
    _, dwr, dbr = train_ops.layer_norm_grads(np64(x[at]), np64(dy[at]), np64(w))
    _, _, ew, eb = bounds(np64(x[at]), np64(dy[at]), np64(w))
    check(dw, dwr, ew, "dweight")
    check(db, dbr, eb, "dbias")
    assert int((dx != 0).any(-1).sum()) == 6


@gpu
def test_gpu_refusals():
    x = rows(4, 16, 0, torch.float32, "cuda").requires_grad_(True)
    w, b = params(16, 0, torch.float32, "cuda")
    C = _ext.require()
    for bad in (w[:8], w.cpu(), w.half(), w.view(4, 4)):
        with pytest.raises(RuntimeError):
            C.layer_norm_forward(x, bad, b)
    with pytest.raises(RuntimeError):
        C.layer_norm_backward(x, x[:2], w)
    with pytest.raises(RuntimeError):
        C.layer_norm_backward(x, x.bfloat16(), w)
    with pytest.raises(RuntimeError):
        C.layer_norm_forward(x.detach().double(), w.double(), b.double())
    with pytest.raises(RuntimeError):
        C.layer_norm_forward(torch.empty(4, 0, device="cuda"))
    with pytest.raises(RuntimeError):
        C.layer_norm_forward(x.detach().cpu(), w, b)
    # a second differentiation is refused, not answered with zeros
    dx, = torch.autograd.grad(layer_norm(x, w, b).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
    # other types run torch's
    y = layer_norm(x.half(), w.half(), b.half())
    assert y.dtype == torch.float16


@gpu
def test_module_on_the_kernels():
    m = LayerNorm((4, 32)).cuda()
    t = torch.nn.LayerNorm((4, 32)).cuda()
    with torch.no_grad():
        for p, q in zip(m.parameters(), t.parameters()):
            p.copy_(torch.randn_like(p))
            q.copy_(p)
    x = rows(50, 128, 0, torch.float32, "cuda").view(50, 4, 32)
    dy = rows(50, 128, 1, torch.float32, "cuda").view(50, 4, 32)
    m(x).backward(dy)
    y, dx, dw, db = run(x.flatten(1), m.weight.flatten(), m.bias.flatten(), dy.flatten(1))
    check_all(x.flatten(1), dy.flatten(1), m.weight.flatten(), m.bias.flatten(), m(x).flatten(1), None,
              m.weight.grad.flatten(), m.bias.grad.flatten())
    assert torch.equal(m.weight.grad.flatten(), dw) and torch.equal(m.bias.grad.flatten(), db)


# ---------------------------------------------------------------------------
# Rows whose spread is small against their offset
# ---------------------------------------------------------------------------
def spread_bounds(x, dy, w, eps=EPS):
    """`bounds` with S, the row's largest |x - mean|, in the place of M: the sums
    are taken of p = x - x_0, which is at most 2 S and off by u times that.  The
    mean of p is off by 2 (adds + 3) u S (with the roundings of 1 / D and of the
    product), so d by a = (2 adds + 9) u S; the relative error of r is a r + (adds
    / 2 + 8) u, as sd / (sd^2 + eps) <= r; both go into h = d r.  With |c1|, |c2|
    <= G, c1 is off by (adds + 3) u G, c2 by G max(eh) + (adds + 5) u G, and dx by
    those, its own roundings and the error of r."""
    D, R = x.shape[-1], x.shape[0]
    adds = D / 64 + 16
    _, h, r = train_ops.layer_norm(x, None, None, eps)
    ah = np.abs(h)
    ar = (2 * adds + 9) * U * np.abs(x - x.mean(-1, keepdims=True)).max(-1, keepdims=True) * r
    er = ar + (adds / 2 + 8) * U
    eh = (1 + ar) * (ar + er * ah)
    g = np.abs(dy if w is None else dy * w).max(-1, keepdims=True)
    edx = (1 + ar) * r * g * ((2 * adds + 13) * U * (1 + ah) + eh.max(-1, keepdims=True) * (1 + ah) + er * (2 + ah))
    chain = R / 16 + 64
    ew = (np.abs(dy) * eh).sum(0) + chain * U * np.abs(dy * h).sum(0)
    return eh, edx, ew, chain * U * np.abs(dy).sum(0)


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [3, 7, 8, 15, 31, 64, 77, 128, 301, 512, 1023, 1100, 2048, 5001, 8200, 16383, 20001])
def test_small_spread_far_from_zero(D, dt):
    """The error follows the spread, not the offset; a row of one value gives the bias."""
    print(f"small spread D={D} {dt}", flush=True)
    gen = torch.Generator().manual_seed(D)
    x = torch.zeros(11, D, dtype=torch.float64)
    x[:4] = torch.tensor([1000.1, 1e5 + 0.1, -7654321.0, 1e30], dtype=torch.float64)[:, None]  # one value
    near = torch.randn(5, D, generator=gen, dtype=torch.float64)
    x[4:9] = near * torch.tensor([1e-2, 0.05, 3.0, 1e-4, 1.0])[:, None].double()
    x[4:9] += torch.tensor([1000.1, 1e5, -1e6, 1.0, 3e5], dtype=torch.float64)[:, None]
    x[8, 0] = -3e5           # an outlier in the first place
    x[9] = 1e8
    x[9, D // 2] += 8        # one value, one step of fp32 higher
    x[10] = near[0]          # around zero
    x = x.to(DT[dt]).cuda()
    dy = rows(11, D, 1, DT[dt], "cuda")
    w, b = params(D, 2, DT[dt], "cuda")
    y, dx, dw, db = run(x, w, b, dy)
    xn, dn, wn, bn = (np64(t) for t in (x, dy, w, b))
    eh, edx, ew, eb = spread_bounds(xn, dn, wn)
    yr, h, _ = train_ops.layer_norm(xn, wn, bn)
    dxr, dwr, dbr = train_ops.layer_norm_grads(xn, dn, wn)
    assert (h[:4] == 0).all() and torch.equal(y[:4], b.expand(4, D))
    check(y, yr, eh * np.abs(wn) + 2 * U * (np.abs(h * wn) + np.abs(bn)), "y")
    check(dx, dxr, edx, "dx")
    check(dw, dwr, ew, "dweight")
    check(db, dbr, eb, "dbias")


# ---------------------------------------------------------------------------
# Forward-mode derivatives
# ---------------------------------------------------------------------------
def check_tangents(device, dt, pdt):
    """The tangent of y along (vx, vw, vb), each alone and all together, against
    64 bits: r (vx - mean(vx) - h mean(vx h)) w + h vw + vb.  The first term is a
    dx (g = vx) times w and the second an h times vw, so they are off by `bounds`'
    edx |w| and eh |vw|, three times that as torch's sums of 48 terms may be one
    chain (adds is 16.75).  In types narrower than fp32 torch rounds up to eight
    steps on the way, each by half a step of the sizes that edx and eh hold."""
    import torch.autograd.forward_ad as fwAD

    D = 48
    x, vx = rows(9, D, 0, DT[dt], device), rows(9, D, 1, DT[dt], device, 0.0)
    w, b = params(D, 2, DT[pdt], device)
    vw, vb = params(D, 3, DT[pdt], device)
    _, h, r = train_ops.layer_norm(np64(x))
    v, wn = np64(vx), np64(w)
    part = (r * (v - v.mean(-1, keepdims=True) - h * (v * h).mean(-1, keepdims=True)) * wn, h * np64(vw),
            np64(vb) + 0 * h)
    eh, edx, _, _ = bounds(np64(x), v, None)
    adds, step = D / 64 + 16, half(DT[dt])
    u = 3 * U + 8 * step / (2 * adds) if dt != "fp32" else 3 * U
    err = (edx * np.abs(wn) * u / U, eh * np.abs(np64(vw)) * u / U, 8 * step * np.abs(np64(vb)))
    for duals in ((0,), (1,), (2,), (0, 1, 2)):
        for grad in (False, True):
            with fwAD.dual_level():
                args = [t.clone().requires_grad_(grad) for t in (x, w, b)]
                args = [fwAD.make_dual(t, tv) if k in duals else t for k, (t, tv) in enumerate(zip(args, (vx, vw, vb)))]
                y, t = fwAD.unpack_dual(layer_norm(*args))
            assert t is not None, f"tangent of {duals} lost"
            assert y.dtype == x.dtype  # the tangent's is torch's: fp32 where its statistics are
            ref = sum(part[k] for k in duals)
            check(t, ref, sum(err[k] for k in duals) + 4 * U * sum(np.abs(part[k]) for k in duals), f"tangent {duals}")


@pytest.mark.parametrize("dt,pdt", [("fp32", "fp32"), ("bf16", "fp32")])
def test_pytorch_path_forward_mode(dt, pdt):
    check_tangents("cpu", dt, pdt)


@gpu
@pytest.mark.parametrize("dt,pdt", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
def test_forward_mode_is_not_dropped(dt, pdt):
    import torch.autograd.forward_ad as fwAD

    check_tangents("cuda", dt, pdt)
    x = rows(3, 16, 0, DT[dt], "cuda")
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        _ext.require().layer_norm(fwAD.make_dual(x, x))


@gpu
@pytest.mark.parametrize("dt,pdt", [("bf16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16"),
                                    ("bf16", None)])
def test_autocast_gives_fp32(dt, pdt):
    """As torch's LayerNorm: computed and returned in fp32, gradients in the
    leaves' own types."""
    x, dy = rows(50, 96, 0, DT[dt], "cuda"), rows(50, 96, 1, torch.float32, "cuda")
    w, b = (None, None) if pdt is None else params(96, 2, DT[pdt], "cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = F.layer_norm(x, (96,), w, b, EPS)
        got = run(x, w, b, dy)
        with torch.autocast("cuda", enabled=False):
            assert layer_norm(x, w, b).dtype == x.dtype
        m = LayerNorm((4, 24), elementwise_affine=False)
        assert m(x.view(50, 4, 24)).dtype == torch.float32
        assert layer_norm(x.half()).dtype == torch.float32
        assert layer_norm(x.double()).dtype == F.layer_norm(x.double(), (96,)).dtype == torch.float64
    assert got[0].dtype == want.dtype == torch.float32 and got[1].dtype == x.dtype
    assert w is None or got[2].dtype == got[3].dtype == w.dtype
    check_all(x, dy, w, b, *got)


def test_module_without_dimensions_is_refused():
    with pytest.raises(RuntimeError, match="normalized_shape"):
        LayerNorm(())(torch.ones(()))


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [5, 64, 100, 1023, 4096, 20001])
def test_lowest_values_in_masked_places(D, dt):
    """The variance is past fp32's range: r = 0 and h = 0, not NaN, wherever the
    lowest values stand; in every place they are a row of one value."""
    x = rows(6, D, 0, DT[dt], "cuda")
    w, b = params(D, 2, DT[dt], "cuda")
    low = torch.finfo(DT[dt]).min
    x[0, 0] = x[1, D // 2] = x[2, D - 1] = low
    x[3, : D // 2] = low
    x[4, D // 2:] = low
    x[5] = low
    assert torch.equal(layer_norm(x, w, b), b.expand(6, D))
    assert torch.equal(run(x, w, b, torch.zeros_like(x))[1], torch.zeros_like(x))
