"""The global gradient norm and clipping (genie_tk.gradients, genie_tk._C.grad_*,
gtk_grad_*): the PyTorch path and the refusals on the CPU, the kernels against
the 64-bit oracle on the GPU.

Tolerances.  u = 2^-24.  Squares and sums are 64-bit: a sum of n terms is off
by at most n 2^-53 relative to the sum of the absolute terms, all of one sign,
which is below u / 8 up to n = 2^26; the norm is rounded once to fp32, so it is
off by 1.25 u.  The factor takes that and its own rounding, the product its
rounding to fp32 and, in bf16, one more half step: (3.5 u + half_t) |out|."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

from genie_tk import _ext, gradients
from genie_tk.gradients import clip_grad_norm_, clip_grads, clip_grads_with_norm_, grad_norm
from oracle import train_ops

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu
INF = math.inf


def np64(t):
    return t.detach().double().cpu().numpy()


def half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def check_norm(norm, grads, p):
    ref = train_ops.global_norm([np64(g) for g in grads], p)
    assert norm.shape == () and norm.dtype == torch.float32
    if ref > torch.finfo(torch.float32).max:
        assert float(norm) == INF
        return ref
    assert abs(float(norm) - ref) <= 1.25 * U * ref + 1e-45, (float(norm), ref)
    return ref


def check_clipped(outs, before, max_norm, ref_norm):
    k = train_ops.clip_factor(ref_norm, max_norm)
    for o, g in zip(outs, before):
        ref = np64(g) * k
        err = np.abs(np64(o) - ref)
        # 2^-133 / 2: half a step among bf16's smallest values
        assert (err <= (3.5 * U + half(o.dtype)) * np.abs(ref) + 2.0 ** -134).all(), err.max()


def make(sizes, seed, dtypes, device="cpu", scale=0.01):
    gen = torch.Generator().manual_seed(seed)
    return [(scale * (1 + k % 5) * torch.randn(n, generator=gen)).to(dtypes[k % len(dtypes)]).to(device)
            for k, n in enumerate(sizes)]


def as_params(grads):
    ps = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        ps.append(p)
    return ps


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("p", [1.0, 2.0, 3.0, INF])
def test_pytorch_path_matches_torch(p):
    # (torch has no largest value of an empty tensor)
    grads = make([5, 130, 1] + [0] * (p != INF), 0, [torch.float32])
    check = [g.clone() for g in grads]
    ours, theirs = as_params(grads), as_params(check)
    norm = clip_grad_norm_(iter(ours), 0.05, p)
    want = torch.nn.utils.clip_grad_norm_(theirs, 0.05, p)
    torch.testing.assert_close(norm, want)
    for a, b in zip(ours, theirs):
        torch.testing.assert_close(a.grad, b.grad)
    torch.testing.assert_close(grad_norm(g for g in check), torch.nn.utils.get_total_norm(check))


def test_pytorch_path_forms():
    grads = make([40, 7], 1, [torch.bfloat16])
    before = [g.clone() for g in grads]
    norm, outs = clip_grads(grads, 0.01, out=[torch.empty(40), torch.empty(7)])
    ref = check_norm(norm, grads, 2.0)
    check_clipped(outs, before, 0.01, ref)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    clip_grads_with_norm_(as_params(grads), 0.01, torch.tensor(ref))
    check_clipped(grads, before, 0.01, ref)
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(clip_grad_norm_(p, 1.0)) == 0.0  # no gradient
    assert float(clip_grad_norm_([], 1.0)) == float(grad_norm([])) == 0.0
    assert clip_grads([], 1.0)[1] == []
    assert [float(grad_norm([torch.empty(0)], q)) for q in (1.0, 2.0, INF)] == [0.0] * 3


def test_pytorch_path_keeps_64_bits():
    grads = make([40, 7], 1, [torch.float64])
    before = [g.clone() for g in grads]
    norm, outs = clip_grads(grads, 0.01)
    ref = train_ops.global_norm([np64(g) for g in grads])
    assert norm.dtype == torch.float64 and abs(float(norm) - ref) < 1e-14
    clip_grads_with_norm_(as_params(grads), 0.01, norm)
    for a, o, b in zip(grads, outs, before):
        np.testing.assert_allclose(np64(a), np64(b) * train_ops.clip_factor(ref, 0.01), rtol=1e-13)
        np.testing.assert_allclose(np64(o), np64(a), rtol=1e-15)


def test_refusals():
    g = [torch.ones(3), torch.ones(2, 2)]
    for call in (lambda: clip_grads(g, -1.0), lambda: clip_grads(g, math.nan), lambda: clip_grads(g, 1.0, out=g[:1]),
                 lambda: clip_grads(g, 1.0, out=[torch.ones(3), torch.ones(4)]),
                 lambda: clip_grad_norm_(as_params(g), -0.5),
                 lambda: grad_norm([torch.ones(3).to_sparse()]), lambda: grad_norm([torch.ones(3, dtype=torch.int64)]),
                 lambda: grad_norm([torch.ones(3, dtype=torch.complex64)]),
                 lambda: clip_grads_with_norm_(as_params(g), 1.0, torch.ones(2))):
        with pytest.raises(ValueError):
            call()
    g[0][1] = math.nan
    before = [t.clone() for t in g]
    with pytest.raises(RuntimeError, match="nan"):
        clip_grad_norm_((p for p in as_params(g)), 1.0, error_if_nonfinite=True)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(g, before))


LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genie-tk_amd", "genie_tk",
                   "libgenie_tk_hip.so")
i64, sz, vp, dp, ci = ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_double, ctypes.c_int


class TensorList(ctypes.Structure):
    _fields_ = [("count", i64), ("data", ctypes.POINTER(vp)), ("numel", ctypes.POINTER(i64)),
                ("dtype", ctypes.POINTER(ci))]


def c_list(entries):
    n = len(entries)
    return TensorList(n, (vp * n)(*(e[0] for e in entries)), (i64 * n)(*(e[1] for e in entries)),
                      (ci * n)(*(e[2] for e in entries)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    L = ctypes.CDLL(LIB)
    L.gtk_last_error.restype = ctypes.c_char_p
    pl = ctypes.POINTER(TensorList)
    L.gtk_grad_norm_workspace_size.restype = sz
    L.gtk_grad_norm_workspace_size.argtypes = [pl]
    L.gtk_grad_norm.argtypes = [pl, ci, vp, vp, sz, vp]
    L.gtk_grad_clip.argtypes = [pl, pl, ci, dp, vp, vp, sz, vp]
    L.gtk_grad_clip_with_norm.argtypes = [pl, pl, dp, vp, vp]
    return L


def test_c_refusals(lib):
    # addresses that are never dereferenced: every call is refused on the host
    ok = c_list([(4096, 8, 0), (8192, 8, 1)])
    big = 1 << 30
    norm = lambda g=ok, kind=0, n=64, ws=64, b=big: lib.gtk_grad_norm(  # noqa: E731
        ctypes.byref(g) if g is not None else None, kind, n, ws, b, None)
    bad_lists = [c_list([(None, 8, 0)]), c_list([(4096, -1, 0)]), c_list([(4096, 8, 2)]), c_list([(4096, 1 << 41, 0)]),
                 TensorList(-1, None, None, None), TensorList(2, None, None, None)]
    for bad in bad_lists:
        assert norm(bad) == 1
        assert lib.gtk_grad_norm_workspace_size(ctypes.byref(bad)) == 0
    assert [norm(None), norm(kind=3), norm(n=None), norm(ws=None), norm(ws=65)] == [1] * 5
    need = lib.gtk_grad_norm_workspace_size(ctypes.byref(ok))
    assert need > 0 and norm(b=need - 1) == 3

    def clip(g=ok, out=None, max_norm=1.0):
        return lib.gtk_grad_clip(ctypes.byref(g), None if out is None else ctypes.byref(out), 0, max_norm, 64, 64, big,
                                 None)

    def scale(g=ok, out=None, max_norm=1.0, n=64):
        return lib.gtk_grad_clip_with_norm(ctypes.byref(g), None if out is None else ctypes.byref(out), max_norm, n,
                                           None)

    for call in (clip, scale):
        assert [call(max_norm=-1.0), call(max_norm=math.nan)] == [1, 1]
        twice = c_list([(4096, 8, 0), (4096, 8, 0)])
        assert call(twice) == 1 and b"twice" in lib.gtk_last_error()
        assert call(c_list([(4112, 8, 0), (4096, 8, 0)])) == 1              # 4096..4128 and 4112..4144
        assert call(ok, c_list([(1 << 20, 8, 0)])) == 1                     # one output for two gradients
        assert call(ok, c_list([(1 << 20, 8, 0), (1 << 21, 9, 0)])) == 1    # another size
        assert call(ok, c_list([(4096, 8, 1), (1 << 21, 8, 0)])) == 1       # onto itself in another type
        assert call(ok, c_list([(8192, 8, 0), (1 << 21, 8, 0)])) == 1       # onto another gradient
        assert call(ok, c_list([(1 << 21, 8, 0), (1 << 21, 8, 0)])) == 1    # one output twice
    assert scale(n=None) == 1
    empty = c_list([])
    assert scale(empty) == 0 and scale(c_list([(None, 0, 0)])) == 0         # nothing to do


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
SETS = {
    "one value": [1],
    "small": [1, 2, 3, 7, 8, 9, 64, 127, 128, 129, 1000],
    "empty ones": [0, 5, 0, 0, 4097, 0],
    "one layer": [128, 128, 16384, 128, 16384, 128, 65536, 512, 65536, 128],
    "many": [17 + 13 * (k % 29) for k in range(731)],
    "uneven": [3_000_001, 5, 70_000, 1, 262_144, 31],
}


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dts", ["fp32", "bf16", "fp32 bf16"])
@pytest.mark.parametrize("name", list(SETS))
def test_sets(name, dts, p):
    print("gradients", name, dts, p, flush=True)
    grads = make(SETS[name], 3, [DT[d] for d in dts.split()], "cuda")
    before = [g.clone() for g in grads]
    ref = check_norm(grad_norm(grads, p), grads, p)
    for limit in (0.3 * ref, 3.0 * ref):
        norm, outs = clip_grads(grads, limit, p)
        assert float(norm) == float(grad_norm(grads, p))
        assert all(o.dtype == g.dtype for o, g in zip(outs, grads))
        check_clipped(outs, before, limit, ref)
        masters = [torch.full_like(g, math.nan, dtype=torch.float32) for g in grads]
        clip_grads(grads, limit, p, out=masters)
        check_clipped(masters, before, limit, ref)
        narrow = [torch.full_like(g, math.nan, dtype=torch.bfloat16) for g in grads]
        clip_grads(grads, limit, p, out=narrow)
        check_clipped(narrow, before, limit, ref)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    # below the limit nothing changes
    assert all(torch.equal(o, g) for o, g in zip(clip_grads(grads, 3.0 * ref, p)[1], grads))
    ps = as_params(grads)
    norm = clip_grad_norm_(iter(ps), 3.0 * ref, p)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    clip_grad_norm_(ps, 0.3 * ref, p)
    check_clipped(grads, before, 0.3 * ref, ref)


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_packed_at_any_alignment(dt):
    """Gradients right behind one another: a tensor's neighbours stay as they are."""
    sizes = [1, 3, 517, 2, 8191, 8192, 8193, 40_001, 5, 65_537]
    flat = torch.randn(sum(sizes) + 40, device="cuda").to(DT[dt])
    at, views = 7, []
    for k, n in enumerate(sizes):
        views.append(flat[at:at + n])
        at += n + k % 3
    before, whole = [v.clone() for v in views], flat.clone()
    ref = check_norm(grad_norm(views), views, 2.0)
    master = torch.full((flat.numel() + 3,), 5.0, device="cuda")
    outs = [master[3 + v.storage_offset():][:v.numel()] for v in views]
    clip_grads(views, 0.5 * ref, out=outs)
    check_clipped(outs, before, 0.5 * ref, ref)
    clip_grad_norm_(as_params(views), 0.5 * ref)
    check_clipped(views, before, 0.5 * ref, ref)
    inside = torch.zeros(flat.numel(), dtype=torch.bool, device="cuda")
    for v in views:
        inside[v.storage_offset():v.storage_offset() + v.numel()] = True
    assert torch.equal(flat[~inside], whole[~inside])
    assert (master[3:][~inside] == 5.0).all() and (master[:3] == 5.0).all()


@gpu
def test_one_behind_the_other():
    """Neighbours are one run only where both sides are neighbours of one type."""
    raw = torch.randn(40_000, device="cuda")
    a, b, c, d = raw[:9000], raw[9000:9000], raw[9000:9003], raw[9003:20_000]
    e = raw[20_000:20_500].view(torch.bfloat16)  # right behind d, another type
    e.copy_(torch.randn(1000))
    f = raw[20_500:30_000]
    every = [a, b, c, d, e, f]
    before = [g.clone() for g in every]
    ref = check_norm(grad_norm(every), every, 2.0)
    apart = [torch.full_like(g, math.nan) for g in every]
    together = torch.full((40_000,), 7.0, device="cuda")
    ends = [0, 9000, 9000, 9003, 20_000, 21_000, 30_500]
    fp32 = [together[lo:hi] for lo, hi in zip(ends, ends[1:])]
    for outs in (apart, fp32, fp32[:3] + apart[3:]):
        clip_grads(every, 0.5 * ref, out=outs)
        check_clipped(outs, before, 0.5 * ref, ref)
    assert (together[30_500:] == 7.0).all()
    order = [5, 3, 0, 4, 2, 1]
    clip_grad_norm_(as_params([every[k] for k in order]), 0.5 * ref)
    check_clipped(every, before, 0.5 * ref, ref)


@gpu
def test_strides():
    base = torch.randn(40, 60, device="cuda")
    dense, gapped, repeated = base.t(), torch.randn(50, 70, device="cuda")[:, 5:23], torch.randn(9, 1, device="cuda").expand(9, 30)
    every = [dense, gapped, repeated]
    ref = check_norm(grad_norm(every), every, 2.0)
    norm, outs = clip_grads(every, 0.5 * ref)
    check_clipped(outs, every, 0.5 * ref, ref)
    outs = [torch.empty(60, 40, device="cuda"), torch.empty(18, 50, device="cuda").t(),
            torch.empty(30, 9, device="cuda", dtype=torch.bfloat16).t()]
    clip_grads(every, 0.5 * ref, out=outs)
    check_clipped(outs, every, 0.5 * ref, ref)
    before = [dense.clone(), gapped.clone()]
    ref = train_ops.global_norm([np64(t) for t in before])
    clip_grad_norm_(as_params([dense, gapped]), 0.5 * ref)
    check_clipped([dense, gapped], before, 0.5 * ref, ref)
    with pytest.raises(RuntimeError):
        _ext.require().grad_clip([repeated], None, 1.0)
    with pytest.raises(RuntimeError, match="twice"):
        _ext.require().grad_clip([gapped, gapped], None, 1.0)


@gpu
def test_sizes_at_the_edges_of_fp32():
    """Squares that 32 bits cannot hold."""
    for scale in (1e30, 1e-30, 3e-39, 2e38):
        g = [torch.randn(5000, device="cuda").clamp(-1.5, 1.5) * scale, torch.full((3,), scale, device="cuda")]
        for p in (2.0, INF):
            check_norm(grad_norm(g, p), g, p)
        h = [t.bfloat16() for t in g]
        check_norm(grad_norm(h), h, 2.0)
    # the norm itself past fp32: infinite, and the factor zero
    g = [torch.full((64,), 3e38, device="cuda")]
    norm, (out,) = clip_grads(g, 1.0)
    assert float(norm) == INF and (out == 0).all()


@gpu
def test_products_among_the_smallest_values():
    """Products below the normal range are rounded to its steps (2^-149 fp32,
    2^-133 bf16), not flushed to zero."""
    g = torch.tensor([1e-38, 5e-39, 7e-41, 3e-45, -2e-39] * 20, device="cuda")
    for t in (g, g.bfloat16()):
        for out in (torch.float32, torch.bfloat16):
            step = 2.0 ** -149 if out == torch.float32 else 2.0 ** -133
            o = torch.empty(100, device="cuda", dtype=out)
            _ext.require().grad_clip_with_norm([t], [o], 0.25, torch.ones(1, device="cuda"))
            ref = np64(t) * train_ops.clip_factor(1.0, 0.25)
            # half a step, and twice where the product is rounded to fp32 before bf16
            assert (np.abs(np64(o) - ref) <= 0.5 * step + 2.0 ** -150 + 4 * U * np.abs(ref)).all()
            assert (np64(o)[np.abs(ref) > step] != 0).all()


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_not_finite(dt, p):
    for bad, want in ((math.nan, math.nan), (INF, INF), (-INF, INF)):
        grads = make([300, 40_000, 11], 5, [DT[dt]], "cuda")
        grads[1][39_999] = bad
        before = [g.clone() for g in grads]
        assert math.isnan(float(grad_norm(grads, p))) if math.isnan(want) else float(grad_norm(grads, p)) == want
        with pytest.raises(RuntimeError, match="nan" if math.isnan(want) else "inf"):
            clip_grad_norm_(as_params(grads), 1.0, p, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(grads, before))
        _, outs = clip_grads(grads, 1.0, p)
        if math.isnan(want):
            assert all(o.isnan().all() for o in outs)
        else:  # 0 * inf is NaN, the rest is 0
            assert outs[1][39_999].isnan() and (outs[1][:39_999] == 0).all() and (outs[0] == 0).all()
    # both in one set: NaN
    grads[0][0], grads[2][1] = INF, math.nan
    assert math.isnan(float(grad_norm(grads, p)))
    grads = make([300, 11], 5, [DT[dt]], "cuda")
    assert all(o.isnan().all() for o in clip_grads(grads + [torch.full((1,), math.nan, device="cuda")], INF, p)[1])
    norm = clip_grad_norm_(as_params(grads), INF, p, error_if_nonfinite=True)
    assert math.isfinite(float(norm))


@gpu
def test_zero_gradients_and_zero_limit():
    grads = [torch.zeros(100, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.bfloat16)]
    norm, outs = clip_grads(grads, 0.0)
    assert float(norm) == 0.0 and all((o == 0).all() for o in outs)
    grads = make([100, 3], 0, [torch.float32], "cuda")
    assert all((o == 0).all() for o in clip_grads(grads, 0.0)[1])
    empty = [torch.empty(0, device="cuda")]
    assert float(grad_norm(empty)) == 0.0 and clip_grads(empty, 1.0)[1][0].numel() == 0


@gpu
def test_given_norm_and_versions():
    grads = make([3000, 5, 129], 8, [torch.float32, torch.bfloat16], "cuda")
    before = [g.clone() for g in grads]
    ps = as_params(grads)
    ps.insert(1, torch.nn.Parameter(torch.zeros(4, device="cuda")))  # without a gradient
    versions = [g._version for g in grads]
    for total in (torch.tensor(8.0), torch.tensor([8.0], device="cuda", dtype=torch.float64)):
        for g, b in zip(grads, before):
            g.copy_(b)
        clip_grads_with_norm_(iter(ps), 2.0, total)
        check_clipped(grads, before, 2.0, 8.0)
    assert all(g._version > v for g, v in zip(grads, versions))


@gpu
def test_same_bits_on_every_call_and_stream():
    grads = make(SETS["many"] + [2_000_003], 4, [torch.float32, torch.bfloat16], "cuda")
    first = clip_grads(grads, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = clip_grads(grads, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], second[0]) and all(torch.equal(a, b) for a, b in zip(first[1], second[1]))


@gpu
def test_captured_and_replayed():
    C = _ext.require()
    grads = make(SETS["many"], 4, [torch.float32], "cuda")
    outs = [torch.empty_like(g) for g in grads]
    C.grad_clip(grads, outs, 0.1)
    torch.cuda.synchronize()
    graphs, norms = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(C.grad_clip(grads, outs, 0.1))
        graphs.append(g)
    for k in range(4):
        for g, new in zip(grads, make(SETS["many"], 20 + k, [torch.float32], "cuda")):
            g.copy_(new)
        ref, want = clip_grads(grads, 0.1)
        for g in graphs:
            for o in outs:
                o.fill_(math.nan)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), k
        assert all(torch.equal(n, ref) for n in norms)


@gpu
def test_sizes_past_32_bits():
    n = (1 << 31) + 4099
    big = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 1 << 30, (1 << 31) - 1, 1 << 31, n - 2, n - 1], device="cuda")
    big[at] = torch.tensor([3.0, 4.0, 1.0, 2.0, 5.0, 3.0], device="cuda", dtype=torch.bfloat16)  # norm 8
    small = [torch.zeros(5, device="cuda")]
    assert float(grad_norm([big] + small)) == 8.0 and float(grad_norm([big], INF)) == 5.0
    assert float(clip_grad_norm_(as_params(small + [big]), 4.0)) == 8.0
    # the factor 4 / (8 + 1e-6) is 0.5 to 2^-23: half the values, which bf16 holds exactly
    assert torch.equal(big[at], torch.tensor([1.5, 2.0, 0.5, 1.0, 2.5, 1.5], device="cuda", dtype=torch.bfloat16))
    assert int((big != 0).sum()) == 6


@gpu
def test_gpu_refusals():
    C = _ext.require()
    g = [torch.ones(8, device="cuda"), torch.ones(4, device="cuda")]
    with pytest.raises(ValueError):
        grad_norm([g[0], torch.ones(3)])
    with pytest.raises(ValueError):
        clip_grads(g, 1.0, out=[torch.ones(8), torch.ones(4)])
    for call in (lambda: C.grad_norm([]), lambda: C.grad_norm([torch.ones(3)]), lambda: C.grad_norm([g[0], torch.ones(3)]),
                 lambda: C.grad_norm([g[0].half()]), lambda: C.grad_norm(g, 3.0), lambda: C.grad_clip(g, None, -1.0),
                 lambda: C.grad_clip(g, g[:1], 1.0), lambda: C.grad_clip(g, [g[1], g[0]], 1.0),
                 lambda: C.grad_clip([g[0], g[0]], None, 1.0), lambda: C.grad_clip([g[0], g[0][2:5]], None, 1.0),
                 lambda: C.grad_clip_with_norm(g, None, 1.0, torch.ones(1)),
                 lambda: C.grad_clip_with_norm(g, None, 1.0, torch.ones(2, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
    assert all((t == 1).all() for t in g)
    # the same gradient may be read twice: only written ones must be apart
    assert float(C.grad_norm([g[0], g[0]])) == 4.0
    # orders and types beyond the kernels' run in PyTorch
    torch.testing.assert_close(grad_norm(g, 3.0), torch.tensor(12.0, device="cuda") ** (1 / 3))
    h = [torch.ones(9, device="cuda", dtype=torch.float16)]
    assert float(clip_grad_norm_(as_params(h), 1.5)) == 3.0 and (h[0] == 0.5).all()


# ---------------------------------------------------------------------------
# Both operators in a training step
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_training_step_with_the_pair_stack(dt):
    """A pair-stack layer and a LayerNorm over its output: the norm of all
    gradients, their clipping, and the LayerNorm's own gradients against 64 bits."""
    from genie_tk.pair_transform import PairTransformNet
    from genie_tk.primitives import LayerNorm
    from tests.test_layer_norm_ops import check_all

    torch.manual_seed(0)
    net = PairTransformNet(64, 1, c_hidden_mul=64, tri_dropout=0.0)
    head = LayerNorm(64)
    with torch.no_grad():
        for p in net.parameters():
            if p.dim() == 2:
                p.normal_(0, p.shape[1] ** -0.5)
    net, head = net.to("cuda", DT[dt]), head.cuda()
    N = 37
    p = torch.randn(1, N, N, 64, device="cuda").to(DT[dt])
    mask = torch.ones(1, N, N, device="cuda")
    mask[:, 30:] = 0
    mask[:, :, 30:] = 0
    up = torch.randn(1, N, N, 64, device="cuda").to(DT[dt])
    trunk = net(p, mask)
    trunk.retain_grad()
    y = head(trunk)
    y.backward(up)
    check_all(trunk, up, head.weight, head.bias, y, trunk.grad, head.weight.grad, head.bias.grad)
    every = [*net.parameters(), *head.parameters()]
    before = [q.grad.clone() for q in every]
    ref = train_ops.global_norm([np64(g) for g in before])
    norm = clip_grad_norm_(every, 0.25 * ref)
    check_norm(norm, before, 2.0)
    check_clipped([q.grad for q in every], before, 0.25 * ref, ref)


# ---------------------------------------------------------------------------
# Written tensors that overlap
# ---------------------------------------------------------------------------
def view_pairs(count, seed, device):
    """Pairs of views of one buffer of distinct values, each without overlap in
    itself, with the answer whether they share a value: by their elements'
    places.  Strides nest or not, dimensions in any order."""
    rng = np.random.default_rng(seed)
    for _ in range(count):
        base = torch.arange(1.0, 4001.0, device=device)
        places = torch.arange(4000)
        pair = []
        strides = [int(rng.choice([1, 1, 2, 3]))]
        for _ in range(2):
            while True:
                if rng.random() < 0.5:  # each its own
                    strides = [int(rng.choice([1, 1, 2, 3]))]
                sizes, mine = [], []
                for k in range(int(rng.integers(1, 4))):
                    if k == len(strides):
                        strides.append(int(strides[-1] * sizes[-1] + rng.integers(0, 9)))
                    sizes.append(int(rng.integers(1, 7)))
                    mine.append(strides[k])
                order = rng.permutation(len(sizes))
                shape, step = [sizes[k] for k in order], [mine[k] for k in order]
                room = 1 + sum((n - 1) * s for n, s in zip(shape, step))
                at = int(rng.integers(0, 60))
                if room + at <= 4000:
                    where = torch.as_strided(places, shape, step, at)
                    if where.unique().numel() == where.numel():
                        break
            pair.append((torch.as_strided(base, shape, step, at), set(where.flatten().tolist())))
        (a, ia), (b, ib) = pair
        yield base, a, b, bool(ia & ib)


def check_view_pairs(device):
    met = apart = 0
    for base, a, b, share in view_pairs(300, 11, device):
        before = base.clone()
        if share:
            met += 1
            with pytest.raises(RuntimeError, match="overlaps another"):
                clip_grad_norm_(as_params([a, b]), 0.5)
            assert torch.equal(base, before)
            continue
        apart += 1
        ga, gb = a.clone(), b.clone()
        norm = clip_grad_norm_(as_params([a, b]), 0.5)
        ref = check_norm(norm, [ga, gb], 2.0)
        check_clipped([a, b], [ga, gb], 0.5, ref)
        assert int((base != before).sum()) == a.numel() + b.numel()  # and nothing between them
    assert met > 60 and apart > 60


def check_overlap_refusals(device):
    """Overlapping written tensors in each of the calls; their neighbours pass."""
    base = torch.arange(1.0, 49.0, device=device).view(6, 8)
    other = torch.arange(1.0, 49.0, device=device).view(6, 8)
    before = base.clone()
    wide = base[:, 0:5]
    half_words = base.view(torch.bfloat16)[:, 7:9]  # the upper half of column 3 and the lower of column 4
    bad = [[wide, base[:, 3:8]], [base, wide], [wide, base.flatten()[17:19]], [wide, wide], [base[::2], base[4:, :3]],
           [base[1:, ::2], base[:3, ::4]], [wide, half_words], [base.t()[2:5], base[5:]]]
    for pair in bad:
        total = torch.ones((), device=device)
        for call in (lambda: clip_grad_norm_(as_params(pair), 0.5), lambda: clip_grads_with_norm_(as_params(pair), 0.5, total),
                     lambda: clip_grad_norm_(as_params(pair), 0.5, 3.0),
                     lambda: clip_grads([other[:t.shape[0], :t.shape[1]] if t.dim() == 2 else other.flatten()[:t.numel()]
                                         for t in pair], 0.5, out=pair)):
            with pytest.raises(RuntimeError, match="overlaps another"):
                call()
    # onto another gradient of the call
    with pytest.raises(RuntimeError, match="overlaps another"):
        clip_grads([wide, other[:, 1:3]], 0.5, out=[other[:, 2:7], torch.empty(6, 2, device=device)])
    assert torch.equal(base, before)
    # read twice, and written onto themselves
    clip_grads([wide, wide, base], 0.5)
    clip_grads([wide, base[:, 5:]], 0.5, out=[wide, base[:, 5:]])
    ref = train_ops.global_norm([np64(before)])
    check_clipped([base], [before], 0.5, ref)


@gpu
def test_overlapping_views_on_the_kernels():
    check_view_pairs("cuda")
    check_overlap_refusals("cuda")


def test_overlapping_views_on_the_pytorch_path():
    check_view_pairs("cpu")
    check_overlap_refusals("cpu")
    p = torch.nn.Parameter(torch.zeros(4))  # a shared parameter listed twice
    p.grad = torch.ones(4)
    for call in (lambda: clip_grad_norm_([p, p], 0.5), lambda: clip_grads_with_norm_([p, p], 0.5, torch.tensor(2.0))):
        with pytest.raises(RuntimeError, match="given twice"):
            call()
    assert torch.equal(p.grad, torch.ones(4))


@gpu
def test_overlapping_views_in_types_beyond_the_kernels():
    base = torch.ones(6, 8, device="cuda", dtype=torch.float16)
    with pytest.raises(RuntimeError, match="overlaps another"):
        clip_grad_norm_(as_params([base[:, :5], base[:, 3:]]), 0.5)
    assert (base == 1).all()
    clip_grad_norm_(as_params([base[:, :5], base[:, 5:]]), 0.5)
    assert (base < 0.1).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_an_expanded_gradient_leaves_the_others_alone(device):
    first = torch.ones(4, device=device)
    grads = [first, torch.ones(3, 1, device=device).expand(3, 5)]
    with pytest.raises(RuntimeError):
        clip_grad_norm_(as_params(grads), 0.5)
    with pytest.raises(RuntimeError):
        clip_grads_with_norm_(as_params(grads), 0.5, torch.tensor(4.0))
    assert torch.equal(first, torch.ones(4, device=device))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gradients_that_require_gradients(device):
    """Clipping is not recorded by autograd (as torch's is not), whatever the strides."""
    for cols in (slice(0, 8), slice(0, 5)):
        leaf = torch.empty_strided((6, 8), (8, 1), device=device)[:, cols].fill_(2.0).requires_grad_(True)
        x = torch.ones(6, 8, device=device, requires_grad=True)
        whole = x * 3.0  # as with create_graph
        graph = whole[:, cols]
        out = torch.empty(6, 8, device=device)[:, cols]
        norm, outs = clip_grads([leaf, graph], 0.5)
        n2, _ = clip_grads([leaf], 0.5, out=[out])
        assert not any(t.requires_grad for t in (norm, n2, out, *outs)) and not grad_norm([graph]).requires_grad
        before = [leaf.detach().clone(), graph.detach().clone()]
        p, q = as_params([before[0], before[1]])  # their gradients are set below
        p.grad, q.grad = leaf, graph
        ref = train_ops.global_norm([np64(b) for b in before])
        clip_grad_norm_([p, q], 0.5)
        check_clipped([leaf, graph], before, 0.5, ref)
        assert leaf.is_leaf and whole.grad_fn.name() == "MulBackward0"  # a recorded copy would be CopySlices


def test_calls_take_torchs_arguments():
    import inspect

    for ours, theirs in ((clip_grad_norm_, torch.nn.utils.clip_grad_norm_),
                         (clip_grads_with_norm_, torch.nn.utils.clip_grads_with_norm_)):
        ours, theirs = ([(p.name, p.default) for p in inspect.signature(f).parameters.values()] for f in (ours, theirs))
        assert ours == theirs
    for foreach in (True, False, None):
        ps = as_params([torch.full((4,), 2.0)])
        assert float(clip_grad_norm_(ps, 1.0, foreach=foreach)) == 4.0
        before = [ps[0].grad.clone()]
        check_clipped(before, [torch.full((4,), 2.0)], 1.0, 4.0)
        clip_grads_with_norm_(ps, 0.5, torch.tensor(1.0), foreach=foreach)
        check_clipped([ps[0].grad], before, 0.5, 1.0)


def test_timed_clipping_does_the_same_work_in_every_call():
    import bench

    grads = make([40, 7, 300], 2, [torch.float32, torch.bfloat16])
    before = [g.clone() for g in grads]
    params = [*as_params(grads), torch.nn.Parameter(torch.zeros(2))]
    ref = train_ops.global_norm([np64(g) for g in before])
    above, below = bench.clip_calls(params).values()
    for _ in range(12):
        norm, outs = above()
        check_norm(norm, before, 2.0)
        check_clipped(outs, before, 0.5 * float(norm), ref)
        check_norm(below(), before, 2.0)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
