"""Dropout with a counter-based generator (genie_tk.primitives.dropout, the row- and
column-shared forms of the pair stack, genie_tk._C.dropout, gtk_dropout): the
generator's published vectors, the oracle, the PyTorch path and the refusals on the
CPU, the kernels against the 64-bit oracle on the GPU.

Tolerances.  Masks are equal.  With u = 2^-24: the scale is rounded to fp32 (u), the
product and the sum to fp32 (u each), the result to its type (half_t of it).  A
dropped value without residual is exactly 0."""
import ctypes
import os

import numpy as np
import pytest
import torch

from genie_tk import PairTransformLayer, PairTransformNet, _ext
from genie_tk.pair_transform import DropoutColumnwise, DropoutRowwise
from genie_tk.primitives import dropout, dropout_mask
from oracle import train_ops

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
SEED = 0x9E3779B97F4A7C15
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().double().cpu().numpy()


def values(shape, seed, dtype, device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * 1.5).to(dtype).to(device)


def check(y, x, p, seed, offset=0, shared_dim=None, residual=None):
    """y = residual + dropout(x) within the roundings."""
    r = None if residual is None else np64(residual)
    ref = train_ops.dropout(np64(x), p, seed, offset, shared_dim, r)
    part = train_ops.dropout(np64(x), p, seed, offset, shared_dim)
    got = np64(y)
    assert got.shape == ref.shape
    err = 2 * U * np.abs(part) + U * np.abs(ref)
    excess = np.abs(got - ref) - ((half(y.dtype) + U) * np.abs(ref) + 2 * err + 1e-38)
    assert (excess <= 0).all(), f"{int((excess > 0).sum())} of {excess.size} out of tolerance"
    if residual is None:
        assert ((got == 0) | (part != 0)).all()
    return ref


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------
def test_published_vectors():
    """The generator's known answers, as distributed with the paper."""
    ones = (1 << 64) - 1
    pi = [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0]
    cases = [((0, 0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
             ((ones, ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
             ((pi[1] << 32 | pi[0], pi[3] << 32 | pi[2], pi[5] << 32 | pi[4]),
              (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for (counter, offset, key), words in cases:
        assert tuple(train_ops.philox([counter], offset, key)[0]) == words


@pytest.mark.parametrize("shape,dim", [((5, 7, 9), None), ((2, 5, 4, 24), -3), ((2, 5, 4, 24), -2), ((3, 6, 11), 1),
                                       ((6, 3), 0), ((4, 10), -1), ((1,), None), ((1, 1, 8), 0), ((0, 4), None),
                                       ((3, 0, 4), 1)])
def test_mask_matches_the_oracle(shape, dim):
    for seed, offset in ((0, 0), (SEED, 3), (-1, 2 ** 40 + 7), (2 ** 63 + 5, 2 ** 64 - 1)):
        got = dropout_mask(shape, 0.3, seed, offset, dim)
        sizes, outer = list(shape), 1
        if dim is not None:
            sizes[dim] = 1
            outer = int(np.prod(shape[:dim % len(shape)]))
        assert list(got.shape) == sizes and got.dtype == torch.bool
        if got.numel():
            ref = train_ops.dropout_keep(outer, got.numel() // outer, 0.3, seed % 2 ** 64, offset)
            assert np.array_equal(got.numpy().reshape(ref.shape), ref)


def test_mask_is_a_function_of_seed_and_offset():
    one = dropout_mask((64, 100), 0.4, SEED, 1)
    assert torch.equal(one, dropout_mask((64, 100), 0.4, SEED, 1))
    assert torch.equal(one, dropout_mask((64, 100), 0.4, torch.tensor(SEED - 2 ** 64), 1))
    for other in (dropout_mask((64, 100), 0.4, SEED + 1, 1), dropout_mask((64, 100), 0.4, SEED, 2)):
        # two independent masks of 6400 agree on 0.52 of them, +- 5 standard deviations
        assert abs((one == other).float().mean().item() - 0.52) < 5 * (0.52 * 0.48 / 6400) ** 0.5
    # what is kept at a larger p is kept at a smaller one too
    assert (dropout_mask((64, 100), 0.6, SEED, 1) <= one).all()


@pytest.mark.parametrize("p", [0.0, 1e-6, 2.0 ** -16, 0.1, 0.25, 0.5, 0.9, 1.0 - 2.0 ** -16, 1.0])
def test_share_of_dropped_values(p):
    n = 1 << 18
    kept = dropout_mask((n,), p, 11).sum().item()
    q = 1 - round(65536 * p) / 65536
    assert abs(kept - n * q) <= 5 * (n * q * (1 - q)) ** 0.5
    x = torch.ones(n, dtype=torch.float64)
    y = dropout(x, p, 11)
    assert y.count_nonzero().item() == kept
    if kept:
        assert y.max().item() == 1 / q
    if p == 0:
        assert torch.equal(y, x)


@pytest.mark.parametrize("dt,rt", [("fp32", None), ("bf16", None), ("fp32", "fp32"), ("bf16", "bf16"),
                                   ("bf16", "fp32"), ("fp32", "bf16")])
def test_pytorch_path(dt, rt):
    x = values((2, 5, 6, 20), 0, DT[dt]).requires_grad_(True)
    r = None if rt is None else values(x.shape, 1, DT[rt]).requires_grad_(True)
    for dim in (None, -3, -2):
        y = dropout(x, 0.25, SEED, 9, dim, r)
        assert y.dtype == (x.dtype if r is None else torch.promote_types(x.dtype, r.dtype))
        check(y, x, 0.25, SEED, 9, dim, r)
        dy = values(x.shape, 2, y.dtype)
        dx, *dr = torch.autograd.grad(y, [x] if r is None else [x, r], dy)
        assert dx.dtype == x.dtype
        check(dx, dy, 0.25, SEED, 9, dim)
        assert not dr or torch.equal(dr[0], dy.to(r.dtype))


def test_pytorch_path_in_other_types():
    x = values((6, 50), 0, torch.float64)
    t = round(65536 * 0.25)
    assert torch.equal(dropout(x, 0.25, 3), torch.where(dropout_mask(x.shape, 0.25, 3), x * (65536 / (65536 - t)), 0.0))
    assert dropout(x.half(), 0.25, 3).dtype == torch.float16
    dual, tangent = torch.autograd.forward_ad, torch.ones_like(x)
    with dual.dual_level():
        out = dual.unpack_dual(dropout(dual.make_dual(x, tangent), 0.25, 3))
    assert torch.equal(out.tangent, dropout(tangent, 0.25, 3))


def test_dropped_values_count_for_nothing():
    keep = dropout_mask((3, 40), 0.5, 7)
    x = torch.where(keep, 1.0, float("nan")).requires_grad_(True)
    r = torch.ones(3, 40)
    y = dropout(x, 0.5, 7, residual=r)
    assert torch.equal(y.detach(), r + 2.0 * keep)
    y.sum().backward()
    assert torch.equal(x.grad, 2.0 * keep)


def test_refusals():
    x = torch.ones(2, 3, 4)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            dropout(x, p, 0)
    for dim in (3, -4):
        with pytest.raises(IndexError, match="shared_dim"):
            dropout(x, 0.5, 0, shared_dim=dim)
    with pytest.raises(ValueError, match="residual"):
        dropout(x, 0.5, 0, residual=x[:1])
    for seed in (torch.ones(1), torch.ones(2, dtype=torch.int64), torch.ones(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="seed tensor"):
            dropout(x, 0.5, seed)
    with pytest.raises(TypeError):
        dropout(x, 0.5, 1.5)
    if _ext.C is not None:
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            _ext.C.dropout(x, 0.5, 0)


def layer_of(c=16, p=0.25, **kw):
    torch.manual_seed(0)
    layer = PairTransformLayer(c_p=c, c_hidden_mul=8, c_hidden_tri_att=8, n_head_tri=2, tri_dropout=p, **kw)
    with torch.no_grad():
        for prm in layer.parameters():
            if not prm.any():
                prm.normal_(std=0.3)
    return layer


def test_shared_dropout_modules():
    x, r = values((2, 5, 6, 16), 0, torch.float32), values((2, 5, 6, 16), 1, torch.float32)
    for mod, dim in ((DropoutRowwise(0.25), -3), (DropoutColumnwise(0.25), -2)):
        assert torch.equal(mod.train()(x, SEED, 4, r), dropout(x, 0.25, SEED, 4, dim, r))
        assert torch.equal(mod(x, SEED), dropout(x, 0.25, SEED, 0, dim))
        assert torch.equal(mod.eval()(x, SEED, 4, r), r + x) and torch.equal(mod(x, SEED), x)
        # without a seed: torch's generator, as before
        torch.manual_seed(1)
        y = mod.train()(x)
        torch.manual_seed(1)
        shape = [2, 5, 6, 16]
        shape[dim] = 1
        assert torch.equal(y, x * torch.nn.functional.dropout(torch.ones(shape), 0.25))


def test_pair_layer_and_net_with_a_seed():
    layer = layer_of().train()
    p, mask = values((1, 6, 6, 16), 0, torch.float32), torch.ones(1, 6, 6)
    out, m = layer((p, mask), 5, 8)
    q = p
    for k, (drop, op) in enumerate(((layer.dropout_row, layer.tri_mul_out), (layer.dropout_row, layer.tri_mul_in),
                                    (layer.dropout_row, layer.tri_att_start), (layer.dropout_col, layer.tri_att_end))):
        q = dropout(op(q, mask), 0.25, 5, 8 + k, drop._shared_dim, q)
    q = (q + layer.pair_transition(q, mask)) * mask.unsqueeze(-1)
    assert m is mask and torch.equal(out, q)
    assert not torch.equal(out, layer((p, mask), 6, 8)[0]) and not torch.equal(out, layer((p, mask), 5, 0)[0])
    # in eval the seed changes nothing
    assert torch.equal(layer.eval()((p, mask), 5)[0], layer((p, mask))[0])
    # without a seed: torch's generator, as before
    torch.manual_seed(3)
    a, _ = layer.train()((p, mask))
    torch.manual_seed(3)
    q = p + layer.dropout_row(layer.tri_mul_out(p, mask))
    q = q + layer.dropout_row(layer.tri_mul_in(q, mask))
    q = q + layer.dropout_row(layer.tri_att_start(q, mask))
    q = q + layer.dropout_col(layer.tri_att_end(q, mask))
    assert torch.equal(a, (q + layer.pair_transition(q, mask)) * mask.unsqueeze(-1))

    net = PairTransformNet(16, 2, c_hidden_mul=8, c_hidden_tri_att=8, n_head_tri=2).train()
    for mine in net.layers:
        mine.load_state_dict(layer.state_dict())
    (q, _) = net.layers[1](net.layers[0]((p, mask), 77, 0), 77, 4)
    assert torch.equal(net(p, mask, 77), q) and torch.equal(net(p, mask, dropout_seed=torch.tensor([77])), q)
    # recomputation under activation checkpoints draws the same masks
    from torch.utils.checkpoint import checkpoint
    plain = torch.autograd.grad(net(p, mask, 77).sum(), list(net.parameters()))
    again = torch.autograd.grad(checkpoint(net, p.requires_grad_(True), mask, 77, use_reentrant=False).sum(),
                                list(net.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(plain, again))


LIB = os.path.join(os.path.dirname(os.path.abspath(_ext.__file__)), "libgenie_tk_hip.so")
i64, u64, vp, f64, ci = ctypes.c_int64, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_double, ctypes.c_int


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    L = ctypes.CDLL(LIB)
    L.gtk_last_error.restype = ctypes.c_char_p
    L.gtk_dropout.argtypes = [vp, ci, vp, ci, vp, ci, i64, i64, i64, f64, u64, vp, u64, vp]
    return L


def test_c_refusals(lib):
    q = 4096  # never dereferenced: every call below is refused on the host, or has nothing to do
    call = lambda x=q, d=0, r=None, rd=0, o=q, od=0, a=2, s=3, i=4, p=0.5: lib.gtk_dropout(  # noqa: E731
        x, d, r, rd, o, od, a, s, i, p, 1, None, 0, None)
    bad = [call(x=None), call(o=None), call(d=2), call(od=-1), call(r=q, rd=1), call(r=q, d=0, rd=1, od=1),
           call(r=q, d=1, rd=0, od=1), call(r=q, d=0, rd=1, od=0), call(a=-1), call(s=-1), call(i=-1), call(p=-0.1),
           call(p=1.5), call(p=float("nan")), call(a=1 << 30, s=1 << 30), call(a=1 << 47, i=1, s=0),
           call(i=(1 << 48) + 1, a=1, s=1)]
    assert bad == [1] * len(bad), bad
    assert b"not in [0, 1]" in (call(p=2.0), lib.gtk_last_error())[1]
    assert [call(a=0, x=None), call(s=0, o=None), call(i=0)] == [0] * 3


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
SHAPES = [(1,), (7,), (8,), (9,), (3, 5), (1, 1, 8), (2, 7, 5, 128), (3, 4, 6, 100), (1, 33, 17, 24), (2, 3, 2, 9),
          (5, 6, 7, 1), (4, 6, 3, 2), (2, 3, 5, 7), (1, 2, 300, 129), (129, 64), (1, 65, 2, 1030)]


@gpu
@pytest.mark.parametrize("dt,rt", [("fp32", None), ("bf16", None), ("fp32", "fp32"), ("bf16", "bf16"),
                                   ("bf16", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dt, rt):
    x = values(shape, 0, DT[dt], "cuda").requires_grad_(True)
    r = None if rt is None else values(shape, 1, DT[rt], "cuda").requires_grad_(True)
    for dim in (None, *range(len(shape))):
        print("dropout", shape, dim, dt, rt, flush=True)
        y = dropout(x, 0.3, SEED, 2 ** 33 + 1, dim, r)
        assert y.dtype == (x.dtype if r is None else torch.promote_types(x.dtype, r.dtype))
        check(y, x, 0.3, SEED, 2 ** 33 + 1, dim, r)
        dy = values(shape, 2, y.dtype, "cuda")
        dx, *dr = torch.autograd.grad(y, [x] if r is None else [x, r], dy)
        assert dx.dtype == x.dtype
        check(dx, dy, 0.3, SEED, 2 ** 33 + 1, dim)
        assert not dr or torch.equal(dr[0], dy.to(r.dtype))


@gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 512, 512, 128), (1, 301, 301, 100), (3, 200, 90, 64), (1, 1000, 7, 8),
                                   (40000, 3, 12), (2, 3, 70001), (300001, 1, 5), (1, 17, 1 << 17)], ids=str)
def test_larger_shapes_against_the_mask(shape, dt):
    """The PyTorch mask (pinned to the oracle above), all shared dimensions."""
    x = values(shape, 0, DT[dt], "cuda")
    t = round(65536 * 0.15)
    for dim in (None, *range(len(shape))):
        print("dropout", shape, dim, dt, flush=True)
        keep = dropout_mask(shape, 0.15, SEED, 1, dim, "cuda")
        ref = torch.where(keep, x.double() * (65536 / (65536 - t)), 0.0)
        for got in (dropout(x, 0.15, SEED, 1, dim), dropout(x, 0.15, torch.tensor([SEED - 2 ** 64], device="cuda"), 1, dim)):
            err = (got.double() - ref).abs()
            assert (err <= (half(x.dtype) + 4 * U) * ref.abs()).all()


@gpu
def test_strides_and_alignment():
    base = values((4, 6, 50, 40), 0, torch.bfloat16, "cuda")
    flat = values((6 * 50 * 40 + 5,), 1, torch.bfloat16, "cuda")
    for x in (base.transpose(1, 2), base[..., 3:30], base[:, ::2], base[:1].expand(4, 6, 50, 40),
              flat[3:3 + 6 * 50 * 40].view(6, 50, 40), flat[1:1 + 7 * 8 * 9].view(7, 8, 9)):
        for r in (None, values(x.shape, 2, torch.float32, "cuda").transpose(0, 1).contiguous().transpose(0, 1)):
            for dim in (None, -3, -2):
                y = dropout(x, 0.25, SEED, 0, dim, r)
                check(y, x, 0.25, SEED, 0, dim, r)
    # an output gradient that is a broadcast value
    x = values((3, 8, 16), 0, torch.float32, "cuda").requires_grad_(True)
    dropout(x, 0.5, 1, shared_dim=1).sum().backward()
    check(x.grad, torch.ones_like(x), 0.5, 1, 0, 1)


@gpu
def test_edges():
    x = values((5, 300), 0, torch.float32, "cuda")
    assert torch.equal(dropout(x, 0.0, 1), x) and not dropout(x, 1.0, 1).any()
    assert torch.equal(dropout(x, 1.0, 1, residual=x), x)
    for shape in ((0,), (0, 4), (3, 0, 4)):
        e = torch.empty(shape, device="cuda", requires_grad=True)
        y = dropout(e, 0.5, 1, shared_dim=0)
        assert y.shape == e.shape and torch.autograd.grad(y.sum(), e)[0].shape == e.shape
    # what is dropped may be anything
    keep = dropout_mask((64, 33), 0.5, 7, device="cuda")
    for v in (float("nan"), float("inf"), -float("inf")):
        for dt in DT.values():
            z = torch.where(keep, 1.0, v).to(dt)
            assert torch.equal(dropout(z, 0.5, 7), (2.0 * keep).to(dt))
            assert torch.equal(dropout(z, 0.5, 7, residual=torch.ones_like(z)), (1 + 2.0 * keep).to(dt))


@gpu
def test_more_than_2_to_the_32_values():
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.5, SEED, 3)
    for at in (0, (1 << 31) - 512, (1 << 32) - 512, n - 4096 - 3):
        at = at // 8 * 8
        size = min(4096, n - at)
        words = train_ops.philox(range(at // 8, (at + size + 7) // 8), 3, SEED)
        bits = np.array([[w >> s & 0xFFFF for w in c for s in (0, 16)] for c in words]).reshape(-1)[:size]
        assert np.array_equal(np64(y[at:at + size]), 2.0 * (bits >= 32768)), at
    del y
    # a shared mask over as many
    z = x[:(1 << 32) + 4096].view(2, (1 << 24) + 16, 128)
    y = dropout(z, 0.5, SEED, 3, -2)
    ref = 2.0 * train_ops.dropout_keep(2, 128, 0.5, SEED, 3)
    for b in range(2):
        for at in (0, (1 << 24) + 15, 1 << 23):
            assert np.array_equal(np64(y[b, at]), ref[b]), (b, at)


@gpu
def test_derivatives():
    x = values((4, 30), 0, torch.float32, "cuda").requires_grad_(True)
    r = values((4, 30), 1, torch.float32, "cuda").requires_grad_(True)
    y = dropout(x.sin(), 0.3, 3, residual=r * r)
    dy = values((4, 30), 2, torch.float32, "cuda").requires_grad_(True)
    gx, gr = torch.autograd.grad(y, (x, r), dy, create_graph=True)
    v = values((4, 30), 3, torch.float32, "cuda")
    hx, hd = torch.autograd.grad((gx * v).sum(), (x, dy), retain_graph=True)
    k = (dropout_mask(x.shape, 0.3, 3, device="cuda") * (65536 / (65536 - round(65536 * 0.3)))).float()
    torch.testing.assert_close(hx, -x.sin() * k * dy * v, rtol=16 * U, atol=1e-6)
    torch.testing.assert_close(hd, x.cos() * k * v, rtol=16 * U, atol=1e-6)
    assert torch.equal(torch.autograd.grad(gr.sum(), dy)[0], 2 * r)
    # mixed types through two derivatives
    b = values((4, 30), 4, torch.bfloat16, "cuda").requires_grad_(True)
    g, = torch.autograd.grad(dropout(b, 0.3, 3, residual=r), b, dy, create_graph=True)
    assert g.dtype == torch.bfloat16
    assert torch.autograd.grad(g.float().sum(), dy)[0].dtype == torch.float32
    # the seed tensor of a forward pass may not change before its backward
    seed = torch.tensor([3], device="cuda")
    y = dropout(x, 0.3, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_tangents_run_the_pytorch_path():
    x, t = values((4, 30), 0, torch.float32, "cuda"), values((4, 30), 1, torch.float32, "cuda")
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        out = ad.unpack_dual(dropout(ad.make_dual(x, t), 0.3, 3))
        with pytest.raises(NotImplementedError):
            _ext.C.dropout(ad.make_dual(x, t), 0.3, 3)
    check(out.primal, x, 0.3, 3)
    check(out.tangent, t, 0.3, 3)


@gpu
def test_refusals_on_the_gpu():
    x = values((4, 30), 0, torch.float32, "cuda")
    with pytest.raises(ValueError, match="seed tensor"):
        dropout(x, 0.5, torch.tensor([1]))
    with pytest.raises(RuntimeError, match="residual"):
        _ext.C.dropout(x, 0.5, 1, residual=x.cpu())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        _ext.C.dropout(x.double(), 0.5, 1)
    with pytest.raises(RuntimeError, match="types"):
        _ext.C.dropout(x, 0.5, 1, residual=x.bfloat16())
    with pytest.raises(IndexError):
        _ext.C.dropout(x, 0.5, 1, shared_dim=2)
    assert dropout(x.double(), 0.5, 1).dtype == torch.float64  # the PyTorch path


@gpu
def test_streams_and_graphs():
    x = values((2, 64, 64, 128), 0, torch.bfloat16, "cuda").requires_grad_(True)
    r = values((2, 64, 64, 128), 1, torch.bfloat16, "cuda").requires_grad_(True)
    dy = values((2, 64, 64, 128), 2, torch.bfloat16, "cuda")
    seed = torch.tensor([40], device="cuda")

    def step():
        y = dropout(x, 0.25, seed, 1, -3, r)
        return (y.detach(), *torch.autograd.grad(y, (x, r), dy))

    eager = {}
    for s in range(40, 44):
        seed.fill_(s)
        eager[s] = [t.clone() for t in step()]
    assert not torch.equal(eager[40][0], eager[41][0])
    seed.fill_(40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, eager[40]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        seed.add_(1)
    seed.fill_(40)
    for s in range(40, 44):  # each replay draws the next mask
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager[s])), s
        values((1000,), 3, torch.float32, "cuda").square().sum().item()


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_pair_stack_trains_with_a_seed(dt):
    """A training step of the stack on the kernels: the masks are dropout_mask's, so
    the same step with them applied by hand (in 64 bits, rounded once as the kernel's
    fused product is) gives the same numbers but for ties, and only a seed decides."""
    torch.manual_seed(0)
    net = PairTransformNet(64, 2, c_hidden_mul=64, tri_dropout=0.25).to("cuda", DT[dt]).train()
    with torch.no_grad():
        for prm in net.parameters():
            if not prm.any():
                prm.normal_(std=0.1)
    p = values((2, 40, 40, 64), 1, DT[dt], "cuda")
    mask = torch.ones(2, 40, 40, device="cuda")
    mask[1, 30:] = 0
    mask[1, :, 30:] = 0

    def run(seed):
        net.zero_grad()
        out = net(p, mask, seed)
        (out.float() * out.float()).mean().backward()
        return [out.detach(), *(q.grad.clone() for q in net.parameters())]

    one = run(5)
    assert all(torch.isfinite(t).all() for t in one)
    assert all(torch.equal(a, b) for a, b in zip(one, run(5)))
    assert all(torch.equal(a, b) for a, b in zip(one, run(torch.tensor([5], device="cuda"))))
    assert not torch.equal(one[0], run(6)[0])

    class ByHand(torch.nn.Module):
        def __init__(self, dim):
            super().__init__()
            self.p, self.dim = 0.25, dim

        def forward(self, x, seed, offset, residual):
            keep = dropout_mask(x.shape, self.p, seed, offset, self.dim, x.device)
            scale = float(np.float32(65536 / 49152))
            return (residual.double() + torch.where(keep, x.double() * scale, 0.0)).to(x.dtype)

    for layer in net.layers:
        layer.dropout_row, layer.dropout_col = ByHand(-3), ByHand(-2)
    for a, b in zip(one, run(5)):
        # a tie that was broken the other way, carried through the layers
        tol = (2 * half(DT[dt]) if dt == "bf16" else 64 * U) * b.float().abs().max()
        assert (a.float() - b.float()).abs().max() <= tol


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_seeds_and_offsets_of_numpy(device):
    x = values((6, 5, 24), 31, torch.float32, device)
    for seed, offset in ((np.int64(-3), np.int32(7)), (np.uint64(SEED), np.uint64(2 ** 63 + 1)), (np.uint8(200), 0)):
        y = dropout(x, 0.3, seed, offset, 1)
        assert torch.equal(y, dropout(x, 0.3, int(seed), int(offset), 1))
        check(y, x, 0.3, int(seed) % 2 ** 64, int(offset), 1)
    for seed, offset in ((1.5, 0), (1, 0.5), (None, 0)):
        with pytest.raises(TypeError):
            dropout(x, 0.3, seed, offset)


@gpu
def test_the_pytorch_path_in_a_captured_step():
    """64-bit values have no kernel; a seed that is a number is no copy from the host."""
    x = values((4, 30), 51, torch.float64, "cuda")
    ref = dropout(x, 0.25, 9, 1)
    assert torch.equal(ref.cpu(), dropout(x.cpu(), 0.25, 9, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.25, 9, 1)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
        values((1000,), 3, torch.float32, "cuda").square().sum().item()
