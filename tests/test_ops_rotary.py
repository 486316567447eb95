"""Rotary positions (``ttc.ops.rotary``) against a pair-by-pair 64-bit form.

A turned component is u c - w s with u, w exact and c, s given in 32 bits: two products and a difference, each rounded
once (or fused), so it is off by at most 2 EPS (|u c| + |w s|), plus the rounding to the output's type."""
import math

import numpy as np
import pytest
import torch

from _ops_oracle import EPS, HALF, quotient, rotary64, within
from ttc.ops import rotary, rotary_table
from ttc.ops.rotary import rotary_torch
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def bound(x, positions, table, layout):
    size = rotary64(x.abs(), positions, torch.stack([table[..., 0].abs(), -table[..., 1].abs()], -1), layout)
    other = rotary64(x.abs(), positions, table.abs(), layout)
    most = np.maximum(np.abs(size), np.abs(other))
    return (2 * EPS + (HALF[x.dtype] if x.dtype != torch.float32 else EPS)) * most * 1.001


def make(shape, dtype, device, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,H,Hk,D,rot", [
    (1, 1, 1, 1, 2, 2), (2, 1, 8, 2, 64, 64), (1, 5, 3, 1, 64, 32), (2, 7, 5, 5, 80, 48), (1, 3, 2, 2, 66, 66),
    (1, 2, 4, 1, 48, 6), (2, 3, 2, 1, 17, 10), (1, 4, 2, 2, 32, 0), (1, 9, 33, 11, 128, 128), (3, 0, 2, 2, 8, 8),
    (0, 3, 2, 2, 8, 8)])
def test_against_pairs(device, dtype, layout, B, T, H, Hk, D, rot):
    table = rotary_table(64, rot, device=device)
    q, k = make((B, T, H, D), dtype, device, 1), make((B, T, Hk, D), dtype, device, 2)
    at = np.arange(T)[None].repeat(B, 0) + 40
    yq, yk = rotary(q, k, table, layout=layout, offset=40)
    for x, y in ((q, yq), (k, yk)):
        assert y.dtype == dtype and y.is_contiguous() and y.shape == x.shape
        within(y, rotary64(x, at, table, layout), bound(x, at, table, layout))
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 10)])
def test_positions(device, index, dtype, D):
    """Given positions: shared or by sequence, repeated, strided, outside the table."""
    table = rotary_table(100, D, device=device)
    q, k = make((3, 4, 2, D), dtype, device, 3), make((3, 4, 1, D), dtype, device, 4)
    each = torch.tensor([[0, 99, 5, 5], [-1, 100, 2 ** 31 - 1, 3], [7, 6, 5, -2 ** 31]], dtype=index, device=device)
    strided = torch.stack([each, each + 1], -1)[..., 0]
    for pos, full in ((each, each), (strided, each), (each[0], each[:1].expand(3, 4)), (each[:1], each[:1].expand(3, 4)),
                      (each[:, :1].expand(3, 4), each[:, :1].expand(3, 4))):
        for x, y in zip((q, k), rotary(q, k, table, pos)):
            at = full.cpu().numpy()
            within(y, rotary64(x, at, table, "half"), bound(x, np.clip(at, 0, 99), table, "half"))


@pytest.mark.gpu
def test_far_positions():
    """A table whose rows start beyond 2^31 bytes, and an index of 8 bytes beyond 2^32."""
    table = torch.zeros(2 ** 22 + 5, 128, 2, device="cuda")
    table[2 ** 22 + 4] = rotary_table(4, 256, device="cuda")[3]
    q = make((1, 2, 2, 256), torch.bfloat16, "cuda", 5)
    pos = torch.tensor([[2 ** 22 + 4, 2 ** 32 + 4]], device="cuda")
    y = rotary(q, None, table, pos)[0]
    want = rotary64(q, np.array([[3, -1]]), rotary_table(4, 256, device="cuda"), "half")
    within(y, want, bound(q, np.array([[3, 3]]), rotary_table(4, 256, device="cuda"), "half"))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views(device, layout, dtype):
    """Views of one projection, transposed and shifted ones, no keys; the inputs stay as they are."""
    table = rotary_table(16, 32, device=device)
    qkv = make((2, 6, 7 * 48 + 1), dtype, device, 6)
    at = np.arange(6)[None].repeat(2, 0)
    for base in (qkv[..., :7 * 48], qkv[..., 1:]):
        x = base.unflatten(-1, (7, 48))
        before = qkv.clone()
        for q, k in ((x[:, :, :4], x[:, :, 4:6]), (x[:, :, ::2], None), (x.transpose(1, 2)[:, :6].transpose(2, 1), x[:, :, 6:])):
            yq, yk = rotary(q, k, table, layout=layout)
            within(yq, rotary64(q, at, table, layout), bound(q, at, table, layout))
            assert (yk is None) == (k is None)
            if k is not None:
                within(yk, rotary64(k, at, table, layout), bound(k, at, table, layout))
        assert torch.equal(qkv, before)
    wide = make((2, 6, 48, 4), dtype, device, 7).transpose(2, 3)  # no unit stride in a head
    within(rotary(wide, None, table, layout=layout)[0], rotary64(wide, at, table, layout), bound(wide, at, table, layout))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,rot", [(64, 32), (10, 6)])
def test_gradients(device, layout, dtype, D, rot):
    """The gradient of a turn is the turn back: against the formula, and against differences in 32 bits."""
    table = rotary_table(32, rot, device=device)
    back = torch.stack([table[..., 0], -table[..., 1]], -1)
    q, k = make((2, 5, 4, D), dtype, device, 8), make((2, 5, 2, D), dtype, device, 9)
    gq, gk = make(q.shape, dtype, device, 10), make(k.shape, dtype, device, 11)
    pos = torch.tensor([[3, 1, 4, 1, 5], [9, 2, 6, 5, 31]], device=device)
    xs = [q.requires_grad_(), k.requires_grad_()]
    out = rotary(*xs, table, pos, layout=layout)
    dq, dk = torch.autograd.grad(out, xs, (gq, gk), retain_graph=True)
    at = pos.cpu().numpy()
    within(dq, rotary64(gq, at, back, layout), bound(gq, at, table, layout))
    within(dk, rotary64(gk, at, back, layout), bound(gk, at, table, layout))
    only = torch.autograd.grad(out[1], xs, gk, allow_unused=True, retain_graph=True)
    assert only[0] is None and torch.equal(only[1], dk)
    shared = torch.autograd.grad(out[0].sum(), q)[0]  # an expanded gradient
    within(shared, rotary64(torch.ones_like(gq), at, back, layout), bound(torch.ones_like(gq), at, table, layout))
    if dtype == torch.float32:
        d = make(q.shape, dtype, device, 12)
        q0 = q.detach()
        got = quotient(lambda x: rotary(x, None, table, pos, layout=layout)[0], [q0], [d], [gq], 0.5)
        want = float((dq.double() * d.double()).sum())
        # linear: the difference has no truncation error; 2 EPS and the rounding of the shifted inputs a term
        assert abs(got - want) <= 8 * EPS * float(((q0.abs() + d.abs()) * 2 * gq.abs()).double().sum()) * 2


@pytest.mark.parametrize("device", DEVICES)
def test_transforms_see_operators(device):
    table = rotary_table(8, 4, device=device)
    q = make((2, 3, 2, 6), torch.float32, device, 13).requires_grad_()
    f = lambda x: rotary(x, None, table)[0]  # noqa: E731
    g, = torch.autograd.grad(f(q).square().sum(), q, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), q)  # |turned|^2 = |x|^2: the second derivative is 2
    assert torch.allclose(gg, torch.full_like(gg, 2.0), atol=1e-5)
    v = torch.func.vmap(f, in_dims=0)(q.detach()[None])
    assert torch.allclose(v[0], f(q.detach()), atol=1e-6)
    _, jvp = torch.func.jvp(f, (q.detach(),), (torch.ones_like(q),))
    assert torch.allclose(jvp, f(torch.ones_like(q)), atol=1e-6)


def test_table():
    """Angles in 64 bits: position times base^(-2 i / dim); scaled forms at their ends and between."""
    t = rotary_table(5000, 8)
    for p in (0, 1, 4999):
        for i in range(4):
            a = p * 10000.0 ** (-2 * i / 8)
            assert abs(float(t[p, i, 0]) - math.cos(a)) <= EPS and abs(float(t[p, i, 1]) - math.sin(a)) <= EPS
    linear = rotary_table(40, 8, scaling="linear", factor=4.0)
    assert torch.allclose(linear[4::4], rotary_table(10, 8)[1:], atol=4 * EPS, rtol=0)
    based = rotary_table(2, 8, scaling="base", factor=4.0)
    angle = torch.atan2(based[1, :, 1].double(), based[1, :, 0].double())
    plain = 10000.0 ** (-torch.arange(4).double() / 4)
    assert abs(float(angle[0]) - 1) < 1e-6 and abs(float(angle[3]) / float(plain[3]) * 4 - 1) < 1e-3
    bands = rotary_table(2, 128, scaling="bands", factor=8.0, original_length=4096)
    m = 0.1 * math.log(8.0) + 1
    ratio = torch.atan2(bands[1, :, 1].double(), bands[1, :, 0].double()) / 10000.0 ** (-torch.arange(64).double() / 64)
    assert torch.allclose(bands.double().square().sum(-1), torch.full((2, 64), m * m, dtype=torch.float64), rtol=1e-6)
    assert abs(float(ratio[0]) - 1) < 1e-6 and abs(float(ratio[63]) - 1 / 8) < 1e-4
    assert (ratio.diff() <= 1e-4).all() and rotary_table(0, 8).shape == (0, 4, 2) and rotary_table(3, 0).shape == (3, 0, 2)


def test_refusals():
    q, t = torch.zeros(2, 3, 4, 8), rotary_table(16, 8)
    for bad in (lambda: rotary(q[0], None, t), lambda: rotary(q, q[:1], t), lambda: rotary(q, q[..., :6], t),
                lambda: rotary(q, None, t[..., 0]), lambda: rotary(q, None, t.double()), lambda: rotary(q, None, t[::2]),
                lambda: rotary(q, None, rotary_table(16, 10)), lambda: rotary(q, None, t, layout="other"),
                lambda: rotary(q, None, t, offset=14), lambda: rotary(q, None, t, offset=-1),
                lambda: rotary(q, None, t, torch.zeros(3)), lambda: rotary(q, None, t, torch.zeros(2, dtype=torch.long)),
                lambda: rotary(q, None, t, torch.zeros(3, dtype=torch.long), offset=1),
                lambda: rotary(q, None, t[:0], torch.zeros(3, dtype=torch.long)),
                lambda: rotary_table(4, 3), lambda: rotary_table(-1, 4), lambda: rotary_table(4, 4, scaling="x"),
                lambda: rotary_table(4, 4, scaling="linear", factor=0.5), lambda: rotary_table(4, 2, scaling="base", factor=2.0),
                lambda: rotary_table(4, 4, scaling="bands", factor=2.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: rotary(q.half(), None, t), lambda: rotary(q, q.bfloat16(), t)):
        with pytest.raises(TypeError):
            bad()


def test_c_entry_refuses():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.rotary import _BLOCK
    good = [0, 1, 1, 8, 8, 0, 0, 1, 1, 64, 64, 8, 8, 8, 8, 8, 8, 64, 64, 64, 4, 0, 0, 0, 0, 0]
    bad = [({0: 7}, 2), ({1: -1}, 1), ({2: -1}, 1), ({3: -2}, 1), ({4: 7}, 1), ({4: 10}, 1), ({7: -1}, 1), ({9: 0}, 1),
           ({10: 0}, 1), ({17: 0}, 1), ({19: 0}, 1), ({20: 0}, 1), ({20: -1}, 1), ({21: 64, 22: 2}, 1), ({7: 1 << 40}, 1),
           ({1: 1 << 40, 2: 1 << 20}, 1), ({1: 1 << 62, 2: 1 << 40}, 1), ({2: 1 << 62, 7: 1 << 20}, 1)]
    for change, code in bad:
        f = list(good)
        for i, v in change.items():
            f[i] = v
        assert lib.ttc_rotary(_BLOCK.pack(*f), None) == code, change
    assert lib.ttc_rotary(None, None) == 1
    for zero in (1, 2):
        f = list(good)
        f[zero] = 0
        assert lib.ttc_rotary(_BLOCK.pack(*f), None) == 0
