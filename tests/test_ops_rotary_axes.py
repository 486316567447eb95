"""Rotary positions with several axes (``ttc.ops.rotary_axes``) against complex numbers in 64 bits.

Bounds, before any run.  A turned component is a sum of two products in 32 bits: off by 3 EPS of the sum of their absolute
values, then rounded once to its type.  The gradient is the same turn back."""
import math

import pytest
import torch

from _ops_oracle import EPS, HALF, quotient, within
from ttc.ops import grid_positions, rotary, rotary_axes, rotary_table
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16]


def make(shape, dtype, device, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def axes64(x, positions, table, sections, layout, sign=1.0):
    """Pair by pair, as complex numbers."""
    x, cs = x.detach().double().cpu(), table.double().cpu()
    B, T = x.shape[:2]
    positions = positions.cpu().expand(B, T, len(sections)).long()
    y, half = x.clone(), cs.shape[1]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(half):
        at = positions[..., axis[i]]
        inside = (at >= 0) & (at < cs.shape[0])
        turn = cs[torch.where(inside, at, 0), i]
        turn = torch.complex(turn[..., 0], sign * turn[..., 1]).unsqueeze(-1)
        u, w = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., u].contiguous(), x[..., w].contiguous()) * turn
        z[~inside] = complex(math.nan, math.nan)
        y[..., u], y[..., w] = z.real, z.imag
    return y


def bound(x, want, dtype):
    """A pair's absolute values, 2 sqrt(2) |pair| at most: the table's entries are cosines and sines (times at most 2 here)."""
    size = x.detach().double().cpu().abs().amax(-1, keepdim=True) * 4
    return 3 * EPS * size + HALF[dtype] * want.abs()


CASES = [  # batch, tokens, heads, key heads, dim, sections
    (1, 1, 1, 1, 2, (1,)), (2, 5, 4, 2, 64, (8, 12, 12)), (1, 33, 3, 1, 32, (0, 8, 8)), (2, 7, 5, 5, 80, (5, 17, 3)),
    (1, 130, 16, 4, 128, (16, 24, 24)), (3, 9, 2, 2, 24, (1, 2, 3, 4)), (1, 40, 2, 2, 16, (8, 0)), (2, 6, 2, 1, 10, (0, 0, 0)),
    (1, 2050, 16, 16, 64, (4, 14, 14)), (1, 11, 2, 2, 18, (3, 3, 3))]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(device, dtype, layout, case):
    B, T, H, Hk, D, sections = case
    q, k = make((B, T, H, D), dtype, device, 1).requires_grad_(), make((B, T, Hk, D), dtype, device, 2).requires_grad_()
    dq, dk = make((B, T, H, D), dtype, device, 3), make((B, T, Hk, D), dtype, device, 4)
    table = (rotary_table(50, 2 * sum(sections)) * 1.25).to(device)
    gen = torch.Generator().manual_seed(5)
    kinds = {"int32": torch.randint(0, 50, (B, T, len(sections)), generator=gen, dtype=torch.int32),
             "shared": torch.randint(0, 50, (T, len(sections)), generator=gen),
             "axis first": torch.randint(0, 50, (len(sections), B, T), generator=gen).permute(1, 2, 0),
             "one row": torch.randint(0, 50, (1, T, len(sections)), generator=gen)}
    for positions in kinds.values():
        positions = positions.to(device)
        with torch.no_grad():
            free = rotary_axes(q, k, table, positions, sections, layout=layout)
        got = rotary_axes(q, k, table, positions, sections, layout=layout)
        for y, z, x in zip(free, got, (q, k)):
            assert torch.equal(y, z) and y.is_contiguous() and y.dtype == dtype
            want = axes64(x, positions, table, sections, layout)
            within(y, want, bound(x, want, dtype))
        grads = torch.autograd.grad(got, (q, k), (dq, dk))
        for g, d in zip(grads, (dq, dk)):
            want = axes64(d, positions, table, sections, layout, -1.0)
            within(g, want, bound(d, want, dtype))
    only, none = rotary_axes(q, None, table, positions, sections, layout=layout)
    assert none is None and torch.equal(only, got[0])
    g, = torch.autograd.grad(rotary_axes(q, k, table, positions, sections, layout=layout)[1], k, dk)
    assert torch.equal(g, grads[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_same_as_one_axis(device, layout):
    """Equal positions on all axes are one position: the same bits as :func:`rotary`."""
    q, k = make((2, 37, 4, 64), torch.bfloat16, device, 1), make((2, 37, 2, 64), torch.bfloat16, device, 2)
    table, at = rotary_table(100, 48).to(device), torch.arange(60, 97, device=device)
    a = rotary(q, k, table, at, layout=layout)
    b = rotary_axes(q, k, table, at[:, None].expand(37, 3), (8, 5, 11), layout=layout)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_outside(device, dtype, layout):
    """A position outside the table turns its axis's components into NaN, those of the other axes stay."""
    q = make((1, 4, 2, 32), dtype, device, 1)
    table, sections = rotary_table(10, 24).to(device), (4, 0, 8)
    positions = torch.tensor([[1, 99, 2], [10, 3, 3], [0, 0, -1], [2 ** 40, -5, 9]], device=device)
    y = rotary_axes(q, None, table, positions, sections, layout=layout)[0]
    want = axes64(q, positions[None], table, sections, layout)
    within(y, want, bound(q, torch.nan_to_num(want), dtype))
    assert torch.isfinite(y[0, 0]).all() and torch.isnan(y[0, 1:]).any(-1).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_views(device, dtype):
    """Parts of a projection, offsets that allow no wide loads, heads in front of tokens, gradients of other strides."""
    wide = make((2, 9, 6, 40), dtype, device, 1)
    table, sections = rotary_table(20, 16).to(device), (2, 3, 3)
    positions = torch.randint(0, 20, (2, 9, 3), generator=torch.Generator().manual_seed(2)).to(device)
    for x in (wide[..., 3:27], wide[:, :, 1:4, :24], wide[..., ::2][..., :18], wide[:1].expand(2, 9, 6, 40),
              wide.transpose(1, 2).contiguous().transpose(1, 2)):
        want = axes64(x, positions, table, sections, "half")
        x = x.detach().requires_grad_()
        y = rotary_axes(x, None, table, positions, sections)[0]
        within(y, want, bound(x, want, dtype))
        d = make(tuple(y.shape[::-1]), dtype, device, 7).permute(3, 2, 1, 0)
        g, = torch.autograd.grad(y, x, d)
        want = axes64(d, positions, table, sections, "half", -1.0)
        within(g, want, bound(d, want, dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_differences(device):
    q, k = make((1, 5, 2, 12), torch.float32, device, 1), make((1, 5, 1, 12), torch.float32, device, 2)
    table, positions = rotary_table(8, 10).to(device), torch.randint(0, 8, (5, 2), device=device)
    f = lambda q, k: rotary_axes(q, k, table, positions, (2, 3))  # noqa: E731
    cs = [make(x.shape, torch.float32, device, 5 + i) for i, x in enumerate((q, k))]
    leaves = [x.clone().requires_grad_() for x in (q, k)]
    grads = torch.autograd.grad(f(*leaves), leaves, cs)
    ds = [make(x.shape, torch.float32, device, 9 + i) for i, x in enumerate((q, k))]
    got = sum(float((g.double() * d.double()).sum()) for g, d in zip(grads, ds))
    # linear: no error but of rounding, 2^-24 of values of at most 8 at steps of 2^-1, for each of 180 components
    assert abs(got - quotient(f, (q, k), ds, cs, 0.5)) <= 180 * 64 * EPS


@pytest.mark.parametrize("device", DEVICES)
def test_learnt_and_observed(device):
    """A table with a gradient, second derivatives: through torch operators."""
    q = make((1, 5, 2, 12), torch.float32, device, 1).requires_grad_()
    table, positions = rotary_table(8, 10).to(device), torch.arange(10, device=device).view(5, 2) % 8
    learnt = table.clone().requires_grad_()
    g, = torch.autograd.grad(rotary_axes(q, None, learnt, positions, (2, 3))[0].square().sum(), learnt)
    assert g.shape == table.shape and g.abs().sum() > 0
    y = rotary_axes(q, None, table, positions, (2, 3))[0]
    first, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    second, = torch.autograd.grad(first.sum(), q)
    assert torch.allclose(second, torch.full_like(second, 2.0), atol=1e-5)  # a turn keeps squares: 2 q, then 2


def test_grid_positions():
    assert grid_positions(2, 1, 3).tolist() == [[0, 0, 0], [0, 0, 1], [0, 0, 2], [1, 0, 0], [1, 0, 1], [1, 0, 2]]
    assert grid_positions(1, 2, start=(5, 7)).tolist() == [[5, 7], [5, 8]] and grid_positions(2, start=3).tolist() == [[3], [4]]
    assert grid_positions(0, 4).shape == (0, 2)
    for bad in (lambda: grid_positions(), lambda: grid_positions(2, -1), lambda: grid_positions(2, 2, start=(1,))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_graph():
    q, table = make((1, 300, 4, 64), torch.bfloat16, "cuda", 1).requires_grad_(), rotary_table(64, 64).cuda()
    positions, d = grid_positions(3, 10, 10, device="cuda"), make((1, 300, 4, 64), torch.bfloat16, "cuda", 3)

    def work():
        leaf = q.detach().requires_grad_()
        y = rotary_axes(leaf, None, table, positions, (8, 12, 12))[0]
        return y.detach(), torch.autograd.grad(y, leaf, d)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        q.data.copy_(make((1, 300, 4, 64), torch.bfloat16, "cuda", 10 + i))
        positions.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, work()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_empty(device):
    table = rotary_table(4, 8).to(device)
    for B, T, H in ((0, 3, 2), (2, 0, 2), (1, 3, 0)):
        q = torch.zeros(B, T, H, 8, device=device)
        y, _ = rotary_axes(q, q, table, torch.zeros(T, 2, dtype=torch.int32, device=device), (1, 3))
        assert y.shape == q.shape


def test_refusals():
    q, t, p = torch.zeros(2, 3, 4, 8), rotary_table(16, 8), torch.zeros(3, 2, dtype=torch.long)
    for bad in (lambda: rotary_axes(q[0], None, t, p, (2, 2)), lambda: rotary_axes(q, q[:1], t, p, (2, 2)),
                lambda: rotary_axes(q, None, t.double(), p, (2, 2)), lambda: rotary_axes(q, None, t, p, (2, 1)),
                lambda: rotary_axes(q, None, t, p, (5, -1)), lambda: rotary_axes(q, None, t, p, ()),
                lambda: rotary_axes(q, None, t, torch.zeros(3, 5, dtype=torch.long), (1, 1, 1, 1, 0)),
                lambda: rotary_axes(q, None, t, p, (4,)), lambda: rotary_axes(q, None, t, p.float(), (2, 2)),
                lambda: rotary_axes(q, None, t, p[:2], (2, 2)), lambda: rotary_axes(q, None, t, p[:, 0], (2, 2)),
                lambda: rotary_axes(q, None, t, p[None].expand(3, 3, 2), (2, 2)),
                lambda: rotary_axes(q, None, t, p, (2, 2), layout="other"), lambda: rotary_axes(q, None, t[:0], p, (2, 2)),
                lambda: rotary_axes(q, None, rotary_table(4, 10), p, (2, 3))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: rotary_axes(q.half(), None, t, p, (2, 2)), lambda: rotary_axes(q, q.bfloat16(), t, p, (2, 2))):
        with pytest.raises(TypeError):
            bad()


def test_c_entry_refuses():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.rotary import _AXES_BLOCK
    names = (["dtype", "B", "T", "D", "inter", "backward", "axes", "s0", "s1", "s2", "s3", "H", "Hk", "q", "k"]
             + [f"x{i}" for i in range(6)] + ["yq", "yk", "table", "length", "pos", "bytes", "pb", "pt", "pa"])
    base = dict.fromkeys(names, 0) | dict(B=1, T=2, D=8, axes=2, s0=1, s1=3, H=1, Hk=1, q=64, k=64, yq=64, yk=64, table=64,
                                          length=4, pos=64, bytes=8)
    pack = lambda **kw: _AXES_BLOCK.pack(*(base | kw).values())  # noqa: E731
    for kw, code in [(dict(dtype=7), 2), (dict(B=-1), 1), (dict(T=-1), 1), (dict(D=-1), 1), (dict(axes=0), 1), (dict(axes=5), 1),
                     (dict(s0=-1), 1), (dict(s1=4), 1), (dict(s0=1 << 40), 1), (dict(axes=4, s3=1), 1), (dict(H=-1), 1),
                     (dict(q=0), 1), (dict(yk=0), 1), (dict(table=0), 1), (dict(length=0), 1), (dict(pos=0), 1),
                     (dict(bytes=2), 1), (dict(B=1 << 40, T=1 << 40), 1), (dict(H=1 << 40), 1)]:
        assert lib.ttc_rotary_axes(pack(**kw), None) == code, kw
    assert lib.ttc_rotary_axes(None, None) == 1 and lib.ttc_rotary_axes(pack(B=0), None) == 0
    assert lib.ttc_rotary_axes(pack(T=0), None) == 0
