"""Group norm with an activation or a gate (``ttc.ops.group_norm``) against a 64-bit form.

Bounds, before any run: with a = max |x| rstd over the data, the normalised value is off by at most K EPS (1 + a): the
mean is a sum of at most 64 terms in one lane and 6 + 8 joins (64 bits above them), the centred square likewise, the
division and the root a rounding each; K = 96 covers 64 + 14 and the products after them.  The weight, the activation
(slope at most 1.1) and the gate multiply that; the output's type rounds once.  Gradients: every term is a product of
such values, the two means over a group sum up to 64 of them in a lane, so K EPS (1 + a)^2 times the largest term."""
import pytest
import torch

from _ops_oracle import EPS, HALF, group_norm64, quotient, within
from ttc.ops import group_norm
from ttc.ops.group_norm import group_norm_torch
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
K = 96
SHAPES = [  # x's shape, groups: rows of one to many lanes, odd sizes, one position and many
    ((1, 4), 1), ((3, 1), 1), ((5, 64), 8), ((16, 256), 2), ((7, 120), 6), ((2, 2048), 1), ((3, 4100), 2), ((9, 10), 10),
    ((4, 1, 48), 3), ((2, 5, 32), 4), ((1, 300, 24), 2), ((2, 9, 7, 15), 5), ((3, 65, 320), 32), ((1, 2, 4096), 2),
    ((300, 96), 12), ((2, 1021, 12), 6), ((1, 9000, 6), 2), ((2, 5000, 32), 2)]


def make(shape, dtype, device, seed, shift=0.0, scale=1.0):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + shift
    return x.to(dtype).to(device)


def tensors(shape, dtype, device, gate, affine, wdtype=None, shift=0.0, scale=1.0):
    C = shape[-1]
    x = make(shape, dtype, device, 1, shift, scale)
    w = make((C,), wdtype or dtype, device, 2, 1.0, 0.3) if affine else None
    b = make((C,), wdtype or dtype, device, 3, 0.0, 0.3) if affine else None
    return x, w, b, make(shape, dtype, device, 4) if gate else None


def reach(x, groups, eps):
    """max |x| rstd."""
    rows = x.detach().double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    rstd = (rows.var((1, 3), unbiased=False) + eps).rsqrt().max()
    return float(rows.abs().max() * rstd)


def big(t):
    return 1.0 if t is None else 1.0 + float(t.detach().abs().max())


def check_forward(x, groups, w, b, eps, act, gate):
    y = group_norm(x, groups, w, b, eps=eps, activation=act, gate=gate)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    want = group_norm64(x, groups, w, b, eps, act, gate)
    within(y, want, HALF[x.dtype] * 1.01 * want.abs() + K * EPS * (1 + reach(x, groups, eps)) * big(w) * big(gate) * 1.1)
    return y


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,gate,affine", [("none", False, False), ("silu", False, True), ("silu", True, True),
                                             ("none", True, False)])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward(device, dtype, act, gate, affine, shape, groups):
    x, w, b, g = tensors(shape, dtype, device, gate, affine)
    check_forward(x, groups, w, b, 1e-5, act, g)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,groups", [((5, 64), 8), ((2, 400, 24), 2), ((2, 4100), 1)])
def test_large_mean(device, shape, groups):
    """A mean 1000 times the deviation costs the digits of the mean, not those of its square."""
    x, w, b, _ = tensors(shape, torch.float32, device, False, True, shift=1000.0)
    check_forward(x, groups, w, b, 1e-5, "none", None)


@pytest.mark.parametrize("device", DEVICES)
def test_other_values(device):
    """fp32 weights with 16-bit data, constant groups, eps, misaligned and strided data, non-finite values."""
    x, w, b, g = tensors((6, 5, 48), torch.bfloat16, device, True, True, wdtype=torch.float32)
    check_forward(x, 4, w, b, 1e-3, "silu", g)
    const = torch.full((3, 32), 2.5, device=device)
    assert torch.equal(group_norm(const, 4), torch.zeros_like(const))
    flat = make((4 * 64 + 1,), torch.float32, device, 5)
    check_forward(flat[1:].reshape(4, 64), 4, None, None, 1e-5, "none", None)
    check_forward(make((64, 5), torch.float32, device, 6).t(), 4, None, None, 1e-5, "silu", None)
    bad = make((4, 32), torch.float32, device, 7)
    bad[1, 3], bad[2, 20] = float("nan"), float("inf")
    y = group_norm(bad, 2)
    lost = torch.isnan(y)
    assert lost[1, :16].all() and lost[2, 16:].all() and int(lost.sum()) == 32
    bad3 = make((2, 50, 32), torch.float32, device, 8)
    bad3[1, 49, 3] = float("inf")
    lost = torch.isnan(group_norm(bad3, 2, activation="silu"))
    assert lost[1, :, :16].all() and int(lost.sum()) == 50 * 16
    far = torch.full((1, 4), 100.0, device=device) * torch.tensor([1.0, -1.0, 1.0, -1.0], device=device)
    z = group_norm(far, 1, activation="silu", gate=torch.tensor([[200.0, -200.0, 1e30, -1e30]], device=device))
    assert torch.isfinite(z).all() and float(z[0, 1]) == 0.0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,groups", [((0, 8), 2), ((3, 0), 1), ((2, 0, 8), 4)])
def test_empty(device, shape, groups):
    x, w, b, g = tensors(shape, torch.bfloat16, device, True, True)
    xs = [t.requires_grad_() for t in (x, w, b, g)]
    y = group_norm(x, groups, w, b, gate=g)
    assert y.shape == shape and y.dtype == x.dtype
    for t, d in zip(xs, torch.autograd.grad(y, xs, torch.zeros_like(y))):
        assert d.shape == t.shape and not d.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,gate,affine", [("none", False, False), ("silu", False, True), ("silu", True, True),
                                             ("none", True, True)])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_gradients(device, dtype, act, gate, affine, shape, groups):
    x, w, b, g = tensors(shape, dtype, device, gate, affine)
    dy = make(shape, dtype, device, 9)
    xs = [None if t is None else t.requires_grad_() for t in (x, w, b, g)]
    have = [t for t in xs if t is not None]
    got = torch.autograd.grad(group_norm(x, groups, w, b, eps=1e-3, activation=act, gate=g), have, dy)
    wide = [None if t is None else t.detach().double().requires_grad_() for t in xs]
    want = torch.autograd.grad(group_norm64(wide[0], groups, wide[1], wide[2], 1e-3, act, wide[3]),
                               [t for t in wide if t is not None], dy.double())
    a = reach(x, groups, 1e-3)
    term = float(dy.abs().max()) * big(w) * big(g) * big(b) * 1.1 * (1 + a) ** 2 * K * EPS
    rows = x.numel() // shape[-1]
    rstd = a / max(float(x.detach().abs().max()), 1e-30)
    bounds = {0: term * max(rstd, 1.0), 1: term * rows, 2: term * rows, 3: term}
    for i, (d, e) in zip([i for i, t in enumerate(xs) if t is not None], zip(got, want)):
        assert d.dtype == xs[i].dtype
        within(d, e, HALF[dtype] * 1.01 * e.abs() + bounds[i])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape,groups", [((6, 40), 5), ((2, 70, 12), 3)])
def test_gradients_against_differences(device, shape, groups):
    """sum(y c) along a direction in 32 bits; the difference's own truncation is computed in 64."""
    x, w, b, g = tensors(shape, torch.float32, device, True, True)
    c = make(shape, torch.float32, device, 10)
    xs, h = [x, w, b, g], 2.0 ** -8
    ds = [make(t.shape, torch.float32, device, 11 + i) for i, t in enumerate(xs)]
    leaves = [t.clone().requires_grad_() for t in xs]
    f = lambda x, w, b, g: group_norm(x, groups, w, b, eps=1e-2, activation="silu", gate=g)  # noqa: E731
    grads = torch.autograd.grad(f(*leaves), leaves, c)
    slope = sum(float((d.double() * e.double()).sum()) for d, e in zip(ds, grads))
    f64 = lambda x, w, b, g: group_norm64(x, groups, w, b, 1e-2, "silu", g)  # noqa: E731
    wide = [t.double().requires_grad_() for t in xs]
    exact = sum(float((d.double() * e).sum()) for d, e in zip(ds, torch.autograd.grad(f64(*wide), wide, c.double())))
    truncation = abs(quotient(f64, [t.double() for t in xs], [d.double() for d in ds], [c], h) - exact)
    noise = K * EPS * (1 + reach(x, groups, 1e-2)) * big(w) * big(g) * 1.2 * float(c.abs().sum()) / h
    assert abs(quotient(f, xs, ds, [c], h) - slope) <= truncation + noise


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((37, 5, 24), 3), ((3, 11, 36), 4), ((1, 5000, 64), 2), ((1, 9000, 15), 3)])
def test_few_and_many_values_a_group(device, dtype, shape, groups):
    """Groups of a few lanes, the last workgroup not full; groups of many slabs, of whole vectors and not."""
    for gate in (False, True):
        x, w, b, g = tensors(shape, dtype, device, gate, True)
        check_forward(x, groups, w, b, 1e-5, "silu", g)
    if dtype == torch.float32:
        x, w, b, _ = tensors(shape, dtype, device, False, True, shift=1000.0)
        check_forward(x, groups, w, b, 1e-5, "none", None)


@pytest.mark.parametrize("device", DEVICES)
def test_needed_gradients_only(device):
    x, w, b, g = tensors((5, 3, 24), torch.float32, device, True, True)
    full = [t.clone().requires_grad_() for t in (x, w, b, g)]
    want = torch.autograd.grad(group_norm(full[0], 3, full[1], full[2], gate=full[3]).sum(), full)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b, g))]
        d, = torch.autograd.grad(group_norm(some[0], 3, some[1], some[2], gate=some[3]).sum(), [some[i]])
        assert torch.allclose(d, want[i], rtol=1e-5, atol=1e-5)
    z = x.clone().requires_grad_()
    d, = torch.autograd.grad(group_norm(z, 3, activation="silu").square().sum(), z, create_graph=True)
    assert torch.autograd.grad(d.square().sum(), z)[0].isfinite().all()
    v = torch.func.vmap(lambda t: group_norm(t, 3))(x[None])
    assert torch.allclose(v[0], group_norm(x, 3), atol=1e-5)


def test_refusals():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for bad in (lambda: group_norm(w, 2), lambda: group_norm(x, 3), lambda: group_norm(x, 0),
                lambda: group_norm(x, 2, w), lambda: group_norm(x, 2, w[:4], w[:4]), lambda: group_norm(x, 2, eps=-1.0),
                lambda: group_norm(x, 2, activation="other"), lambda: group_norm(x, 2, gate=x[:1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: group_norm(x.half(), 2), lambda: group_norm(x, 2, gate=x.bfloat16()),
                lambda: group_norm(x, 2, w.bfloat16(), w.bfloat16()), lambda: group_norm(x, 2, w, w.bfloat16())):
        with pytest.raises(TypeError):
            bad()


def test_c_entry_refuses():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.group_norm import _BLOCK
    names = ["dtype", "wdtype", "n", "l", "c", "groups", "act", "backward", "eps", "x", "gate", "weight", "bias", "mean",
             "rstd", "y", "dy", "dx", "dgate", "dweight", "dbias", "ws", "size"]
    base = dict.fromkeys(names, 0) | dict(n=2, l=9000, c=8, groups=2, eps=1e-5, x=64, y=64, ws=64, size=1 << 20)
    pack = lambda **kw: _BLOCK.pack(*(base | kw).values())  # noqa: E731
    need = lib.ttc_group_norm_workspace_bytes(pack())
    assert need > 0 and lib.ttc_group_norm_workspace_bytes(pack(n=0)) == 0
    for c in range(1, 9):  # fewer channels than a vector
        for dtype in (0, 1):
            assert lib.ttc_group_norm_workspace_bytes(pack(c=c, groups=1, l=90000, dtype=dtype)) > 0
            assert lib.ttc_group_norm_workspace_bytes(pack(c=c, groups=c, l=2, dtype=dtype, backward=1)) > 0
    assert lib.ttc_group_norm_workspace_bytes(None) == 0 and lib.ttc_group_norm_workspace_bytes(pack(groups=3)) == 0
    for kw, code in [(dict(dtype=3), 2), (dict(wdtype=-1), 2), (dict(groups=3), 1), (dict(groups=0), 1), (dict(n=-1), 1),
                     (dict(l=-1), 1), (dict(c=-8), 1), (dict(act=2), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
                     (dict(x=0), 1), (dict(y=0), 1), (dict(weight=64), 1), (dict(mean=64), 1), (dict(ws=0), 1),
                     (dict(size=need - 1), 1), (dict(backward=1), 1), (dict(backward=1, dy=64), 1), (dict(c=1 << 40), 1),
                     (dict(backward=1, dy=64, mean=64, rstd=64, dgate=64), 1),
                     (dict(n=1 << 40, l=1, c=1 << 20, groups=1 << 20, size=(1 << 62)), 1)]:
        assert lib.ttc_group_norm(pack(**kw), None) == code, kw
    assert lib.ttc_group_norm(None, None) == 1
    for kw in (dict(n=0), dict(l=0), dict(c=0, groups=1)):
        assert lib.ttc_group_norm(pack(**kw), None) == 0


def term_bounds(x, groups, w, b, eps, act, gate, dy):
    """Bounds of dx, dweight, dbias and dgate from their terms' absolute values in 64 bits.  In units of EPS: a normalised
    value is off by K (|xhat| + |x| rstd), what depends on it by that times the weight and slopes below 1.1 (K (1 + |y0|) in
    all), a product by each factor's error times the other; a sum adds at most N of its terms one after the other in 32 bits
    (4 positions and 256 rows of a workgroup, 64 values of a lane and 6 joins), the rest in 64."""
    N = 300
    n, c = x.shape[0], x.shape[-1]
    d = lambda t: t.detach().double()  # noqa: E731
    grouped = lambda t: t.reshape(n, -1, groups, c // groups)  # noqa: E731
    mean_of = lambda t: grouped(t).mean((1, 3), keepdim=True)  # noqa: E731
    back = lambda t: (t + torch.zeros_like(grouped(d(x)))).reshape(x.shape)  # noqa: E731
    rstd = back((mean_of((d(x) - back(mean_of(d(x)))) ** 2) + eps).rsqrt())
    xh = (d(x) - back(mean_of(d(x)))) * rstd
    raw = xh.abs() + d(x).abs() * rstd
    weight, bias = (1.0, 0.0) if w is None else (d(w).abs(), d(b).abs())
    y0 = 1 + weight * raw + bias
    on = 1.1 if gate is None else 1.1 + d(gate).abs()
    d0 = d(dy).abs() * on
    e0 = d0 * y0                        # what d0 is off by, in units of K EPS
    dh, eh = d0 * weight, e0 * weight
    s1 = back(mean_of((N + K) * dh + K * eh))
    s2 = back(mean_of((N + K) * dh * xh.abs() + K * (dh * raw + eh * xh.abs())))
    rows = lambda t: t.reshape(-1, c).sum(0)  # noqa: E731
    return {"x": EPS * rstd * (K * (dh + eh) + s1 + xh.abs() * s2 + K * raw * back(mean_of(dh * xh.abs()))),
            "w": EPS * rows((N + K) * d0 * xh.abs() + K * (d0 * raw + e0 * xh.abs())), "b": EPS * rows((N + K) * d0 + K * e0),
            "gate": EPS * K * 1.1 * d(dy).abs() * y0}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,gate", [("none", False), ("silu", False), ("silu", True)])
@pytest.mark.parametrize("shape,groups", [((300, 96), 12), ((2, 5000, 32), 2), ((1, 9000, 6), 2), ((50000, 24), 3),
                                          ((20000, 7), 1), ((3, 4100), 1), ((700, 3, 40), 5), ((9, 2048), 2)])
def test_gradients_term_by_term(device, dtype, act, gate, shape, groups):
    """Sums over many rows, several rows a thread and slabs, with bounds that a wrong or missing part of a sum passes."""
    x, w, b, g = tensors(shape, dtype, device, gate, True)
    dy = make(shape, dtype, device, 9)
    xs = {n: t.requires_grad_() for n, t in (("x", x), ("w", w), ("b", b), ("gate", g)) if t is not None}
    got = dict(zip(xs, torch.autograd.grad(group_norm(x, groups, w, b, eps=1e-3, activation=act, gate=g), list(xs.values()), dy)))
    wide = {n: t.detach().double().requires_grad_() for n, t in xs.items()}
    y = group_norm64(wide["x"], groups, wide["w"], wide["b"], 1e-3, act, wide.get("gate"))
    want = dict(zip(wide, torch.autograd.grad(y, list(wide.values()), dy.double())))
    bound = term_bounds(x, groups, w, b, 1e-3, act, g, dy)
    for name in xs:
        assert float(bound[name].max()) < 0.05 * float(want[name].abs().max()), name
        within(got[name], want[name], bound[name] + HALF[dtype] * 1.01 * want[name].abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,l", [(0, 1), (0, 9), (3, 0)])
def test_c_backward_of_nothing(dtype, n, l):
    """No rows or no positions: the weights' gradients are written, as zeros."""
    from ttc.ops._call import DTYPES
    from ttc.ops.group_norm import _BLOCK
    w = torch.ones(24, dtype=dtype, device="cuda")
    dw, db = torch.full_like(w, 7), torch.full_like(w, 7)
    block = _BLOCK.pack(DTYPES[dtype], DTYPES[dtype], n, l, 24, 4, 0, 1, 1e-5, 0, 0, w.data_ptr(), w.data_ptr(), 0, 0, 0, 0, 0, 0,
                        dw.data_ptr(), db.data_ptr(), 0, 0)
    assert lib.ttc_group_norm_workspace_bytes(block) == 0
    assert lib.ttc_group_norm(block, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()


def test_c_backward_of_nothing_that_is_wanted():
    """No gradients asked for: nothing is launched (no GPU is touched)."""
    from ttc.ops.group_norm import _BLOCK
    assert lib.ttc_group_norm(_BLOCK.pack(0, 0, 0, 1, 24, 4, 0, 1, 1e-5, *(0,) * 14), None) == 0
