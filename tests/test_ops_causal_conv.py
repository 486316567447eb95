"""Causal convolution (``ttc.ops.causal_conv`` and ``..._step``) against its definition in 64 bits.

Bounds, before any run.  The sum p of a token has taps + 1 terms: off by (taps + 2) EPS of the sum of their absolute values.
SiLU has a slope within [-0.1, 1.1] and a second derivative of at most 1/2; its own evaluation (an exponential of an argument
rounded to 24 digits, a division, a product) is off by (16 + 2 |p|) EPS of the value.  So e = dy act'(p) is off by |dy| times
(error of p) / 2 + 1.1 (16 + 2 |p|) EPS; the gradients are sums of e times taps or inputs, each term with two more roundings and
one for each term added.  Each result is rounded once more to its type."""
import math

import pytest
import torch

from _ops_oracle import EPS, HALF, quotient, within
from ttc.ops import causal_conv, causal_conv_step
from ttc.ops._call import with_spaces
from ttc.ops.causal_conv import causal_conv_torch
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16]


def make(shape, dtype, device, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def conv64(x, w, bias, state, act, dy=None, dfinal=None):
    """Values and gradients token by token and tap by tap, and the bounds above (without the last rounding)."""
    d = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, w, bias, state, dy, dfinal = d(x), d(w), d(bias), d(state), d(dy), d(dfinal)
    B, T, C = x.shape
    K = w.shape[1]
    wide = torch.cat([torch.zeros(B, K - 1, C, dtype=torch.float64) if state is None else state, x], 1)
    p = torch.zeros(B, T, C, dtype=torch.float64) + (0 if bias is None else bias)
    size = torch.zeros(B, T, C, dtype=torch.float64) + (0 if bias is None else bias.abs())
    for j in range(K):
        p, size = p + wide[:, j:j + T] * w[:, j], size + wide[:, j:j + T].abs() * w[:, j].abs()
    off = (K + 2) * EPS * size
    s = 1 / (1 + torch.exp(-p))
    silu = act == "silu"
    y = p * s if silu else p
    out = {"y": (y, 1.1 * off + (16 + 2 * p.abs()) * EPS * y.abs() if silu else off), "final": (wide[:, T:], 0 * wide[:, T:])}
    if dy is None:
        return out
    slope = s * (1 + p * (1 - s)) if silu else torch.ones_like(p)
    e = dy * slope
    e_off = dy.abs() * (off / 2 + 1.1 * (16 + 2 * p.abs()) * EPS) if silu else 0 * e
    dwide, dsize = torch.zeros_like(wide), torch.zeros_like(wide)
    dw, dw_size = torch.zeros_like(w), torch.zeros_like(w)
    for j in range(K):
        rows = wide[:, j:j + T]
        dwide[:, j:j + T] += e * w[:, j]
        dsize[:, j:j + T] += (e_off + (K + 4) * EPS * e.abs()) * w[:, j].abs()
        dw[:, j] = (e * rows).sum((0, 1))
        dw_size[:, j] = ((e_off + (B * T + 4) * EPS * e.abs()) * rows.abs()).sum((0, 1))
    if dfinal is not None:
        dwide[:, T:] += dfinal
        dsize[:, T:] += EPS * (dfinal.abs() + dwide[:, T:].abs())
    out.update(x=(dwide[:, K - 1:], dsize[:, K - 1:]), state=(dwide[:, :K - 1], dsize[:, :K - 1]), weight=(dw, dw_size),
               bias=(e.sum((0, 1)), (e_off + (B * T + 4) * EPS * e.abs()).sum((0, 1))))
    return out


def check(got, want):
    value, bound = want
    within(got, value, bound + HALF[got.dtype] * (value.abs() + bound) + 1e-37)


CASES = [  # batch, tokens, channels, taps
    (1, 1, 1, 1), (2, 3, 8, 4), (1, 2, 16, 8), (3, 1, 5, 2), (2, 8, 64, 4), (1, 9, 24, 3), (3, 64, 40, 4), (2, 65, 33, 5),
    (1, 130, 24, 8), (2, 200, 520, 2), (1, 7, 1111, 6), (1, 700, 136, 4), (1, 257, 8, 7), (2, 1030, 7, 1)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(device, dtype, act, state, case):
    B, T, C, K = case
    wdtype = torch.float32 if C % 3 == 0 else dtype
    x, w = make((B, T, C), dtype, device, 1).requires_grad_(), make((C, K), wdtype, device, 2, 0.5).requires_grad_()
    bias = make((C,), wdtype, device, 3).requires_grad_() if K % 2 == 0 else None
    s = make((B, K - 1, C), dtype, device, 4).requires_grad_() if state else None
    dy, dfinal = make((B, T, C), dtype, device, 5), make((B, K - 1, C), dtype, device, 6) if state else None
    want = conv64(x, w, bias, s, act, dy, dfinal)
    with torch.no_grad():
        y, final = causal_conv(x, w, bias, activation=act, initial_state=s, output_state=True)
    assert y.dtype == final.dtype == dtype and y.is_contiguous() and final.is_contiguous()
    check(y, want["y"])
    assert torch.equal(final.double().cpu(), want["final"][0])
    y2, final2 = causal_conv(x, w, bias, activation=act, initial_state=s, output_state=True)
    assert torch.equal(y, y2) and torch.equal(final, final2)
    names = {"x": x, "weight": w, "bias": bias, "state": s}
    names = {n: t for n, t in names.items() if t is not None}
    outs, ds = ((y2, final2), (dy, dfinal)) if state else ((y2,), (dy,))
    for n, g in zip(names, torch.autograd.grad(outs, list(names.values()), ds)):
        assert g.dtype == names[n].dtype
        check(g, want[n])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_differences(device, act):
    """Gradients in fp32 against central differences of the sum in 64 bits."""
    B, T, C, K = 2, 21, 12, 4
    xs = [make(s, torch.float32, device, i) for i, s in enumerate([(B, T, C), (C, K), (C,), (B, K - 1, C)])]
    cs = [make((B, T, C), torch.float32, device, 8), make((B, K - 1, C), torch.float32, device, 9)]
    f = lambda x, w, b, s: causal_conv(x, w, b, activation=act, initial_state=s, output_state=True)  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in xs]
    grads = torch.autograd.grad(f(*leaves), leaves, cs)
    for i, (t, g) in enumerate(zip(xs, grads)):
        d = torch.zeros_like(t)
        d.view(-1)[::3] = make(((t.numel() + 2) // 3,), torch.float32, device, 20 + i)
        ds = [d if j == i else torch.zeros_like(u) for j, u in enumerate(xs)]
        h = 2.0 ** -7
        want = quotient(f, xs, ds, cs, h)
        # of third derivatives (below 1 for SiLU, |d| and |w| of some units): h^2 / 6 of some thousands of terms; rounding EPS / h
        size = float(sum((c.abs() * 8).sum() for c in cs))
        assert abs(float((g * d).sum()) - want) <= size * (h * h + 64 * EPS / h), i


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_views(device, dtype):
    """Parts of a projection, odd offsets, rows shared by a batch, gradients of other strides."""
    wide = make((2, 37, 50), dtype, device, 1)
    w = make((24, 4), dtype, device, 2)
    dy = make((37, 2, 24), dtype, device, 3).transpose(0, 1)
    for x in (wide[..., :24], wide[..., 3:27], wide[..., ::2][..., :24], wide[:1, :, 16:40].expand(2, 37, 24),
              wide.transpose(0, 1)[:, :, :24].contiguous().transpose(0, 1)):
        want = conv64(x, w, None, None, "silu", dy)
        leaf, wl = x.detach(), w.clone().requires_grad_()
        leaf.requires_grad_()
        y = causal_conv(leaf, wl, activation="silu")
        check(y, want["y"])
        dx, dw = torch.autograd.grad(y, (leaf, wl), dy)
        check(dx, want["x"])
        check(dw, want["weight"])
    base = make((1, 37, 24), dtype, device, 1).requires_grad_()  # one sequence for a whole batch: its gradient is the sum
    dx, = torch.autograd.grad(causal_conv(base.expand(2, 37, 24), w), base, dy)
    parts = [conv64(base, w, None, None, "none", dy[i:i + 1])["x"] for i in range(2)]
    bound = sum(p[1] + HALF[dtype] * p[0].abs() for p in parts)
    total = sum(p[0] for p in parts)
    within(dx, total, bound + HALF[dtype] * (total.abs() + bound))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_and_steps(device, dtype):
    """A sequence in pieces of any length, then token by token, gives the same bits as the whole one."""
    B, T, C, K = 2, 40, 24, 4
    x, w, b = make((B, T, C), dtype, device, 1), make((C, K), dtype, device, 2), make((C,), dtype, device, 3)
    whole, end = causal_conv(x, w, b, activation="silu", output_state=True)
    state, got, at = None, [], 0
    for n in (1, 2, 0, 9, 17):
        y, state = causal_conv(x[:, at:at + n], w, b, activation="silu", initial_state=state, output_state=True)
        got.append(y)
        at += n
    for t in range(at, T):
        version = state._version
        got.append(causal_conv_step(x[:, t], state, w, b, activation="silu")[:, None])
        assert state._version > version
    # the CPU's torch operators sum in the same order, but evaluate exp by vectors and single values
    same = torch.equal if device == "cuda" else lambda a, c: torch.allclose(a.float(), c.float(), rtol=2 * HALF[dtype], atol=64 * EPS)
    assert same(torch.cat(got, 1), whole) and torch.equal(state, end)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels,taps", [(40, 4), (33, 3), (8, 1), (16, 8)])
def test_step_slots(device, dtype, channels, taps):
    """A pool in any order; rows outside it are skipped; the other slots stay as they are."""
    x, w = make((5, channels), dtype, device, 1), make((channels, taps), torch.float32, device, 2)
    pool = make((9, taps - 1, channels), dtype, device, 3)
    before, index = pool.clone(), torch.tensor([7, -1, 2, 9, 0], dtype=torch.int32, device=device)
    y = causal_conv_step(x, pool, w, slots=index, activation="silu")
    assert not y[1].any() and not y[3].any()
    live = torch.tensor([0, 2, 4], device=device)
    rows = index[live].long()
    want = conv64(x[live][:, None], w, None, before[rows], "silu")
    check(y[live][:, None], want["y"])
    assert torch.equal(pool[rows].double().cpu(), want["final"][0])
    rest = [i for i in range(9) if i not in (7, 2, 0)]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_not_finite(device, dtype):
    """A NaN or an infinity reaches the tokens whose window holds it, and no other token's output or gradient."""
    x, w = make((1, 50, 16), dtype, device, 1), make((16, 4), dtype, device, 2)
    dy = make((1, 50, 16), dtype, device, 3)
    x[0, 20, 3], x[0, 31, 5] = math.nan, math.inf
    w[7, 0] = math.inf
    leaf = x.clone().requires_grad_()
    y = causal_conv(leaf, w, activation="silu")
    dx, = torch.autograd.grad(y, leaf, dy)
    bad = ~torch.isfinite(y[0])
    want = torch.zeros(50, 16, dtype=torch.bool)
    want[20:24, 3] = True
    assert torch.equal(bad[:, 3].cpu(), want[:, 3]) and not bad[:, [0, 1, 2, 4, 6]].any()
    assert not bad[:31, 5].any() and not bad[35:, 5].any() and bad[31:33, 5].any()
    assert torch.isfinite(dx[0, :, [0, 1, 2, 4, 6]]).all() and torch.isfinite(dx[0, 24:, 3]).all()
    assert torch.isfinite(dx[0, :17, 3]).all()
    linear, = torch.autograd.grad(causal_conv(leaf, w), leaf, dy)  # tap 0 of the last 3 tokens' gradients meets no token
    assert torch.isfinite(linear[0, 47:, 7]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_empty(device):
    w = torch.randn(8, 4, device=device)
    for shape in ((0, 5, 8), (2, 0, 8)):
        y, s = causal_conv(torch.zeros(shape, device=device), w, output_state=True)
        assert y.shape == shape and s.shape == (shape[0], 3, 8) and not s.any()
    s0 = torch.randn(2, 3, 8, device=device)
    y, s = causal_conv(torch.zeros(2, 0, 8, device=device), w, initial_state=s0, output_state=True)
    assert torch.equal(s, s0)
    assert causal_conv(torch.zeros(2, 3, 0, device=device), torch.zeros(0, 4, device=device)).shape == (2, 3, 0)
    assert causal_conv_step(torch.zeros(0, 8, device=device), torch.zeros(0, 3, 8, device=device), w).shape == (0, 8)


@pytest.mark.parametrize("device", DEVICES)
def test_observed(device):
    """Second derivatives, per-sample gradients: through torch operators."""
    x, w = make((2, 9, 6), torch.float32, device, 1).requires_grad_(), make((6, 3), torch.float32, device, 2).requires_grad_()
    g, = torch.autograd.grad(causal_conv(x, w, activation="silu").square().sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), w)
    r, = torch.autograd.grad(causal_conv_torch(x, w, activation="silu")[0].square().sum(), x, create_graph=True)
    k, = torch.autograd.grad(r.sum(), w)
    assert torch.allclose(h, k, rtol=1e-4, atol=1e-4)
    each = torch.func.vmap(torch.func.grad(lambda x, w: causal_conv(x[None], w).square().sum(), argnums=1), (0, None))(x, w)
    for i in range(2):
        one, = torch.autograd.grad(causal_conv(x[i:i + 1], w).square().sum(), w)
        assert torch.allclose(each[i], one, rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
def test_graph_and_stream():
    """Captured: forward, backward and a step, replayed on new inputs between eager calls; eager on another stream."""
    x, w = make((2, 300, 64), torch.bfloat16, "cuda", 1), make((64, 4), torch.bfloat16, "cuda", 2).requires_grad_()
    dy, pool = make((2, 300, 64), torch.bfloat16, "cuda", 3), make((2, 3, 64), torch.bfloat16, "cuda", 4)

    def work():
        leaf = x.detach().requires_grad_()
        y = causal_conv(leaf, w, activation="silu")
        with torch.no_grad():
            z = causal_conv_step(x[:, 0], pool, w, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, (leaf, w), dy), z)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        x.copy_(make((2, 300, 64), torch.bfloat16, "cuda", 10 + i))
        start = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        after = pool.clone()
        pool.copy_(start)
        for a, b in zip(held, work()):
            assert torch.equal(a, b)
        assert torch.equal(pool, after)


@pytest.mark.gpu
def test_far_offsets():
    """Rows more than 2^32 elements from the first one."""
    far = torch.zeros(2 ** 32 + 4096, dtype=torch.bfloat16, device="cuda")
    x = far.as_strided((2, 20, 64), (2 ** 32, 64, 1))
    x.copy_(make((2, 20, 64), torch.bfloat16, "cuda", 1))
    w = make((64, 4), torch.bfloat16, "cuda", 2)
    check(causal_conv(x, w), conv64(x, w, None, None, "none")["y"])
    assert torch.equal(causal_conv_step(x[:, 3], torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda"), w),
                       causal_conv(x[:, 3:4].contiguous(), w)[:, 0])


def test_refusals():
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    s = torch.zeros(2, 3, 8)
    for bad in (lambda: causal_conv(x[0], w), lambda: causal_conv(x, w[:4]), lambda: causal_conv(x, w[:, 0]),
                lambda: causal_conv(x, torch.zeros(8, 9)), lambda: causal_conv(x, torch.zeros(8, 0)),
                lambda: causal_conv(x, w, torch.zeros(4)), lambda: causal_conv(x, w, activation="relu"),
                lambda: causal_conv(x, w, initial_state=s[:1]), lambda: causal_conv(x, w, initial_state=s.double()),
                lambda: causal_conv_step(x, s, w), lambda: causal_conv_step(x[:, 0], s[:1], w),
                lambda: causal_conv_step(x[:, 0], s.transpose(1, 2), w), lambda: causal_conv_step(x[:, 0], s.bfloat16(), w),
                lambda: causal_conv_step(x[:, 0], s, w, slots=torch.zeros(2, dtype=torch.long)),
                lambda: causal_conv_step(x[:, 0], s, w, slots=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: causal_conv(x.half(), w), lambda: causal_conv(x, w.bfloat16()),
                lambda: causal_conv(x, w, torch.zeros(8).bfloat16()), lambda: causal_conv(x.double(), w.double())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        causal_conv_step(x[:, 0], s, w.clone().requires_grad_())


def test_c_entries_refuse():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.causal_conv import _BLOCK, _STEP_BLOCK
    names = ["dtype", "wdtype", "B", "T", "C", "K", "act", "backward", "x", "xb", "xt", "w", "bias", "state", "y", "final", "dy",
             "yb", "yt", "dfinal", "dx", "dw", "db", "dstate", "ws", "size"]
    base = dict.fromkeys(names, 0) | dict(B=1, T=9, C=8, K=4, x=64, w=64, y=64)
    pack = lambda **kw: _BLOCK.pack(*(base | kw).values())  # noqa: E731
    back = dict(backward=1, dy=64, dx=64, dw=64)
    need = lib.ttc_causal_conv_workspace_bytes(pack(**back))
    assert need >= 5 * 8 * 4 and lib.ttc_causal_conv_workspace_bytes(None) == 0 == lib.ttc_causal_conv_workspace_bytes(pack())
    for kw, code in [(dict(dtype=2), 2), (dict(wdtype=1), 2), (dict(B=-1), 1), (dict(T=-1), 1), (dict(C=-1), 1), (dict(K=0), 1),
                     (dict(K=9), 1), (dict(act=2), 1), (dict(x=0), 1), (dict(w=0), 1), (dict(y=0), 1), (back, 1),
                     (back | dict(ws=64, size=need - 1), 1), (back | dict(dy=0, ws=64, size=need), 1),
                     (dict(B=1 << 40, T=1 << 40), 1), (dict(T=(1 << 63) - 1), 1), (dict(C=1 << 40), 1)]:
        assert lib.ttc_causal_conv(pack(**kw), None) == code, kw
    assert lib.ttc_causal_conv(None, None) == 1 and lib.ttc_causal_conv(pack(B=0), None) == 0
    assert lib.ttc_causal_conv(pack(C=0), None) == 0
    names = ["dtype", "wdtype", "B", "C", "K", "act", "slots", "x", "xb", "w", "bias", "state", "index", "y"]
    base = dict.fromkeys(names, 0) | dict(B=2, C=8, K=4, slots=2, x=64, w=64, state=64, y=64)
    pack = lambda **kw: _STEP_BLOCK.pack(*(base | kw).values())  # noqa: E731
    for kw, code in [(dict(dtype=2), 2), (dict(wdtype=1), 2), (dict(B=-1), 1), (dict(K=9), 1), (dict(slots=3), 1),
                     (dict(slots=-1, index=64), 1), (dict(x=0), 1), (dict(w=0), 1), (dict(state=0), 1), (dict(y=0), 1),
                     (dict(act=3), 1)]:
        assert lib.ttc_causal_conv_step(pack(**kw), None) == code, kw
    assert lib.ttc_causal_conv_step(None, None) == 1 and lib.ttc_causal_conv_step(pack(B=0, slots=0), None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,K", [(0, 5, 4), (0, 0, 1), (2, 0, 1), (2, 0, 3)])
def test_c_backward_of_nothing(dtype, B, T, K):
    """No sequences or no tokens: the weights' gradients are written, as zeros, and the state's is the final state's."""
    from ttc.ops.causal_conv import _block
    x = torch.empty(B, T, 24, dtype=dtype, device="cuda")
    w, bias = torch.ones(24, K, dtype=dtype, device="cuda"), torch.ones(24, dtype=dtype, device="cuda")
    dw, db, d_final = torch.full_like(w, 7), torch.full_like(bias, 7), make((B, K - 1, 24), dtype, "cuda", 1)
    d_state, space = torch.full_like(d_final, 7), torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    block = _block(x, w, bias, "silu", None, None, None, 1, x, d_final, x, dw, db, d_state)
    need = lib.ttc_causal_conv_workspace_bytes(block)
    assert need <= space.numel() and (B > 0 or need == 0)
    if need:
        block = with_spaces(block, space)
    assert lib.ttc_causal_conv(block, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert not dw.any() and not db.any() and torch.equal(d_state, d_final)
