"""Linear attention with a decay for each head (``ttc.ops.linear_attention`` and ``..._step``) against the recurrence in 64
bits.

Bounds, before any run.  Every output is a sum of products of q, k, v, d_o, states and decays; with the same sums taken over
absolute values (``linear64`` of the absolute inputs) it is off by at most n EPS times that, n the roundings on a term's way:
the head's size in each of two products, the tokens it passes (a rounding of the state and two of the decay each), 64 for
the rest.  In bfloat16 the products' weights, the state in front of a chunk and the output are rounded to 8 digits: 3 HALF
on the same sum (states and the decays' gradient, returned in fp32, are not rounded on the way).  The decays' gradient
is a sum over later tokens of q.dq - k.dk: the sum of those absolute values, n EPS."""
import math

import pytest
import torch

from _ops_oracle import EPS, HALF, linear64, quotient, within
from ttc.ops import linear_attention, linear_attention_step
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(shape, dtype, device, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def gates(B, T, H, device, kind="mixed", dtype=torch.float32):
    g = -torch.rand(B, T, H, generator=torch.Generator().manual_seed(77)) * torch.logspace(-3, 0.3, H)
    if kind == "none":
        g = torch.zeros(B, T, H)
    elif kind == "strong":  # decays of up to e^-100 beside ones of almost 1
        g = g * torch.where(torch.rand(B, T, H, generator=torch.Generator().manual_seed(78)) < 0.3, 60.0, 0.01)
    elif kind == "reset":
        g[torch.rand(B, T, H, generator=torch.Generator().manual_seed(79)) < 0.05] = -math.inf
        g[torch.rand(B, T, H, generator=torch.Generator().manual_seed(80)) < 0.05] = -1e30
        g[torch.rand(B, T, H, generator=torch.Generator().manual_seed(81)) < 0.03] = torch.finfo(torch.float32).min
        g[:, :1, :1] = -math.inf
    elif kind == "growing":
        g = -g * 0.02
    return g.to(dtype).to(device)


def inputs(B, T, H, Hq, Hk, Hv, dk, dv, dtype, device, state, kind="mixed", gdtype=torch.float32):
    return dict(q=make((B, T, Hq, dk), dtype, device, 1), k=make((B, T, Hk, dk), dtype, device, 2, dk ** -0.5),
                v=make((B, T, Hv, dv), dtype, device, 3), g=gates(B, T, H, device, kind, gdtype),
                state=make((B, H, dk, dv), torch.float32, device, 4) if state else None)


def magnitudes(x, scale, d_o=None, d_state=None):
    a = lambda t: None if t is None else t.detach().abs()  # noqa: E731
    return linear64(a(x["q"]), a(x["k"]), a(x["v"]), x["g"], abs(scale), a(x["state"]), a(d_o), a(d_state))


def roundings(x, T):
    return 2 * max(x["q"].shape[-1], x["v"].shape[-1]) + 3 * T + 64


def check_out(x, o, final, scale):
    want, size = linear64(x["q"], x["k"], x["v"], x["g"], scale, x["state"]), magnitudes(x, scale)
    n, dt = roundings(x, o.shape[1]), o.dtype
    within(o, want["o"], size["o"] * (n * EPS + (3 * HALF[dt] if dt != torch.float32 else 0)) + 1e-30)
    if final is not None:
        within(final, want["state"], size["state"] * n * EPS + 1e-30)


CASES = [  # batch, tokens, heads of the output, of q, k, v, dk, dv
    (1, 1, 1, 1, 1, 1, 1, 1), (2, 1, 4, 4, 4, 4, 64, 64), (1, 2, 2, 2, 2, 2, 16, 16), (1, 63, 2, 2, 1, 1, 32, 16),
    (2, 64, 3, 3, 3, 3, 64, 128), (1, 65, 4, 2, 2, 4, 128, 64), (1, 17, 2, 2, 2, 2, 5, 3), (2, 130, 6, 6, 2, 3, 48, 80),
    (1, 129, 2, 1, 1, 2, 128, 128), (1, 300, 2, 2, 2, 2, 33, 127), (3, 0, 2, 2, 2, 2, 8, 8), (0, 5, 2, 2, 2, 2, 8, 8),
    (1, 40, 1, 1, 1, 1, 127, 20), (1, 1100, 2, 2, 2, 2, 16, 24)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_forward(device, dtype, state, case):
    x = inputs(*case, dtype, device, state)
    scale = case[6] ** -0.5
    o, final = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["state"], output_state=True)
    assert o.dtype == dtype and o.is_contiguous() and final.dtype == torch.float32
    check_out(x, o, final, scale)
    assert torch.equal(linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["state"]), o)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["none", "strong", "reset", "growing"])
@pytest.mark.parametrize("T", [5, 64, 200])
def test_decays(device, dtype, kind, T):
    x = inputs(2, T, 3, 3, 3, 3, 32, 48, dtype, device, True, kind)
    o, final = linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.3, initial_state=x["state"], output_state=True)
    check_out(x, o, final, 0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(device, dtype):
    """Views of one projection, decays per head and in 16 bits, expanded and transposed inputs."""
    qkv = make((2, 90, 4 * 32 + 2 * 32 + 4 * 40 + 1), dtype, device, 5)
    for base in (qkv[..., :-1], qkv[..., 1:]):
        q, k, v = torch.split(base, [128, 64, 160], dim=-1)
        x = dict(q=q.unflatten(-1, (4, 32)), k=k.unflatten(-1, (2, 32)) * 0.2, v=v.unflatten(-1, (4, 40)),
                 g=gates(2, 90, 4, device), state=None)
        check_out(x, *linear_attention(x["q"], x["k"], x["v"], x["g"], scale=1.0, output_state=True), 1.0)
    head = torch.tensor([-0.01, -0.3, -2.0, -40.0], device=device)
    for g in (head, head.to(dtype)):
        x["g"] = g.float().expand(2, 90, 4)
        check_out(x, *linear_attention(x["q"], x["k"], x["v"], g, scale=1.0, output_state=True), 1.0)
    g16 = gates(2, 90, 4, device, dtype=dtype)
    x["g"] = g16.float()
    check_out(x, *linear_attention(x["q"], x["k"], x["v"], g16, scale=1.0, output_state=True), 1.0)
    y = dict(q=make((2, 4, 90, 32), dtype, device, 6).transpose(1, 2), k=make((2, 90, 1, 32), dtype, device, 7, 0.2),
             v=make((1, 90, 2, 24), dtype, device, 8).expand(2, 90, 2, 24), state=None,
             g=gates(2, 4, 90, device).transpose(1, 2))
    check_out(y, *linear_attention(y["q"], y["k"], y["v"], y["g"], scale=1.0, output_state=True), 1.0)
    w = dict(y, q=make((2, 90, 32, 4), dtype, device, 6).transpose(2, 3))  # no unit stride in a head
    check_out(w, *linear_attention(w["q"], w["k"], w["v"], w["g"], scale=1.0, output_state=True), 1.0)


def put(x, name, at, value):
    t = x[name].clone()
    t[at] = value
    return dict(x, **{name: t})


@pytest.mark.parametrize("device", DEVICES[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [12, 64, 150])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_masked_places(device, dtype, T, value):
    """What is not finite has no effect on earlier tokens, on other heads, or past a reset."""
    x = inputs(1, T, 2, 2, 2, 2, 32, 48, dtype, device, False)
    run = lambda y, **kw: linear_attention(y["q"], y["k"], y["v"], y["g"], output_state=True, **kw)  # noqa: E731
    o, final = run(x)
    bad = T // 2
    for name in ("q", "k", "v"):
        z, zf = run(put(x, name, (0, bad, 0, 3), value))
        assert torch.equal(z[:, :, 1], o[:, :, 1]) and torch.equal(zf[:, 1], final[:, 1])
        within(z[:, :bad, 0], o[:, :bad, 0].float(), 2 * HALF[dtype] * o[:, :bad, 0].abs().float() + 0.02)
        assert not torch.isfinite(z[:, bad, 0]).all()
        if name == "q":
            within(z[:, bad + 1:, 0], o[:, bad + 1:, 0].float(), 2 * HALF[dtype] * o[:, bad + 1:, 0].abs().float() + 0.02)
        cut = dict(x, g=x["g"].clone())
        cut["g"][0, bad + 1, 0] = -math.inf
        oc, fc = run(cut)
        z, zf = run(put(cut, name, (0, bad, 0, 3), value))
        within(z[:, bad + 1:], oc[:, bad + 1:].float(), 2 * HALF[dtype] * oc[:, bad + 1:].abs().float() + 0.02)
        within(zf, fc, 64 * EPS * fc.abs() + 1e-4)
    cut = dict(x, g=x["g"].clone())
    cut["g"][0, 0, 0] = -math.inf
    dirty = torch.full((1, 2, 32, 48), value, device=device)
    dirty[:, 1] = 0
    z, zf = run(cut, initial_state=dirty)
    assert torch.isfinite(z).all() and torch.isfinite(zf).all()


def grads(x, d_o, d_state, scale, per_head=None):
    leaf = {n: t.detach().clone().requires_grad_() for n, t in x.items() if t is not None}
    g = leaf["g"] if per_head is None else per_head.detach().clone().requires_grad_()
    out = linear_attention(leaf["q"], leaf["k"], leaf["v"], g, scale=scale, initial_state=leaf.get("state"),
                           output_state=True)
    wrt = [leaf["q"], leaf["k"], leaf["v"], g] + ([leaf["state"]] if "state" in leaf else [])
    got = torch.autograd.grad(out if d_state is not None else out[:1], wrt, (d_o, d_state) if d_state is not None else (d_o,))
    return dict(zip(("q", "k", "v", "g", "d_state"), got))


def gate_size(x, size):
    H = x["g"].shape[-1]
    wide = lambda t: t.detach().abs().double().cpu()  # noqa: E731
    # of shared heads: the sums over each group bound its heads' terms
    r = (wide(x["q"]) * size["q"]).sum(-1).repeat_interleave(H // x["q"].shape[2], 2)
    c = (wide(x["k"]) * size["k"]).sum(-1).repeat_interleave(H // x["k"].shape[2], 2)
    return (r + c).flip(1).cumsum(1).flip(1)


def check_grads(x, got, d_o, d_state, scale):
    want = linear64(x["q"], x["k"], x["v"], x["g"], scale, x["state"], d_o, d_state)
    size = magnitudes(x, scale, d_o, d_state)
    n, dt = roundings(x, d_o.shape[1]), d_o.dtype
    for name in ("q", "k", "v"):
        assert got[name].dtype == dt and got[name].shape == x[name].shape
        within(got[name], want[name], size[name] * (n * EPS + (3 * HALF[dt] if dt != torch.float32 else 0)) + 1e-30)
    end = 0 if d_state is None else (size["state"] * d_state.detach().abs().double().cpu()).sum((-1, -2))[:, None]
    within(got["g"], want["g"], (gate_size(x, size) + end) * n * EPS + HALF[got["g"].dtype] * want["g"].abs() + 1e-30)
    if x["state"] is not None:
        within(got["d_state"], want["d_state"], size["d_state"] * n * EPS + 1e-30)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("case", [c for c in CASES if c[1] < 400])
def test_gradients(device, dtype, state, case):
    x = inputs(*case, dtype, device, state)
    B, T, H, dv = case[0], case[1], case[2], case[7]
    d_o = make((B, T, H, dv), dtype, device, 9)
    d_state = make((B, H, case[6], dv), torch.float32, device, 10) if state else None
    check_grads(x, grads(x, d_o, d_state, 0.4), d_o, d_state, 0.4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["none", "strong", "reset"])
@pytest.mark.parametrize("T", [9, 64, 140])
def test_gradients_of_decays(device, dtype, kind, T):
    x = inputs(2, T, 3, 3, 1, 3, 32, 24, dtype, device, True, kind)
    d_o, d_state = make((2, T, 3, 24), dtype, device, 9), make((2, 3, 32, 24), torch.float32, device, 10)
    got = grads(x, d_o, d_state, 0.4)
    check_grads(x, got, d_o, d_state, 0.4)
    assert not got["g"][x["g"] < -104].any()
    if kind != "reset":
        head = x["g"][0, 0].clone()
        y = dict(x, g=head.expand(2, T, 3))
        each = grads(y, d_o, d_state, 0.4)["g"]
        one = grads(dict(x, g=head), d_o, d_state, 0.4)["g"]
        assert one.shape == (3,)
        within(one, each.double().sum((0, 1)), 2 * T * 2 * EPS * each.abs().sum((0, 1)) + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind,case", [
    (torch.float32, "mixed", (1, 1100, 2, 2, 1, 2, 24, 40)), (torch.bfloat16, "mixed", (1, 2100, 2, 2, 2, 2, 40, 24)),
    (torch.bfloat16, "reset", (1, 1025, 1, 1, 1, 1, 64, 64)), (torch.float32, "none", (2, 513, 1, 1, 1, 1, 16, 16))])
def test_gradients_of_long_inputs(dtype, kind, case):
    """Several stretches of the decays' gradient."""
    x = inputs(*case, dtype, "cuda", True, kind)
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    d_o, d_state = make((B, T, H, dv), dtype, "cuda", 9), make((B, H, dk, dv), torch.float32, "cuda", 10)
    got = grads(x, d_o, d_state, 0.2)
    check_grads(x, got, d_o, d_state, 0.2)
    want = linear64(x["q"], x["k"], x["v"], x["g"], 0.2, x["state"], d_o, d_state)["g"]
    assert float((got["g"].double().cpu() - want).norm() / want.norm()) < 1e-5  # the bounds above grow with the length


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [7, 100])
def test_gradients_against_differences(device, T):
    """sum(o c) + sum(state d) along a direction in 32 bits; the difference's own truncation is computed in 64."""
    x = inputs(1, T, 2, 2, 1, 2, 24, 40, torch.float32, device, True)
    c = [make((1, T, 2, 40), torch.float32, device, 20), make((1, 2, 24, 40), torch.float32, device, 21)]
    got = grads(x, c[0], c[1], 0.4)
    names, h = ("q", "k", "v", "g", "state"), 2.0 ** -7
    ds = [make(x[n].shape, torch.float32, device, 22 + i, 0.05 if n == "g" else 1.0) for i, n in enumerate(names)]
    slope = sum(float((d.double() * got["d_state" if n == "state" else n].double()).sum()) for n, d in zip(names, ds))

    def f(q, k, v, g, s):
        return linear_attention(q, k, v, g, scale=0.4, initial_state=s, output_state=True)

    def f64(q, k, v, g, s):
        r = linear64(q, k, v, g, 0.4, s)
        return r["o"], r["state"]
    xs = [x[n] for n in names]
    want = linear64(*xs[:4], 0.4, xs[4], c[0], c[1])
    exact = sum(float((d.double().cpu() * want["d_state" if n == "state" else n]).sum()) for n, d in zip(names, ds))
    truncation = abs(quotient(f64, [t.double() for t in xs], [d.double() for d in ds], c, h) - exact)
    size = magnitudes(x, 0.4)
    noise = roundings(x, T) * EPS * 1.2 * float((size["o"] * c[0].abs().double().cpu()).sum() +
                                                (size["state"] * c[1].abs().double().cpu()).sum()) / h
    assert abs(quotient(f, xs, ds, c, h) - slope) <= truncation + noise


@pytest.mark.parametrize("device", DEVICES)
def test_needed_gradients_only(device):
    x = inputs(1, 70, 2, 2, 1, 2, 16, 20, torch.float32, device, True)
    d_o, d_state = make((1, 70, 2, 20), torch.float32, device, 9), make((1, 2, 16, 20), torch.float32, device, 10)
    want = grads(x, d_o, d_state, 0.4)
    for name, key in (("q", "q"), ("k", "k"), ("v", "v"), ("g", "g"), ("state", "d_state")):
        leaf = {n: t.detach().clone().requires_grad_(n == name) for n, t in x.items()}
        out = linear_attention(leaf["q"], leaf["k"], leaf["v"], leaf["g"], scale=0.4, initial_state=leaf["state"],
                               output_state=True)
        pairs = [(o, d) for o, d in zip(out, (d_o, d_state)) if o.requires_grad]
        d, = torch.autograd.grad([o for o, _ in pairs], [leaf[name]], [d for _, d in pairs])
        assert torch.allclose(d, want[key], rtol=1e-4, atol=1e-4)
    leaf = {n: t.detach().clone().requires_grad_() for n, t in x.items()}
    out = linear_attention(leaf["q"], leaf["k"], leaf["v"], leaf["g"], initial_state=leaf["state"], output_state=True)
    d, = torch.autograd.grad(out[1].sum(), leaf["k"])  # the state's gradient alone
    assert d.isfinite().all() and d.abs().max() > 0


@pytest.mark.parametrize("device", DEVICES)
def test_transforms_see_operators(device):
    x = inputs(1, 20, 2, 2, 1, 2, 16, 20, torch.float32, device, False)
    f = lambda v: linear_attention(x["q"], x["k"], v, x["g"])  # noqa: E731
    v = x["v"].clone().requires_grad_()
    d, = torch.autograd.grad(f(v).square().sum(), v, create_graph=True)
    dd, = torch.autograd.grad(d.sum(), v)
    twice = 2 * torch.autograd.grad(f(v), v, f(torch.ones_like(v)).detach())[0]  # of |A v|^2: 2 A' A 1
    assert torch.allclose(dd, twice, rtol=1e-3, atol=1e-3)
    assert torch.allclose(torch.func.vmap(f)(x["v"][None])[0], f(x["v"]), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 1, 1, 1), (5, 8, 8, 8, 8, 64, 64), (3, 6, 2, 3, 6, 48, 80),
                                  (2, 4, 4, 1, 1, 128, 128), (7, 2, 2, 2, 2, 33, 127), (2, 3, 3, 3, 3, 5, 6),
                                  (0, 2, 2, 2, 2, 8, 8)])
def test_step(device, dtype, case):
    B, H, Hq, Hk, Hv, dk, dv = case
    x = inputs(B, 3, H, Hq, Hk, Hv, dk, dv, dtype, device, True)
    S = x["state"].clone()
    for t in range(3):
        now = {n: x[n][:, t:t + 1] for n in ("q", "k", "v", "g")} | {"state": S.clone()}
        o = linear_attention_step(x["q"][:, t], x["k"][:, t], x["v"][:, t], x["g"][:, t], S)
        assert o.shape == (B, H, dv) and o.dtype == dtype
        check_out(now, o[:, None], S, dk ** -0.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_slots(device, dtype):
    """A pool in any order; rows outside it are skipped; the other slots stay as they are."""
    x = inputs(5, 1, 2, 2, 2, 2, 32, 40, dtype, device, False)
    pool = make((9, 2, 32, 40), torch.float32, device, 11)
    before, index = pool.clone(), torch.tensor([7, -1, 2, 9, 0], dtype=torch.int32, device=device)
    x["g"][0, 0, 0] = -math.inf
    pool[7, 0], before[7, 0] = math.nan, math.nan
    o = linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["g"][:, 0], pool, slots=index)
    assert not o[1].any() and not o[3].any()
    live = torch.tensor([0, 2, 4], device=device)
    now = {n: x[n][live] for n in ("q", "k", "v", "g")} | {"state": before[index[live].long()]}
    now["state"][0, 0] = 0
    check_out(now, o[live][:, None], pool[index[live].long()], 32 ** -0.5)
    rest = [i for i in range(9) if i not in (7, 2, 0)]
    assert torch.equal(pool[rest], before[rest])
    head = torch.tensor([-0.5, -1.0], device=device)
    p1, p2 = before.clone(), before.clone()
    a = linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], head, p1, slots=index)
    b = linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], head.expand(5, 2).contiguous(), p2, slots=index)
    assert torch.equal(a[1:], b[1:]) and torch.equal(p1[:7], p2[:7])


@pytest.mark.gpu
def test_step_far_slots():
    """A pool of more than 2^32 bytes and elements."""
    pool = torch.zeros(2 ** 18 + 8, 1, 128, 128, device="cuda")
    assert pool.numel() > 2 ** 32
    x = inputs(2, 1, 1, 1, 1, 1, 128, 128, torch.bfloat16, "cuda", False)
    index = torch.tensor([2 ** 18 + 5, 3], dtype=torch.int32, device="cuda")
    pool[2 ** 18 + 5] = 1.5
    x["state"] = torch.stack([torch.full((1, 128, 128), 1.5, device="cuda"), torch.zeros(1, 128, 128, device="cuda")])
    o = linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["g"][:, 0], pool, slots=index)
    check_out(x, o[:, None], pool[index.long()], 128 ** -0.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(device, dtype):
    """A prompt's state carried on token by token gives what the whole sequence gives."""
    x = inputs(2, 90, 4, 4, 2, 4, 48, 64, dtype, device, False)
    o, S = linear_attention(x["q"][:, :70], x["k"][:, :70], x["v"][:, :70], x["g"][:, :70], output_state=True)
    tail = [linear_attention_step(x["q"][:, t], x["k"][:, t], x["v"][:, t], x["g"][:, t], S) for t in range(70, 90)]
    check_out(x, torch.cat([o, torch.stack(tail, 1)], 1), S, 48 ** -0.5)


def test_refusals():
    q, g = torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 4)
    s = torch.zeros(2, 4, 8, 8)
    for bad in (lambda: linear_attention(q[0], q, q, g), lambda: linear_attention(q, q[:, :2], q, g),
                lambda: linear_attention(q, q[..., :4], q, g), lambda: linear_attention(q, q, q, g[:, :2]),
                lambda: linear_attention(q, q, q, g[..., :3]), lambda: linear_attention(q, q[:, :, :3], q, g),
                lambda: linear_attention(q, q, q, g, initial_state=s[:1]),
                lambda: linear_attention(q, q, q, g, initial_state=s.double()),
                lambda: linear_attention(torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 8), g[:1, :1, :1]),
                lambda: linear_attention(q[..., :0], q[..., :0], q, g), lambda: linear_attention(q, q, q[:, :, :0], g),
                lambda: linear_attention_step(q, q, q, g, s), lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], s[:1]),
                lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], s.transpose(2, 3)),
                lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], s, slots=torch.zeros(2, dtype=torch.long)),
                lambda: linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], s, slots=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear_attention(q.half(), q.half(), q.half(), g), lambda: linear_attention(q, q.bfloat16(), q, g),
                lambda: linear_attention(q, q, q, g.double())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        linear_attention_step(q[:, 0].requires_grad_(), q[:, 0], q[:, 0], g[:, 0], s)


def test_c_entries_refuse():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.linear_attention import _BLOCK, _STEP_BLOCK
    names = (["dtype", "gdtype", "per_head", "backward", "B", "T", "H", "Hq", "Hk", "Hv", "dk", "dv", "scale", "q", "k", "v",
              "g"] + [f"s{i}" for i in range(12)] + ["state", "o", "final", "d_o", "d0", "d1", "d2", "d_final", "dq", "dk_",
                                                     "dv_", "dg", "d_state", "saved", "saved_size", "ws", "size"])
    base = dict.fromkeys(names, 0) | dict(B=1, T=2, H=4, Hq=4, Hk=2, Hv=4, dk=8, dv=8, scale=1.0, q=64, k=64, v=64, g=64, o=64)
    pack = lambda **kw: _BLOCK.pack(*(base | kw).values())  # noqa: E731
    back = dict(backward=1, d_o=64, dq=64, dk_=64, dv_=64, dg=64)
    need = lib.ttc_linear_attention_workspace_bytes(pack(**back))
    assert need > 0 and lib.ttc_linear_attention_workspace_bytes(None) == 0
    for kw, code in [(dict(dtype=2), 2), (dict(gdtype=1), 2), (dict(B=-1), 1), (dict(T=-1), 1), (dict(H=0), 1), (dict(Hk=3), 1),
                     (dict(Hq=0), 1), (dict(dk=0), 1), (dict(dk=129), 1), (dict(dv=129), 1), (dict(q=0), 1), (dict(k=0), 1),
                     (dict(v=0), 1), (dict(g=0), 1), (dict(o=0), 1), (dict(B=1 << 40, T=1 << 40), 1), (back, 1),
                     (back | dict(ws=64, size=need - 1), 1), (back | dict(d_o=0, ws=64, size=need), 1)]:
        assert lib.ttc_linear_attention(pack(**kw), None) == code, kw
    long = back | dict(T=4096, ws=64, size=1 << 40)
    kept = lib.ttc_linear_attention_saved_bytes(pack(**long))
    assert kept > 0 and lib.ttc_linear_attention_saved_bytes(pack()) == 0
    assert lib.ttc_linear_attention(pack(**long, saved=64, saved_size=kept - 1), None) == 1
    assert lib.ttc_linear_attention(None, None) == 1 and lib.ttc_linear_attention(pack(B=0), None) == 0
    names = ["dtype", "gdtype", "B", "H", "Hq", "Hk", "Hv", "dk", "dv", "slots", "scale", "q", "k", "v", "g"] + \
        [f"s{i}" for i in range(8)] + ["state", "index", "o"]
    base = dict.fromkeys(names, 0) | dict(B=2, H=4, Hq=4, Hk=2, Hv=4, dk=8, dv=8, slots=2, scale=1.0, q=64, k=64, v=64, g=64,
                                          state=64, o=64)
    pack = lambda **kw: _STEP_BLOCK.pack(*(base | kw).values())  # noqa: E731
    for kw, code in [(dict(dtype=2), 2), (dict(gdtype=1), 2), (dict(B=-1), 1), (dict(Hv=3), 1), (dict(dv=200), 1),
                     (dict(slots=3), 1), (dict(slots=-1), 1), (dict(q=0), 1), (dict(state=0), 1), (dict(o=0), 1), (dict(g=0), 1)]:
        assert lib.ttc_linear_attention_step(pack(**kw), None) == code, kw
    assert lib.ttc_linear_attention_step(None, None) == 1 and lib.ttc_linear_attention_step(pack(B=0, slots=0), None) == 0
