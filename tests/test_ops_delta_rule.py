"""The gated delta rule (``ttc.ops.delta_rule`` and ``..._step``) against the recurrence in 64 bits; bounds, before any run, in
``_delta_oracle.py``."""
import math

import pytest
import torch

from _delta_oracle import delta64, near
from _ops_oracle import EPS, HALF, quotient, within
from ttc.ops import delta_rule, delta_rule_step, linear_attention
from ttc.ops.delta_rule import delta_rule_torch
from ttc.solvers._lib import lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16]
NAMES = ("q", "k", "v", "g", "beta", "state")


def make(shape, dtype, device, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def gates(B, T, H, kind):
    rand = lambda seed: torch.rand(B, T, H, generator=torch.Generator().manual_seed(seed))  # noqa: E731
    g = -rand(77) * torch.logspace(-3, 0.3, H)
    if kind == "none":
        g = torch.zeros(B, T, H)
    elif kind == "strong":  # decays of up to e^-100 beside ones of almost 1
        g = g * torch.where(rand(78) < 0.3, 60.0, 0.01)
    elif kind == "reset":
        g[rand(79) < 0.05] = -math.inf
        g[rand(80) < 0.05] = -1e30
        g[rand(81) < 0.03] = torch.finfo(torch.float32).min
        g[:, :1, :1] = -math.inf
    elif kind == "growing":
        g = -g * 0.02
    return g


def inputs(B, T, H, Hq, Hk, Hv, dk, dv, dtype, device, state, kind="mixed", gdtype=torch.float32, bdtype=torch.float32,
           normalize=False):
    k = make((B, T, Hk, dk), torch.float32, "cpu", 2)
    if not normalize:
        k = 0.99 * k / k.norm(dim=-1, keepdim=True).clamp_min(1e-6)
    beta = torch.rand(B, T, H, generator=torch.Generator().manual_seed(5))
    return dict(q=make((B, T, Hq, dk), dtype, device, 1), k=k.to(dtype).to(device), v=make((B, T, Hv, dv), dtype, device, 3),
                g=gates(B, T, H, kind).to(gdtype).to(device), beta=beta.to(bdtype).to(device),
                state=make((B, H, dk, dv), torch.float32, device, 4) if state else None)


def call(x, scale, normalize=False, **kw):
    return delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], scale=scale, initial_state=x["state"], output_state=True,
                      normalize=normalize, **kw)


def oracle(x, scale, d_o=None, d_state=None, normalize=False, **kw):
    return delta64(x["q"], x["k"], x["v"], x["g"], x["beta"], scale, x["state"], d_o, d_state, normalize, **kw)


def grads(x, d_o, d_state, scale, normalize=False, names=NAMES):
    leaves = {n: x[n].detach().clone().requires_grad_() if n in names and x[n] is not None else x[n] for n in NAMES}
    o, final = call(leaves, scale, normalize)
    wanted = [n for n in names if x[n] is not None]
    outs, ds = zip(*[(y, d) for y, d in ((o, d_o), (final, d_state)) if d is not None and y.requires_grad])
    got = dict(zip(wanted, torch.autograd.grad(outs, [leaves[n] for n in wanted], ds)))
    got["o"], got["final"] = o.detach(), final.detach()
    return got


def check(got, want, names, ordinary=False):
    for n in names:
        ref = {"state": "d_state", "final": "state"}.get(n, n)
        within(got[n], *want[ref])
        if ordinary and want[ref][0].any():  # the decay of a first token without a state has no effect: no size to go by
            near(got[n], want[ref])


CASES = [  # batch, tokens, heads of the output, of q, k, v, dk, dv
    (1, 1, 1, 1, 1, 1, 1, 1), (2, 1, 4, 4, 4, 4, 64, 64), (1, 2, 2, 2, 2, 2, 16, 16), (2, 4, 2, 2, 2, 1, 128, 40),
    (1, 5, 3, 3, 1, 3, 24, 8), (1, 63, 2, 2, 1, 1, 32, 16), (2, 64, 3, 3, 3, 3, 64, 128), (1, 65, 4, 2, 2, 4, 128, 64),
    (1, 17, 2, 2, 2, 2, 5, 3), (2, 130, 6, 6, 2, 3, 48, 80), (1, 129, 2, 1, 1, 2, 128, 128), (1, 300, 2, 2, 2, 2, 33, 127),
    (3, 0, 2, 2, 2, 2, 8, 8), (0, 5, 2, 2, 2, 2, 8, 8), (1, 40, 1, 1, 1, 1, 127, 20), (1, 700, 2, 2, 2, 2, 16, 24),
    (2, 33, 2, 2, 2, 2, 32, 100), (1, 97, 2, 2, 2, 2, 100, 32)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state,normalize", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("case", CASES)
def test_forward(device, dtype, state, normalize, case):
    x = inputs(*case, dtype, device, state, normalize=normalize)
    scale = case[6] ** -0.5
    o, final = call(x, scale, normalize)
    assert o.dtype == dtype and o.is_contiguous() and final.dtype == torch.float32
    want = oracle(x, scale, normalize=normalize)
    within(o, *want["o"])
    within(final, *want["state"])
    near(o, want["o"])
    near(final, want["state"])
    default = delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["state"], normalize=normalize)
    assert torch.equal(default, o)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state,normalize", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("case", CASES)
def test_gradients(device, dtype, state, normalize, case):
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    x = inputs(*case, dtype, device, state, normalize=normalize, gdtype=dtype if dk % 3 == 0 else torch.float32,
               bdtype=dtype if dv % 4 == 0 else torch.float32)
    d_o = make((B, T, H, dv), dtype, device, 9)
    d_state = make((B, H, dk, dv), torch.float32, device, 10) if state else None
    got, want = grads(x, d_o, d_state, 0.4, normalize), oracle(x, 0.4, d_o, d_state, normalize)
    # a vector of one element has the same length whatever it is: its gradient, but for eps, is a difference of equal terms
    check(got, want, ("o", "final") + (NAMES if state else NAMES[:5]), dk > 1 or not normalize)
    for n in NAMES[:5]:
        assert got[n].dtype == x[n].dtype and got[n].shape == x[n].shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "strong", "reset", "growing"])
@pytest.mark.parametrize("case", [(2, 200, 3, 3, 3, 3, 24, 32), (1, 150, 2, 2, 2, 2, 128, 128), (1, 90, 2, 2, 1, 2, 64, 40)])
def test_decays(device, dtype, kind, case):
    """Outputs and all gradients under decays of 1, very strong ones, resets at any token, and growth."""
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    x = inputs(*case, dtype, device, True, kind)
    d_o, d_state = make((B, T, H, dv), dtype, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    check(grads(x, d_o, d_state, 0.3), oracle(x, 0.3, d_o, d_state), ("o", "final") + NAMES)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keys", ["same", "two", "zero", "opposite"])
@pytest.mark.parametrize("strength", [0.0, 1.0, 2.0])
def test_keys_and_strengths(device, dtype, keys, strength):
    """Keys that repeat (the triangle is full), none at all, strengths of 0 (nothing is taken up), 1 (what is held at the key is
    replaced) and 2 (it changes its sign)."""
    case = (1, 140, 2, 2, 2, 2, 32, 24)
    x = inputs(*case, dtype, device, True, "none")
    row = x["k"][:, :1]
    if keys == "same":
        x["k"] = row.expand_as(x["k"]).contiguous()
    elif keys == "two":
        x["k"][:, ::2] = row
    elif keys == "opposite":
        x["k"] = row * torch.where(torch.arange(140, device=device) % 2 == 0, 1, -1).to(dtype)[None, :, None, None]
    else:
        x["k"].zero_()
    x["beta"].fill_(strength)
    d_o, d_state = make((1, 140, 2, 24), dtype, device, 9), make((1, 2, 32, 24), torch.float32, device, 10)
    check(grads(x, d_o, d_state, 0.4), oracle(x, 0.4, d_o, d_state), ("o", "final") + NAMES)
    if keys == "zero":  # of length sqrt(eps): no key, and gradients that are finite
        got = grads(x, d_o, d_state, 0.4, True)
        check(got, oracle(x, 0.4, d_o, d_state, True), ("o", "final") + NAMES)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("normalize", [False, True])
def test_differences(device, normalize):
    """Gradients in fp32 against central differences of the sum in 64 bits."""
    B, T, H, dk, dv = 1, 70, 2, 12, 8
    x = inputs(B, T, H, 1, 2, 1, dk, dv, torch.float32, device, True, normalize=normalize)
    d_o, d_state = make((B, T, H, dv), torch.float32, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    got = grads(x, d_o, d_state, 0.4, normalize)
    xs = [x[n] for n in NAMES]
    f = lambda *t: call(dict(zip(NAMES, t)), 0.4, normalize)  # noqa: E731
    h = 2.0 ** -9
    for i, n in enumerate(NAMES):
        one = make(x[n].shape, torch.float32, device, 30 + i)
        one = one / one.norm()
        ds = [one if j == i else torch.zeros_like(t) for j, t in enumerate(xs)]
        want = quotient(f, xs, ds, (d_o, d_state), h)
        mine = float((got[n].double() * one.double()).sum())
        # steps along a unit vector: third derivatives of the outputs are below 8^3 of their size; outputs of size |o| are
        # rounded at some hundred terms each, which a step of h divides
        size = float((d_o.norm() + d_state.norm()) * (got["o"].norm() + got["final"].norm()))
        assert abs(mine - want) <= size * (8 ** 3 * h * h / 6 + 400 * EPS / h * 0.1), (n, mine, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_views(device, dtype):
    """Parts of a projection, odd offsets, one row for a whole batch, gates and gradients of other strides."""
    B, T, H, dk, dv = 2, 75, 4, 24, 16
    x = inputs(B, T, H, 4, 4, 4, dk, dv, dtype, device, False, normalize=True, bdtype=dtype)
    wide = make((B, T, 2 * H * dk + H * dv + 7), dtype, device, 20)
    d_o = make((dv, T, H, B), dtype, device, 21).permute(3, 1, 2, 0)
    gh = x["g"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    bh = x["beta"].repeat_interleave(2, dim=1)[:, ::2]
    for off in (0, 7):
        q, k, v = torch.split(wide[..., off:off + 2 * H * dk + H * dv], [H * dk, H * dk, H * dv], dim=-1)
        y = dict(q=q.unflatten(-1, (H, dk)), k=k.unflatten(-1, (H, dk)), v=v.unflatten(-1, (H, dv)), g=gh, beta=bh, state=None)
        leaves = {n: y[n].detach().requires_grad_() for n in NAMES[:5]}
        o = delta_rule(*(leaves[n] for n in NAMES[:5]), scale=0.5, normalize=True)
        got = dict(zip(NAMES, torch.autograd.grad(o, list(leaves.values()), d_o)), o=o.detach())
        check(got, oracle(y, 0.5, d_o, None, True), ("o",) + NAMES[:5])
    swapped = {n: x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")}
    assert torch.equal(delta_rule(*(dict(x, **swapped)[n] for n in NAMES[:5]), normalize=True),
                       delta_rule(*(x[n] for n in NAMES[:5]), normalize=True))
    every = x["q"][..., ::2]
    y = dict(x, q=every, k=x["k"][..., ::2])
    within(call(y, 0.4, True)[0], *oracle(y, 0.4, normalize=True)["o"])
    one = x["k"][:1].clone().requires_grad_()  # one sequence's keys for the whole batch: its gradient is the sum
    o = delta_rule(x["q"], one.expand_as(x["k"]), x["v"], x["g"], x["beta"], scale=0.5, normalize=True)
    dk_, = torch.autograd.grad(o, one, d_o)
    want = oracle(dict(x, k=one.expand_as(x["k"])), 0.5, d_o, None, True)["k"]
    total, off = want[0].sum(0, keepdim=True), want[1].sum(0, keepdim=True)
    within(dk_, total, off + HALF[dtype] * (total.abs() + off))


@pytest.mark.parametrize("device", DEVICES)
def test_part_of_the_gradients(device):
    """Any subset of inputs that require gradients, and of outputs that have them, gives the bits of the whole."""
    B, T, H, dk, dv = 1, 80, 2, 32, 32
    x = inputs(B, T, H, 1, 2, 1, dk, dv, torch.bfloat16, device, True)
    d_o, d_state = make((B, T, H, dv), torch.bfloat16, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    full = grads(x, d_o, d_state, 0.4)
    for names in (("q",), ("k",), ("v",), ("g",), ("beta",), ("state",), ("v", "state"), ("q", "beta")):
        part = grads(x, d_o, d_state, 0.4, names=names)
        for n in names:
            assert torch.equal(part[n], full[n]), n
    leaf = dict(x, k=x["k"].clone().requires_grad_())
    final = call(leaf, 0.4)[1]
    dk_, = torch.autograd.grad(final, leaf["k"], d_state)
    within(dk_, *oracle(x, 0.4, torch.zeros_like(d_o), d_state)["k"])


SPOILT = [("k", math.nan), ("v", math.nan), ("v", math.inf), ("beta", math.nan), ("g", math.nan), ("g", math.inf), ("q", math.inf),
          ("k", -math.inf), ("beta", math.inf)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what,value", SPOILT)
@pytest.mark.parametrize("at", [0, 63, 100])
def test_not_finite(device, dtype, what, value, at):
    """What is not finite has no effect on outputs in front of it, nor on outputs and gradients behind a reset; and a spoilt text
    has none on the gradients of the text in front of it."""
    B, T, H, dk, dv, cut = 1, 170, 2, 32, 40, 110
    x = inputs(B, T, H, 2, 2, 2, dk, dv, dtype, device, True)
    x["g"][:, cut] = -math.inf
    d_o, d_state = make((B, T, H, dv), dtype, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    clean = oracle(x, 0.4, d_o, d_state)
    bad = dict(x, **{what: x[what].clone()})
    bad[what][0, at, 0] = value if x[what].dim() == 3 else bad[what][0, at, 0].index_fill(0, torch.tensor([3], device=device), value)
    got = grads(bad, d_o, d_state, 0.4)
    pick = lambda t, rows: t[:, rows]  # noqa: E731
    within(got["o"][:, :at], *(pick(t, slice(0, at)) for t in clean["o"]))
    for n in ("o", "q", "k", "v", "beta"):
        within(got[n][:, cut:], *(pick(t, slice(cut, T)) for t in clean[n]))
    within(got["g"][:, cut + 1:], *(pick(t, slice(cut + 1, T)) for t in clean["g"]))
    within(got["final"], *clean["state"])
    for n in ("o", "q", "k", "v", "g", "beta"):  # the other head
        within(got[n][:, :, 1], *(t[:, :, 1] for t in clean[n]))
    assert not got["o"][:, at:cut, 0].isfinite().all()
    late = dict(x, **{what: x[what].clone()})  # in the second text: the first one's gradients stay
    late[what][0, cut + 1 + at // 3, 0] = bad[what][0, at, 0]
    got = grads(late, d_o, d_state, 0.4)
    for n in ("o", "q", "k", "v", "beta", "g"):
        within(got[n][:, :cut], *(pick(t, slice(0, cut)) for t in clean[n]))
    within(got["state"], *clean["d_state"])


@pytest.mark.parametrize("device", DEVICES)
def test_spoilt_state_and_gradients(device):
    """A state that is not finite in one column spoils that column until a reset; so does an output's gradient, backwards."""
    B, T, H, dk, dv = 1, 150, 1, 24, 20
    x = inputs(B, T, H, 1, 1, 1, dk, dv, torch.float32, device, True)
    x["g"][:, 70] = -math.inf
    d_o, d_state = make((B, T, H, dv), torch.float32, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    clean = oracle(x, 0.4, d_o, d_state)
    bad = dict(x, state=x["state"].clone())
    bad["state"][0, 0, 5, 7] = math.nan
    got = grads(bad, d_o, d_state, 0.4)
    rest = [i for i in range(dv) if i != 7]
    within(got["o"][..., rest], *(t[..., rest] for t in clean["o"]))
    within(got["o"][:, 70:], *(t[:, 70:] for t in clean["o"]))
    assert got["o"][:, :70, :, 7].isnan().all()
    within(got["v"], *clean["v"])
    within(got["state"], *clean["d_state"])
    if device == "cpu":  # torch operators do not see a gradient before it is there
        return
    spoilt = d_o.clone()
    spoilt[0, 90, 0, 3] = math.nan
    got = grads(x, spoilt, d_state, 0.4)
    for n in ("q", "k", "v", "g", "beta"):
        within(got[n][:, :70], *(t[:, :70] for t in clean[n]))
        within(got[n][:, 91:], *(t[:, 91:] for t in clean[n]))
    within(got["state"], *clean["d_state"])


@pytest.mark.parametrize("device", DEVICES)
def test_overflow_stays_behind(device):
    """Finite inputs whose sums overflow within a chunk: tokens in front of that are as they were."""
    x = inputs(1, 100, 1, 1, 1, 1, 16, 16, torch.float32, device, False, "none")
    clean = oracle(x, 1.0)["o"]
    x["v"][0, 40:] = 3e38
    x["beta"][0, 40:] = 2.0
    o = call(x, 1.0)[0]
    within(o[:, :40], *(t[:, :40] for t in clean))
    assert not o[:, 40:].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("heads", [(4, 4, 4, 4), (4, 2, 1, 4), (6, 3, 6, 2)])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (17, 33), (1, 1), (128, 5)])
def test_step(device, dtype, normalize, heads, dims):
    B, (dk, dv) = 3, dims
    x = inputs(B, 3, *heads, dk, dv, dtype, device, True, normalize=normalize, bdtype=dtype)
    S = x["state"].clone()
    for t in range(3):
        now = {n: x[n][:, t:t + 1] for n in NAMES[:5]} | {"state": S.clone()}
        o = delta_rule_step(*(x[n][:, t] for n in NAMES[:5]), S, normalize=normalize)
        assert o.shape == (B, heads[0], dv) and o.dtype == dtype
        want = oracle(now, dk ** -0.5, normalize=normalize)
        within(o[:, None], *want["o"])
        within(S, *want["state"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_step_slots(device, dtype):
    """A pool in any order; rows outside it are skipped; the other slots stay as they are; a reset drops a spoilt state."""
    x = inputs(5, 1, 2, 2, 2, 2, 32, 40, dtype, device, False)
    pool = make((9, 2, 32, 40), torch.float32, device, 11)
    before, index = pool.clone(), torch.tensor([7, -1, 2, 9, 0], dtype=torch.int32, device=device)
    x["g"][0, 0, 0] = -math.inf
    pool[7, 0], before[7, 0] = math.nan, math.nan
    version = pool._version
    o = delta_rule_step(*(x[n][:, 0] for n in NAMES[:5]), pool, slots=index)
    assert pool._version > version and not o[1].any() and not o[3].any()
    live = torch.tensor([0, 2, 4], device=device)
    now = {n: x[n][live] for n in NAMES[:5]} | {"state": before[index[live].long()]}
    now["state"][0, 0] = 0
    want = oracle(now, 32 ** -0.5)
    within(o[live][:, None], *want["o"])
    within(pool[index[live].long()], *want["state"])
    rest = [i for i in range(9) if i not in (7, 2, 0)]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompt", [3, 70])
def test_prompt_then_tokens(device, dtype, prompt):
    """A prompt's state carried on in pieces and token by token gives what the whole sequence gives."""
    x = inputs(2, 90, 4, 4, 2, 4, 48, 64, dtype, device, False, normalize=True)
    part = lambda a, b: [x[n][:, a:b] for n in NAMES[:5]]  # noqa: E731
    o, S = delta_rule(*part(0, prompt), output_state=True, normalize=True)
    o2, S = delta_rule(*part(prompt, 80), output_state=True, normalize=True, initial_state=S)
    tail = [delta_rule_step(*(x[n][:, t] for n in NAMES[:5]), S, normalize=True) for t in range(80, 90)]
    want = oracle(x, 48 ** -0.5, normalize=True)
    within(torch.cat([o, o2, torch.stack(tail, 1)], 1), *want["o"])
    within(S, *want["state"])


@pytest.mark.parametrize("device", DEVICES)
def test_orthogonal_keys_are_linear_attention(device):
    """Keys at right angles meet nothing that is held: linear attention with the values b v."""
    T = 16
    x = inputs(1, T, 1, 1, 1, 1, 16, 12, torch.float32, device, False)
    x["k"] = torch.eye(16, device=device)[None, :, None]
    a = delta_rule(*(x[n] for n in NAMES[:5]))
    b = linear_attention(x["q"], x["k"], x["v"] * x["beta"].unsqueeze(-1), x["g"])
    within(a, b, 32 * EPS * (b.abs().double().cpu() + 1))


@pytest.mark.parametrize("device", DEVICES)
def test_observed(device):
    """Second derivatives, transforms: through torch operators; partial derivatives where one input is computed from another."""
    x = inputs(2, 20, 2, 2, 2, 2, 8, 6, torch.float32, device, True, normalize=True)
    leaves = [x[n].clone().requires_grad_() for n in NAMES]
    loss = lambda *t: call(dict(zip(NAMES, t)), 0.4, True)[0].square().sum()  # noqa: E731
    first = torch.autograd.grad(loss(*leaves), leaves, create_graph=True)
    second = torch.autograd.grad(sum(g.square().sum() for g in first), leaves)
    ref = torch.autograd.grad(delta_rule_torch(*leaves[:5], 0.4, leaves[5], True)[0].square().sum(), leaves, create_graph=True)
    again = torch.autograd.grad(sum(g.square().sum() for g in ref), leaves)
    for a, b in zip((*first, *second), (*ref, *again)):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * float(b.abs().max()) + 1e-5)
    each = torch.func.vmap(torch.func.grad(lambda v: delta_rule(x["q"][:1], x["k"][:1], v[None], x["g"][:1], x["beta"][:1])
                                           .square().sum()))(x["v"])
    assert each.shape == x["v"].shape
    k = x["k"].clone().requires_grad_()
    q = 2 * k  # q is computed from k
    g, = torch.autograd.grad(delta_rule(q, k, x["v"], x["g"], x["beta"], normalize=True).square().sum(), k, create_graph=True)
    p = k.detach().clone().requires_grad_()
    plain, = torch.autograd.grad(delta_rule_torch(2 * p, p, x["v"], x["g"], x["beta"], 8 ** -0.5, None, True)[0].square().sum(), p)
    assert torch.allclose(g, plain, rtol=1e-3, atol=1e-4)


@pytest.mark.gpu
def test_graph_and_stream():
    """Captured: training, a prompt and a step, replayed on new inputs between eager calls; two graphs in turn."""
    shape = (1, 200, 2, 2, 2, 2, 64, 64)
    xs = [inputs(*shape, torch.bfloat16, "cuda", True, normalize=True) for _ in range(2)]
    d_o, d_state = make((1, 200, 2, 64), torch.bfloat16, "cuda", 9), make((1, 2, 64, 64), torch.float32, "cuda", 10)
    pools = [make((1, 2, 64, 64), torch.float32, "cuda", 11) for _ in range(2)]

    def work(x, pool):
        leaves = [x[n].detach().requires_grad_() for n in NAMES]
        o, final = call(dict(zip(NAMES, leaves)), 0.4, True)
        got = torch.autograd.grad((o, final), leaves, (d_o, d_state))
        with torch.no_grad():
            return (o.detach(), final.detach(), *got, call(x, 0.4, True)[0],
                    delta_rule_step(*(x[n][:, 0] for n in NAMES[:5]), pool, normalize=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apart = work(xs[0], pools[0].clone())
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(apart, work(xs[0], pools[0].clone())):
        assert torch.equal(a, b)
    graphs, held = [], []
    for x, pool in zip(xs, pools):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(work(x, pool))
        graphs.append(graph)
    for i in range(3):
        for x in xs:
            x["v"].copy_(make((1, 200, 2, 64), torch.bfloat16, "cuda", 50 + i))
        starts = [p.clone() for p in pools]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, pool, start, mine in zip(xs, pools, starts, held):
            after = pool.clone()
            pool.copy_(start)
            for a, b in zip(mine, work(x, pool)):
                assert torch.equal(a, b)
            assert torch.equal(pool, after)


@pytest.mark.gpu
def test_many_heads_and_far_rows():
    """More chunks than one workgroup number holds in 16 bits; rows more than 2^32 elements apart; a far slot."""
    x = inputs(1500, 66, 40, 40, 40, 40, 8, 8, torch.bfloat16, "cuda", False, normalize=True)
    o, S = call(x, 0.4, True)
    for b in (0, 777, 1499):
        one = {n: x[n][b:b + 1] if x[n] is not None else None for n in NAMES}
        want = oracle(one, 0.4, normalize=True)
        within(o[b:b + 1], *want["o"])
        within(S[b:b + 1], *want["state"])
    far = torch.zeros(2 ** 32 + 70 * 64, dtype=torch.bfloat16, device="cuda")
    y = inputs(2, 70, 1, 1, 1, 1, 64, 64, torch.bfloat16, "cuda", False)
    v = far.as_strided((2, 70, 1, 64), (2 ** 32, 64, 64, 1))
    v.copy_(y["v"])
    assert torch.equal(call(dict(y, v=v), 0.4)[0], call(y, 0.4)[0])
    del far, v
    pool = torch.zeros(2 ** 18 + 8, 1, 128, 128, device="cuda")
    assert pool.numel() > 2 ** 32
    z = inputs(2, 1, 1, 1, 1, 1, 128, 128, torch.bfloat16, "cuda", False)
    index = torch.tensor([2 ** 18 + 5, 3], dtype=torch.int32, device="cuda")
    pool[2 ** 18 + 5] = 1.5
    z["state"] = torch.stack([torch.full((1, 128, 128), 1.5, device="cuda"), torch.zeros(1, 128, 128, device="cuda")])
    o = delta_rule_step(*(z[n][:, 0] for n in NAMES[:5]), pool, slots=index)
    want = oracle(z, 128 ** -0.5)
    within(o[:, None], *want["o"])
    within(pool[index.long()], *want["state"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["mixed", "reset"])
@pytest.mark.parametrize("case", [(1, 1800, 2, 2, 2, 2, 128, 128), (2, 1111, 1, 1, 1, 1, 64, 32), (1, 900, 3, 1, 3, 1, 20, 70),
                                  (1, 777, 2, 2, 2, 1, 128, 24), (1, 650, 1, 1, 1, 1, 30, 128)])
def test_long(case, kind, dtype):
    """Inputs whose chunks are split into segments."""
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    x = inputs(*case, dtype, "cuda", True, kind, normalize=True)
    d_o, d_state = make((B, T, H, dv), dtype, "cuda", 9), make((B, H, dk, dv), torch.float32, "cuda", 10)
    got, want = grads(x, d_o, d_state, 0.1, True), oracle(x, 0.1, d_o, d_state, True)
    check(got, want, ("o", "final") + NAMES, kind == "mixed")
    with torch.no_grad():
        o, S = call(x, 0.1, True)
    assert torch.equal(o, got["o"]) and torch.equal(S, got["final"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["k", "v", "g", "beta", "q"])
def test_not_finite_in_segments(dtype, what):
    """A spoilt text among others, far apart: no effect in front of it, nor behind the reset after it, nor (its gradients) on the
    text in front of it."""
    B, T, H, dk, dv, first, second = 1, 1500, 1, 64, 48, 420, 1010
    x = inputs(B, T, H, 1, 1, 1, dk, dv, dtype, "cuda", True)
    x["g"][:, [first, second]] = -math.inf
    d_o, d_state = make((B, T, H, dv), dtype, "cuda", 9), make((B, H, dk, dv), torch.float32, "cuda", 10)
    clean = oracle(x, 0.4, d_o, d_state)
    x[what][0, 700] = math.nan
    got = grads(x, d_o, d_state, 0.4)
    within(got["o"][:, :700], *(t[:, :700] for t in clean["o"]))
    for n in ("o", "q", "k", "v", "beta", "g"):
        within(got[n][:, :first], *(t[:, :first] for t in clean[n]))
        within(got[n][:, second + 1:], *(t[:, second + 1:] for t in clean[n]))
    within(got["final"], *clean["state"])
    within(got["state"], *clean["d_state"])
    assert not got["o"][:, 700:second].isfinite().all()


def test_refusals():
    q, g = torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 4)
    s = torch.zeros(2, 4, 8, 8)
    for bad in (lambda: delta_rule(q[0], q, q, g, g), lambda: delta_rule(q, q[:, :2], q, g, g),
                lambda: delta_rule(q, q[..., :4], q, g, g), lambda: delta_rule(q, q, q, g[:, :2], g[:, :2]),
                lambda: delta_rule(q, q, q, g, g[..., :2]), lambda: delta_rule(q, q, q, g[0, 0], g), lambda: delta_rule(q, q, q, g, g[0]),
                lambda: delta_rule(q, q, q, g[..., :3], g[..., :3]), lambda: delta_rule(q, q[:, :, :3], q, g, g),
                lambda: delta_rule(q, q, q, g, g, initial_state=s[:1]), lambda: delta_rule(q, q, q, g, g, initial_state=s.double()),
                lambda: delta_rule(torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 8), g[:1, :1, :1], g[:1, :1, :1]),
                lambda: delta_rule(q[..., :0], q[..., :0], q, g, g), lambda: delta_rule(q, q, q[:, :, :0], g, g),
                lambda: delta_rule(q, q, q, g, g, normalize=True, eps=-1.0), lambda: delta_rule(q, q, q, g, g, eps=math.nan),
                lambda: delta_rule_step(q, q, q, g, g, s),
                lambda: delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s[:1]),
                lambda: delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s.transpose(2, 3)),
                lambda: delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s, slots=torch.zeros(2, dtype=torch.long)),
                lambda: delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], g[:, 0], s, slots=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: delta_rule(q.half(), q.half(), q.half(), g, g), lambda: delta_rule(q, q.bfloat16(), q, g, g),
                lambda: delta_rule(q, q, q, g.double(), g), lambda: delta_rule(q, q, q, g, g.bfloat16())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        delta_rule_step(q[:, 0].requires_grad_(), q[:, 0], q[:, 0], g[:, 0], g[:, 0], s)


def test_c_entries_refuse():
    """Codes come back before anything is launched (no GPU is touched)."""
    from ttc.ops.delta_rule import _BLOCK, _STEP_BLOCK
    names = (["dtype", "gdtype", "bdtype", "norm", "backward", "B", "T", "H", "Hq", "Hk", "Hv", "dk", "dv", "scale", "eps", "q",
              "k", "v", "g", "beta"] + [f"s{i}" for i in range(15)]
             + ["state", "o", "final", "d_o", "d0", "d1", "d2", "d_final", "dq", "dk_", "dv_", "dg", "db", "d_state", "saved",
                "saved_size", "ws", "size"])
    base = dict.fromkeys(names, 0) | dict(B=1, T=70, H=4, Hq=4, Hk=2, Hv=4, dk=8, dv=8, scale=1.0, eps=0.0, q=64, k=64, v=64,
                                          g=64, beta=64, o=64)
    pack = lambda **kw: _BLOCK.pack(*(base | kw).values())  # noqa: E731
    need = lib.ttc_delta_rule_workspace_bytes(pack())
    kept = lib.ttc_delta_rule_saved_bytes(pack())
    back = dict(backward=1, d_o=64, dq=64, dk_=64, dv_=64, dg=64, db=64, saved=64, saved_size=kept)
    wants = lib.ttc_delta_rule_workspace_bytes(pack(**back))
    assert need > 0 and kept > need and wants > 0 and lib.ttc_delta_rule_workspace_bytes(pack(T=4)) == 0
    assert lib.ttc_delta_rule_workspace_bytes(pack(saved=64)) == 0 == lib.ttc_delta_rule_workspace_bytes(None)
    room = dict(ws=64, size=1 << 40)
    for kw, code in [(dict(dtype=2), 2), (dict(gdtype=1), 2), (dict(bdtype=1), 2), (dict(B=-1), 1), (dict(T=-1), 1), (dict(H=0), 1),
                     (dict(Hk=3), 1), (dict(Hq=0), 1), (dict(dk=0), 1), (dict(dk=129), 1), (dict(dv=129), 1), (dict(eps=-1.0), 1),
                     (dict(eps=math.nan), 1), (dict(q=0), 1), (dict(k=0), 1), (dict(v=0), 1), (dict(g=0), 1), (dict(beta=0), 1),
                     (dict(o=0), 1), (dict(B=1 << 40, T=1 << 40), 1), (back | dict(saved=0), 1), (back | dict(saved_size=kept - 1), 1),
                     (back | dict(d_o=0), 1), (dict(saved=64, saved_size=kept - 1), 1), (dict(ws=72), 1),
                     (dict(saved=72, saved_size=kept), 1)]:
        assert lib.ttc_delta_rule(pack(**(room | kw)), None) == code, kw
    assert lib.ttc_delta_rule(pack(ws=64, size=need - 1), None) == 1 and lib.ttc_delta_rule(pack(), None) == 1
    assert lib.ttc_delta_rule(pack(**back, ws=64, size=wants - 1), None) == 1
    assert lib.ttc_delta_rule(None, None) == 1 and lib.ttc_delta_rule(pack(B=0), None) == 0
    names = ["dtype", "gdtype", "bdtype", "norm", "B", "H", "Hq", "Hk", "Hv", "dk", "dv", "slots", "scale", "eps", "q", "k", "v", "g",
             "beta"] + [f"s{i}" for i in range(10)] + ["state", "index", "o"]
    base = dict.fromkeys(names, 0) | dict(B=2, H=4, Hq=4, Hk=2, Hv=4, dk=8, dv=8, slots=2, scale=1.0, eps=0.0, q=64, k=64, v=64,
                                          g=64, beta=64, state=64, o=64)
    pack = lambda **kw: _STEP_BLOCK.pack(*(base | kw).values())  # noqa: E731
    for kw, code in [(dict(dtype=2), 2), (dict(gdtype=1), 2), (dict(bdtype=1), 2), (dict(B=-1), 1), (dict(Hv=3), 1), (dict(dv=200), 1),
                     (dict(slots=3), 1), (dict(slots=-1, index=64), 1), (dict(q=0), 1), (dict(state=0), 1), (dict(o=0), 1),
                     (dict(g=0), 1), (dict(beta=0), 1), (dict(eps=-1.0), 1)]:
        assert lib.ttc_delta_rule_step(pack(**kw), None) == code, kw
    assert lib.ttc_delta_rule_step(None, None) == 1 and lib.ttc_delta_rule_step(pack(B=0, slots=0), None) == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("case", [(5, 25, 8, 8, 8, 8, 128, 32), (2, 256, 4, 4, 4, 4, 41, 128), (3, 130, 4, 1, 2, 4, 64, 64),
                                  (2, 90, 6, 6, 6, 6, 30, 20), (2, 70, 5, 5, 5, 5, 128, 128)])
def test_sums_of_16_bit_outputs(device, train, case):
    """Outputs in 16 bits are sums in 32, rounded once.  Some 400 roundings on a term's way, each of at most EPS and independent of
    each other, leave a sum off by e = 20 EPS of the outputs' size.  One of z times that size, whose neighbours are at least 2^-8 z
    of it apart, then rounds to the other one as often as e 2^8 / z, at most always: with z as normal values are, 0.8 dz near 0,
    the mean of 1 / z from e 2^8 = 3e-4 on is 0.8 ln(1 / 3e-4) = 6.5, and 6.5 e 2^8 = 0.2 % of all differ from the rounded 64-bit
    values; a count of n scatters by sqrt(n), four of which are added.  Their number and not their size is bounded: in the first
    case one output of the largest, off by a step, is 2^-7 of 38 in the norm, more than all others together.  (Operands cut to 16
    digits, the state and the scores, made 0.7 to 1.1 % differ.)"""
    x = inputs(*case, torch.bfloat16, device, True, normalize=True)
    leaves = {n: x[n].clone().requires_grad_(train) for n in NAMES}
    o = call(leaves, 0.3, True)[0].detach().cpu()
    want = oracle(x, 0.3, normalize=True)["o"][0].to(torch.bfloat16)
    most = 6.5 * 20 * EPS * 2 ** 8 * o.numel()
    assert int((o != want).sum()) <= most + 4 * math.sqrt(most), float((o != want).double().mean())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", [(8, 100, 8, 8, 8, 8, 64, 64), (4, 64, 16, 16, 16, 16, 32, 40), (4, 90, 8, 8, 8, 8, 128, 64)])
def test_sums_of_16_bit_gradients(device, case):
    """As above: a term of these gradients has passed the state and the gradient of the state, twice as many roundings, so they
    are off by sqrt(800) EPS.  (Score tiles cut to 16 digits made up to 0.36 % of dq and dk differ.)"""
    x = inputs(*case, torch.bfloat16, device, True)
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    d_o, d_state = make((B, T, H, dv), torch.bfloat16, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    got, want = grads(x, d_o, d_state, 0.3), oracle(x, 0.3, d_o, d_state)
    for n in ("q", "k", "v"):
        most = 6.5 * math.sqrt(800) * EPS * 2 ** 8 * got[n].numel()
        differ = int((got[n].cpu() != want[n][0].to(torch.bfloat16)).sum())
        assert differ <= most + 4 * math.sqrt(most), (n, differ / got[n].numel())
