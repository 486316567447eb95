"""``DeltaRuleLayer`` (``ttc.layers``): the short convolution, turned keys, the gated delta rule and the gated norm run together.

Tolerances: the output is a sum of ``num_heads * value_dim`` products of normalised values of about 1 and weights of a random
initialisation, so of about 1; 32-bit rounding of some hundred products and sums per value stays below 1e-4 of it.  In bfloat16
each of the six stages (projection, convolution, turn, mixing, norm, projection) rounds once to 2^-8 a value, and a key's
rounding meets the state twice (what is read at it, what is written): about 3 % of a value of 1 at the output, 0.1 absolute at
its largest."""
import sys

import pytest
import torch
import torch.nn.functional as F

from _delta_oracle import delta64
from _ops_oracle import group_norm64
from test_ops_rotary_axes import axes64
from ttc import DeltaRuleLayer, LinearAttentionLayer
from ttc.ops import grid_positions

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TOL = {torch.float32: 1e-4, torch.bfloat16: 0.1}


def make(device, dtype, **kw):
    torch.manual_seed(3)
    args = dict(dim=48, num_heads=4, key_dim=16, value_dim=24, key_heads=2, rotary_sections=(2, 3, 2), max_positions=64)
    return DeltaRuleLayer(**(args | kw)).to(device).to(dtype)


def tokens(B, T, seed, device, dtype):
    return torch.randn(B, T, 48, generator=torch.Generator().manual_seed(seed)).to(device).to(dtype)


def oracle(layer, x, positions):
    """The layer's formulas in 64 bits."""
    w = lambda p: p.detach().double().cpu()  # noqa: E731
    B, T, _ = x.shape
    H, K = layer.num_heads, layer.taps
    mixed, z, b, g = torch.split(w(x) @ w(layer.in_proj.weight).t(), [sum(layer._mixed), H * layer.value_dim, H, H], dim=-1)
    wide = torch.cat([torch.zeros(B, K - 1, mixed.shape[-1], dtype=torch.float64), mixed], 1)
    mixed = F.silu(sum(wide[:, j:j + T] * w(layer.conv_weight)[:, j] for j in range(K)))
    q, k, v = torch.split(mixed, layer._mixed, dim=-1)
    heads = lambda t, d: t.unflatten(-1, (-1, d))  # noqa: E731
    q, k, v = heads(q, layer.key_dim), heads(k, layer.key_dim), heads(v, layer.value_dim)
    if layer.rotary_sections:
        q, k = (axes64(t, positions.cpu(), layer.angles, layer.rotary_sections, layer.layout) for t in (q, k))
    r = delta64(q, k, v, -F.softplus(g + w(layer.bias_gamma)), torch.sigmoid(b), layer.key_dim ** -0.5, normalize=True)
    o = group_norm64(r["o"][0].flatten(0, 1).flatten(1), H, w(layer.norm_weight), w(layer.norm_bias), layer.eps, "silu",
                     z.flatten(0, 1))
    return o.reshape(B, T, -1) @ w(layer.out_proj.weight).t(), (wide[:, T:], r["state"][0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 7, 150])
@pytest.mark.parametrize("kw", [{}, dict(rotary_sections=(), key_heads=4, taps=1), dict(layout="interleaved", key_heads=1, taps=3)])
def test_forward(device, dtype, T, kw):
    layer = make(device, dtype, **kw)
    x, positions = tokens(2, T, 1, device, dtype), grid_positions(6, 5, 5, device=device)[:T]
    with torch.no_grad():
        y, (before, S) = layer(x, positions=positions, output_state=True)
        want, (want_before, want_S) = oracle(layer, x, positions)
        assert y.dtype == before.dtype == dtype and S.dtype == torch.float32 and layer.angles.dtype == torch.float32
        assert float((y.double().cpu() - want).abs().max()) < TOL[dtype]
        assert float((S.double().cpu() - want_S).abs().max()) < TOL[dtype] * (1 + float(want_S.abs().max()))
        if layer.taps > 1:
            assert float((before.double().cpu() - want_before).abs().max()) < TOL[dtype]
        assert torch.equal(layer(x, positions=positions), y)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_steps(device, dtype):
    """Prompts of two lengths, in one and in two pieces, then tokens one by one with the states in a pool: what the whole
    sequences give."""
    layer = make(device, dtype)
    x, positions = tokens(2, 30, 2, device, dtype), grid_positions(2, 3, 5, device=device)
    with torch.no_grad():
        whole = layer(x, positions=positions)
        pool, slots = layer.new_state(5), torch.tensor([3, -1, 1], dtype=torch.int32, device=device)
        length = [20, 11]
        for b, at in enumerate((3, 1)):
            _, state = layer(x[b:b + 1, :7], positions=positions[:7], output_state=True)
            _, state = layer(x[b:b + 1, 7:length[b]], state, positions[7:length[b]], output_state=True)
            for mine, one in zip(pool, state):
                mine[at] = one[0]
        for i in range(8):
            now = torch.stack([x[0, 20 + i], x[0, 0], x[1, 11 + i]])
            y = layer.step(now, pool, positions[[20 + i, 0, 11 + i]], slots)
            for row, (b, t) in ((0, (0, 20 + i)), (2, (1, 11 + i))):
                assert float((y[row] - whole[b, t]).abs().max()) < 2 * TOL[dtype]
        assert not any(mine[[0, 2, 4]].any() for mine in pool)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients(device):
    """Beside linear attention: gradients reach every parameter, and are those of differences along a direction."""
    torch.manual_seed(5)
    mixer, other = make(device, torch.float32), LinearAttentionLayer(48, 4, 16, 24).to(device)
    x, positions = tokens(2, 70, 4, device, torch.float32), grid_positions(4, 4, 5, device=device)[:70]
    params = [*mixer.parameters(), *other.parameters()]

    def loss():
        h = x + mixer(x, positions=positions)
        return (h + other(h)).square().mean()

    grads = torch.autograd.grad(loss(), params)
    assert all(g.isfinite().all() and g.abs().max() > 0 for g in grads)
    norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    h = 2.0 ** -6  # along the gradient, of all parameters together: of unit length
    with torch.no_grad():
        for p, g in zip(params, grads):
            p += g * (h / norm)
        up = float(loss().double())
        for p, g in zip(params, grads):
            p -= g * (2 * h / norm)
        down = float(loss().double())
    # a loss of about 2 in 32 bits, over 2 h: 2^-23 / 2^-5; third derivatives of at most 100 norms: 100 h^2 / 6
    assert abs((up - down) / (2 * h) - norm) <= 64 * 2.0 ** -18 + norm * 100 * h * h / 6


@pytest.mark.gpu
def test_same_on_both_devices():
    layer = make("cpu", torch.float32)
    x, positions = tokens(2, 100, 6, "cpu", torch.float32), grid_positions(4, 5, 5)
    a = x.clone().requires_grad_()
    y = layer(a, positions=positions)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(7))
    want = torch.autograd.grad(y, [a, *layer.parameters()], dy)
    layer = layer.cuda()
    b = x.cuda().requires_grad_()
    z = layer(b, positions=positions.cuda())
    assert torch.allclose(z.cpu(), y, atol=1e-4)
    for g, e in zip(torch.autograd.grad(z, [b, *layer.parameters()], dy.cuda()), want):
        assert float((g.cpu() - e).abs().max()) < 1e-4 * (1 + float(e.abs().max()))


@pytest.mark.gpu
def test_step_in_a_graph():
    """A captured step replayed several times, with eager work between the replays, gives the eager steps bit for bit."""
    layer = make("cuda", torch.bfloat16)
    pool, eager = layer.new_state(3), layer.new_state(3)
    x, pos = torch.randn(3, 48, device="cuda").bfloat16(), torch.zeros(3, 3, dtype=torch.int64, device="cuda")
    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, pool, pos, slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.step(x, pool, pos, slots)
    for s in pool:
        s.zero_()
    for i in range(4):
        x.copy_(torch.randn(3, 48, generator=torch.Generator().manual_seed(i)))
        pos.fill_(i)
        graph.replay()
        want = layer.step(x, eager, pos, slots)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(pool, eager))


def test_angles_and_refusals():
    layer = make("cpu", torch.bfloat16)
    assert layer.angles.dtype == torch.float32 and "angles" not in layer.state_dict()
    with torch.device("meta"):
        empty = DeltaRuleLayer(16, 2, 8, 8, rotary_sections=(1, 2))
    assert torch.equal(empty.to_empty(device="cpu").angles, DeltaRuleLayer(16, 2, 8, 8, rotary_sections=(1, 2)).angles)
    with pytest.raises(AssertionError):
        DeltaRuleLayer(16, 4, key_heads=3)
    with pytest.raises(ValueError):
        layer(torch.zeros(1, 5, 48).bfloat16())
    with pytest.raises(ValueError):
        DeltaRuleLayer(16, 2, 8, 8, taps=9)(torch.zeros(1, 5, 16))


def apart(got, want):
    """The distance's part of the norm."""
    return float((got.detach().double().cpu() - want).norm() / want.norm())


@pytest.mark.parametrize("device", DEVICES)
def test_autocast(device):
    """32-bit weights under autocast: prompts in pieces behind a new state and tokens one by one, the states in the weights' type,
    as without autocast but for the projections' rounding; a state from either side goes on at the other.

    Bound: as for a layer in 16 bits, eight roundings of 2^-8 (six stages, a key's roundings meet the state twice) of the norm."""
    layer = make(device, torch.float32)
    x, positions = tokens(2, 30, 2, device, torch.float32), grid_positions(2, 3, 5, device=device)
    cast = lambda: torch.autocast(device, dtype=torch.bfloat16)  # noqa: E731
    want, (want_before, want_S) = oracle(layer, x, positions)
    with torch.no_grad():
        state = layer.new_state(2)
        assert state[0].dtype == torch.float32
        with cast():
            whole = layer(x, positions=positions)
            y, state = layer(x[:, :20], state, positions[:20], output_state=True)
            assert whole.dtype == y.dtype == torch.bfloat16 and state[0].dtype == torch.float32
            got = [y]
            for t in range(20, 30):
                got.append(layer.step(x[:, t], state, positions[t].expand(2, 3))[:, None])
        got = torch.cat(got, 1)
        assert got.dtype == torch.bfloat16
        for mine, ref in ((whole, want), (got, want), (state[0], want_before), (state[1], want_S)):
            assert apart(mine, ref) <= 8 * 2.0 ** -8
        with cast():  # a state of a prompt without one has the projection's type
            _, state = layer(x[:, :20], positions=positions[:20], output_state=True)
            assert state[0].dtype == torch.bfloat16
            y, _ = layer(x[:, 20:], state, positions[20:], output_state=True)
        assert apart(y, want[:, 20:]) <= 8 * 2.0 ** -8
        y, after = layer(x[:, 20:], state, positions[20:], output_state=True)  # goes on in 32 bits
        assert y.dtype == after[0].dtype == torch.float32 and apart(y, want[:, 20:]) <= 8 * 2.0 ** -8
        with pytest.raises(ValueError):  # in place it cannot hold what comes
            layer.step(x[:, 20], state, positions[20].expand(2, 3))
    with cast():
        loss = layer(x, layer.new_state(2), positions).float().square().sum()
    for p, g in zip(layer.parameters(), torch.autograd.grad(loss, list(layer.parameters()))):
        assert g.dtype == p.dtype and g.isfinite().all() and g.any()


@pytest.mark.parametrize("device", DEVICES)
def test_wider_state(device):
    """A layer in 16 bits with its convolution's state in 32: the same bits as with a state in 16, which hold its inputs exactly."""
    layer = make(device, torch.bfloat16)
    x, positions = tokens(2, 12, 2, device, torch.bfloat16), grid_positions(2, 2, 3, device=device)
    with torch.no_grad():
        narrow, wide = layer.new_state(2), tuple(s.float() for s in layer.new_state(2))
        a, narrow = layer(x[:, :9], narrow, positions[:9], output_state=True)
        b, wide = layer(x[:, :9], wide, positions[:9], output_state=True)
        assert narrow[0].dtype == torch.bfloat16 and wide[0].dtype == torch.float32
        for t in range(9, 12):
            at = positions[t].expand(2, 3)
            a, b = (torch.cat([y, layer.step(x[:, t], s, at)[:, None]], 1) for y, s in ((a, narrow), (b, wide)))
        assert torch.equal(a, b) and torch.equal(narrow[0].float(), wide[0]) and torch.equal(narrow[1], wide[1])


# Parts of the norm: in 16 bits eight roundings of 2^-8 (six stages; a key's meets the state twice), in 32 bits eight stages of
# some 160 EPS, as for the mixer alone
PART = {torch.float32: 8 * 160 * 2.0 ** -24, torch.bfloat16: 8 * 2.0 ** -8}
KINDS = [{}, dict(rotary_sections=(), key_heads=4, taps=1), dict(layout="interleaved", key_heads=1, taps=3)]


def places(T, device):
    """Far from each other on every axis, so that turns matter between any two tokens."""
    return torch.randint(0, 64, (T, 3), generator=torch.Generator().manual_seed(8)).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 7, 60])
@pytest.mark.parametrize("kw", KINDS)
def test_by_the_norm(device, dtype, T, kw):
    """Outputs and states by the size that they have: whole sequences, and the last five tokens one by one behind a prompt."""
    layer = make(device, dtype, **kw)
    x, positions, first = tokens(2, T, 1, device, dtype), places(T, device), max(T - 5, 0)
    want, (want_before, want_S) = oracle(layer, x, positions)
    with torch.no_grad():
        y, state = layer(x, positions=positions, output_state=True)
        part, pool = layer(x[:, :first], layer.new_state(2), positions[:first], output_state=True)
        rows = [part, *(layer.step(x[:, t], pool, positions[t].expand(2, 3))[:, None] for t in range(first, T))]
    for got, (before, S) in ((y, state), (torch.cat(rows, 1), pool)):
        assert apart(got, want) <= PART[dtype] and apart(S, want_S) <= PART[dtype]
        assert layer.taps == 1 or apart(before, want_before) <= PART[dtype]


@pytest.mark.parametrize("T", [7, 60])
@pytest.mark.parametrize("kw", KINDS)
def test_mistakes_are_seen(monkeypatch, T, kw):
    """Formulas without the turns, the decays, the strengths or the keys' lengths are further off than the bounds in 16 bits."""
    layer, positions = make("cpu", torch.bfloat16, **kw), places(T, "cpu")
    x = tokens(2, T, 1, "cpu", torch.bfloat16)
    want, (_, want_S) = oracle(layer, x, positions)
    plain = delta64
    mistakes = {"decays": lambda q, k, v, g, b, *a, **kw: plain(q, k, v, 0 * g, b, *a, **kw),
                "strengths": lambda q, k, v, g, b, *a, **kw: plain(q, k, v, g, 0 * b + 1, *a, **kw),
                "lengths": lambda *a, normalize: plain(*a)}
    for form in mistakes.values():
        with monkeypatch.context() as m:
            m.setattr(sys.modules[__name__], "delta64", form)
            got, (_, S) = oracle(layer, x, positions)
        assert apart(got, want) > 2 * PART[torch.bfloat16] and apart(S, want_S) > 2 * PART[torch.bfloat16]
    if layer.rotary_sections:
        with monkeypatch.context() as m:
            m.setattr(sys.modules[__name__], "axes64", lambda t, *a: t.double())
            got, (_, S) = oracle(layer, x, positions)
        assert apart(got, want) > 2 * PART[torch.bfloat16] and apart(S, want_S) > 2 * PART[torch.bfloat16]
