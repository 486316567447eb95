"""``LinearAttentionLayer`` (``ttc.layers``): the sequence operators run together, beside ``TTCLayer``.

Tolerances: the layer's output is a sum of ``num_heads * value_dim`` products of normalised values of about 1 and weights
of a random initialisation, so of about 1; 32-bit rounding of some hundred products and sums per value stays below 1e-4 of
it.  In bfloat16 each of the five stages (projection, rotation, mixing, norm, projection) rounds once to 2^-8 a value, or
about 2 % of a value of 1 at the output: 0.06 absolute."""
import math

import pytest
import torch
import torch.nn.functional as F

from _ops_oracle import group_norm64, linear64, rotary64
from ttc import LinearAttentionLayer, TTCLayer

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TOL = {torch.float32: 1e-4, torch.bfloat16: 0.06}


def make(device, dtype, **kw):
    torch.manual_seed(3)
    args = dict(dim=48, num_heads=4, key_dim=16, value_dim=24, kv_heads=2, rotary_dim=8, max_positions=256)
    return LinearAttentionLayer(**(args | kw)).to(device).to(dtype)


def oracle(layer, x, state=None, offset=0):
    """The layer's formulas in 64 bits."""
    w = lambda p: p.detach().double().cpu()  # noqa: E731
    B, T, _ = x.shape
    q, k, v, z, g = torch.split(w(x) @ w(layer.in_proj.weight).t(), layer._split, dim=-1)
    heads = lambda t, d: t.unflatten(-1, (-1, d))  # noqa: E731
    at = (torch.arange(T) + offset)[None].expand(B, T).numpy()
    turn = lambda t: torch.from_numpy(rotary64(heads(t, layer.key_dim), at, layer.angles, layer.layout))  # noqa: E731
    r = linear64(turn(q), turn(k), heads(v, layer.value_dim), -F.softplus(g + w(layer.bias_gamma)), layer.key_dim ** -0.5,
                 state)
    o = group_norm64(r["o"].flatten(0, 1).flatten(1), layer.num_heads, w(layer.norm_weight), w(layer.norm_bias), layer.eps,
                     "silu", z.flatten(0, 1))
    return o.reshape(B, T, -1) @ w(layer.out_proj.weight).t(), r["state"]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 7, 150])
@pytest.mark.parametrize("kw", [{}, dict(layout="interleaved", kv_heads=4, rotary_dim=None), dict(rotary_dim=0, kv_heads=1)])
def test_forward(device, dtype, T, kw):
    layer = make(device, dtype, **kw)
    x = torch.randn(2, T, 48, generator=torch.Generator().manual_seed(1)).to(device).to(dtype)
    with torch.no_grad():
        y, state = layer(x, offset=5, output_state=True)
        want, want_state = oracle(layer, x, offset=5)
        assert y.dtype == dtype and layer.angles.dtype == torch.float32 and state.dtype == torch.float32
        assert float((y.double().cpu() - want).abs().max()) < TOL[dtype]
        assert float((state.double().cpu() - want_state).abs().max()) < TOL[dtype] * (1 + float(want_state.abs().max()))
        assert torch.equal(layer(x, offset=5), y)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_steps(device, dtype):
    """Prompts of two lengths, then tokens one by one with the states in a pool: what the whole sequences give."""
    layer = make(device, dtype)
    x = torch.randn(2, 30, 48, generator=torch.Generator().manual_seed(2)).to(device).to(dtype)
    with torch.no_grad():
        whole = layer(x)
        pool, slots = layer.new_state(5), torch.tensor([3, -1, 1], dtype=torch.int32, device=device)
        length = [20, 11]
        for b, at in enumerate((3, 1)):
            _, S = layer(x[b:b + 1, :length[b]], output_state=True)
            pool[at] = S[0]
        for i in range(8):
            now = torch.stack([x[0, 20 + i], x[0, 0], x[1, 11 + i]])
            y = layer.step(now, pool, torch.tensor([20 + i, 0, 11 + i], device=device), slots)
            for row, (b, t) in ((0, (0, 20 + i)), (2, (1, 11 + i))):
                assert float((y[row] - whole[b, t]).abs().max()) < 2 * TOL[dtype]
        assert not pool[[0, 2, 4]].any()


@pytest.mark.parametrize("device", DEVICES)
def test_training_beside_the_control_layer(device):
    """A block of both layers: gradients reach every parameter, and a descent step lowers the loss."""
    torch.manual_seed(5)
    mixer = make(device, torch.float32)
    control = TTCLayer(12, 12, 16, 4, 4, 4, solver_impl="hip" if device == "cuda" else "riccati").to(device)
    x = torch.randn(2, 16, 48, generator=torch.Generator().manual_seed(4)).to(device)

    def loss():
        h = x + mixer(x)
        h = h + control(h.unflatten(-1, (4, 12)), T=8).flatten(-2)
        return (h.roll(1, 1) - x).square().mean()
    params = [*mixer.parameters(), *control.parameters()]
    first = loss()
    grads = torch.autograd.grad(first, params)
    assert all(g.isfinite().all() and g.abs().max() > 0 for g in grads)
    norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
    with torch.no_grad():
        for p, g in zip(params, grads):
            p -= g * (0.05 / norm)
    assert float(loss()) < float(first)


@pytest.mark.gpu
def test_same_on_both_devices():
    layer = make("cpu", torch.float32)
    x = torch.randn(2, 100, 48, generator=torch.Generator().manual_seed(6))
    a = [x.clone().requires_grad_()]
    y = layer(*a)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(7))
    want = torch.autograd.grad(y, [*a, *layer.parameters()], dy)
    layer = layer.cuda()
    b = [x.cuda().requires_grad_()]
    z = layer(*b)
    assert torch.allclose(z.cpu(), y, atol=1e-4)
    for g, e in zip(torch.autograd.grad(z, [*b, *layer.parameters()], dy.cuda()), want):
        assert float((g.cpu() - e).abs().max()) < 1e-4 * (1 + float(e.abs().max()))


@pytest.mark.gpu
def test_step_in_a_graph():
    """A captured step replayed several times, with eager work between the replays, gives the eager steps bit for bit."""
    layer = make("cuda", torch.bfloat16)
    pool, eager = layer.new_state(3), layer.new_state(3)
    x, pos = torch.randn(3, 48, device="cuda").bfloat16(), torch.zeros(3, dtype=torch.int64, device="cuda")
    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, pool, pos, slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.step(x, pool, pos, slots)
    pool.zero_()
    for i in range(4):
        x.copy_(torch.randn(3, 48, generator=torch.Generator().manual_seed(i)))
        pos.fill_(i)
        graph.replay()
        want = layer.step(x, eager, pos, slots)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(pool, eager)


@pytest.mark.gpu
def test_on_another_stream():
    """Operators run on the current stream, forward and backward."""
    layer = make("cuda", torch.float32)
    x = torch.randn(2, 200, 48, device="cuda")
    leaf = x.clone().requires_grad_()
    want = layer(leaf)
    dwant, = torch.autograd.grad(want.sum(), leaf)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-2  # keeps the stream busy while the layer's launches queue up behind it
        leaf2 = (x + 0 * big[0, 0]).nan_to_num().detach().requires_grad_()
        y = layer(leaf2)
        dy, = torch.autograd.grad(y.sum(), leaf2)
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(dy, dwant)


def test_refusals():
    with pytest.raises(AssertionError):
        LinearAttentionLayer(16, 4, kv_heads=3)
    layer = LinearAttentionLayer(16, 2, 8, 8, max_positions=4)
    with pytest.raises(ValueError):
        layer(torch.zeros(1, 5, 16))
