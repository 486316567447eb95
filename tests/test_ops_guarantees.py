"""What the sequence operators (``ttc.ops``) promise beyond their formulas: how often a value is rounded, what masked places
can reach, whose derivative a gradient is, and which calls are taken at all.  Tolerances stand at each test."""
import math

import pytest
import torch

from _ops_oracle import EPS, HALF, linear64, within
from test_ops_linear_attention import DEVICES, grads, inputs, magnitudes, make, roundings
from ttc import LinearAttentionLayer
from ttc.layers.front_end import front_end, front_end_torch
from ttc.ops import group_norm, linear_attention, linear_attention_step, rotary, rotary_table
from ttc.ops._call import recorded_backward
from ttc.ops.group_norm import group_norm_torch
from ttc.ops.linear_attention import linear_attention_torch


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", [(2, 200, 2, 2, 2, 2, 64, 64), (1, 150, 2, 2, 1, 1, 128, 128), (2, 130, 3, 3, 3, 1, 32, 20),
                                  (1, 700, 1, 1, 1, 1, 128, 33), (2, 3, 2, 2, 2, 2, 16, 40)])
def test_outputs_in_16_bits_are_rounded_once(device, case):
    """Scores and states keep 16 digits or more on the way (the first 8 of a value, then 8 of the rest, which is below 2^-7
    of it: 2^-15 for each term), and the output, a gradient of a head that is not shared included, is rounded once."""
    x = inputs(*case, torch.bfloat16, device, True)
    B, T, H, dk, dv = case[0], case[1], case[2], case[6], case[7]
    d_o, d_state = make((B, T, H, dv), torch.bfloat16, device, 9), make((B, H, dk, dv), torch.float32, device, 10)
    got = grads(x, d_o, d_state, 0.4)
    got["o"] = linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.4, initial_state=x["state"])
    want = linear64(x["q"], x["k"], x["v"], x["g"], 0.4, x["state"], d_o, d_state)
    size = magnitudes(x, 0.4, d_o, d_state)
    for name in ("o", "q", "k", "v"):
        once = HALF[torch.bfloat16] * 1.01 * want[name].abs()
        within(got[name], want[name], once + size[name] * (roundings(x, T) * EPS + 2.0 ** -15) + 1e-30)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("slots", [False, True])
def test_a_state_that_a_backward_needs_is_not_overwritten_unnoticed(device, slots):
    x = inputs(2, 20, 2, 2, 2, 2, 16, 24, torch.float32, device, True)
    index = torch.tensor([1, 0], dtype=torch.int32, device=device) if slots else None
    q = x["q"].clone().requires_grad_()
    o = linear_attention(q, x["k"], x["v"], x["g"], initial_state=x["state"])
    before = x["state"]._version
    linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["g"][:, 0], x["state"], slots=index)
    assert x["state"]._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.sum(), q)
    with torch.inference_mode():  # where tensors have no versions
        state = x["state"].clone()
        linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["g"][:, 0], state, slots=index)
    assert not torch.equal(state, x["state"])


def from_token(t, got, x, scale, d_o, d_state):
    """Outputs and gradients of tokens t on, and the final state, are those of the recurrence."""
    o, final = linear_attention(x["q"], x["k"], x["v"], x["g"], scale=scale, initial_state=x["state"], output_state=True)
    want = linear64(x["q"], x["k"], x["v"], x["g"], scale, x["state"], d_o, d_state)
    size, n, dt = magnitudes(x, scale, d_o, d_state), roundings(x, o.shape[1]) * EPS, o.dtype
    near = n + (2.0 ** -15 if dt != torch.float32 else 0)
    within(final, want["state"], size["state"] * n + 1e-30)
    for name, out in (("o", o), ("q", got["q"]), ("k", got["k"]), ("v", got["v"])):
        within(out[:, t:], want[name][:, t:], HALF[dt] * 1.01 * want[name][:, t:].abs() + size[name][:, t:] * near + 1e-30)
    d = (x["q"].detach().double().cpu().abs() * size["q"]).sum(-1) + (x["k"].detach().double().cpu().abs() * size["k"]).sum(-1)
    end = (size["state"] * d_state.detach().double().cpu().abs()).sum((-1, -2))[:, None]
    within(got["g"][:, t:], want["g"][:, t:], (d.flip(1).cumsum(1).flip(1) + end)[:, t:] * n + EPS * want["g"][:, t:].abs())


@pytest.mark.parametrize("device", DEVICES[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [100.0, math.inf, math.nan])
def test_a_reset_behind_decays_that_overflow(device, dtype, value):
    """In the next chunk (32 tokens in 32 bits, 64 in 16) of the same part of a long input, which has two chunks here: nothing
    of what came before is left."""
    C = 64 if dtype == torch.bfloat16 else 32
    x = inputs(1, 512, 2, 2, 2, 2, 32, 48, dtype, device, True)
    x["g"][:, C // 2, 0], reset = value, C + C // 2
    x["g"][:, reset, 0] = -math.inf
    d_o = make((1, 512, 2, 48), dtype, device, 9)
    d_o[:, :reset, 0] = 0
    d_state = make((1, 2, 32, 48), torch.float32, device, 10)
    from_token(reset, grads(x, d_o, d_state, 0.3), x, 0.3, d_o, d_state)


@pytest.mark.parametrize("device", DEVICES[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [4, 64, 200])
def test_a_reset_just_below_the_limit(device, dtype, T):
    """-105 drops the state as -inf does, where later tokens grow by more than it took away too."""
    x = inputs(1, T, 2, 2, 2, 2, 32, 48, dtype, device, True)
    x["g"][:, 2, 0] = -105.0
    x["g"][:, 3:20, 0] = 3.0 if T > 4 else 40.0
    x["k"][:, 2:20, 0] = 0  # so that nothing but what leaks is left in the state
    x["state"] *= 1e30
    d_o, d_state = make((1, T, 2, 48), dtype, device, 9), make((1, 2, 32, 48), torch.float32, device, 10)
    got = grads(x, d_o, d_state, 0.3)
    from_token(0, got, x, 0.3, d_o, d_state)
    cut = dict(x, g=x["g"].clone())
    cut["g"][:, 2, 0] = -math.inf
    for name, d in grads(cut, d_o, d_state, 0.3).items():
        assert torch.equal(d, got[name]), name


def with_lost_token(T, bad, reset, dtype, device, value, parts):
    """Inputs of which one token is lost (all of `parts` not finite, in the first head) and a later one resets."""
    x = inputs(1, T, 2, 2, 2, 2, 32, 48, dtype, device, True)
    for name in parts:
        x[name][0, bad, 0] = value
    x["g"][0, reset, 0] = -math.inf
    d_o, d_state = make((1, T, 2, 48), dtype, device, 9), make((1, 2, 32, 48), torch.float32, device, 10)
    d_o[:, :reset, 0] = 0
    return x, d_o, d_state


@pytest.mark.parametrize("device", DEVICES[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,bad,reset", [(4, 1, 2), (12, 3, 4), (64, 20, 29), (200, 70, 90), (130, 128, 129)])
@pytest.mark.parametrize("value,parts", [(math.nan, "g"), (math.inf, "g"), (math.nan, "qkvg")])
def test_a_lost_token_stays_in_its_text(device, dtype, T, bad, reset, value, parts):
    """A decay that is not finite has no effect past a reset, in one chunk too; nor has a token that is NaN altogether."""
    x, d_o, d_state = with_lost_token(T, bad, reset, dtype, device, value, parts)
    o = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["state"])
    assert not torch.isfinite(o[0, bad, 0]).all() and torch.isfinite(o[0, :bad]).all() and torch.isfinite(o[0, :, 1]).all()
    from_token(reset, grads(x, d_o, d_state, 0.3), x, 0.3, d_o, d_state)


class Recorded(torch.autograd.Function):
    """A form whose backward is recorded_backward, as that of the kernels' Functions where it is itself recorded."""

    @staticmethod
    def forward(ctx, form, *xs):
        ctx.form = form
        ctx.save_for_backward(*xs)
        return form(*xs)

    @staticmethod
    def backward(ctx, *grads):
        return (None, *recorded_backward(ctx.form, ctx.saved_tensors, ctx.needs_input_grad[1:], grads,
                                         torch.is_grad_enabled()))


def related(name, x, w):
    """An operator's inputs that are computed from one another."""
    if name == "norm":  # the gate from what is normalised, the weights from a mean of it
        return x, x.mean((0, 1)), x.sum((0, 1)) * 0.1, x @ w
    heads = lambda t: t.unflatten(-1, (2, 8))  # noqa: E731
    if name == "same":  # queries and keys are one tensor, values and decays functions of it
        q = heads(x)
        return q, q, torch.tanh(heads(x @ w)), -torch.sigmoid(x[..., :2]), None
    q = heads(x @ w)
    return q, torch.tanh(q), q * q, -torch.sigmoid(q[..., 0]), q.mean(1).unsqueeze(-1) * q.mean(1).unsqueeze(-2)


FORMS = {"norm": (lambda x, w, b, g: group_norm(x, 2, w, b, activation="silu", gate=g),
                  lambda x, w, b, g: group_norm_torch(x, 2, w, b, activation="silu", gate=g))}
FORMS["same"] = FORMS["chain"] = (lambda q, k, v, g, s: linear_attention(q, k, v, g, scale=0.3, initial_state=s),
                                  lambda q, k, v, g, s: linear_attention_torch(q, k, v, g, 0.3, s)[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["norm", "same", "chain"])
def test_recorded_gradients_are_partial(device, name):
    """An input's gradient leaves out what reaches the output through other inputs, with create_graph too: first and second
    derivatives are those of the torch operators.  Both are 32-bit sums of at most 20 x 16 terms over three stages with slopes
    below 8: 2^10 EPS of the largest value."""
    x = make((2, 20, 16), torch.float32, device, 30)
    w = make((16, 16), torch.float32, device, 31, 0.25)
    op, form = FORMS[name]

    def derivatives(f):
        leaf = x.clone().requires_grad_()
        first, = torch.autograd.grad(f(*related(name, leaf, w)).sin().sum(), leaf, create_graph=True)
        return first.detach(), torch.autograd.grad(first.sin().sum(), leaf)[0]

    want = derivatives(form)
    for f in (op, lambda *xs: Recorded.apply(form, *xs)):
        for d, e in zip(derivatives(f), want):
            assert float((d - e).abs().max()) <= 2 ** 10 * EPS * max(1.0, float(e.abs().max()))


@pytest.mark.gpu
def test_recorded_gradients_of_the_front_end_are_partial():
    """The bias computed from the projection: the kernel's first derivatives under create_graph and the second ones against
    the operators', both 32-bit sums of at most 80 terms with slopes below 8: 2^10 EPS of the largest."""
    dims = (2, 6, 5, 3, 4)
    x = make((3, 73), torch.float32, "cuda", 40)

    def derivatives(f):
        leaf = x.clone().requires_grad_()
        y = f(leaf, leaf.mean(0)[:12] - 1.0, dims)
        first, = torch.autograd.grad(sum(t.sin().sum() for t in y), leaf, create_graph=True)
        return first.detach(), torch.autograd.grad(first.sin().sum(), leaf)[0]

    for d, e in zip(derivatives(front_end), derivatives(front_end_torch)):
        assert float((d - e).abs().max()) <= 2 ** 10 * EPS * max(1.0, float(e.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,bad,reset", [(10, 5, 6), (64, 20, 29), (200, 70, 90), (130, 128, 129)])
@pytest.mark.parametrize("value,parts", [(math.nan, "v"), (math.inf, "k"), (math.nan, "q"), (math.nan, "g"), (math.inf, "g"),
                                         (math.nan, "qkvg"), (100.0, "g")])
def test_torch_form_drops_what_is_masked(dtype, T, bad, reset, value, parts):
    """The CPU's form as the kernels: no effect on earlier tokens, on other heads or past a reset, outputs or gradients."""
    x, d_o, d_state = with_lost_token(T, bad, reset, dtype, "cpu", value, parts)
    o = linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.3, initial_state=x["state"])
    clean = linear64(x["q"][:, :bad], x["k"][:, :bad], x["v"][:, :bad], x["g"][:, :bad], 0.3, x["state"])["o"]
    early = {n: x[n][:, :bad] for n in "qkvg"} | {"state": x["state"]}
    size = magnitudes(early, 0.3)["o"]
    within(o[:, :bad], clean, HALF[dtype] * 1.01 * clean.abs() + size * roundings(x, T) * EPS + 1e-30)
    assert torch.isfinite(o[:, :, 1]).all() and (value == 100.0 or not torch.isfinite(o[0, bad, 0]).all())
    from_token(reset, grads(x, d_o, d_state, 0.3), x, 0.3, d_o, d_state)


def test_torch_form_drops_a_state_that_is_not_finite():
    x, d_o, d_state = with_lost_token(70, 3, 5, torch.float32, "cpu", 0.0, "v")
    x["state"][0, 0, 3, 4] = math.nan
    from_token(5, grads(x, d_o, d_state, 0.3), x, 0.3, d_o, d_state)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("observed", [False, True])
def test_autocast_does_not_narrow_the_arithmetic(device, observed):
    """32-bit inputs have 32-bit results under autocast as outside of it, in the kernels' form and the operators'."""
    x = inputs(1, 90, 2, 2, 2, 2, 32, 48, torch.float32, device, True)
    run = lambda s: linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.3, initial_state=s, output_state=True)  # noqa: E731
    with torch.autocast(device, torch.bfloat16):
        o, final = torch.func.vmap(run)(x["state"][None]) if observed else run(x["state"])
    o, final = (o[0], final[0]) if observed else (o, final)
    want, size = linear64(x["q"], x["k"], x["v"], x["g"], 0.3, x["state"]), magnitudes(x, 0.3)
    assert o.dtype == final.dtype == torch.float32
    within(o, want["o"], size["o"] * roundings(x, 90) * EPS)
    within(final, want["state"], size["state"] * roundings(x, 90) * EPS)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("narrow", [False, True])
def test_compiles_as_one_graph(device, narrow):
    """Operators and their order are those of the torch form: 4 EPS of the largest value."""
    x = inputs(1, 20, 2, 2, 2, 2, 8, 8, torch.float32, device, True)
    f = lambda q, s: linear_attention(q, x["k"], x["v"], x["g"], scale=0.3, initial_state=s)  # noqa: E731
    want = linear_attention_torch(x["q"], x["k"], x["v"], x["g"], 0.3, x["state"])[0]
    with torch.autocast(device, torch.bfloat16, enabled=narrow):
        got = torch.compile(f, fullgraph=True, backend="eager")(x["q"], x["state"])
    assert float((got - want).abs().max()) <= 4 * EPS * float(want.abs().max())


@pytest.mark.parametrize("device", DEVICES)
def test_a_layer_without_positions_has_no_longest_input(device):
    """One call on 9 tokens against two on 5 and 4 and against single steps; some hundred 32-bit terms of about 1: 1e-5."""
    torch.manual_seed(3)
    layer = LinearAttentionLayer(16, 2, 8, 8, rotary_dim=0, max_positions=4).to(device)
    x = make((1, 9, 16), torch.float32, device, 50)
    with torch.no_grad():
        y, state = layer(x, output_state=True)
        first, S = layer(x[:, :5], output_state=True)
        rest, S2 = layer(x[:, 5:], S, offset=5, output_state=True)
        steps = torch.cat([layer.step(x[:, t], S, torch.tensor([t], device=device)) for t in range(5, 9)])
    assert float((torch.cat([first, rest], 1) - y).abs().max()) < 1e-5 and float((S2 - state).abs().max()) < 1e-5
    assert float((steps - y[0, 5:]).abs().max()) < 1e-5 and float((S - state).abs().max()) < 1e-5


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_a_table_that_is_learnt_has_a_gradient(device, layout):
    """d cos = sum (x_a d_a + x_b d_b), d sin = sum (x_a d_b - x_b d_a) over the 2 x 3 heads at a position: 12 products and
    their sums of values below 5, 32 EPS x 25 x 12."""
    q, k = make((2, 6, 2, 8), torch.float32, device, 60), make((2, 6, 1, 8), torch.float32, device, 61)
    dq, dk = make(q.shape, torch.float32, device, 62), make(k.shape, torch.float32, device, 63)
    table = rotary_table(9, 6, device=device).requires_grad_()
    got, = torch.autograd.grad(rotary(q, k, table, offset=2, layout=layout), table, (dq, dk))
    want = torch.zeros(9, 3, 2, dtype=torch.float64)
    for x, d in ((q, dq), (k, dk)):
        x, d = x.double().cpu()[..., :6], d.double().cpu()[..., :6]
        a, b = (slice(0, 3), slice(3, 6)) if layout == "half" else (slice(0, 6, 2), slice(1, 6, 2))
        want[2:8, :, 0] += (x[..., a] * d[..., a] + x[..., b] * d[..., b]).sum((0, 2))
        want[2:8, :, 1] += (x[..., a] * d[..., b] - x[..., b] * d[..., a]).sum((0, 2))
    within(got, want, torch.tensor(32 * EPS * 25 * 12))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("where", ["meta", "cpu"])
def test_a_layer_without_storage_gets_its_angles(device, where):
    """Made on the meta device or emptied, then filled from a checkpoint, which holds no angles."""
    args = dict(dim=16, num_heads=2, key_dim=8, value_dim=8, max_positions=64, rotary=dict(scaling="linear", factor=2.0))
    torch.manual_seed(3)
    layer = LinearAttentionLayer(**args)
    with torch.device(where):
        other = LinearAttentionLayer(**args)
    other = other.to_empty(device=device)
    other.load_state_dict(layer.state_dict())
    assert other.angles.device.type == device and torch.equal(other.angles.cpu(), layer.angles)
    x = make((1, 5, 16), torch.float32, device, 51)
    assert torch.equal(other(x), layer.to(device)(x))
    assert torch.equal(other.bfloat16().angles, layer.angles) and other.to("meta").angles.is_meta


@pytest.mark.gpu
def test_more_heads_than_one_launch_holds():
    """2^26 and 2^24 (sequence, head) pairs and more, one by one and in chunks: what the pieces of the batch give, bit for bit."""
    B, H = 2 ** 13, 2 ** 13 + 1
    q, k, v, d_o = (make((B, 1, 1, 1), torch.bfloat16, "cuda", 70 + i) * make((1, 1, H, 1), torch.bfloat16, "cuda", 75 + i)
                    for i in range(4))
    g = -torch.rand(1, 1, H, device="cuda").expand(B, 1, H).contiguous()

    def run(rows):
        leaves = [t[rows].detach().requires_grad_() for t in (q, k, v, g)]
        o = linear_attention(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, d_o[rows]))

    whole = run(slice(None))
    for at in range(0, B, 1024):
        for a, b in zip(whole, run(slice(at, at + 1024))):
            assert torch.equal(a[at:at + 1024], b)
    del whole, q, k, v, d_o, g
    B, H = 2 ** 12 + 1, 2 ** 12
    q, k, v = (make((B, 5, 1, d), torch.bfloat16, "cuda", 80 + d) for d in (8, 8, 33))
    g = -torch.rand(H, device="cuda")
    whole = linear_attention(q, k, v, g)
    for at in range(0, B, 512):
        assert torch.equal(whole[at:at + 512], linear_attention(*(t[at:at + 512] for t in (q, k, v)), g))


@pytest.mark.gpu
def test_rows_of_2_31_elements():
    """2^24 heads of 128, the most there are: all have the decay of the first one, and so its outputs."""
    H = 2 ** 24
    q, k, v = (make((1, 5, 1, d), torch.bfloat16, "cuda", 90 + i) for i, d in enumerate((8, 8, 128)))
    o = linear_attention(q, k, v, torch.full((1,), -0.3, device="cuda").expand(H))
    want = linear_attention(q, k, v, torch.full((1,), -0.3, device="cuda"))
    for t in range(5):
        assert bool((o[0, t] == want[0, t, 0]).all())
