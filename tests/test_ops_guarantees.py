"""What the sequence operators (``ttc.ops``) promise beyond their formulas: how often a value is rounded, what masked places
can reach, whose derivative a gradient is, and which calls are taken at all.  Tolerances stand at each test."""
import math

import pytest
import torch

from _ops_oracle import EPS, HALF, linear64, within
from test_ops_linear_attention import DEVICES, grads, inputs, magnitudes, make, roundings
from ttc.ops import linear_attention, linear_attention_step


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
