"""What the entry points of ``ttc.ops`` share: what a call copies for its kernel lives until the kernel has been enqueued."""
import importlib
import weakref

import pytest
import torch

from ttc.ops import rotary_table


def skewed(*shape):
    """A tensor whose rows are not of unit stride."""
    return torch.randn(*shape[:-1], 2 * shape[-1])[..., ::2]


def conv(m):
    m._forward(skewed(2, 5, 8), torch.randn(8, 4), None, "silu", None, True)


def conv_backward(m):
    x = skewed(2, 5, 8)
    state = torch.randn(2, 8, 3).transpose(1, 2)

    class Left:  # what the forward leaves
        saved_tensors, needs_input_grad, activation = (x, torch.randn(8, 4), None, state), (True, True, False, True, False, False), "silu"

    m._CausalConvFunc.backward(Left, skewed(2, 5, 8), torch.randn(2, 8, 3).transpose(1, 2))


def qkv():
    return skewed(1, 70, 2, 8), skewed(1, 70, 2, 8), skewed(1, 70, 2, 8), -torch.rand(1, 70, 2)


def delta(m):
    q, k, v, g = qkv()
    m._forward(q, k, v, g, torch.rand(1, 70, 2), 1.0, False, 0.0, None, True, True)


def delta_backward(m):
    q, k, v, g = qkv()

    class Left:
        saved_tensors = (q, k, v, g, torch.rand(1, 70, 2), None, torch.empty(1 << 20, dtype=torch.uint8))
        needs_input_grad, args = (True,) * 5 + (False,) * 5, (1.0, False, 0.0)

    m._DeltaRuleFunc.backward(Left, skewed(1, 70, 2, 8), torch.randn(1, 2, 8, 8).transpose(2, 3))


def linear(m):
    m._forward(*qkv(), 1.0, None, True, True)


def linear_backward(m):
    class Left:
        saved_tensors, needs_input_grad, scale = (*qkv(), None, None), (True,) * 4 + (False,) * 3, 1.0

    m._LinearAttentionFunc.backward(Left, skewed(1, 70, 2, 8), torch.randn(1, 2, 8, 8).transpose(2, 3))


def turn(m):
    m._launch((skewed(1, 9, 2, 8), skewed(1, 9, 2, 8)), rotary_table(16, 8), None, 0, "half", 0)


def turn_axes(m):
    m._launch_axes((skewed(1, 9, 2, 8), skewed(1, 9, 2, 8)), rotary_table(16, 8), torch.zeros(9, 2, dtype=torch.long), (1, 3), "half", 0)


@pytest.mark.parametrize("name,work,copies", [
    ("causal_conv", conv, 1), ("causal_conv", conv_backward, 4), ("delta_rule", delta, 3), ("delta_rule", delta_backward, 5),
    ("linear_attention", linear, 3), ("linear_attention", linear_backward, 5), ("rotary", turn, 2), ("rotary", turn_axes, 2)])
def test_copies_live_until_the_launch(monkeypatch, name, work, copies):
    """The block holds addresses only: a copy that is dropped before the launch can be handed to someone else first."""
    made, launches = [], []
    contiguous = torch.Tensor.contiguous

    def copy(x, *args, **kw):
        y = contiguous(x, *args, **kw)
        if y is not x and y.data_ptr() != x.data_ptr():
            made.append(weakref.ref(y))
        return y

    def launch(fn, what, block, device):
        launches.append(what)
        assert len(made) == copies and all(ref() is not None for ref in made), [ref() is not None for ref in made]

    module = importlib.import_module(f"ttc.ops.{name}")
    monkeypatch.setattr(torch.Tensor, "contiguous", copy)
    monkeypatch.setattr(module, "launch", launch)
    with torch.no_grad():
        work(module)
    assert len(launches) == 1
