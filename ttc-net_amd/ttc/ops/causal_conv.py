"""Causal convolution of each channel over a few tokens, with an activation: what stands in front of a token mixer whose
queries, keys and values are to see their nearest tokens.

    y_t = act(bias + sum_j weight[:, j] w_{t + j}),    w = the state's taps - 1 rows, then x

:func:`causal_conv` runs it over whole sequences (prompts, training), :func:`causal_conv_step` over one token of each
sequence of a serving batch, whose states (the last ``taps - 1`` inputs) it updates in place.  CUDA tensors go through the
kernels of ``ttc_causal_conv`` and ``ttc_causal_conv_step``; CPU tensors, and any call that something observes operator by
operator, run :func:`causal_conv_torch`.
"""
from __future__ import annotations

import struct

import torch

from .._dispatch import traced
from ..solvers._lib import lib
from ._call import DTYPES, check_device, check_types, launch, ptr, recorded_backward, unit_rows, with_spaces

__all__ = ["causal_conv", "causal_conv_step", "causal_conv_torch", "MAX_TAPS"]

MAX_TAPS = 8  # TTC_CAUSAL_CONV_MAX_TAPS
_ACTIVATIONS = {"none": 0, "silu": 1}
_BLOCK = struct.Struct("8qq2q3q2qq2qq4qqq")
_STEP_BLOCK = struct.Struct("7qqq2qqqq")


def causal_conv_torch(x, weight, bias=None, *, activation: str = "none", initial_state=None):
    """:func:`causal_conv` as torch operators: ``(y, final state)``."""
    B, T, C = x.shape
    K = weight.shape[1]
    front = x.new_zeros(B, K - 1, C) if initial_state is None else initial_state
    wide, w = torch.cat([front, x], 1).float(), weight.float()
    y = wide[:, :T] * w[:, 0]
    for j in range(1, K):
        y = y + wide[:, j:j + T] * w[:, j]
    if bias is not None:
        y = y + bias.float()
    if activation == "silu":
        y = y * torch.sigmoid(y)
    return y.to(x.dtype), wide[:, T:].to(x.dtype, copy=True).contiguous()  # exact, and its gradient is joined in 32 bits


def _block(x, weight, bias, activation, initial, y, final, backward=0, d_y=None, d_final=None, dx=None, dweight=None,
           dbias=None, d_initial=None):
    B, T, C = x.shape
    return _BLOCK.pack(DTYPES[x.dtype], DTYPES[weight.dtype], B, T, C, weight.shape[1], _ACTIVATIONS[activation], backward,
                       ptr(x), *x.stride()[:2], ptr(weight), ptr(bias), ptr(initial), ptr(y), ptr(final), ptr(d_y),
                       *((0, 0) if d_y is None else d_y.stride()[:2]), ptr(d_final), ptr(dx), ptr(dweight), ptr(dbias),
                       ptr(d_initial), 0, 0)


def _forward(x, weight, bias, activation, initial, want_state):
    B, T, C = x.shape
    y = x.new_empty((B, T, C))
    final = x.new_empty((B, weight.shape[1] - 1, C)) if want_state else None
    x = unit_rows(x)  # a copy lives until the launch
    launch(lib.ttc_causal_conv, "ttc_causal_conv", _block(x, weight, bias, activation, initial, y, final), x.device)
    return y, final


class _CausalConvFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, initial, activation, want_state):
        ctx.save_for_backward(x, weight, bias, initial)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return _forward(x, weight, bias, activation, None if initial is None else initial.contiguous(), want_state)

    @staticmethod
    def backward(ctx, d_y, d_final):
        x, weight, bias, initial = ctx.saved_tensors
        needs = ctx.needs_input_grad[:4]
        if d_y is None and d_final is None:
            return (None,) * 6
        recorded = torch.is_grad_enabled()
        if recorded or traced(d_y, d_final, x, weight, bias, initial):
            form = lambda x, w, b, s: causal_conv_torch(x, w, b, activation=ctx.activation, initial_state=s)  # noqa: E731
            return (*recorded_backward(form, (x, weight, bias, initial), needs, (d_y, d_final), recorded), None, None)
        if d_y is None:
            d_y = torch.zeros_like(x, memory_format=torch.contiguous_format)
        new = lambda t, wanted: torch.empty(t.shape, dtype=t.dtype, device=t.device) if wanted else None  # noqa: E731
        dx, dweight, dbias, d_initial = (new(t, n) for t, n in zip((x, weight, bias, initial), needs))
        args = (unit_rows(x), weight, bias, ctx.activation, None if initial is None else initial.contiguous(), None, None, 1,
                unit_rows(d_y), None if d_final is None else d_final.contiguous(), dx, dweight, dbias, d_initial)
        block = _block(*args)
        size = lib.ttc_causal_conv_workspace_bytes(block)
        if size:
            space = torch.empty(size, dtype=torch.uint8, device=x.device)
            block = with_spaces(block, space)
        launch(lib.ttc_causal_conv, "ttc_causal_conv", block, x.device)
        return dx, dweight, dbias, d_initial, None, None


def _check(name, x, dims, weight, bias, activation):
    if x.dim() != dims:
        raise ValueError(f"{name}: x {'[batch, tokens, channels]' if dims == 3 else '[batch, channels]'} is needed")
    C = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != C or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"{name}: a weight [{C}, taps] of 1 to {MAX_TAPS} taps is needed, got {tuple(weight.shape)}")
    if bias is not None and bias.shape != (C,):
        raise ValueError(f"{name}: a bias [{C}] is needed, got {tuple(bias.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name}: unknown activation {activation!r}")
    check_types(name, x)
    if weight.dtype not in (x.dtype, torch.float32) or (bias is not None and bias.dtype != weight.dtype):
        raise TypeError(f"{name}: weight and bias of type {x.dtype} or float32 are needed")
    check_device(name, x, weight, bias)
    return weight.contiguous(), None if bias is None else bias.contiguous()


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
                initial_state: torch.Tensor | None = None, output_state: bool = False):
    """``y [batch, tokens, channels]``, with ``output_state`` also the final state; new contiguous tensors.

    ``x [batch, tokens, channels]``: float32 or bfloat16, any strides over batch and tokens.  ``weight [channels, taps]`` (1
    to 8 taps, the last one meets the token itself) and ``bias [channels]`` of ``x``'s type or float32; sums in 32 bits.
    ``activation``: ``"none"`` or ``"silu"``.  States are the last ``taps - 1`` inputs, ``[batch, taps - 1, channels]`` of
    ``x``'s type; without one there are zeros in front of the first token.  Differentiable in all tensors.
    """
    name = "causal_conv"
    weight, bias = _check(name, x, 3, weight, bias, activation)
    B, T, C = x.shape
    if initial_state is not None:
        shape = (B, weight.shape[1] - 1, C)
        if initial_state.shape != shape or initial_state.dtype != x.dtype:
            raise ValueError(f"{name}: a state {list(shape)} of type {x.dtype} is needed")
        check_device(name, x, initial_state)
    if not x.is_cuda or x.numel() == 0 or traced(x, weight, bias, initial_state):
        y, final = causal_conv_torch(x, weight, bias, activation=activation, initial_state=initial_state)
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, initial_state)):
        y, final = _CausalConvFunc.apply(x, weight, bias, initial_state, activation, output_state)
    else:
        y, final = _forward(x, weight, bias, activation, None if initial_state is None else initial_state.contiguous(),
                            output_state)
    return (y, final) if output_state else y


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     activation: str = "none", slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each sequence: ``y [batch, channels]``; ``state`` is updated in place.

    ``x [batch, channels]``, ``weight`` and ``bias`` as in :func:`causal_conv`.  ``state [slots, taps - 1, channels]`` of
    ``x``'s type, contiguous; ``slots`` (int32 ``[batch]``) names each row's place in it, without it row ``b`` has place
    ``b``.  A row whose slot lies outside (-1: a row that fills up a batch of fixed size) is skipped: its output is 0.  Rows
    must not share a slot.  Not differentiable.
    """
    name = "causal_conv_step"
    weight, bias = _check(name, x, 2, weight, bias, activation)
    B, C = x.shape
    K = weight.shape[1]
    if state.shape[1:] != (K - 1, C) or state.dtype != x.dtype or not state.is_contiguous():
        raise ValueError(f"{name}: a contiguous state [slots, {K - 1}, {C}] of type {x.dtype} is needed")
    check_device(name, x, state, slots)
    if slots is None:
        if state.shape[0] != B:
            raise ValueError(f"{name}: {B} sequences, {state.shape[0]} states")
    else:
        if slots.shape != (B,) or slots.dtype != torch.int32:
            raise ValueError(f"{name}: int32 slots [{B}] are needed")
        slots = slots.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state)):
        raise RuntimeError(f"{name} is not differentiable: call it under torch.no_grad(), or use causal_conv")
    if not x.is_cuda or traced(x, weight, bias, state, slots):
        return _step_torch(x, state, weight, bias, activation, slots)
    x = unit_rows(x)
    y = x.new_empty((B, C))
    block = _STEP_BLOCK.pack(DTYPES[x.dtype], DTYPES[weight.dtype], B, C, K, _ACTIVATIONS[activation], state.shape[0],
                             x.data_ptr(), x.stride(0), weight.data_ptr(), ptr(bias), state.data_ptr(), ptr(slots),
                             y.data_ptr())
    launch(lib.ttc_causal_conv_step, "ttc_causal_conv_step", block, x.device)
    torch.autograd.graph.increment_version(state)  # whoever saved it for a backward has to find out
    return y


def _step_torch(x, state, weight, bias, activation, slots):
    rows = torch.arange(x.shape[0], device=x.device) if slots is None else slots.long()
    inside = (rows >= 0) & (rows < state.shape[0])
    rows = rows[inside]
    y, after = causal_conv_torch(x[inside].unsqueeze(1), weight, bias, activation=activation, initial_state=state[rows])
    state[rows] = after
    out = x.new_zeros(x.shape)
    out[inside] = y[:, 0]
    return out
