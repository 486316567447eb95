"""Group norm with an activation or a gate, channels last.

CUDA tensors go through the kernels of ``ttc_group_norm``; CPU tensors, and any call that something observes operator by
operator, run :func:`group_norm_torch`.
"""
from __future__ import annotations

import struct

import torch

from .._dispatch import traced
from ..solvers._lib import lib
from ._call import DTYPES, check_device, check_types, launch, ptr, recorded_backward

__all__ = ["group_norm", "group_norm_torch"]

_ACTIVATIONS = {"none": 0, "silu": 1}
_BLOCK = struct.Struct("8qd4q2qqq4qqq")


def group_norm_torch(x, groups, weight=None, bias=None, *, eps=1e-5, activation="none", gate=None):
    """:func:`group_norm` as torch operators."""
    C = x.shape[-1]
    grouped = x.float().reshape(x.shape[0], x[0, ..., 0].numel() if x.shape[0] else 1, groups, C // groups)
    centred = grouped - grouped.mean((1, 3), keepdim=True)
    y = (centred * torch.rsqrt(centred.square().mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    if weight is not None:
        y = y * weight.float() + bias.float()
    z = y if gate is None else gate.float()
    on = z * torch.sigmoid(z) if activation == "silu" else z
    return (on if gate is None else y * on).to(x.dtype).contiguous()


def _block(x, groups, weight, bias, eps, activation, gate, mean, rstd, y, dy=None, dx=None, dgate=None, dweight=None,
           dbias=None):
    n, c = x.shape[0], x.shape[-1]
    fields = [DTYPES[x.dtype], 0 if weight is None else DTYPES[weight.dtype], n, x.numel() // (n * c), c, groups,
              _ACTIVATIONS[activation], 0 if dy is None else 1, eps, ptr(x), ptr(gate), ptr(weight), ptr(bias), ptr(mean),
              ptr(rstd), ptr(y), ptr(dy), ptr(dx), ptr(dgate), ptr(dweight), ptr(dbias), 0, 0]
    block = _BLOCK.pack(*fields)
    size = lib.ttc_group_norm_workspace_bytes(block)
    if size:
        space = torch.empty(size, dtype=torch.uint8, device=x.device)
        fields[-2:] = space.data_ptr(), size
        return _BLOCK.pack(*fields), space
    return block, None


def _forward(x, groups, weight, bias, eps, activation, gate, keep):
    y = torch.empty_like(x)  # x is contiguous
    mean = rstd = None
    if keep:
        mean, rstd = torch.empty(2, x.shape[0], groups, dtype=torch.float32, device=x.device)
    block, space = _block(x, groups, weight, bias, eps, activation, gate, mean, rstd, y)
    launch(lib.ttc_group_norm, "ttc_group_norm", block, x.device)
    return y, mean, rstd


class _GroupNormFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, gate, groups, eps, activation):
        y, mean, rstd = _forward(x.contiguous(), groups, weight, bias, eps, activation,
                                 None if gate is None else gate.contiguous(), True)
        ctx.save_for_backward(x, weight, bias, gate, mean, rstd)
        ctx.args = (groups, eps, activation)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, gate, mean, rstd = ctx.saved_tensors
        groups, eps, activation = ctx.args
        needs = ctx.needs_input_grad[:4]
        recorded = torch.is_grad_enabled()
        if recorded or traced(dy, x, weight, bias, gate):
            form = lambda x, w, b, g: group_norm_torch(x, groups, w, b, eps=eps, activation=activation, gate=g)  # noqa: E731
            return (*recorded_backward(form, (x, weight, bias, gate), needs, (dy,), recorded), None, None, None)
        x, dy = x.contiguous(), dy.contiguous()
        gate = None if gate is None else gate.contiguous()
        new = lambda t, wanted: torch.empty_like(t) if wanted else None  # noqa: E731
        dx, dweight, dbias, dgate = (new(t, n) for t, n in zip((x, weight, bias, gate), needs))
        block, space = _block(x, groups, weight, bias, eps, activation, gate, mean, rstd, None, dy, dx, dgate, dweight,
                              dbias)
        launch(lib.ttc_group_norm, "ttc_group_norm", block, x.device)
        return dx, dweight, dbias, dgate, None, None, None


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5, activation: str = "none", gate: torch.Tensor | None = None) -> torch.Tensor:
    """``x [n, ..., channels]`` normalised over the channels of each group and all positions between the first and the
    last dimension (none: over the channels of each row alone), times ``weight`` plus ``bias`` (``[channels]``, both or
    neither), then passed through ``activation`` (``"none"`` or ``"silu"``); with a ``gate`` of ``x``'s shape the
    activation is the gate's: ``norm(x) * activation(gate)``.

    float32 or bfloat16 (``weight`` and ``bias`` of ``x``'s type or float32); statistics and arithmetic in 32 bits, biased
    variance of the centred values.  Differentiable in all tensors; a new contiguous tensor.
    """
    if x.dim() < 2:
        raise ValueError("group_norm: x [n, ..., channels] is needed")
    C = x.shape[-1]
    if groups <= 0 or C % groups:
        raise ValueError(f"group_norm: {C} channels do not divide into {groups} groups")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"group_norm: unknown activation {activation!r}")
    if not eps >= 0:
        raise ValueError(f"group_norm: eps of at least 0 is needed, got {eps}")
    if (weight is None) != (bias is None):
        raise ValueError("group_norm: weight and bias, or neither")
    check_types("group_norm", x, gate)
    if gate is not None and gate.shape != x.shape:
        raise ValueError("group_norm: a gate of x's shape is needed")
    if weight is not None:
        if weight.shape != (C,) or bias.shape != (C,):
            raise ValueError(f"group_norm: weight and bias [{C}] are needed")
        if weight.dtype != bias.dtype or weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"group_norm: weight and bias of type {x.dtype} or float32 are needed")
        check_device("group_norm", x, weight, bias)
        weight, bias = weight.contiguous(), bias.contiguous()
    if x.numel() == 0:  # no elements, so no statistics: every gradient is zero
        y = x.clone() if gate is None else x * gate
        return y if weight is None else (y * weight + bias).to(x.dtype)
    if not x.is_cuda or traced(x, weight, bias, gate):
        return group_norm_torch(x, groups, weight, bias, eps=eps, activation=activation, gate=gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, gate)):
        return _GroupNormFunc.apply(x, weight, bias, gate, groups, eps, activation)
    return _forward(x.contiguous(), groups, weight, bias, eps, activation, None if gate is None else gate.contiguous(),
                    False)[0]
