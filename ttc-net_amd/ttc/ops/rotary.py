"""Rotary positions: pairs of a head's components turned by the token's angle.

:func:`rotary_table` makes the cosines and sines of every position once, :func:`rotary` turns queries and keys by
them.  CUDA tensors go through one kernel each way for queries and keys together (``ttc_rotary``); CPU tensors, and
any call that something observes operator by operator, run :func:`rotary_torch`.
"""
from __future__ import annotations

import math
import struct

import torch

from .._dispatch import traced
from ..solvers._lib import lib
from ._call import DTYPES, check_device, check_types, launch, ptr, unit_rows

__all__ = ["rotary", "rotary_table", "rotary_torch"]

_LAYOUTS = {"half": 0, "interleaved": 1}
_BLOCK = struct.Struct("7q2q2q6q2qqqqq2qq")


def rotary_table(length: int, dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_length: int | None = None, fast: float = 32.0, slow: float = 1.0,
                 device=None) -> torch.Tensor:
    """``[length, dim / 2, 2]`` fp32: cosine and sine of ``position * base^(-2 i / dim)``, computed in 64 bits.

    For contexts ``factor`` times longer than the ``original_length`` that a model was trained on, ``scaling`` is

    * ``"linear"``: positions divided by ``factor``;
    * ``"base"``: ``base`` raised to ``base * factor^(dim / (dim - 2))``, which keeps the fastest pair's angle and
      divides the slowest one's by ``factor``;
    * ``"bands"``: pairs that turn more than ``fast`` times over ``original_length`` are kept, those that turn less than
      ``slow`` times divided by ``factor``, those between interpolated linearly in the number of turns' logarithm's
      place (the pair's index); the table is multiplied by ``0.1 ln(factor) + 1``, which raises the scores of longer
      contexts.
    """
    if not (length >= 0 and dim >= 0 and dim % 2 == 0):
        raise ValueError(f"rotary_table: length and an even dim are needed, got {length}, {dim}")
    if scaling not in ("none", "linear", "base", "bands"):
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    if not (base > 0 and (scaling == "none" or factor >= 1)):
        raise ValueError("rotary_table: a positive base and a factor of at least 1 are needed")
    if scaling == "base":
        if dim == 2 and factor != 1:
            raise ValueError("rotary_table: scaling 'base' needs more than one pair")
        if dim > 2:
            base = base * factor ** (dim / (dim - 2))
    pair = torch.arange(dim // 2, dtype=torch.float64, device=device)
    speed = torch.pow(base, -2.0 * pair / max(dim, 1))
    magnitude = 1.0
    if scaling == "linear":
        speed = speed / factor
    elif scaling == "bands":
        if not (original_length is not None and original_length > 0 and fast > slow > 0):
            raise ValueError("rotary_table: scaling 'bands' needs original_length and fast > slow > 0")
        at = lambda turns: dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), dim - 1)
        kept = 1 - ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        speed = speed / factor * (1 - kept) + speed * kept
        magnitude = 0.1 * math.log(factor) + 1
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * speed
    return (torch.stack([angle.cos(), angle.sin()], -1) * magnitude).float()


def _turn(x: torch.Tensor, cs: torch.Tensor, layout: str) -> torch.Tensor:
    rot = 2 * cs.shape[-2]
    wide = x.float()
    cos, sin = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    if layout == "half":
        a, b = wide[..., :rot // 2], wide[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = wide[..., 0:rot:2], wide[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, wide[..., rot:]], -1).to(x.dtype)


def rotary_torch(q, k, table, positions=None, *, offset: int = 0, layout: str = "half"):
    """:func:`rotary` as torch operators."""
    if positions is None:
        cs = table[offset:offset + q.shape[1]]
    else:
        inside = (positions >= 0) & (positions < table.shape[0])
        cs = table[positions.long().clamp(0, max(table.shape[0] - 1, 0))]
        cs = cs.masked_fill(~inside[..., None, None], math.nan)
    return _turn(q, cs, layout), None if k is None else _turn(k, cs, layout)


def _launch(xs, table, positions, offset, layout, backward):
    """The kernel over ``xs`` (queries, keys or None): the turned copies."""
    q, k = xs
    B, T, H, D = q.shape
    xs = [None if x is None else unit_rows(x) for x in xs]
    ys = [None if x is None else x.new_empty(x.shape) for x in xs]
    strides = [0] * 6
    for i, x in enumerate(xs):
        if x is not None:
            strides[3 * i:3 * i + 3] = x.stride()[:3]
    pos_bytes, pos_b, pos_t = 0, 0, 0
    if positions is not None:
        pos_bytes, pos_t = positions.element_size(), positions.stride(-1)
        pos_b = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    block = _BLOCK.pack(DTYPES[q.dtype], B, T, D, 2 * table.shape[1], _LAYOUTS[layout], backward, H,
                        0 if k is None else k.shape[2], ptr(xs[0]), ptr(xs[1]), *strides, ptr(ys[0]), ptr(ys[1]),
                        table.data_ptr(), table.shape[0], ptr(positions), pos_bytes, pos_b, pos_t, offset)
    launch(lib.ttc_rotary, "ttc_rotary", block, q.device)
    return ys


class _RotaryFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, table, positions, offset, layout):
        ctx.save_for_backward(table, positions)
        ctx.args = (offset, layout)
        ctx.shapes = (q.shape, None if k is None else k.shape)
        ctx.set_materialize_grads(False)
        yq, yk = _launch((q, k), table, positions, offset, layout, 0)
        return yq, yk

    @staticmethod
    def backward(ctx, dq, dk):
        table, positions = ctx.saved_tensors
        offset, layout = ctx.args
        if dq is None and dk is None:
            return (None,) * 6
        if torch.is_grad_enabled() or traced(dq, dk):  # the turn back is a turn by the table's conjugate
            conjugate = table * table.new_tensor([1.0, -1.0])
            one = lambda d: None if d is None else rotary_torch(d, None, conjugate, positions, offset=offset,  # noqa: E731
                                                                layout=layout)[0]
            return one(dq), one(dk), None, None, None, None
        if dq is None:
            return None, _launch((dk, None), table, positions, offset, layout, 1)[0], None, None, None, None
        return (*_launch((dq, dk), table, positions, offset, layout, 1), None, None, None, None)


def rotary(q: torch.Tensor, k: torch.Tensor | None, table: torch.Tensor, positions: torch.Tensor | None = None, *,
           offset: int = 0, layout: str = "half"):
    """Queries ``[batch, tokens, heads, dim]`` and keys ``[batch, tokens, key heads, dim]`` (or None) turned by their
    positions: ``(q', k')``, new contiguous tensors.

    ``table``: :func:`rotary_table`'s, ``[length, rot / 2, 2]`` fp32; the first ``rot`` components of a head turn, the
    others are copied.  ``positions``: int32 or int64 ``[tokens]`` or ``[batch, tokens]``; without them token ``t`` has
    position ``offset + t``.  A given position outside the table makes that token's turned components NaN (nothing is read
    outside, and nothing waits for the device to find out).  ``layout``: pairs ``(i, i + rot / 2)`` (``"half"``) or
    ``(2 i, 2 i + 1)`` (``"interleaved"``).  ``q`` and ``k`` may be views with any strides over batch, tokens and heads;
    float32 or bfloat16, turned in 32 bits.  Differentiable in ``q`` and ``k``; with a ``table`` that requires a gradient the torch operators run
    instead of the kernel, and it has one too.
    """
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("rotary: q and k [batch, tokens, heads, dim] are needed")
    if k is not None and (k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]):
        raise ValueError("rotary: q and k of one batch, number of tokens and head size are needed")
    check_types("rotary", q, k)
    check_device("rotary", q, table, positions)
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("rotary: a contiguous float32 table [length, rot / 2, 2] is needed")
    if 2 * table.shape[1] > q.shape[3]:
        raise ValueError(f"rotary: a table for {2 * table.shape[1]} components, heads of {q.shape[3]}")
    if layout not in _LAYOUTS:
        raise ValueError(f"rotary: unknown layout {layout!r}")
    if positions is None:
        if offset < 0 or offset + q.shape[1] > table.shape[0]:
            raise ValueError(f"rotary: positions {offset} to {offset + q.shape[1] - 1}, a table of {table.shape[0]}")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("rotary: int32 or int64 positions are needed")
        if offset != 0:
            raise ValueError("rotary: either positions or an offset")
        if positions.shape != q.shape[:2] and positions.shape != q.shape[1:2] and positions.shape != (1, q.shape[1]):
            raise ValueError(f"rotary: positions [tokens] or [batch, tokens] are needed, got {tuple(positions.shape)}")
        if table.shape[0] == 0 and q.numel() > 0:
            raise ValueError("rotary: an empty table")
    learnt = table.requires_grad and torch.is_grad_enabled()  # the kernel's backward has no gradient for the table
    if not q.is_cuda or learnt or traced(q, k, table, positions):
        return rotary_torch(q, k, table, positions, offset=offset, layout=layout)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RotaryFunc.apply(q, k, table, positions, offset, layout)
    return tuple(_launch((q, k), table, positions, offset, layout, 0))
