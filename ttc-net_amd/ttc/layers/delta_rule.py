"""``DeltaRuleLayer``: a token mixer to put beside :class:`ttc.TTCLayer`, whose state replaces what it holds at a key.

Queries, keys and values pass a short convolution (:func:`ttc.ops.causal_conv`), queries and keys may be turned by positions on
several axes (:func:`ttc.ops.rotary_axes`), the gated delta rule mixes them (:func:`ttc.ops.delta_rule`, keys brought to length
1 there), and each head is normalised and gated (:func:`ttc.ops.group_norm`):

    q, k, v, z, b, g = in_proj(x);   q, k, v = silu(conv(q, k, v))
    o = delta_rule(q, k, v, log_gamma = -softplus(g + bias_gamma), beta = sigmoid(b));   y = out_proj(group_norm(o) * silu(z))

:meth:`forward` takes whole sequences (training, prompts) of one text each, :meth:`step` one token of each sequence of a batch, whose
states it updates in place.  A sequence's state, whatever its length, is the last ``taps - 1`` inputs of the convolution and
``[heads, key_dim, value_dim]`` float32.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._angles import Angles
from ..ops import causal_conv, causal_conv_step, delta_rule, delta_rule_step, group_norm, rotary_axes, rotary_table

__all__ = ["DeltaRuleLayer"]


class DeltaRuleLayer(Angles, nn.Module):
    """``dim``: width of the model; ``key_dim``, ``value_dim``: a head's sizes (up to 128); ``key_heads`` divides ``num_heads``
    (shared queries and keys); ``taps``: of the convolution (1 to 8); ``rotary_sections``: how many pairs of a key each axis of
    the positions turns (none by default: no positions), from a table of ``max_positions`` with the further arguments
    ``rotary`` of :func:`ttc.ops.rotary_table`; ``memory``: the heads' decays start, spread evenly over their logarithm, at
    memories of this many tokens."""

    def __init__(self, dim: int, num_heads: int, key_dim: int = 64, value_dim: int = 64, key_heads: int | None = None,
                 taps: int = 4, rotary_sections: tuple[int, ...] = (), max_positions: int = 8192, layout: str = "half",
                 memory: tuple[float, float] = (4.0, 512.0), eps: float = 1e-5, bias: bool = False,
                 rotary: dict | None = None):
        super().__init__()
        key_heads = num_heads if key_heads is None else key_heads
        assert num_heads % key_heads == 0, f"{key_heads} heads of queries and keys do not divide {num_heads} heads"
        self.dim, self.num_heads, self.key_heads = dim, num_heads, key_heads
        self.key_dim, self.value_dim, self.taps, self.layout, self.eps = key_dim, value_dim, taps, layout, eps
        self.rotary_sections = tuple(rotary_sections)
        # queries | keys | values (what the convolution sees) | output gates | strengths | log-decays
        self._mixed = [key_heads * key_dim, key_heads * key_dim, num_heads * value_dim]
        self.in_proj = nn.Linear(dim, sum(self._mixed) + num_heads * (value_dim + 2), bias=bias)
        self.out_proj = nn.Linear(num_heads * value_dim, dim, bias=bias)
        self.conv_weight = nn.Parameter((torch.rand(sum(self._mixed), taps) * 2 - 1) / math.sqrt(taps))
        self.norm_weight = nn.Parameter(torch.ones(num_heads * value_dim))
        self.norm_bias = nn.Parameter(torch.zeros(num_heads * value_dim))
        # softplus(bias_gamma) = 1 / memory where the projection gives 0
        rate = torch.exp(torch.linspace(math.log(1 / memory[1]), math.log(1 / memory[0]), num_heads))
        self.bias_gamma = nn.Parameter(torch.log(torch.expm1(rate)))
        self._table = dict(rotary or {}, length=max_positions if self.rotary_sections else 0, dim=2 * sum(self.rotary_sections))
        self.register_buffer("angles", rotary_table(**self._table), persistent=False)

    def _project(self, x):
        H = self.num_heads
        mixed, z, b, g = torch.split(self.in_proj(x), [sum(self._mixed), H * self.value_dim, H, H], dim=-1)
        return mixed, z, torch.sigmoid(b.float()), -F.softplus(g.float() + self.bias_gamma.float())

    def _beside(self, mixed, before):
        """The convolution's inputs and taps in a type that holds a state of another one too."""
        wide = mixed.dtype if before is None else torch.promote_types(mixed.dtype, before.dtype)
        return mixed.to(wide), self.conv_weight.to(torch.promote_types(self.conv_weight.dtype, wide))

    def _heads(self, mixed, positions):
        q, k, v = torch.split(mixed, self._mixed, dim=-1)
        q, k, v = (t.unflatten(-1, (t.shape[-1] // d, d)) for t, d in ((q, self.key_dim), (k, self.key_dim), (v, self.value_dim)))
        if self.rotary_sections:
            if positions is None:
                raise ValueError(f"DeltaRuleLayer: positions on {len(self.rotary_sections)} axes are needed")
            q, k = rotary_axes(q, k, self.angles, positions, self.rotary_sections, layout=self.layout)
        return q, k, v

    def _finish(self, o, z):
        rows = group_norm(o.reshape(-1, self.num_heads * self.value_dim), self.num_heads, self.norm_weight, self.norm_bias,
                          eps=self.eps, activation="silu", gate=z.reshape(-1, self.num_heads * self.value_dim))
        return self.out_proj(rows.view(*z.shape))

    def new_state(self, slots: int) -> tuple[torch.Tensor, torch.Tensor]:
        """States of ``slots`` sequences that have not begun: the convolution's, of the weights' type (which holds exactly what a
        projection in fewer bits gives under autocast), and the mixer's."""
        w = self.in_proj.weight
        return (torch.zeros(slots, self.taps - 1, sum(self._mixed), dtype=w.dtype, device=w.device),
                torch.zeros(slots, self.num_heads, self.key_dim, self.value_dim, dtype=torch.float32, device=w.device))

    def forward(self, x: torch.Tensor, state: tuple[torch.Tensor, torch.Tensor] | None = None,
                positions: torch.Tensor | None = None, output_state: bool = False):
        """``x [batch, tokens, dim]`` behind ``state``, with ``rotary_sections`` at ``positions [tokens, axes]`` or ``[batch,
        tokens, axes]``; with ``output_state`` also the state behind the last token, the convolution's of the projection's type or
        that of ``state``, whichever is wider."""
        mixed, z, beta, log_gamma = self._project(x)
        before, S = (None, None) if state is None else state
        rows, weight = self._beside(mixed, before)
        rows, before = causal_conv(rows, weight, activation="silu", output_state=True,
                                   initial_state=None if before is None else before.to(rows.dtype))
        q, k, v = self._heads(rows.to(mixed.dtype), positions)
        out = delta_rule(q, k, v, log_gamma, beta, initial_state=S, output_state=output_state, normalize=True)
        o, S = out if output_state else (out, None)
        y = self._finish(o, z)
        return (y, (before, S)) if output_state else y

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: tuple[torch.Tensor, torch.Tensor], positions: torch.Tensor | None = None,
             slots: torch.Tensor | None = None) -> torch.Tensor:
        """``x [batch, dim]``, one token of each sequence, with ``rotary_sections`` at ``positions [batch, axes]``; ``state``
        (:meth:`new_state`, or of a type no narrower than the projection's) is updated in place, row ``b``'s at ``slots[b]`` (int32;
        outside: the row is skipped) or ``b``."""
        mixed, z, beta, log_gamma = self._project(x)
        rows, weight = self._beside(mixed, state[0])
        rows = causal_conv_step(rows, state[0], weight, activation="silu", slots=slots)
        q, k, v = self._heads(rows.to(mixed.dtype).unsqueeze(1), None if positions is None else positions.unsqueeze(1))
        o = delta_rule_step(q.squeeze(1), k.squeeze(1), v.squeeze(1), log_gamma, beta, state[1], slots=slots, normalize=True)
        return self._finish(o, z)
