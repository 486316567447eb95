"""``LinearAttentionLayer``: a token mixer to put beside :class:`ttc.TTCLayer`, which treats every token on its own.

Queries and keys are turned by their positions (:func:`ttc.ops.rotary`), mixed by linear attention with a decay for each
token and head (:func:`ttc.ops.linear_attention`), normalised head by head and gated (:func:`ttc.ops.group_norm`):

    q, k, v, z, g = in_proj(x);   o = linear_attention(rotary(q), rotary(k), v, log_gamma = -softplus(g + bias_gamma))
    y = out_proj(group_norm(o) * silu(z))

:meth:`forward` takes whole sequences (training, prompts), :meth:`step` one token of each sequence of a batch, whose
states it updates in place.  The state of a sequence is ``[heads, key_dim, value_dim]`` float32, whatever its length.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import group_norm, linear_attention, linear_attention_step, rotary, rotary_table

__all__ = ["LinearAttentionLayer"]


class LinearAttentionLayer(nn.Module):
    """``dim``: width of the model; ``key_dim``, ``value_dim``: a head's sizes (up to 128); ``kv_heads`` divides
    ``num_heads`` (shared keys and values); ``rotary_dim``: how much of a key is turned (``key_dim`` by default, 0: none, so that positions have no limit);
    ``max_positions``: of the table of angles; ``memory``: the heads' decays start, spread evenly over their logarithm, at
    memories of this many tokens; ``rotary``: further arguments of :func:`ttc.ops.rotary_table`."""

    def __init__(self, dim: int, num_heads: int, key_dim: int = 64, value_dim: int = 64, kv_heads: int | None = None,
                 rotary_dim: int | None = None, max_positions: int = 8192, layout: str = "half",
                 memory: tuple[float, float] = (4.0, 512.0), eps: float = 1e-5, bias: bool = False,
                 rotary: dict | None = None):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        assert num_heads % kv_heads == 0, f"{kv_heads} heads of keys and values do not divide {num_heads} heads"
        self.dim, self.num_heads, self.kv_heads = dim, num_heads, kv_heads
        self.key_dim, self.value_dim, self.layout, self.eps = key_dim, value_dim, layout, eps
        # queries | keys | values | output gates | log-decays
        self._split = [num_heads * key_dim, kv_heads * key_dim, kv_heads * value_dim, num_heads * value_dim, num_heads]
        self.in_proj = nn.Linear(dim, sum(self._split), bias=bias)
        self.out_proj = nn.Linear(num_heads * value_dim, dim, bias=bias)
        self.norm_weight = nn.Parameter(torch.ones(num_heads * value_dim))
        self.norm_bias = nn.Parameter(torch.zeros(num_heads * value_dim))
        # softplus(bias_gamma) = 1 / memory where the projection gives 0
        rate = torch.exp(torch.linspace(math.log(1 / memory[1]), math.log(1 / memory[0]), num_heads))
        self.bias_gamma = nn.Parameter(torch.log(torch.expm1(rate)))
        self._table = dict(rotary or {}, length=max_positions, dim=key_dim if rotary_dim is None else rotary_dim)
        self.register_buffer("angles", rotary_table(**self._table), persistent=False)

    def _apply(self, fn, recurse=True):
        angles = self.angles
        super()._apply(fn, recurse)
        # No checkpoint holds the angles: whatever is done to the parameters (another type, to_empty), they keep their values
        # in 32 bits, or get them where the layer was made without any
        if angles.is_meta and not self.angles.is_meta:
            self.angles = rotary_table(**dict(self._table, device=self.angles.device))
        elif self.angles is not angles:
            self.angles = angles.to(self.angles.device)
        return self

    def _project(self, x):
        q, k, v, z, g = torch.split(self.in_proj(x), self._split, dim=-1)
        heads = lambda t, d: t.unflatten(-1, (t.shape[-1] // d, d))  # noqa: E731
        log_gamma = -F.softplus(g.float() + self.bias_gamma.float())
        return heads(q, self.key_dim), heads(k, self.key_dim), heads(v, self.value_dim), z, log_gamma

    def _turn(self, q, k, positions=None, offset=0):
        if self.angles.shape[1] == 0:  # rotary_dim = 0: no positions, so any number of tokens
            return q, k
        return rotary(q, k, self.angles, positions, offset=offset, layout=self.layout)

    def _finish(self, o, z):
        rows = group_norm(o.reshape(-1, self.num_heads * self.value_dim), self.num_heads, self.norm_weight, self.norm_bias,
                          eps=self.eps, activation="silu", gate=z.reshape(-1, self.num_heads * self.value_dim))
        return self.out_proj(rows.view(*z.shape))

    def new_state(self, slots: int) -> torch.Tensor:
        """States of ``slots`` sequences that have not begun."""
        return torch.zeros(slots, self.num_heads, self.key_dim, self.value_dim, dtype=torch.float32,
                           device=self.in_proj.weight.device)

    def forward(self, x: torch.Tensor, state: torch.Tensor | None = None, offset: int = 0, output_state: bool = False):
        """``x [batch, tokens, dim]``, whose first token has position ``offset`` and follows ``state``; with
        ``output_state`` also the state behind the last token."""
        q, k, v, z, log_gamma = self._project(x)
        q, k = self._turn(q, k, offset=offset)
        out = linear_attention(q, k, v, log_gamma, initial_state=state, output_state=output_state)
        o, state = out if output_state else (out, None)
        y = self._finish(o, z)
        return (y, state) if output_state else y

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, positions: torch.Tensor,
             slots: torch.Tensor | None = None) -> torch.Tensor:
        """``x [batch, dim]``, one token of each sequence at ``positions [batch]``; ``state`` (:meth:`new_state`) is
        updated in place, row ``b``'s at ``slots[b]`` (int32; outside: the row is skipped) or ``b``."""
        q, k, v, z, log_gamma = self._project(x)
        q, k = (t.squeeze(1) for t in self._turn(q.unsqueeze(1), k.unsqueeze(1), positions.unsqueeze(1)))
        return self._finish(linear_attention_step(q, k, v, log_gamma, state, slots=slots), z)
