"""Sequence operators for models that hold the test-time control layer: rotary positions (with one axis or several), causal
convolution over a few tokens, linear attention with a decay for each head, the gated delta rule, group norm with an activation
or a gate.  Hand-written gfx950 kernels for CUDA tensors (``include/ttc_ops.h``), the same formulas as torch operators for CPU
tensors."""
from .causal_conv import causal_conv, causal_conv_step
from .delta_rule import delta_rule, delta_rule_step
from .group_norm import group_norm
from .linear_attention import linear_attention, linear_attention_step
from .rotary import grid_positions, rotary, rotary_axes, rotary_table

__all__ = ["causal_conv", "causal_conv_step", "delta_rule", "delta_rule_step", "grid_positions", "group_norm", "linear_attention",
           "linear_attention_step", "rotary", "rotary_axes", "rotary_table"]
