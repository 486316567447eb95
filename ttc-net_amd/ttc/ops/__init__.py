"""Sequence operators for models that hold the test-time control layer: rotary positions, linear attention with a
decay for each head, group norm with an activation or a gate.  Hand-written gfx950 kernels for CUDA tensors
(``include/ttc_ops.h``), the same formulas as torch operators for CPU tensors."""
from .group_norm import group_norm
from .linear_attention import linear_attention, linear_attention_step
from .rotary import rotary, rotary_table

__all__ = ["group_norm", "linear_attention", "linear_attention_step", "rotary", "rotary_table"]
