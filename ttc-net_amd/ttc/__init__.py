"""TTC-Net's Test-Time Control layer on AMD MI355X (gfx950).

``from ttc import TTCLayer`` as with the reference package (``ttc/__init__.py``);
the LQR solve inside runs in hand-written HIP kernels (``libttc_lqr.so``).  ``LinearAttentionLayer`` mixes
tokens beside it, from the sequence operators of ``ttc.ops`` (kernels in the same library).
"""
from .layers.linear_attention import LinearAttentionLayer
from .layers.ttc_layer import TTCLayer

__all__ = ["LinearAttentionLayer", "TTCLayer"]
