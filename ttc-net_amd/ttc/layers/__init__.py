from .linear_attention import LinearAttentionLayer
from .ttc_layer import TTCLayer, LQR_SOLVER_IMPL_MAP

__all__ = ["LinearAttentionLayer", "TTCLayer", "LQR_SOLVER_IMPL_MAP"]
