"""When a call must be made of torch operators that something else observes, instead of one kernel."""
from __future__ import annotations

import torch

__all__ = ["traced"]

_PLAIN = (torch.Tensor, torch.nn.Parameter)


def traced(*xs) -> bool:
    """Whether operators are observed one by one (functorch transforms, batched gradients, forward-mode
    tangents, tracing and compilation, dispatch modes such as ``make_fx``'s, tensor subclasses such as fake
    tensors): none of these sees the kernel."""
    if torch.compiler.is_compiling():  # first: a full-graph compilation can trace none of the rest
        return True
    if (torch._C._are_functorch_transforms_active() or torch._C._len_torch_dispatch_stack() > 0
            or torch.autograd.forward_ad._current_level >= 0 or torch.jit.is_tracing()):
        return True
    for x in xs:
        if x is not None and (type(x) not in _PLAIN or not torch._C._has_storage(x)):
            return True
    return False
