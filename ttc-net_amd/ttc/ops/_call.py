"""What the operators' entry points share: types, argument blocks, streams, and the derivative of a backward
that is itself recorded."""
from __future__ import annotations

import struct

import torch

from ..solvers._lib import check

DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # TTC_DTYPE_*


def ptr(x) -> int:
    return 0 if x is None else x.data_ptr()


def check_types(name: str, first, *xs) -> None:
    """All of one type that has kernels, all on one device."""
    if first.dtype not in DTYPES:
        raise TypeError(f"{name}: float32 and bfloat16 tensors are supported, got {first.dtype}")
    for x in xs:
        if x is not None:
            if x.dtype != first.dtype:
                raise TypeError(f"{name}: tensors of one type are needed, got {first.dtype} and {x.dtype}")
            if x.device != first.device:
                raise ValueError(f"{name}: tensors on one device are needed, got {first.device} and {x.device}")


def check_device(name: str, first, *xs) -> None:
    for x in xs:
        if x is not None and x.device != first.device:
            raise ValueError(f"{name}: tensors on one device are needed, got {first.device} and {x.device}")


def unit_rows(x: torch.Tensor) -> torch.Tensor:
    """``x``, or a copy of it where its last dimension does not have stride 1."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def with_spaces(block: bytes, *spaces) -> bytes:
    """``block`` with these as its last fields: an address and a number of bytes each."""
    tail = [n for x in spaces for n in ((0, 0) if x is None else (x.data_ptr(), x.numel()))]
    return block[:-8 * len(tail)] + struct.pack(f"{len(tail)}q", *tail)


def launch(fn, name: str, block: bytes, device: torch.device) -> None:
    """``fn(block, stream)`` on the device's current stream."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(block, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(block, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


def recorded_backward(form, inputs, needs, grads, create_graph: bool):
    """Gradients of ``form(*inputs)`` (torch operators; a tensor or a tuple) for the inputs flagged in ``needs``, with
    operators that can be differentiated or observed again."""
    with torch.enable_grad():
        # Partial derivatives: with respect to aliases, since one input may be computed from another, or be the same tensor
        inputs = [x if x is None else x.view_as(x) if create_graph else x.detach().requires_grad_(n)
                  for x, n in zip(inputs, needs)]
        out = form(*inputs)
        pairs = [(o, g) for o, g in zip(out if isinstance(out, tuple) else (out,), grads) if g is not None]
        wrt = [x for x, n in zip(inputs, needs) if n]
        got = iter(torch.autograd.grad([o for o, _ in pairs], wrt, [g for _, g in pairs],
                                       create_graph=create_graph, allow_unused=True))
    return tuple(next(got) if n else None for n in needs)
