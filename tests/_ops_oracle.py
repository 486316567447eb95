"""Plain 64-bit forms of the sequence operators (``ttc.ops``), written from their definitions, and what the tests
derive their tolerances from.  Test infrastructure only."""
import math

import numpy as np
import torch

EPS = 2.0 ** -24  # half a unit in the last place of 1 in 32 bits
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8}  # relative error of one rounding (24 and 8 digits)


def rotary64(x, positions, table, layout):
    """Pair by pair.  ``positions`` [batch, tokens] (numpy); a position outside the table turns into NaN."""
    x, cs = x.detach().double().cpu().numpy(), table.double().cpu().numpy()
    y, half = x.copy(), cs.shape[1]
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            p = int(positions[b, t])
            for i in range(half):
                c, s = cs[p, i] if 0 <= p < cs.shape[0] else (math.nan, math.nan)
                u, w = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
                y[b, t, :, u] = x[b, t, :, u] * c - x[b, t, :, w] * s
                y[b, t, :, w] = x[b, t, :, u] * s + x[b, t, :, w] * c
    return y


def group_norm64(x, groups, weight, bias, eps, activation, gate):
    """As torch operators in 64 bits, differentiable."""
    n, c = x.shape[0], x.shape[-1]
    rows = x.double().reshape(n, -1, groups, c // groups).transpose(1, 2).reshape(n, groups, -1)
    mean = rows.mean(-1, keepdim=True)
    var = ((rows - mean) ** 2).mean(-1, keepdim=True)
    y = ((rows - mean) / torch.sqrt(var + eps)).reshape(n, groups, -1, c // groups).transpose(1, 2).reshape(x.shape)
    if weight is not None:
        y = y * weight.double() + bias.double()
    f = (lambda z: z / (1 + torch.exp(-z))) if activation == "silu" else (lambda z: z)
    return f(y) if gate is None else y * f(gate.double())


def within(got, want, bound):
    """|got - want| <= bound element by element, NaN and infinities in the same places."""
    got = got.detach().double().cpu().numpy()
    want = want.detach().double().cpu().numpy() if isinstance(want, torch.Tensor) else np.asarray(want)
    bound = bound.detach().double().cpu().numpy() if isinstance(bound, torch.Tensor) else np.asarray(bound)
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), "other infinities"
    off = np.abs(got - want)
    over = np.where(fine, off - bound, -1.0)
    assert (over <= 0).all(), f"off by {off[fine].max():.3e}, {np.nanmax(off[fine] / np.broadcast_to(bound, off.shape)[fine]):.2f} of the bound"


def quotient(f, xs, ds, cs, h):
    """Central difference of sum(f(xs) * cs) along ds, the sum in 64 bits."""
    def at(sign):
        out = f(*[None if x is None else x + sign * h * d for x, d in zip(xs, ds)])
        out = out if isinstance(out, tuple) else (out,)
        return sum(float((o.detach().double().cpu() * c.double().cpu()).sum()) for o, c in zip(out, cs) if c is not None)
    return (at(1.0) - at(-1.0)) / (2 * h)
