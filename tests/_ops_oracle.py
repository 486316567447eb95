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


def linear64(q, k, v, g, scale, state=None, d_o=None, d_state=None):
    """Token by token: o, the final state, and for gradients d_o (and d_state) those of q, k, v, g and the state, from the
    formulas (R: the gradient of the state).  ``g`` [batch, tokens, heads]; shared heads' gradients are summed.  A decay
    of 0 drops the state whatever it holds."""
    H = g.shape[-1]
    wide = lambda x: x.detach().double().cpu().repeat_interleave(H // x.shape[2], dim=2)  # noqa: E731
    Q, K, V, G = wide(q), wide(k), wide(v), g.detach().double().cpu()
    (B, T), dk, dv = Q.shape[:2], Q.shape[-1], V.shape[-1]
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state is None else state.detach().double().cpu()
    before, after, o = [], [], torch.zeros(B, T, H, dv, dtype=torch.float64)
    decay, gone = G.exp(), (G < -104)[..., None, None]
    kept = lambda t, X: torch.where(gone[:, t], torch.zeros_like(X), X * decay[:, t, :, None, None])  # noqa: E731
    for t in range(T):
        before.append(S)
        S = kept(t, S) + K[:, t, :, :, None] * V[:, t, :, None, :]
        after.append(S)
        o[:, t] = scale * (S * Q[:, t, :, :, None]).sum(-2)
    if d_o is None:
        return {"o": o, "state": S}
    D = d_o.detach().double().cpu()
    R = torch.zeros_like(S) if d_state is None else d_state.detach().double().cpu()
    dq, dk_, dv_, dg = torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V), torch.zeros_like(G)
    for t in reversed(range(T)):
        dq[:, t] = scale * (after[t] * D[:, t, :, None, :]).sum(-1)
        R = R + scale * Q[:, t, :, :, None] * D[:, t, :, None, :]
        dk_[:, t] = (R * V[:, t, :, None, :]).sum(-1)
        dv_[:, t] = (R * K[:, t, :, :, None]).sum(-2)
        dg[:, t] = (R * kept(t, before[t])).sum((-1, -2))
        R = kept(t, R)
    shared = lambda x, d: d.unflatten(2, (x.shape[2], -1)).sum(3)  # noqa: E731
    return {"o": o, "state": S, "q": shared(q, dq), "k": shared(k, dk_), "v": shared(v, dv_), "g": dg, "d_state": R}
