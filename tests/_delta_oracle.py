"""The gated delta rule token by token in 64 bits, forwards and backwards, with a bound on what 32 bits may be off by.  Test
infrastructure only.

Bounds, in 2-norms for each token and head (an entry is off by at most its row's norm).  One step maps the state by
e^g (I - b k k'), whose norm is e^g max(1, |1 - b |k|^2|), so an error made earlier grows by no more than that; a step adds n EPS
of the sizes of what it sums: the state, the value, and, as tokens are taken 64 at a time, what the 64 tokens in front of it added
(behind it, backwards).  n counts the roundings on a term's way: a head's size for each of two products, 64 terms of a chunk in the
triangular system, in its inverse and in the products, each rounded a few times: 2 max(dk, dv) + 5 * 64.  Products carry errors on
by the product rule.  Values that the kernels hold in 16 digits on the way to a 16-bit result (their first 8, and 8 of the rest,
which is below 2^-7) add 2^-15 of the same sizes; a result is rounded once more to its type."""
import torch

from _ops_oracle import EPS, HALF

RESET = -104.0
CHUNK = 64


def delta64(q, k, v, g, beta, scale, state=None, d_o=None, d_state=None, normalize=False, eps=1e-6):
    """{name: (value, bound)}: o, state, and for gradients d_o (and d_state) those of q, k, v, g, beta, d_state."""
    dt, H = q.dtype if q.dtype in HALF else torch.float32, g.shape[-1]  # 64 bits: of a larger computation, whose bound counts
    d = lambda x: x.detach().double().cpu()  # noqa: E731
    wide = lambda x: x.repeat_interleave(H // x.shape[2], dim=2)  # noqa: E731
    length = lambda x: (d(x).square().sum(-1, keepdim=True) + (eps if normalize else 0)).sqrt()  # noqa: E731
    lq, lk = length(q), length(k)
    Q, K = (wide(d(q) / lq), wide(d(k) / lk)) if normalize else (wide(d(q)), wide(d(k)))
    Q, V, G, Be = Q * scale, wide(d(v)), d(g), d(beta)
    (B, T), dk, dv = Q.shape[:2], Q.shape[-1], V.shape[-1]
    n = (2 * max(dk, dv) + 5 * CHUNK) * EPS
    near = 2.0 ** -15 if dt != torch.float32 else 0.0
    cut, decay = G < RESET, G.exp()
    norm = lambda x: x.norm(dim=-1)  # noqa: E731
    size = lambda S: S.flatten(-2).norm(dim=-1)  # noqa: E731
    drop = lambda t, X: torch.where(cut[:, t].reshape(B, H, *(1,) * (X.dim() - 2)), torch.zeros_like(X),  # noqa: E731
                                    X * decay[:, t].reshape(B, H, *(1,) * (X.dim() - 2)))
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state is None else d(state)
    eS = torch.zeros(B, H, dtype=torch.float64)
    o, eo = torch.zeros(B, T, H, dv, dtype=torch.float64), torch.zeros(B, T, H, dtype=torch.float64)
    e, ee, held, eheld, around = o.clone(), eo.clone(), [], [], []
    added = torch.zeros(T, B, H, dtype=torch.float64)  # |k_s| |u_s|
    for t in range(T):
        S, eS = drop(t, S), drop(t, eS)
        kt, bt, nk = K[:, t], Be[:, t], norm(K[:, t])
        before = added[max(t - CHUNK, 0):t].sum(0)
        held.append(S), eheld.append(eS), around.append(size(S) + before)
        e[:, t] = V[:, t] - (S * kt.unsqueeze(-1)).sum(-2)
        local = n * (norm(V[:, t]) + (size(S) + before) * nk)
        ee[:, t] = eS * nk + local
        u = bt.unsqueeze(-1) * e[:, t]
        eS = torch.clamp((1 - bt * nk ** 2).abs(), min=1) * eS + bt.abs() * nk * local + n * (size(S) + nk * norm(u))
        S = S + kt.unsqueeze(-1) * u.unsqueeze(-2)
        added[t] = nk * norm(u)
        o[:, t] = (S * Q[:, t].unsqueeze(-1)).sum(-2)
        eo[:, t] = norm(Q[:, t]) * (eS + (n + near) * (size(S) + before + added[t]))
    last = lambda x, off: off + HALF[dt] * (x.abs() + off) + 1e-30  # noqa: E731
    out = {"o": (o, last(o, eo.unsqueeze(-1))), "state": (S, eS[..., None, None] * (1 + EPS) + EPS * S.abs() + 1e-30)}
    if d_o is None:
        return out
    D = d(d_o)
    R = torch.zeros_like(S) if d_state is None else d(d_state)
    eR = torch.zeros(B, H, dtype=torch.float64)
    dq, dK, dV, dg, db = (torch.zeros_like(x) for x in (Q, K, V, G, Be))
    eq, ek, ev, eg, eb = (torch.zeros_like(G) for _ in range(5))
    behind = torch.zeros(T, B, H, dtype=torch.float64)  # |k_s| |dv_s| + |q_s| |do_s|
    for t in reversed(range(T)):
        kt, bt, nk, u = K[:, t], Be[:, t], norm(K[:, t]), Be[:, t].unsqueeze(-1) * e[:, t]
        nq, nd, nu, eu = norm(Q[:, t]), norm(D[:, t]), norm(u), bt.abs() * ee[:, t]
        now = held[t] + kt.unsqueeze(-1) * u.unsqueeze(-2)
        sS = around[t] + nk * nu
        dq[:, t] = scale * (now * D[:, t].unsqueeze(-2)).sum(-1)
        eq[:, t] = scale * nd * (eheld[t] + nk * eu + (n + near) * sS)
        R = R + Q[:, t].unsqueeze(-1) * D[:, t].unsqueeze(-2)
        after = behind[t + 1:t + 1 + CHUNK].sum(0) + nq * nd
        sR = size(R) + after
        x = (R * kt.unsqueeze(-1)).sum(-2)
        ex = eR * nk + n * nk * sR
        dV[:, t], ev[:, t] = bt.unsqueeze(-1) * x, bt.abs() * ex
        db[:, t] = (x * e[:, t]).sum(-1)
        eb[:, t] = ex * norm(e[:, t]) + norm(x) * ee[:, t] + n * nk * sR * norm(e[:, t])
        nv, edv = norm(dV[:, t]), bt.abs() * ex
        dK[:, t] = (R * u.unsqueeze(-2)).sum(-1) - (held[t] * dV[:, t].unsqueeze(-2)).sum(-1)
        ek[:, t] = eR * nu + sR * eu + eheld[t] * nv + sS * edv + (n + near) * (sR * nu + sS * nv)
        R = R - kt.unsqueeze(-1) * dV[:, t].unsqueeze(-2)
        eR = torch.clamp((1 - bt * nk ** 2).abs(), min=1) * eR + bt.abs() * nk * n * nk * sR + n * sR
        behind[t] = nk * nv + nq * nd
        dg[:, t] = torch.where(cut[:, t], torch.zeros_like(sS), (held[t] * R).sum((-1, -2)))
        eg[:, t] = eheld[t] * sR + sS * eR + n * sS * (sR + nk * nv)
        R, eR = drop(t, R), drop(t, eR)

    def shared(y, off, x, l):
        y = y.unflatten(2, (x.shape[2], -1))
        off = (off.unflatten(2, (x.shape[2], -1)) + n * y.norm(dim=-1)).sum(3).unsqueeze(-1)
        y = y.sum(3)
        if normalize:
            unit = d(x) / l
            y, off = (y - unit * (unit * y).sum(-1, keepdim=True)) / l, 2 * off / l
        return y, last(y, off)

    one = lambda y, off, dtype: (y, off + HALF[dtype] * (y.abs() + off) + 1e-30)  # noqa: E731
    unit = torch.ones(1, dtype=torch.float64)
    plain = lambda y, off, x: (y.unflatten(2, (x.shape[2], -1)).sum(3),  # noqa: E731
                               last(y.unflatten(2, (x.shape[2], -1)).sum(3),
                                    (off.unflatten(2, (x.shape[2], -1)) + n * y.unflatten(2, (x.shape[2], -1)).norm(dim=-1)).sum(3).unsqueeze(-1) * unit))
    out.update(q=shared(dq, eq, q, lq), k=shared(dK, ek, k, lk), v=plain(dV, ev, v), g=one(dg, eg, g.dtype),
               beta=one(db, eb, beta.dtype), d_state=(R, eR[..., None, None] + EPS * R.abs() + 1e-30))
    return out


def near(got, want):
    """Of ordinary inputs, in the 2-norm of a whole result, where roundings are independent of each other: some 400 of them on a
    term's way, each below EPS of terms whose squares' sum is at most 8^2 times the result's: 8 * 20 EPS; and one rounding."""
    off = (got.detach().double().cpu() - want[0]).norm()
    assert off <= (160 * EPS + HALF[got.dtype]) * want[0].norm(), f"off by {float(off / want[0].norm()):.2e} of the norm"
