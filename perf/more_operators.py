"""Further sequence operators of this package (``ttc.ops``) as cases that can be timed and checked: the gated
delta rule (prompts, training, single tokens), rotary positions with several axes, and the short causal
convolution in front of a token mixer.

``run`` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the
end), or through the package's entry points where ``own`` is true; ``exact`` in 64 bits from their
definitions.  Everything is made from the seed.

Keys of a case (those that its ``op`` uses):
``op``       "delta" (prompt or training pass) | "step" (one token, state updated in place) | "axes" | "conv" |
             "conv step" (one token, state updated in place)
``B, T``     sequences and tokens;  ``H`` heads of the output;  ``Hk`` heads of queries and keys (and of the turned keys)
``Dk, Dv``   sizes of a key and a value;  ``state``: an initial state comes in and the final one goes out
``norm``     the operator brings queries and keys to length 1 itself (otherwise the keys come so)
``pool``     state slots of a serving process, B of which are in the batch (0: the state is the batch's own)
``D``        size of a head;  ``s0, s1, s2``: pairs that each axis turns;  ``layout`` "half" | "interleaved"
``C, K``     channels and taps;  ``act`` "silu" | "none";  ``bias``
``bf16``     16-bit data (otherwise 32-bit);  ``train``: forward and backward, with all gradients
"""
import math
import os
import sys

import torch

own = False

CHUNK = 64
EPS = 1e-6


def _entry():
    """The package's operators."""
    path = os.path.join(os.getcwd(), "ttc-net_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ttc import ops
    return ops


# ---- cases -----------------------------------------------------------------------------------

def _delta(B, T, H, Dk, Dv, Hk=None, bf16=True, train=False, state=False, norm=True):
    return dict(op="delta", B=B, T=T, H=H, Hk=Hk or H, Dk=Dk, Dv=Dv, bf16=bf16, train=train, state=state, norm=norm)


def _step(B, H, Dk, Dv, Hk=None, bf16=True, pool=0, norm=True):
    return dict(op="step", B=B, H=H, Hk=Hk or H, Dk=Dk, Dv=Dv, bf16=bf16, pool=pool, norm=norm)


def _axes(B, T, H, Hk, D, sections, layout="half", bf16=True, train=False):
    s0, s1, s2 = sections
    return dict(op="axes", B=B, T=T, H=H, Hk=Hk, D=D, s0=s0, s1=s1, s2=s2, layout=layout, bf16=bf16, train=train)


def _conv(B, T, C, K, act="silu", bias=False, bf16=True, train=False, state=False):
    return dict(op="conv", B=B, T=T, C=C, K=K, act=act, bias=bias, bf16=bf16, train=train, state=state)


def _conv_step(B, C, K, act="silu", bias=False, bf16=True, pool=0):
    return dict(op="conv step", B=B, C=C, K=K, act=act, bias=bias, bf16=bf16, pool=pool)


def listed():
    return [
        # one token of one sequence, 8 heads of 64 in fp32: the latency of a single decode step
        dict(_step(1, 8, 64, 64, bf16=False), name="step one sequence"),
        # a serving batch of 192 sequences, their states in a pool of 256 slots
        dict(_step(192, 16, 128, 128, pool=256), name="step batch in a pool"),
        # one long prompt of ragged length: few heads, one chunk after the other
        dict(_delta(1, 16381, 16, 128, 128, state=True), name="delta prompt long"),
        # training on x [4, 2048, .] with the 32 heads of the wide configurations
        dict(_delta(4, 2048, 32, 64, 64, train=True), name="delta train"),
        # fp32 training with shared queries and keys, odd sizes, a state that comes in and goes out, keys already of length 1
        dict(_delta(3, 509, 12, 48, 80, Hk=4, bf16=False, train=True, state=True, norm=False),
             name="delta train ragged fp32"),
        # one decode step for 16 sequences whose text follows pictures: time, height and width, 8 shared key heads
        dict(_axes(16, 1, 32, 8, 128, (16, 24, 24)), name="axes decode"),
        # the prompt of one long video
        dict(_axes(1, 16381, 16, 16, 128, (16, 24, 24)), name="axes prompt long"),
        # fp32 training on pictures (height and width), neighbouring pairs, half of each head turned
        dict(_axes(4, 2048, 16, 16, 64, (0, 8, 8), layout="interleaved", bf16=False, train=True),
             name="axes train interleaved"),
        # one decode step for 16 sequences: queries, keys and values of 16 heads of 128, their states in a pool
        dict(_conv_step(16, 6144, 4, pool=24), name="conv decode"),
        # the same channels over one long prompt
        dict(_conv(1, 16381, 6144, 4), name="conv prompt long"),
        # training on x [4, 2048, .]: 32 heads of 64, and half as many shared ones of keys and values
        dict(_conv(4, 2048, 4096, 4, train=True), name="conv train"),
        # fp32 training with a bias and a state, three taps, odd sizes
        dict(_conv(3, 509, 1111, 3, act="none", bias=True, bf16=False, train=True, state=True), name="conv train odd fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges, below the largest listed one."""
    most = max(_cost(c) for c in listed())
    while True:
        c = _any(rng)
        if _cost(c) <= most:
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _any(rng):
    op = rng.choice(["delta", "delta", "delta", "step", "axes", "conv", "conv step"])
    bf16 = rng.random() < 0.6
    if op in ("delta", "step"):
        H = rng.choice([4, 8, 16, 32, 6, 12, rng.randint(1, 24)])
        Hk = rng.choice([x for x in range(1, H + 1) if H % x == 0] + [H] * 6)
        Dk, Dv = (rng.choice([16, 32, 64, 64, 128, 128, rng.randint(8, 127)]) for _ in range(2))
        norm = rng.random() < 0.6
        if op == "step":
            B = _log_int(rng, 1, max(1, min(512, 48 * 2**20 // (H * Dk * Dv))))
            return _step(B, H, Dk, Dv, Hk, bf16, pool=rng.choice([0, B + rng.randint(0, 16)]), norm=norm)
        train = rng.random() < 0.5
        most = (2**25 if train else 2**26) // (H * max(Dk, 32) * 2)
        B = _log_int(rng, 1, 16)
        return _delta(B, _log_int(rng, 2, max(2, min(8192 if train else 16384, most // B))), H, Dk, Dv, Hk, bf16,
                      train, rng.random() < 0.4, norm)
    if op == "axes":
        D = rng.choice([32, 64, 128, 2 * rng.randint(8, 80)])
        H = rng.choice([4, 8, 16, 32, rng.randint(1, 24)])
        B = _log_int(rng, 1, 64)
        most = 2**26 // (2 * H * D * B)
        pairs = rng.choice([D // 2, rng.randint(3, D // 2)])
        cuts = sorted(rng.choice([(pairs // 4, pairs // 4 + 3 * pairs // 8),
                                  (rng.randint(0, pairs), rng.randint(0, pairs))]))
        return _axes(B, _log_int(rng, 1, max(1, min(16384, most))), H, rng.choice([H, max(1, H // 4)]), D,
                     (cuts[0], cuts[1] - cuts[0], pairs - cuts[1]), rng.choice(["half", "interleaved"]), bf16,
                     rng.random() < 0.5)
    C = rng.choice([8 * _log_int(rng, 8, 1024), _log_int(rng, 16, 8192)])
    K, act, bias = rng.choice([2, 3, 4, 4, 4]), rng.choice(["silu", "silu", "none"]), rng.random() < 0.4
    if op == "conv step":
        B = _log_int(rng, 1, 512)
        return _conv_step(B, C, K, act, bias, bf16, rng.choice([0, B + rng.randint(0, 16)]))
    B = _log_int(rng, 1, 16)
    return _conv(B, _log_int(rng, 1, max(1, min(16384, 2**26 // (B * C)))), C, K, act, bias, bf16, rng.random() < 0.5,
                 rng.random() < 0.4)


def work(c):
    e = 2 if c["bf16"] else 4
    if c["op"] == "step":  # read out at the key, update, read out at the query
        one = c["H"] * c["Dk"] * c["Dv"]
        row = e * (2 * c["Hk"] * c["Dk"] + 2 * c["H"] * c["Dv"] + c["H"]) + 4 * c["H"]
        return {"bytes": c["B"] * (8 * one + row), "flops": c["B"] * 7 * one}
    if c["op"] == "delta":  # the recurrence's own products, and theirs backward
        n, one = c["B"] * c["T"], c["H"] * c["Dk"] * c["Dv"]
        qkv = 2 * c["Hk"] * c["Dk"] + c["H"] * c["Dv"]
        o, gates = c["H"] * c["Dv"], (4 + e) * c["H"]
        states = 8 * c["B"] * one if c["state"] else 0
        if c["train"]:
            return {"bytes": n * (e * (3 * qkv + 2 * o) + 3 * gates) + 3 * states, "flops": n * one * 18}
        return {"bytes": n * (e * (qkv + o) + gates) + states, "flops": n * one * 6}
    if c["op"] == "axes":
        n, passes, pairs = c["B"] * c["T"], 2 if c["train"] else 1, c["s0"] + c["s1"] + c["s2"]
        heads = c["H"] + c["Hk"]
        return {"bytes": passes * (2 * e * n * heads * c["D"] + 24 * n), "flops": passes * 6 * n * heads * pairs}
    if c["op"] == "conv step":
        return {"bytes": e * c["C"] * (c["B"] * 2 * c["K"] + c["K"]), "flops": c["B"] * c["C"] * (2 * c["K"] + 4)}
    n = c["B"] * c["T"] * c["C"]
    return {"bytes": e * n * (5 if c["train"] else 2), "flops": n * (2 * c["K"] + 4) * (3 if c["train"] else 1)}


# ---- inputs ----------------------------------------------------------------------------------

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    c, dev = case, _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = torch.bfloat16 if c["bf16"] else torch.float32
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    s = {"case": c}
    if c["op"] in ("delta", "step"):
        B, T, H, Hk, Dk, Dv = c["B"], c.get("T", 1), c["H"], c["Hk"], c["Dk"], c["Dv"]
        # one projection holds queries, keys and values: the operators get views of it
        qkv = rand(B, T, (2 * Hk * Dk + H * Dv))
        sizes = [Hk * Dk, Hk * Dk, H * Dv]
        if not c["norm"]:  # keys of length 1, as a layer that does that itself hands them over
            k = qkv[..., Hk * Dk:2 * Hk * Dk].unflatten(-1, (Hk, Dk))
            k /= (k * k).sum(-1, keepdim=True).sqrt()
        q, k, v = torch.split(qkv.to(dt), sizes, dim=-1)
        # decays from a memory of 4 tokens to one of 512, head by head, modulated by the data; strengths within (0, 1)
        rate = torch.exp(torch.linspace(math.log(1 / 512), math.log(1 / 4), H, device=dev))
        log_gamma = -rate * torch.nn.functional.softplus(rand(B, T, H))
        s.update(q=q.unflatten(-1, (Hk, Dk)), k=k.unflatten(-1, (Hk, Dk)), v=v.unflatten(-1, (H, Dv)),
                 log_gamma=log_gamma, beta=torch.sigmoid(rand(B, T, H)).to(dt))
        if c["op"] == "step":
            for name in ("q", "k", "v", "log_gamma", "beta"):
                s[name] = s[name].squeeze(1)
            s["state"] = rand(c["pool"] or B, H, Dk, Dv)
            s["slots"] = torch.randperm(c["pool"], generator=gen, device=dev)[:B].to(torch.int32) if c["pool"] else None
        else:
            s["state"] = rand(B, H, Dk, Dv) if c["state"] else None
            if c["train"]:
                s["d_o"] = rand(B, T, H, Dv).to(dt)
                s["d_state"] = rand(B, H, Dk, Dv) * 0.1 if c["state"] else None
    elif c["op"] == "axes":
        B, T, H, Hk, D = (c[n] for n in ("B", "T", "H", "Hk", "D"))
        qkv = rand(B, T, (H + 2 * Hk) * D).to(dt).unflatten(-1, (H + 2 * Hk, D))
        sections = (c["s0"], c["s1"], c["s2"])
        pairs = sum(sections)
        length = max(2 * T, 4096)
        angle = torch.arange(length, dtype=torch.float64, device=dev)[:, None] * torch.pow(
            10000.0, -torch.arange(pairs, dtype=torch.float64, device=dev) / pairs)
        # frames of 16 x 16 patches (a token of text has one position on all axes: the decode step's)
        at = torch.arange(T, device=dev)
        grid = torch.stack([at // 256, at // 16 % 16, at % 16], -1)
        start = torch.randint(0, length - T + 1, (B, 1, 1), generator=gen, device=dev)
        s.update(q=qkv[:, :, :H], k=qkv[:, :, H:H + Hk], table=torch.stack([angle.cos(), angle.sin()], -1).float(),
                 positions=start + grid, sections=sections)
        if c["train"]:
            s.update(d_q=rand(B, T, H, D).to(dt), d_k=rand(B, T, Hk, D).to(dt))
    else:
        B, T, C, K = c["B"], c.get("T", 1), c["C"], c["K"]
        # queries, keys and values are a part of a wider projection
        s.update(x=rand(B, T, C + 16).to(dt)[..., :C], weight=(rand(C, K) / math.sqrt(K)).to(dt),
                 bias=(0.1 * rand(C)).to(dt) if c["bias"] else None)
        if c["op"] == "conv step":
            s["x"] = s["x"].squeeze(1)
            s["state"] = rand(c["pool"] or B, K - 1, C).to(dt)
            s["slots"] = torch.randperm(c["pool"], generator=gen, device=dev)[:B].to(torch.int32) if c["pool"] else None
        else:
            s["state"] = rand(B, K - 1, C).to(dt) if c["state"] else None
            if c["train"]:
                s["d_y"] = rand(B, T, C).to(dt)
                s["d_state"] = rand(B, K - 1, C).to(dt) if c["state"] else None
    return s


# ---- plain forms -----------------------------------------------------------------------------

def _heads(x, H):
    """[B, T, heads, D] in 32 bits as [B, H, T, D], shared heads repeated."""
    return x.float().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2).contiguous()


def _unit(x):
    x = x.float()
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _inverse(low):
    """Of the unit lower triangles I + low, [.., n, n] with n a power of two: from blocks of 1 to blocks twice as
    large, [[a, 0], [c, b]]^-1 = [[a^-1, 0], [-b^-1 c a^-1, b^-1]]."""
    n, size = low.shape[-1], 1
    inv = torch.ones(*low.shape[:-2], n, 1, 1, device=low.device)
    while size < n:
        blocks = low.unflatten(-2, (-1, 2 * size)).unflatten(-1, (-1, 2 * size))
        same = torch.arange(n // (2 * size), device=low.device)
        c = blocks[..., same, :, same, :].movedim(0, -3)[..., size:, :size].contiguous()
        a, b = inv[..., 0::2, :, :].contiguous(), inv[..., 1::2, :, :].contiguous()
        joined = -torch.matmul(torch.matmul(b, c), a)
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([joined, b], -1)], -2)
        size *= 2
    return inv.squeeze(-3)


def _plain_delta(q, k, v, log_gamma, beta, state, norm):
    """Chunks of 64 tokens: what each token adds to the state is a triangular system in the chunk and a product
    with the state in front of it, chunk after chunk."""
    B, T, H = log_gamma.shape
    Dk, Dv, dt = q.shape[-1], v.shape[-1], q.dtype
    if norm:
        q, k = _unit(q), _unit(k)
    n = -(-T // CHUNK)
    pad = lambda x: torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - T)).unflatten(2, (n, CHUNK))  # noqa: E731
    q, k, v = pad(_heads(q, H)) * Dk ** -0.5, pad(_heads(k, H)), pad(_heads(v, H))
    gate = lambda x: pad(x.float().transpose(1, 2).unsqueeze(-1))  # noqa: E731
    g, strength = gate(log_gamma).squeeze(-1).cumsum(-1), gate(beta)                     # [B, H, n, CHUNK(, 1)]
    late = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).triu(1)
    w = (g.unsqueeze(-1) - g.unsqueeze(-2)).masked_fill(late, -math.inf).exp()
    kt = k.transpose(-1, -2).contiguous()
    inverse = _inverse((torch.matmul(k * strength, kt) * w).tril(-1))
    grown = g.exp().unsqueeze(-1)
    own_part = torch.matmul(inverse, v * strength)
    read = torch.matmul(inverse, k * (strength * grown))
    scores = torch.matmul(q, kt) * w
    late_keys = (k * (g[..., -1:] - g).exp().unsqueeze(-1)).transpose(-1, -2).contiguous()
    S = torch.zeros(B, H, Dk, Dv, device=q.device) if state is None else state
    out = []
    for i in range(n):
        u = own_part[:, :, i] - torch.matmul(read[:, :, i], S)
        out.append(torch.matmul(q[:, :, i] * grown[:, :, i], S) + torch.matmul(scores[:, :, i], u))
        S = S * grown[:, :, i, -1:] + torch.matmul(late_keys[:, :, i], u)
    o = torch.cat(out, 2)[:, :, :T].transpose(1, 2).contiguous().to(dt)
    return (o, S) if state is not None else (o, None)


def _plain_step(q, k, v, log_gamma, beta, pool, slots, norm):
    H = log_gamma.shape[1]
    Dk, dt = q.shape[-1], q.dtype
    if norm:
        q, k = _unit(q), _unit(k)
    q, k, v = (x.float().repeat_interleave(H // x.shape[1], dim=1) for x in (q, k, v))
    state = (pool if slots is None else pool[slots.long()]) * log_gamma.exp()[..., None, None]
    u = beta.float().unsqueeze(-1) * (v - (state * k.unsqueeze(-1)).sum(-2))
    state = state + k.unsqueeze(-1) * u.unsqueeze(-2)
    o = (state * (q * Dk ** -0.5).unsqueeze(-1)).sum(-2)
    if slots is None:
        pool.copy_(state)
    else:
        pool[slots.long()] = state
    return o.to(dt)


def _plain_axes(q, k, table, positions, sections, layout):
    at = torch.repeat_interleave(torch.arange(3, device=q.device), torch.tensor(sections, device=q.device),
                                 output_size=table.shape[1])
    cs = table[positions[..., at], torch.arange(table.shape[1], device=q.device)]        # [B, T, pairs, 2]
    cos, sin = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    rot = 2 * table.shape[1]

    def turn(x):
        xf = x.float()
        if layout == "half":
            a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([turned, xf[..., rot:]], -1).to(x.dtype)

    return turn(q), turn(k)


def _act(y, act):
    return y * torch.sigmoid(y) if act == "silu" else y


def _plain_conv(x, weight, bias, state, act):
    B, T, C = x.shape
    K = weight.shape[1]
    front = x.new_zeros(B, K - 1, C) if state is None else state
    wide = torch.cat([front, x], 1)
    wf, w = wide.float(), weight.float()
    y = sum(wf[:, j:j + T] * w[:, j] for j in range(K))
    if bias is not None:
        y = y + bias.float()
    return _act(y, act).to(x.dtype), wide[:, T:] if state is not None else None


def _plain_conv_step(x, pool, weight, bias, slots, act):
    rows = slice(None) if slots is None else slots.long()
    wide = torch.cat([pool[rows], x.unsqueeze(1)], 1)
    y = (wide.float() * weight.float().t()).sum(1)
    if bias is not None:
        y = y + bias.float()
    pool[rows] = wide[:, 1:]
    return _act(y, act).to(x.dtype)


# ---- one pass --------------------------------------------------------------------------------

def _with_grads(f, inputs, names, d_out):
    """f(inputs) and the gradients of the named inputs for the outputs' gradients d_out."""
    leaves = {n: inputs[n].detach().requires_grad_() for n in names if inputs[n] is not None}
    out = f(dict(inputs, **leaves))
    pairs = [(o, d) for o, d in zip(out, d_out) if o is not None and d is not None]
    got = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs])
    res = {"out%d" % i: o.detach() for i, o in enumerate(out) if o is not None}
    res.update(("d_" + n, g) for n, g in zip(leaves, got))
    return res


def run(s):
    c = s["case"]
    if c["op"] == "step":
        args = (s["q"], s["k"], s["v"], s["log_gamma"], s["beta"], s["state"])
        if own:
            o = _entry().delta_rule_step(*args, slots=s["slots"], normalize=c["norm"], eps=EPS)
        else:
            o = _plain_step(*args, s["slots"], c["norm"])
        return {"out0": o, "state": s["state"]}
    if c["op"] == "conv step":
        if own:
            y = _entry().causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"],
                                          activation=c["act"])
        else:
            y = _plain_conv_step(s["x"], s["state"], s["weight"], s["bias"], s["slots"], c["act"])
        return {"out0": y, "state": s["state"]}
    if c["op"] == "delta":
        def delta(x):
            args = (x["q"], x["k"], x["v"], x["log_gamma"], x["beta"])
            if own:
                o = _entry().delta_rule(*args, initial_state=x["state"], output_state=c["state"], normalize=c["norm"],
                                        eps=EPS)
                return o if c["state"] else (o, None)
            return _plain_delta(*args, x["state"], c["norm"])
        f, names, d_out = delta, ("q", "k", "v", "log_gamma", "beta", "state"), ("d_o", "d_state")
    elif c["op"] == "axes":
        def turn(x):
            args = (x["q"], x["k"], x["table"], x["positions"], x["sections"])
            return _entry().rotary_axes(*args, layout=c["layout"]) if own else _plain_axes(*args, c["layout"])
        f, names, d_out = turn, ("q", "k"), ("d_q", "d_k")
    else:
        def conv(x):
            if own:
                y = _entry().causal_conv(x["x"], x["weight"], x["bias"], activation=c["act"], initial_state=x["state"],
                                         output_state=c["state"])
                return y if c["state"] else (y, None)
            return _plain_conv(x["x"], x["weight"], x["bias"], x["state"], c["act"])
        f, names, d_out = conv, ("x", "weight", "bias", "state"), ("d_y", "d_state")
    if c["train"]:
        return _with_grads(f, s, names, [s[d] for d in d_out])
    return {"out%d" % i: o for i, o in enumerate(f(s)) if o is not None}


# ---- 64 bits ---------------------------------------------------------------------------------

def _exact_delta(s, c, d_o=None, d_state=None):
    """Token by token, forwards for the outputs and queries' gradients, backwards for the others."""
    H, Dk, Dv, B, T = c["H"], c["Dk"], c["Dv"], c["B"], c.get("T", 1)
    scale = Dk ** -0.5
    length = lambda x: (x.double().square().sum(-1, keepdim=True) + EPS).sqrt() if c["norm"] else 1.0  # noqa: E731
    wide = lambda x: x.double().repeat_interleave(H // x.shape[2], dim=2)  # noqa: E731
    lq, lk = length(s["q"]), length(s["k"])
    q, k, v = wide(s["q"] / lq), wide(s["k"] / lk), wide(s["v"])
    decay, beta = s["log_gamma"].double().exp(), s["beta"].double()
    S = q.new_zeros(B, H, Dk, Dv) if s["state"] is None else s["state"].double()
    do = None if d_o is None else d_o.double() * scale
    o, e = q.new_empty(B, T, H, Dv), q.new_empty(B, T, H, Dv)
    before = None if do is None else q.new_empty(T, B, H, Dk, Dv)  # the decayed state that token t meets
    for t in range(T):
        S = S * decay[:, t, :, None, None]
        if before is not None:
            before[t] = S
        e[:, t] = v[:, t] - (S * k[:, t, :, :, None]).sum(-2)
        S = S + k[:, t, :, :, None] * (beta[:, t, :, None] * e[:, t])[:, :, None, :]
        o[:, t] = (S * q[:, t, :, :, None]).sum(-2) * scale
    res = {"out0": o}
    if c.get("state") or c["op"] == "step":
        res["out1"] = S
    if do is None:
        return res
    R = torch.zeros_like(S) if d_state is None else d_state.double()
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, decay, beta))
    for t in reversed(range(T)):
        kt, bt = k[:, t, :, :, None], beta[:, t, :, None]
        u = bt * e[:, t]
        now = before[t] + kt * u[:, :, None, :]
        dq[:, t] = (now * do[:, t, :, None, :]).sum(-1)
        R = R + q[:, t, :, :, None] * do[:, t, :, None, :]
        du = (R * kt).sum(-2)
        db[:, t], dv[:, t] = (du * e[:, t]).sum(-1), bt * du
        dk[:, t] = (R * u[:, :, None, :]).sum(-1) - (before[t] * dv[:, t, :, None, :]).sum(-1)
        R = R - kt * dv[:, t, :, None, :]
        dg[:, t] = (R * before[t]).sum((-1, -2))
        R = R * decay[:, t, :, None, None]
    del before

    def shared(d, x, length):
        d = d.unflatten(2, (x.shape[2], -1)).sum(3)
        if not c["norm"]:
            return d
        unit = x.double() / length
        return (d - unit * (unit * d).sum(-1, keepdim=True)) / length

    res.update(d_q=shared(dq, s["q"], lq), d_k=shared(dk, s["k"], lk), d_v=dv, d_log_gamma=dg, d_beta=db)
    if s["state"] is not None:
        res["d_state"] = R
    return res


def _exact_axes(x, s, c, sign):
    """Complex numbers times the table's, pair by pair."""
    parts, first = [], 0
    for axis, n in enumerate(s["sections"]):
        parts.append(s["table"].double()[s["positions"][..., axis], first:first + n])
        first += n
    cs = torch.cat(parts, -2)
    z = torch.complex(cs[..., 0], sign * cs[..., 1]).unsqueeze(-2)
    rot, xd = 2 * first, x.double()
    part = xd[..., :rot].unflatten(-1, (2, first) if c["layout"] == "half" else (first, 2))
    along = -2 if c["layout"] == "half" else -1
    turned = torch.complex(part.select(along, 0).contiguous(), part.select(along, 1).contiguous()) * z
    return torch.cat([torch.stack([turned.real, turned.imag], along).flatten(-2), xd[..., rot:]], -1)


def _exact_conv(s, c):
    B, C, K, T = c["B"], c["C"], c["K"], c["T"]
    w = s["weight"].double()
    front = torch.zeros(B, K - 1, C, dtype=torch.float64, device=w.device) if s["state"] is None else s["state"].double()
    wide = torch.cat([front, s["x"].double()], 1)
    y = torch.zeros(B, T, C, dtype=torch.float64, device=w.device) if s["bias"] is None else (
        s["bias"].double().expand(B, T, C).clone())
    for lag in range(K):  # the input `lag` tokens back meets tap K - 1 - lag
        y += wide[:, K - 1 - lag:K - 1 - lag + T] * w[:, K - 1 - lag]
    sig = torch.sigmoid(y)
    res = {"out0": y * sig if c["act"] == "silu" else y}
    if c["state"]:
        res["out1"] = wide[:, wide.shape[1] - (K - 1):]
    if not c["train"]:
        return res
    d = s["d_y"].double()
    if c["act"] == "silu":
        d = d * (sig * (1 + y * (1 - sig)))
    d_wide = torch.zeros_like(wide)
    dw = torch.empty_like(w)
    for j in range(K):
        d_wide[:, j:j + T] += d * w[:, j]
        dw[:, j] = (d * wide[:, j:j + T]).sum((0, 1))
    if c["state"]:
        d_wide[:, d_wide.shape[1] - (K - 1):] += s["d_state"].double()
        res["d_state"] = d_wide[:, :K - 1]
    res.update(d_x=d_wide[:, K - 1:], d_weight=dw)
    if s["bias"] is not None:
        res["d_bias"] = d.sum((0, 1))
    return res


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "delta":
        return _exact_delta(s, c, s.get("d_o"), s.get("d_state"))
    if c["op"] == "step":
        rows = slice(None) if s["slots"] is None else s["slots"].long()
        at = dict(s, state=s["state"][rows],
                  **{n: s[n].unsqueeze(1) for n in ("q", "k", "v", "log_gamma", "beta")})
        got = _exact_delta(at, c)
        pool = s["state"].double()
        pool[rows] = got["out1"]
        return {"out0": got["out0"][:, 0], "state": pool}
    if c["op"] == "axes":
        res = {"out%d" % i: _exact_axes(s[n], s, c, 1.0) for i, n in enumerate("qk")}
        if c["train"]:
            res.update(("d_" + n, _exact_axes(s["d_" + n], s, c, -1.0)) for n in "qk")
        return res
    if c["op"] == "conv step":
        rows = slice(None) if s["slots"] is None else s["slots"].long()
        at = dict(s, x=s["x"].unsqueeze(1), state=s["state"][rows])
        got = _exact_conv(at, dict(c, T=1, state=True, train=False))
        pool = s["state"].double()
        pool[rows] = got["out1"]
        return {"out0": got["out0"][:, 0], "state": pool}
    return _exact_conv(s, c)
