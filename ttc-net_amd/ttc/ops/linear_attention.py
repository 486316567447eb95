"""Linear attention with a decay for each head.

With a state ``S [dk, dv]`` for each sequence and head, and ``g = log_gamma`` of the token and head,

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t.

:func:`linear_attention` runs it over whole sequences (prompts, training), :func:`linear_attention_step` over one token
of each sequence of a serving batch, whose states it updates in place.  CUDA tensors go through the kernels of
``ttc_linear_attention`` and ``ttc_linear_attention_step``; CPU tensors, and any call that something observes operator by
operator, run :func:`linear_attention_torch`.
"""
from __future__ import annotations

import struct

import torch

from .._dispatch import traced
from ..solvers._lib import lib
from ._call import DTYPES, check_device, check_types, launch, ptr, recorded_backward, unit_rows

__all__ = ["linear_attention", "linear_attention_step", "linear_attention_torch", "MAX_DIM"]

MAX_DIM = 128         # TTC_LINEAR_ATTENTION_MAX_DIM
RESET = -104.0        # TTC_RESET_LOG_GAMMA
_CHUNK = 64
_BLOCK = struct.Struct("12qd4q12qqqqq3qq4qqqqqq")
_STEP_BLOCK = struct.Struct("10qd4q8qqqq")


def _token_by_token(q, k, v, g, S):
    """A chunk as its recurrence: a token meets nothing but the state, and a reset selects."""
    out = []
    for t in range(q.shape[2]):
        cut = g[:, :, t] < RESET
        S = torch.where(cut[..., None, None], torch.zeros_like(S), S)
        S = S * g[:, :, t].masked_fill(cut, 0.0).exp()[..., None, None] + k[:, :, t].unsqueeze(-1) * v[:, :, t].unsqueeze(-2)
        out.append((S * q[:, :, t].unsqueeze(-1)).sum(-2))
    return torch.stack(out, 2), S


def linear_attention_torch(q, k, v, log_gamma, scale, initial_state=None):
    """:func:`linear_attention` as torch operators: ``(o, final state)``.  Chunks of 64 tokens, products within a chunk,
    the state from chunk to chunk.  A product with a weight of 0 does not drop what is not finite: a chunk that holds such
    values goes token by token.  Where nothing can look at them (operators that are observed; a CUDA tensor, for which the host
    would have to wait) it does not, and they can reach every output of their chunk and head and of those after it."""
    if q.device.type in ("cpu", "cuda"):
        with torch.autocast(q.device.type, enabled=False):  # products in 32 bits, whatever a model's own are in
            return _in_chunks(q, k, v, log_gamma, scale, initial_state)
    return _in_chunks(q, k, v, log_gamma, scale, initial_state)


def _in_chunks(q, k, v, log_gamma, scale, initial_state):
    look = not (q.is_cuda or traced(q, k, v, log_gamma, initial_state))
    finite = lambda *xs: all(bool(x.detach().sum().isfinite()) for x in xs)  # noqa: E731  (or else sums that overflow)
    B, T = q.shape[:2]
    H, dk, dv = log_gamma.shape[-1], q.shape[-1], v.shape[-1]
    wide = lambda x: x.float().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2)  # noqa: E731
    qs, ks, vs = wide(q) * scale, wide(k), wide(v)
    g = log_gamma.float().expand(B, T, H).transpose(1, 2)
    S = q.new_zeros((B, H, dk, dv), dtype=torch.float32) if initial_state is None else initial_state
    whole = look and finite(q, k, v) and bool((log_gamma < torch.inf).all())
    nothing = (qs * ks).sum(-1, keepdim=True) * vs * g.unsqueeze(-1)  # of no tokens: empty, and depends on everything
    out = [nothing] if T == 0 else []
    for at in range(0, T, _CHUNK):
        qc, kc, vc, gc = (x[:, :, at:at + _CHUNK] for x in (qs, ks, vs, g))
        if look and not (finite(S) and (whole or finite(qc, kc, vc) and bool((gc < torch.inf).all()))):
            o, S = _token_by_token(qc, kc, vc, gc, S)
            out.append(o)
            continue
        n = gc.shape[-1]
        reset = gc < RESET  # drops the state: no weight crosses it
        part = reset.long().cumsum(-1)
        sums = gc.masked_fill(reset, 0.0).double().cumsum(-1)  # differences of large sums
        weight = lambda a, ok: torch.where(ok, a, torch.full_like(a, -torch.inf)).exp().float()  # noqa: E731
        low = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        w = weight(sums.unsqueeze(-1) - sums.unsqueeze(-2), low & (part.unsqueeze(-1) == part.unsqueeze(-2)))
        first, last = part == 0, part == part[..., -1:]
        keep = lambda ok, x: torch.where(ok.unsqueeze(-1), x, torch.zeros_like(x))  # noqa: E731
        o = ((qc @ kc.transpose(-1, -2).contiguous()) * w) @ vc
        o = o + keep(first, weight(sums, first).unsqueeze(-1) * (qc @ S))
        S = keep(first[..., -1:], weight(sums[..., -1:], first[..., -1:]).unsqueeze(-1) * S)
        S = S + (kc * weight(sums[..., -1:] - sums, last).unsqueeze(-1)).transpose(-1, -2).contiguous() @ vc
        out.append(o)
    return torch.cat(out, 2).transpose(1, 2).contiguous().to(q.dtype), S + 0


def _gamma_strides(log_gamma):
    """Over batch, tokens and heads; [heads]: one decay for each head."""
    if log_gamma.dim() == 1:
        return 0, 0, log_gamma.stride(0)
    return log_gamma.stride()


def _block(dtype, log_gamma, q, k, v, scale, initial, o, final, backward=0, d_o=None, d_final=None, dq=None, dk=None,
           dv=None, d_gamma=None, d_initial=None, saved=None, space=None):
    B, T = q.shape[:2]
    return _BLOCK.pack(DTYPES[dtype], DTYPES[log_gamma.dtype], log_gamma.dim() == 1, backward, B, T, log_gamma.shape[-1],
                       q.shape[2], k.shape[2], v.shape[2], q.shape[3], v.shape[3], scale, ptr(q), ptr(k), ptr(v),
                       ptr(log_gamma), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *_gamma_strides(log_gamma),
                       ptr(initial), ptr(o), ptr(final), ptr(d_o), *((0, 0, 0) if d_o is None else d_o.stride()[:3]),
                       ptr(d_final), ptr(dq), ptr(dk), ptr(dv), ptr(d_gamma), ptr(d_initial), ptr(saved),
                       0 if saved is None else 4 * saved.numel(), ptr(space), 0 if space is None else space.numel())


def _run(*args, **kw):
    q = args[2]
    block = _block(*args, **kw)
    size = lib.ttc_linear_attention_workspace_bytes(block)
    if size:
        space = torch.empty(size, dtype=torch.uint8, device=q.device)
        block = _block(*args, **kw, space=space)
    launch(lib.ttc_linear_attention, "ttc_linear_attention", block, q.device)


def _forward(q, k, v, log_gamma, scale, initial, want_state, train=False):
    """``(o, final state or None, what the backward wants kept or None)``."""
    B, T = q.shape[:2]
    H = log_gamma.shape[-1]
    o = torch.empty(B, T, H, v.shape[-1], dtype=q.dtype, device=q.device)
    final = torch.empty(B, H, q.shape[-1], v.shape[-1], dtype=torch.float32, device=q.device) if want_state else None
    args = (q.dtype, log_gamma, unit_rows(q), unit_rows(k), unit_rows(v), scale, initial, o, final)
    saved = None
    if train:
        size = lib.ttc_linear_attention_saved_bytes(_block(*args))
        saved = torch.empty(size // 4, dtype=torch.float32, device=q.device) if size else None
    _run(*args, saved=saved)
    return o, final, saved


class _LinearAttentionFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, log_gamma, initial, scale, want_state):
        o, final, saved = _forward(q, k, v, log_gamma, scale, None if initial is None else initial.contiguous(),
                                   want_state, True)
        ctx.save_for_backward(q, k, v, log_gamma, initial, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    def backward(ctx, d_o, d_final):
        q, k, v, log_gamma, initial, saved = ctx.saved_tensors
        needs = ctx.needs_input_grad[:5]
        if d_o is None and d_final is None:
            return (None,) * 7
        recorded = torch.is_grad_enabled()
        if recorded or traced(d_o, d_final, q, k, v, log_gamma, initial):
            form = lambda q, k, v, g, s: linear_attention_torch(q, k, v, g, ctx.scale, s)  # noqa: E731
            return (*recorded_backward(form, (q, k, v, log_gamma, initial), needs, (d_o, d_final), recorded), None, None)
        if d_o is None:
            d_o = torch.zeros(q.shape[0], q.shape[1], log_gamma.shape[-1], v.shape[-1], dtype=q.dtype, device=q.device)
        new = lambda x, wanted: torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None  # noqa: E731
        dq, dk, dv, d_gamma, d_initial = (new(x, n) for x, n in zip((q, k, v, log_gamma, initial), needs))
        _run(q.dtype, log_gamma, unit_rows(q), unit_rows(k), unit_rows(v), ctx.scale,
             None if initial is None else initial.contiguous(), None, None, backward=1, d_o=unit_rows(d_o),
             d_final=None if d_final is None else d_final.contiguous(), dq=dq, dk=dk, dv=dv, d_gamma=d_gamma,
             d_initial=d_initial, saved=saved)
        return dq, dk, dv, d_gamma, d_initial, None, None


def _check(name, q, k, v, log_gamma, dims):
    lead = "[batch, tokens, heads, dim]" if dims == 4 else "[batch, heads, dim]"
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise ValueError(f"{name}: q, k and v {lead} are needed")
    *lead, qh, dk = q.shape
    *k_lead, kh, k_dk = k.shape
    *v_lead, vh, dv = v.shape
    if k_lead != lead or v_lead != lead or k_dk != dk:
        raise ValueError(f"{name}: q, k and v of one batch and number of tokens, q and k of one head size are needed")
    if not (1 <= dk <= MAX_DIM and 1 <= dv <= MAX_DIM):
        raise ValueError(f"{name}: head sizes of 1 to {MAX_DIM} are supported, got {dk} and {dv}")
    check_types(name, q, k, v)
    check_device(name, q, log_gamma)
    if log_gamma.dtype not in (torch.float32, q.dtype):
        raise TypeError(f"{name}: log_gamma of type float32 or {q.dtype} is needed, got {log_gamma.dtype}")
    *g_lead, H = log_gamma.shape
    if g_lead and g_lead != lead:
        raise ValueError(f"{name}: log_gamma [heads] or one for each token and head is needed, got "
                         f"{tuple(log_gamma.shape)}")
    if not (H and qh and kh and vh) or H % qh or H % kh or H % vh:
        raise ValueError(f"{name}: the heads of q, k and v ({qh}, {kh}, {vh}) have to divide those of log_gamma ({H})")
    return H


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_gamma: torch.Tensor, *,
                     scale: float | None = None, initial_state: torch.Tensor | None = None, output_state: bool = False):
    """``o [batch, tokens, heads, dv]``, with ``output_state`` also the final state.

    ``q, k [batch, tokens, heads, dk]``, ``v [batch, tokens, heads, dv]``: float32 or bfloat16, ``dk`` and ``dv`` up to 128,
    any strides over batch, tokens and heads.  ``log_gamma [batch, tokens, heads]``, or ``[heads]`` (one decay for each
    head), float32 or of ``q``'s type; its heads are the output's, and the head counts of ``q``, ``k`` and ``v`` divide
    them: output head ``h`` uses head ``h // (heads // q_heads)`` of ``q`` (a value longer than 128 is several heads that
    share ``q`` and ``k``).  ``scale``: ``dk ** -0.5`` by default.  States are float32 ``[batch, heads, dk, dv]``.

    A ``log_gamma`` below -104 (``exp`` is 0 in 32 bits; ``-inf`` included) drops the state, so that several texts can
    follow each other in one sequence: nothing before it has any effect on what follows, whatever it holds.  Of CUDA calls
    that are observed operator by operator (compiled, under a transform, gradients with ``create_graph``) that holds for
    finite values only.  Differentiable in all tensors.
    """
    H = _check("linear_attention", q, k, v, log_gamma, 4)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if initial_state is not None:
        shape = (q.shape[0], H, q.shape[-1], v.shape[-1])
        if initial_state.shape != shape or initial_state.dtype != torch.float32:
            raise ValueError(f"linear_attention: a float32 state {list(shape)} is needed")
        check_device("linear_attention", q, initial_state)
    if not q.is_cuda or traced(q, k, v, log_gamma, initial_state):
        o, final = linear_attention_torch(q, k, v, log_gamma, scale, initial_state)
    elif torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, log_gamma, initial_state)):
        o, final = _LinearAttentionFunc.apply(q, k, v, log_gamma, initial_state, scale, output_state)
    else:
        o, final, _ = _forward(q, k, v, log_gamma, scale, None if initial_state is None else initial_state.contiguous(),
                               output_state)
    return (o, final) if output_state else o


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_gamma: torch.Tensor, state: torch.Tensor,
                          *, scale: float | None = None, slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each sequence: ``o [batch, heads, dv]``; ``state`` is updated in place.

    ``q, k [batch, heads, dk]``, ``v [batch, heads, dv]``, ``log_gamma [batch, heads]`` or ``[heads]`` as in
    :func:`linear_attention`.  ``state [slots, heads, dk, dv]`` float32 contiguous; ``slots`` (int32 ``[batch]``) names
    each row's place in it, without it row ``b`` has place ``b``.  A row whose slot lies outside (-1: a row that fills up
    a batch of fixed size) is skipped: its output is 0.  Rows must not share a slot.  Not differentiable.
    """
    name = "linear_attention_step"
    H = _check(name, q, k, v, log_gamma, 3)
    B, dk, dv = q.shape[0], q.shape[-1], v.shape[-1]
    scale = dk ** -0.5 if scale is None else float(scale)
    if state.shape[1:] != (H, dk, dv) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{name}: a contiguous float32 state [slots, {H}, {dk}, {dv}] is needed")
    check_device(name, q, state, slots)
    if slots is None:
        if state.shape[0] != B:
            raise ValueError(f"{name}: {B} sequences, {state.shape[0]} states")
    else:
        if slots.shape != (B,) or slots.dtype != torch.int32:
            raise ValueError(f"{name}: int32 slots [{B}] are needed")
        slots = slots.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_gamma.requires_grad
                                    or state.requires_grad):
        raise RuntimeError(f"{name} is not differentiable: call it under torch.no_grad(), or use linear_attention")
    if not q.is_cuda or traced(q, k, v, log_gamma, state, slots):
        return _step_torch(q, k, v, log_gamma, state, scale, slots)
    q, k, v = unit_rows(q), unit_rows(k), unit_rows(v)
    o = q.new_empty((B, H, dv))
    gb, gh = (0, log_gamma.stride(0)) if log_gamma.dim() == 1 else log_gamma.stride()
    block = _STEP_BLOCK.pack(DTYPES[q.dtype], DTYPES[log_gamma.dtype], B, H, q.shape[1], k.shape[1], v.shape[1], dk, dv,
                             state.shape[0], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_gamma.data_ptr(),
                             *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], gb, gh, state.data_ptr(), ptr(slots),
                             o.data_ptr())
    launch(lib.ttc_linear_attention_step, "ttc_linear_attention_step", block, q.device)
    torch.autograd.graph.increment_version(state)  # whoever saved it for a backward has to find out
    return o


def _step_torch(q, k, v, log_gamma, state, scale, slots):
    rows = torch.arange(q.shape[0], device=q.device) if slots is None else slots.long()
    inside = (rows >= 0) & (rows < state.shape[0])
    rows = rows[inside]
    one = lambda x: x[inside].unsqueeze(1)  # noqa: E731
    g = log_gamma if log_gamma.dim() == 1 else one(log_gamma)
    o, S = linear_attention_torch(one(q), one(k), one(v), g, scale, state[rows])
    state[rows] = S
    out = q.new_zeros((q.shape[0], log_gamma.shape[-1], v.shape[-1]))
    out[inside] = o[:, 0]
    return out
