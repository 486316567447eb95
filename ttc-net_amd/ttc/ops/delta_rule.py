"""The gated delta rule: linear attention whose state forgets, before it takes up a value, what it holds at that key.

With a state ``S [dk, dv]`` for each sequence and head, ``g = log_gamma`` and ``b = beta`` of the token and head,

    S_t = exp(g_t) (I - b_t k_t k_t^T) S_{t-1} + b_t k_t v_t^T,    o_t = scale * S_t^T q_t.

:func:`delta_rule` runs it over whole sequences (prompts, training), :func:`delta_rule_step` over one token of each sequence
of a serving batch, whose states it updates in place.  CUDA tensors go through the kernels of ``ttc_delta_rule`` and
``ttc_delta_rule_step``; CPU tensors, and any call that something observes operator by operator, run
:func:`delta_rule_torch`.
"""
from __future__ import annotations

import struct

import torch

from .._dispatch import traced
from ..solvers._lib import lib
from ._call import DTYPES, check_device, check_types, launch, ptr, recorded_backward, unit_rows, with_spaces
from .linear_attention import MAX_DIM, RESET

__all__ = ["delta_rule", "delta_rule_step", "delta_rule_torch"]

_CHUNK = 64
_BLOCK = struct.Struct("13q2d5q15q3qq3qq5qq4q")
_STEP_BLOCK = struct.Struct("12q2d5q10q3q")


def _token_by_token(q, k, v, g, beta, S):
    """A chunk as its recurrence: a token meets nothing but the state, and a reset selects."""
    out = []
    for t in range(q.shape[2]):
        cut = g[:, :, t] < RESET
        S = torch.where(cut[..., None, None], torch.zeros_like(S), S)
        S = S * g[:, :, t].masked_fill(cut, 0.0).exp()[..., None, None]
        u = beta[:, :, t, None] * (v[:, :, t] - (S * k[:, :, t].unsqueeze(-1)).sum(-2))
        S = S + k[:, :, t].unsqueeze(-1) * u.unsqueeze(-2)
        out.append((S * q[:, :, t].unsqueeze(-1)).sum(-2))
    return torch.stack(out, 2), S


def delta_rule_torch(q, k, v, log_gamma, beta, scale, initial_state=None, normalize=False, eps=1e-6):
    """:func:`delta_rule` as torch operators: ``(o, final state)``.  Chunks of 64 tokens: a triangular system and products in
    a chunk, the state from chunk to chunk.  A product with a weight of 0 does not drop what is not finite: a chunk that holds
    such values goes token by token.  Where nothing can look at them (operators that are observed; a CUDA tensor, for which the
    host would have to wait) it does not, and they can reach every output of their chunk and head and of those after it."""
    if q.device.type in ("cpu", "cuda"):
        with torch.autocast(q.device.type, enabled=False):  # products in 32 bits, whatever a model's own are in
            return _in_chunks(q, k, v, log_gamma, beta, scale, initial_state, normalize, eps)
    return _in_chunks(q, k, v, log_gamma, beta, scale, initial_state, normalize, eps)


def _in_chunks(q, k, v, log_gamma, beta, scale, initial_state, normalize, eps):
    look = not (q.is_cuda or traced(q, k, v, log_gamma, beta, initial_state))
    finite = lambda *xs: all(bool(x.detach().sum().isfinite()) for x in xs)  # noqa: E731  (or else sums that overflow)
    B, T, H = log_gamma.shape
    dk, dv = q.shape[-1], v.shape[-1]
    wide = lambda x: x.float().repeat_interleave(H // x.shape[2], dim=2).transpose(1, 2)  # noqa: E731
    unit = lambda x: x * torch.rsqrt((x * x).sum(-1, keepdim=True) + eps) if normalize else x  # noqa: E731
    qs, ks, vs = unit(wide(q)) * scale, unit(wide(k)), wide(v)
    g, be = log_gamma.float().transpose(1, 2), beta.float().transpose(1, 2)
    S = q.new_zeros((B, H, dk, dv), dtype=torch.float32) if initial_state is None else initial_state
    # In a call that holds such values, chunks with a reset go token by token too: their gradients pass it otherwise
    whole = look and finite(qs, ks, vs, be) and bool((g < torch.inf).all())
    # of no tokens: empty, and depends on everything
    out = [(qs * ks).sum(-1, keepdim=True) * vs * (g * be).unsqueeze(-1)] if T == 0 else []
    for at in range(0, T, _CHUNK):
        qc, kc, vc, gc, bc = (x[:, :, at:at + _CHUNK] for x in (qs, ks, vs, g, be))
        if look and not (finite(S) and (whole or (finite(qc, kc, vc, bc) and bool(((gc < torch.inf) & (gc >= RESET)).all())))):
            o, S = _token_by_token(qc, kc, vc, gc, bc, S)
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
        kt, grown = kc.transpose(-1, -2).contiguous(), weight(sums, first).unsqueeze(-1)
        triangle = (kc @ kt) * w.tril(-1) * bc.unsqueeze(-2)
        e = torch.linalg.solve_triangular(triangle, vc - keep(first, grown * (kc @ S)), upper=False, unitriangular=True)
        u = bc.unsqueeze(-1) * e
        out.append(((qc @ kt) * w) @ u + keep(first, grown * (qc @ S)))
        S = keep(first[..., -1:], weight(sums[..., -1:], first[..., -1:]).unsqueeze(-1) * S)
        S = S + (kc * weight(sums[..., -1:] - sums, last).unsqueeze(-1)).transpose(-1, -2).contiguous() @ u
    return torch.cat(out, 2).transpose(1, 2).contiguous().to(q.dtype), S + 0


def _block(q, k, v, log_gamma, beta, scale, normalize, eps, initial, o, final, backward=0, d_o=None, d_final=None, dq=None,
           dk=None, dv=None, d_gamma=None, d_beta=None, d_initial=None):
    B, T = q.shape[:2]
    return _BLOCK.pack(DTYPES[q.dtype], DTYPES[log_gamma.dtype], DTYPES[beta.dtype], normalize, backward, B, T,
                       log_gamma.shape[-1], q.shape[2], k.shape[2], v.shape[2], q.shape[3], v.shape[3], scale, eps, ptr(q),
                       ptr(k), ptr(v), ptr(log_gamma), ptr(beta), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                       *log_gamma.stride(), *beta.stride(), ptr(initial), ptr(o), ptr(final), ptr(d_o),
                       *((0, 0, 0) if d_o is None else d_o.stride()[:3]), ptr(d_final), ptr(dq), ptr(dk), ptr(dv), ptr(d_gamma),
                       ptr(d_beta), ptr(d_initial), 0, 0, 0, 0)  # what is kept for the backward, the workspace


def _run(block, saved, device):
    if saved is not None:
        block = with_spaces(block, saved, None)  # the workspace holds what is not kept
    size = lib.ttc_delta_rule_workspace_bytes(block)
    if size:
        space = torch.empty(size, dtype=torch.uint8, device=device)
        block = with_spaces(block, space)
    launch(lib.ttc_delta_rule, "ttc_delta_rule", block, device)


def _forward(q, k, v, log_gamma, beta, scale, normalize, eps, initial, want_state, train=False):
    """``(o, final state or None, what the backward needs kept or None)``."""
    B, T = q.shape[:2]
    H = log_gamma.shape[-1]
    o = torch.empty(B, T, H, v.shape[-1], dtype=q.dtype, device=q.device)
    final = torch.empty(B, H, q.shape[-1], v.shape[-1], dtype=torch.float32, device=q.device) if want_state else None
    args = (unit_rows(q), unit_rows(k), unit_rows(v), log_gamma, beta, scale, normalize, eps, initial, o, final)
    block, saved = _block(*args), None  # args: what was copied for the block lives until the launch
    if train:
        saved = torch.empty(max(lib.ttc_delta_rule_saved_bytes(block), 1), dtype=torch.uint8, device=q.device)
    _run(block, saved, q.device)
    return o, final, saved


class _DeltaRuleFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, log_gamma, beta, initial, scale, normalize, eps, want_state):
        o, final, saved = _forward(q, k, v, log_gamma, beta, scale, normalize, eps,
                                   None if initial is None else initial.contiguous(), want_state, True)
        ctx.save_for_backward(q, k, v, log_gamma, beta, initial, saved)
        ctx.args = (scale, normalize, eps)
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    def backward(ctx, d_o, d_final):
        q, k, v, log_gamma, beta, initial, saved = ctx.saved_tensors
        needs = ctx.needs_input_grad[:6]
        if d_o is None and d_final is None:
            return (None,) * 10
        recorded = torch.is_grad_enabled()
        if recorded or traced(d_o, d_final, q, k, v, log_gamma, beta, initial):
            scale, normalize, eps = ctx.args
            form = lambda q, k, v, g, b, s: delta_rule_torch(q, k, v, g, b, scale, s, normalize, eps)  # noqa: E731
            return (*recorded_backward(form, (q, k, v, log_gamma, beta, initial), needs, (d_o, d_final), recorded), None, None,
                    None, None)
        if d_o is None:
            d_o = torch.zeros(q.shape[0], q.shape[1], log_gamma.shape[-1], v.shape[-1], dtype=q.dtype, device=q.device)
        new = lambda x, wanted: torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None  # noqa: E731
        grads = tuple(new(x, n) for x, n in zip((q, k, v, log_gamma, beta, initial), needs))
        args = (unit_rows(q), unit_rows(k), unit_rows(v), log_gamma, beta, *ctx.args, None, None, None, 1, unit_rows(d_o),
                None if d_final is None else d_final.contiguous(), *grads)
        _run(_block(*args), saved, q.device)
        return (*grads, None, None, None, None)


def _check(name, q, k, v, log_gamma, beta, eps, dims):
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
    check_device(name, q, log_gamma, beta)
    for x, what in ((log_gamma, "log_gamma"), (beta, "beta")):
        if x.dtype not in (torch.float32, q.dtype):
            raise TypeError(f"{name}: {what} of type float32 or {q.dtype} is needed, got {x.dtype}")
        if x.dim() != dims - 1 or list(x.shape[:-1]) != lead or x.shape != log_gamma.shape:
            raise ValueError(f"{name}: one {what} for each token and head is needed, got {tuple(x.shape)}")
    H = log_gamma.shape[-1]
    if not (H and qh and kh and vh) or H % qh or H % kh or H % vh:
        raise ValueError(f"{name}: the heads of q, k and v ({qh}, {kh}, {vh}) have to divide those of log_gamma ({H})")
    if not eps >= 0:
        raise ValueError(f"{name}: eps of at least 0 is needed, got {eps}")
    return H


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_gamma: torch.Tensor, beta: torch.Tensor, *,
               scale: float | None = None, initial_state: torch.Tensor | None = None, output_state: bool = False,
               normalize: bool = False, eps: float = 1e-6):
    """``o [batch, tokens, heads, dv]``, with ``output_state`` also the final state.

    ``q, k [batch, tokens, heads, dk]``, ``v [batch, tokens, heads, dv]``: float32 or bfloat16, ``dk`` and ``dv`` up to 128,
    any strides over batch, tokens and heads.  ``log_gamma`` and ``beta [batch, tokens, heads]``: float32 or of ``q``'s type,
    any strides; their heads are the output's, and the head counts of ``q``, ``k`` and ``v`` divide them: output head ``h``
    uses head ``h // (heads // q_heads)`` of ``q``.  ``scale``: ``dk ** -0.5`` by default.  States are float32
    ``[batch, heads, dk, dv]``.

    ``normalize`` takes ``q / sqrt(|q|^2 + eps)`` and ``k / sqrt(|k|^2 + eps)`` in the place of ``q`` and ``k`` (in 32 bits,
    without copies of them).  Where it is not set, keys have to be of about length 1: each ``beta |k|^2`` above 2 makes the state
    grow, as the recurrence itself does.

    A ``log_gamma`` below -104 (``exp`` is 0 in 32 bits; ``-inf`` included) drops the state, so that several texts can
    follow each other in one sequence: nothing before it has any effect on what follows, whatever it holds.  Tokens have no
    effect on earlier ones, whatever they hold.  Of CUDA calls that are observed operator by operator (compiled, under a
    transform, gradients with ``create_graph``) both hold for finite values only.  Differentiable in all tensors; a call that
    is to be differentiated keeps, for each chunk of 64 tokens (32 in float32) and head, the state in front of it and some
    values of each token in 32 bits.
    """
    name = "delta_rule"
    H = _check(name, q, k, v, log_gamma, beta, eps, 4)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if initial_state is not None:
        shape = (q.shape[0], H, q.shape[-1], v.shape[-1])
        if initial_state.shape != shape or initial_state.dtype != torch.float32:
            raise ValueError(f"{name}: a float32 state {list(shape)} is needed")
        check_device(name, q, initial_state)
    tensors = (q, k, v, log_gamma, beta, initial_state)
    if not q.is_cuda or traced(*tensors):
        o, final = delta_rule_torch(q, k, v, log_gamma, beta, scale, initial_state, normalize, eps)
    elif torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        o, final = _DeltaRuleFunc.apply(*tensors, scale, bool(normalize), float(eps), output_state)
    else:
        o, final, _ = _forward(q, k, v, log_gamma, beta, scale, bool(normalize), float(eps),
                               None if initial_state is None else initial_state.contiguous(), output_state)
    return (o, final) if output_state else o


def delta_rule_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_gamma: torch.Tensor, beta: torch.Tensor,
                    state: torch.Tensor, *, scale: float | None = None, slots: torch.Tensor | None = None,
                    normalize: bool = False, eps: float = 1e-6) -> torch.Tensor:
    """One token of each sequence: ``o [batch, heads, dv]``; ``state`` is updated in place.

    ``q, k [batch, heads, dk]``, ``v [batch, heads, dv]``, ``log_gamma`` and ``beta [batch, heads]`` and the other arguments as
    in :func:`delta_rule`.  ``state [slots, heads, dk, dv]`` float32 contiguous; ``slots`` (int32 ``[batch]``) names each row's
    place in it, without it row ``b`` has place ``b``.  A row whose slot lies outside (-1: a row that fills up a batch of fixed
    size) is skipped: its output is 0.  Rows must not share a slot.  Not differentiable.
    """
    name = "delta_rule_step"
    H = _check(name, q, k, v, log_gamma, beta, eps, 3)
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
                                    or beta.requires_grad or state.requires_grad):
        raise RuntimeError(f"{name} is not differentiable: call it under torch.no_grad(), or use delta_rule")
    if not q.is_cuda or traced(q, k, v, log_gamma, beta, state, slots):
        return _step_torch(q, k, v, log_gamma, beta, state, scale, slots, normalize, eps)
    q, k, v = unit_rows(q), unit_rows(k), unit_rows(v)
    o = q.new_empty((B, H, dv))
    block = _STEP_BLOCK.pack(DTYPES[q.dtype], DTYPES[log_gamma.dtype], DTYPES[beta.dtype], bool(normalize), B, H, q.shape[1],
                             k.shape[1], v.shape[1], dk, dv, state.shape[0], scale, eps, q.data_ptr(), k.data_ptr(),
                             v.data_ptr(), log_gamma.data_ptr(), beta.data_ptr(), *q.stride()[:2], *k.stride()[:2],
                             *v.stride()[:2], *log_gamma.stride(), *beta.stride(), state.data_ptr(), ptr(slots), o.data_ptr())
    launch(lib.ttc_delta_rule_step, "ttc_delta_rule_step", block, q.device)
    torch.autograd.graph.increment_version(state)  # whoever saved it for a backward has to find out
    return o


def _step_torch(q, k, v, log_gamma, beta, state, scale, slots, normalize, eps):
    rows = torch.arange(q.shape[0], device=q.device) if slots is None else slots.long()
    inside = (rows >= 0) & (rows < state.shape[0])
    rows = rows[inside]
    one = lambda x: x[inside].unsqueeze(1)  # noqa: E731
    o, S = delta_rule_torch(one(q), one(k), one(v), one(log_gamma), one(beta), scale, state[rows], normalize, eps)
    state[rows] = S
    out = q.new_zeros((q.shape[0], log_gamma.shape[-1], v.shape[-1]))
    out[inside] = o[:, 0]
    return out
