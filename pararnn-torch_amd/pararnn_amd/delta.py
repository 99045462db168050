"""The gated delta rule: whole sequences, their gradients, single tokens.

For every head, with a state ``S`` ``(Dk, Dv)`` held in float32, a log decay ``g_t`` and a rate
``beta_t``, a token writes what the decayed state lacks of its value at its key:

    u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t),
    S_t = exp(g_t) S_{t-1} + k_t u_t^T,            o_t = scale S_t^T q_t.

``delta_rule`` runs prompts and training sequences in chunks of 64 tokens (a triangular system per
chunk, the state from chunk to chunk), ``delta_rule_step`` one token per session on a state or a
pool of states, in place.  Layouts, packed sequences, shared heads, states and pools are
:func:`linear_attention`'s, so the two serve side by side on the same pages.

The rule is stable where ``beta_t |k_t|^2`` lies in 0 .. 2: keys of unit length and rates in (0, 1),
or up to 2 where a state may also be reflected.  float32, bfloat16 and float16; arithmetic and
states are float32 (bfloat16 of widths in eights on bfloat16 matrix products, whose operands are all 24
bits of a float32 value in three parts), results are rounded once.  Sums run in a fixed order: equal calls
give equal bits.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor
from torch.autograd import forward_ad

from pararnn_amd import _lib
from pararnn_amd.attention import (
    _at,
    _check_state,
    _check_table,
    _decay_code,
    _enqueue,
    _heads,
    _no_tangents,
    _once,
    _Problem,
    _rows,
    _tiles,
    _view,
    _writes,
)
from pararnn_amd.ops import _DTYPES, _validate, _workspace
from pararnn_amd.ragged import PackedSequences


def _rate_code(what: str, beta: Tensor, q: Tensor) -> int:
    if beta.device != q.device:
        raise RuntimeError(f"{what}: tensors on different devices ({beta.device} vs {q.device})")
    if beta.dtype != q.dtype and beta.dtype != torch.float32:
        raise TypeError(f"{what}: beta must be float32 or {q.dtype}, got {beta.dtype}")
    return _DTYPES[beta.dtype]


class _DeltaProblem(_Problem):
    what = "delta_rule"

    def __init__(self, q, k, v, g, beta, h0, table, packed, scale):
        self.b, self.b_code = beta, None
        super().__init__(q, k, v, g, h0, table, packed, scale)

    def _fill(self) -> None:
        super()._fill()
        if self.b_code is None:  # (q, whose type it may be, has been checked by now)
            self.b_code = _rate_code(self.what, self.b, self.q)
        batch, time, heads, _, _ = self.dims
        if tuple(self.b.shape) != (batch, time, heads):
            raise ValueError(f"{self.what}: beta must be {(batch, time, heads)}, got "
                             f"{tuple(self.b.shape)}")
        self.c = _lib.DeltaProblem(self.c, self.b.data_ptr(), *self.b.stride(), self.b_code)

    def with_rates(self, q, k, v, g, beta, h0) -> _DeltaProblem:
        """The same checked call on tensors like those it was made of (backward)."""
        p = object.__new__(_DeltaProblem)
        p.b, p.b_code = beta, self.b_code
        return self._onto(p, q, k, v, g, h0)

    def forget(self) -> _DeltaProblem:
        self.b = None
        super().forget()
        return self


def _forward(p: _DeltaProblem, state_out: Tensor | None, table: Tensor | None,
             kept: bool) -> tuple[Tensor, Tensor | None]:
    batch, time, heads, _, dv = p.dims
    lib, dev, c = _lib.load(), p.q.device, ctypes.byref(p.c)
    out = p.q.new_empty(batch, time, heads, dv)
    keep = _workspace(lib.prnn_delta_rule_kept_size(c), dev) if kept else None
    need = lib.prnn_delta_rule_workspace_size(c, int(kept))
    ws = _workspace(need, dev) if need else None
    rc = _enqueue(lib.prnn_delta_rule, dev, c, ctypes.byref(_view(out)), _at(state_out), _at(table),
                  0 if state_out is None else state_out.shape[0], _at(keep), _at(ws), need)
    _lib.check(rc, "delta_rule")
    return out, keep


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, packed, scale, want_state):
        p = _DeltaProblem(q, k, v, g, beta, h0, None, packed, scale)
        _, _, heads, dk, dv = p.dims
        state = q.new_empty(p.sequences, heads, dk, dv, dtype=torch.float32) if want_state else None
        out, keep = _forward(p, state, None, True)
        ctx.save_for_backward(q, k, v, g, beta, h0, keep)
        ctx.call = p.forget()
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @_once
    def backward(ctx, go, gs):
        q, k, v, g, beta, h0, keep = ctx.saved_tensors
        if go is None and gs is None:
            return (None,) * 9
        p = ctx.call.with_rates(q, k, v, g, beta, h0)
        batch, time, heads, _, dv = p.dims
        if go is None:
            go = q.new_zeros(1).expand(batch, time, heads, dv)
        if go.dtype != q.dtype:
            go = go.to(q.dtype)
        need = ctx.needs_input_grad
        lib, dev, c = _lib.load(), q.device, ctypes.byref(p.c)
        go = _tiles(go)
        gs = None if gs is None else gs.contiguous()
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (p.q, p.k, p.v)]
        make = torch.empty if p.sequences else torch.zeros
        dg = make(p.g.shape, dtype=p.g.dtype, device=dev) if need[3] else None
        db = torch.empty(p.b.shape, dtype=p.b.dtype, device=dev) if need[4] else None
        dh0 = torch.empty_like(p.h0) if need[5] else None
        size = lib.prnn_delta_rule_backward_workspace_size(c, int(need[3]))
        ws = _workspace(size, dev) if size else None
        rc = _enqueue(lib.prnn_delta_rule_backward, dev, c, ctypes.byref(_view(go)), _at(gs),
                      keep.data_ptr(), *(t.data_ptr() for t in grads), _at(dg), _at(db), _at(dh0),
                      _at(ws), size)
        _lib.check(rc, "delta_rule backward")
        return (*(t if n else None for t, n in zip(grads, need)), dg, db, dh0, None, None, None)


def delta_rule(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, *,
               scale: float | None = None, h0: Tensor | None = None,
               cu_seqlens: Tensor | PackedSequences | None = None,
               block_table: Tensor | None = None, state_out: Tensor | None = None,
               state_table: Tensor | None = None,
               return_state: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """The gated delta rule over whole sequences; ``(B, T, H, Dv)`` in ``q``'s type.

    ``q`` ``(B, T, Hq, Dk)``, ``k`` ``(B, T, Hk, Dk)``, ``v`` ``(B, T, Hv, Dv)``, ``log_decay``
    ``(H,)`` or ``(B, T, H)`` (at most zero in use, ``-inf`` forgets the state), ``beta``
    ``(B, T, H)``: both float32 or ``q``'s type.  ``scale`` defaults to ``Dk ** -0.5``.  ``h0``,
    ``cu_seqlens``, ``block_table``, ``state_out``, ``state_table`` and ``return_state`` are
    :func:`linear_attention`'s.  Gradients of the output and of the returned states flow to ``q``,
    ``k``, ``v``, ``log_decay``, ``beta`` and ``h0``; between the passes a call keeps what its tokens
    wrote and the states before its chunks of 64 tokens, 4 bytes an element, and 26 KB of a chunk's
    system per head.

    What is not finite in a token's inputs reaches no earlier token's output, and in its output's gradient
    no later token's gradients; a ``q``, key, decay or rate that is not finite may leave NaN in the
    gradients of all tokens of its chunk.
    """
    what = "delta_rule"
    _no_tangents(what, q, k, v, log_decay, beta, h0)
    packed = cu_seqlens
    if packed is not None and not isinstance(packed, PackedSequences):
        packed = PackedSequences(packed)
    grads = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, log_decay, beta, h0))
    if block_table is not None and h0 is None and (state_out is None or state_table is not None):
        raise ValueError(f"{what}: block_table needs h0, or without a state_table state_out, as a "
                         "pool (C, ...)")
    if state_table is not None and state_out is None:
        raise ValueError(f"{what}: state_table needs state_out as a pool (C, ...)")
    if grads and block_table is None and state_out is None:
        out, state = _DeltaRule.apply(q, k, v, log_decay, beta, h0, packed, scale, return_state)
        return (out, state) if return_state else out
    if grads:
        raise RuntimeError(f"{what}: block_table and state_out are inference-only; call it under "
                           "torch.no_grad()")
    p = _DeltaProblem(q, k, v, log_decay, beta, h0, None if h0 is None else block_table, packed,
                      scale)
    dest, table = p.destination(block_table, state_out, state_table, return_state)
    out, _ = _forward(p, dest, table, False)
    return (out, dest) if return_state else out


def delta_rule_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor,
                    state: Tensor, *, scale: float | None = None,
                    block_table: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """One token for every row; ``state`` ``(B, H, Dk, Dv)`` float32 advances in place.

    ``q`` ``(B, Hq, Dk)``, ``k`` ``(B, Hk, Dk)``, ``v`` ``(B, Hv, Dv)`` (a time axis of 1 after
    ``B`` is allowed on all of them), ``log_decay`` ``(H,)`` or ``(B, H)``, ``beta`` ``(B, H)``.
    Returns ``(B, H, Dv)`` in ``q``'s type (with the time axis if ``q`` has it), in ``out`` where
    given.  ``block_table`` as for :func:`linear_attention_step`: ``state`` is a pool, a slot outside
    it (-1) an idle row, and no two rows may name one slot.  No autograd.  With contiguous operands
    and ``out=`` it allocates nothing and can be captured in a HIP graph.
    """
    what = "delta_rule_step"
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or log_decay.requires_grad or beta.requires_grad
                                    or state.requires_grad):
        raise RuntimeError(f"{what} has no autograd; call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _no_tangents(what, q, k, v, log_decay, beta, state)
    timed = q.dim() == 4
    if timed:
        if q.shape[1] != 1 or k.dim() != 4 or k.shape[1] != 1 or v.dim() != 4 or v.shape[1] != 1:
            raise ValueError(f"{what} takes one token per row, got q {tuple(q.shape)}")
        q, k, v = q[:, 0], k[:, 0], v[:, 0]
        if log_decay.dim() == 3:
            if log_decay.shape[1] != 1:
                raise ValueError(f"{what}: log_decay must be (H,) or (B, H), got "
                                 f"{tuple(log_decay.shape)}")
            log_decay = log_decay[:, 0]
        if beta.dim() == 3 and beta.shape[1] == 1:
            beta = beta[:, 0]
    code = _DTYPES.get(q.dtype)
    # the quick look first: calls of small sizes are bound by the host
    if not (code is not None and q.is_cuda and k.dtype is q.dtype and v.dtype is q.dtype
            and k.device == q.device and v.device == q.device):
        code = _validate(what, q, k, v)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k and v must be (B, heads, width), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    (batch, hq, dk), (bk, hk, dk2), (bv, hv, dv) = q.shape, k.shape, v.shape
    if bk != batch or bv != batch or dk2 != dk:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v "
                         f"{tuple(v.shape)} do not fit")
    if batch > 65535:
        raise ValueError(f"{what}: {batch} rows are more than 65535")
    g_code, b_code = _decay_code(what, log_decay, q), _rate_code(what, beta, q)
    heads = log_decay.shape[-1] if log_decay.dim() else 0
    if _heads(what, hq, hk, hv, heads) != heads:
        raise ValueError(f"{what}: log_decay has {heads} heads, q, k and v have "
                         f"{max(hq, hk, hv)}")
    if log_decay.dim() == 1:
        g_sb, g_sh = 0, log_decay.stride(0)
    elif log_decay.dim() == 2 and log_decay.shape[0] == batch:
        g_sb, g_sh = log_decay.stride()
    else:
        raise ValueError(f"{what}: log_decay must be (H,) or (B, H), got "
                         f"{tuple(log_decay.shape)}")
    if tuple(beta.shape) != (batch, heads):
        raise ValueError(f"{what}: beta must be {(batch, heads)}, got {tuple(beta.shape)}")
    dev = q.device
    _check_state(what, "state", state, q, (heads, dk, dv), None if block_table is not None
                 else batch)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous (it is advanced in place)")
    table = None if block_table is None else _check_table(what, "block_table", block_table, batch, dev)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if out is None:
        res = q.new_empty(batch, heads, dv)
        _writes(what, state)
    else:
        if out.shape != ((batch, 1, heads, dv) if timed else (batch, heads, dv)):
            raise ValueError(f"{what}: out {tuple(out.shape)} != {(batch, heads, dv)}")
        if out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
            raise ValueError(f"{what}: out must be contiguous, of q's type and on its device")
        res = out
        _writes(what, state, out)
    rc = _enqueue(
        _lib.load().prnn_delta_rule_step, dev,
        q.data_ptr(), q.stride(0), q.stride(1), hq, k.data_ptr(), k.stride(0), k.stride(1), hk,
        v.data_ptr(), v.stride(0), v.stride(1), hv, log_decay.data_ptr(), g_sb, g_sh, g_code,
        beta.data_ptr(), beta.stride(0), beta.stride(1), b_code, state.data_ptr(),
        None if table is None else table.data_ptr(), state.shape[0], res.data_ptr(), batch, heads,
        dk, dv, dk ** -0.5 if scale is None else scale, code)
    _lib.check(rc, what)
    if out is not None:
        return out
    return res[:, None] if timed else res
