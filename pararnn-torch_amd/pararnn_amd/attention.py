"""Linear attention with a decay per head: whole sequences, their gradients, single tokens.

For every head, with a state ``S`` ``(Dk, Dv)`` held in float32 and a log decay ``g_t``:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,        o_t = scale q_t^T S_t.

``linear_attention`` runs prompts and training sequences in the chunked form (matrix products
inside a chunk, the state from chunk to chunk), ``linear_attention_step`` one token per session
on a state or a pool of states, in place.  Both keep the state in the same layout, so a prompt's
final state is what decoding goes on from; it lies next to the recurrent cells' states in a
serving program and is paged in the same way (``block_table``).

Layouts: ``q`` ``(B, T, Hq, Dk)``, ``k`` ``(B, T, Hk, Dk)``, ``v`` ``(B, T, Hv, Dv)`` with any
strides whose last one is 1 (views of one fused projection are read as they are).  ``H`` is the
largest of the head counts and of the decay's; each count divides it, and consecutive heads share
an array that has fewer.  Widths up to 256.  float32, bfloat16 and float16; arithmetic and states
are float32 (bfloat16 products take operands of 16 bits or more in bfloat16 parts, see the
kernels), results are rounded once.  What an infinity or NaN reaches is not finite, whether the sum
would be infinite or not a number.  Results do not depend on the order in which workgroups run: no
atomics.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch import Tensor
from torch.autograd import forward_ad

from pararnn_amd import _lib
from pararnn_amd.ops import _DTYPES, _validate, _workspace
from pararnn_amd.ragged import PackedSequences


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_increment_version = torch._C._increment_version  # of torch.autograd.graph, without its wrapper


def _enqueue(fn, dev: torch.device, *args) -> int:
    """``fn(*args, stream)`` with ``dev`` as the current device and its current stream.  Small calls
    are bound by the host: the stream object that ``torch.cuda.current_stream`` builds and a guard
    for a device that is current already take 3 us of a step's 12."""
    index = dev.index
    if index == _current_device():
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(dev):
        return fn(*args, _raw_stream(index))


def _once(fn):
    """``once_differentiable``, whose guards an ordinary backward pass (no graph of it wanted, grad
    mode off already) goes without: 4 us of a small call."""
    guarded = torch.autograd.function.once_differentiable(fn)

    @functools.wraps(fn)
    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return backward


def _no_tangents(what: str, *tensors: Tensor | None) -> None:
    """Refuses forward-mode duals: the kernels would drop their tangents unnoticed."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def _writes(what: str, *tensors: Tensor) -> None:
    """Tells autograd that a call is about to write ``tensors`` in place, which it cannot see: a
    backward pass that saved one of them must not read the new values unnoticed."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{what} writes in place and has no autograd; call it under "
                                   "torch.no_grad()")
    _increment_version(tensors)


def _rows(t: Tensor) -> Tensor:
    """``t`` with its heads' values side by side."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _tiles(t: Tensor) -> Tensor:
    """``t`` as the walks read it.  Which walk runs goes by type and widths alone, so that equal
    values give equal bits: the bfloat16 one (widths in eights) reads 16 bytes at a time, and rows
    that do not lie for that (a view of a fused projection with an odd offset, a row expanded over
    time) are copied."""
    sb, st, sh, sd = t.stride()
    time, width = t.shape[1], t.shape[3]
    if time == 1:
        st = width  # whatever it is, the kernels do not use it
    # at most 16 MiB between tokens: the kernels' offsets inside a chunk
    if (sd != 1 and width != 1) or st > 1 << 22:
        t = t.contiguous()
        sb, st, sh, _ = t.stride()
    if t.dtype is not torch.bfloat16 or width % 8:
        return t
    if (sb | st | sh) % 8 == 0 and t.data_ptr() % 16 == 0 and st >= width:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _view(t: Tensor) -> _lib.LaView:
    sb, st, sh, _ = t.stride()
    return _lib.LaView(t.data_ptr(), sb, st, sh, t.shape[2])


def _heads(what: str, *counts: int) -> int:
    h = max(counts)
    for n in counts:
        if n < 1 or h % n:
            raise ValueError(f"{what}: head counts {counts} do not divide {h}")
    return h


def _decay_code(what: str, g: Tensor, q: Tensor) -> int:
    if g.device != q.device:
        raise RuntimeError(f"{what}: tensors on different devices ({g.device} vs {q.device})")
    if g.dtype != q.dtype and g.dtype != torch.float32:
        raise TypeError(f"{what}: log_decay must be float32 or {q.dtype}, got {g.dtype}")
    return _DTYPES[g.dtype]


def _check_state(what: str, name: str, t: Tensor, q: Tensor, tail: tuple[int, ...],
                 rows: int | None) -> None:
    if t.device != q.device:
        raise RuntimeError(f"{what}: tensors on different devices ({t.device} vs {q.device})")
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be float32, got {t.dtype}")
    if t.dim() != 4 or tuple(t.shape[1:]) != tail or (rows is not None and t.shape[0] != rows):
        want = ("C" if rows is None else rows, *tail)
        raise ValueError(f"{what}: {name} shape {tuple(t.shape)} != {want}")
    # counts go to the kernels in 32 bits
    if t.shape[0] >= 1 << 31:
        raise ValueError(f"{what}: {name} has {t.shape[0]} rows, more than 2^31 - 1")


_INTS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _slots(what: str, name: str, t: Tensor, dev: torch.device) -> Tensor:
    """A list of slots as the kernels read it: int32, contiguous, on ``dev``."""
    if t.dtype not in _INTS:
        raise TypeError(f"{what}: {name} must be whole numbers, got {t.dtype}")
    if t.dim() != 1:
        raise ValueError(f"{what}: {name} must be one-dimensional, got {tuple(t.shape)}")
    if t.shape[0] > 1 << 30:
        raise ValueError(f"{what}: {name} has {t.shape[0]} entries, more than 2^30")
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} under graph capture needs a contiguous int32 {name} on the "
                           "device of what it names")
    if t.dtype is torch.int64:
        t = t.clamp(-1, (1 << 31) - 1)  # what int32 cannot hold names no slot either
    return t.to(device=dev, dtype=torch.int32).contiguous()


def _check_table(what: str, name: str, table: Tensor, rows: int, dev: torch.device) -> Tensor:
    if table.dim() != 1 or table.numel() != rows:
        raise ValueError(f"{what}: {name} must be ({rows},), got {tuple(table.shape)}")
    return _slots(what, name, table, dev)


def _at(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class _Problem:
    """A checked call: the C problem and the tensors that it points to."""

    what = "linear_attention"

    def __init__(self, q: Tensor, k: Tensor, v: Tensor, g: Tensor, h0: Tensor | None,
                 table: Tensor | None, packed: PackedSequences | None, scale: float | None):
        what = self.what
        code = _DTYPES.get(q.dtype)
        # the quick look first: calls of small sizes are bound by the host
        if not (code is not None and q.is_cuda and k.dtype is q.dtype and v.dtype is q.dtype
                and k.device == q.device and v.device == q.device):
            code = _validate(what, q, k, v)
        for n, t in (("q", q), ("k", k), ("v", v)):
            if t.dim() != 4:
                raise ValueError(f"{what}: {n} must be (B, T, heads, width), got "
                                 f"{tuple(t.shape)}")
        (batch, time, hq, dk), (bk, tk, hk, dk2), (bv, tv, hv, dv) = q.shape, k.shape, v.shape
        if bk != batch or bv != batch or tk != time or tv != time:
            raise ValueError(f"{what}: q, k and v disagree on (B, T): {(batch, time)}, "
                             f"{(bk, tk)}, {(bv, tv)}")
        if dk2 != dk:
            raise ValueError(f"{what}: q has width {dk}, k {dk2}")
        if max(batch, 1) * max(time, 1) > 1 << 30:
            raise ValueError(f"{what}: {batch} x {time} tokens are more than 2^30")
        g_code = _decay_code(what, g, q)
        if g.dim() not in (1, 3) or (g.dim() == 3 and g.shape[:2] != (batch, time)):
            raise ValueError(f"{what}: log_decay must be (H,) or (B, T, H), got "
                             f"{tuple(g.shape)}")
        heads = max(hq, hk, hv, g.shape[-1])
        if heads < 1 or (hq != heads and (hq < 1 or heads % hq)) or (
                hk != heads and (hk < 1 or heads % hk)) or (
                hv != heads and (hv < 1 or heads % hv)):
            raise ValueError(f"{what}: head counts {(hq, hk, hv)} do not divide {heads}")
        if g.shape[-1] != heads:
            raise ValueError(f"{what}: log_decay has {g.shape[-1]} heads, q, k and v have {heads}")
        self.q, self.k, self.v, self.g = _tiles(q), _tiles(k), _tiles(v), g
        if not 1 <= dk <= 256 or not 1 <= dv <= 256:
            raise ValueError(f"{what}: head widths ({dk}, {dv}) are not in 1 .. 256")
        self.dims = (batch, time, heads, dk, dv)
        self.sequences = batch
        self.offsets, self.longest = None, 0
        if packed is not None:
            if batch != 1:
                raise ValueError(f"{what}: cu_seqlens packs q with batch=1, got batch={batch}")
            if packed.tokens != time:
                raise ValueError(f"cu_seqlens[-1] must equal time={time}, got {packed.tokens}")
            self.sequences = packed.sequences
            self.offsets, self.longest = packed.offsets(q.device), packed.longest
        self.table = None if table is None else _check_table(what, "block_table", table,
                                                             self.sequences, q.device)
        self.h0 = None
        if h0 is not None:
            _check_state(what, "h0", h0, q, (heads, dk, dv),
                         None if table is not None else self.sequences)
            self.h0 = h0.contiguous()
        self.scale = float(dk ** -0.5 if scale is None else scale)
        self.codes = (g_code, code)
        self._fill()

    def _fill(self) -> None:
        g, batch, time = self.g, self.dims[0], self.dims[1]
        at = g.stride() if g.dim() == 3 else (0, 0, g.stride(0))
        if at[0] == 0 and at[1] == 0 and g.dim() == 3 and time * batch > 0:
            # expanded, not per head: the gradient's layout tells them apart
            g = self.g = g.contiguous()
            at = g.stride()
        self.c = _lib.LaProblem(
            _view(self.q), _view(self.k), _view(self.v), g.data_ptr(), *at, _at(self.h0),
            _at(self.table), _at(self.offsets), 0 if self.h0 is None else self.h0.shape[0],
            0 if self.offsets is None else self.sequences, *self.dims, *self.codes, self.scale,
            self.longest)

    def again(self, q: Tensor, k: Tensor, v: Tensor, g: Tensor, h0: Tensor | None) -> _Problem:
        """The same checked call on tensors like those it was made of (backward)."""
        return self._onto(object.__new__(_Problem), q, k, v, g, h0)

    def _onto(self, p, q: Tensor, k: Tensor, v: Tensor, g: Tensor, h0: Tensor | None):
        p.q, p.k, p.v, p.g = _tiles(q), _tiles(k), _tiles(v), g
        p.h0 = None if h0 is None else h0.contiguous()
        p.dims, p.codes, p.scale = self.dims, self.codes, self.scale
        p.sequences, p.offsets, p.table = self.sequences, self.offsets, None
        p.longest = self.longest
        p._fill()
        return p

    def destination(self, block_table: Tensor | None, state_out: Tensor | None,
                    state_table: Tensor | None, return_state: bool):
        """(where the final states go, the table of their rows) of a call without gradients."""
        _, _, heads, dk, dv = self.dims
        q, what = self.q, self.what
        if state_out is None:
            if not return_state:
                return None, None
            return q.new_empty(self.sequences, heads, dk, dv, dtype=torch.float32), None
        if return_state:
            raise ValueError(f"{what}: state_out and return_state exclude each other")
        table = None
        if state_table is not None:
            table = _check_table(what, "state_table", state_table, self.sequences, q.device)
        elif block_table is not None:
            table = self.table if self.table is not None else _check_table(
                what, "block_table", block_table, self.sequences, q.device)
        _check_state(what, "state_out", state_out, q, (heads, dk, dv),
                     self.sequences if table is None else None)
        if not state_out.is_contiguous():
            raise ValueError(f"{what}: state_out must be contiguous")
        _writes(what, state_out)
        return state_out, table

    def forget(self) -> _Problem:
        """Keeps what was checked, not the tensors."""
        self.q = self.k = self.v = self.g = self.h0 = self.c = None
        return self


def _forward(p: _Problem, state_out: Tensor | None, table: Tensor | None) -> Tensor:
    batch, time, heads, _, dv = p.dims
    lib, dev, c = _lib.load(), p.q.device, ctypes.byref(p.c)
    out = p.q.new_empty(batch, time, heads, dv)
    need = lib.prnn_linear_attention_workspace_size(c)
    ws = _workspace(need, dev) if need else None
    rc = _enqueue(lib.prnn_linear_attention, dev, c, ctypes.byref(_view(out)), _at(state_out),
                  _at(table), 0 if state_out is None else state_out.shape[0], _at(ws), need)
    _lib.check(rc, "linear_attention")
    return out


def _backward(p: _Problem, go: Tensor, gs: Tensor | None, need_g: bool, need_h0: bool):
    lib, dev, c = _lib.load(), p.q.device, ctypes.byref(p.c)
    go = _tiles(go)
    gs = None if gs is None else gs.contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (p.q, p.k, p.v))
    make = torch.empty if p.sequences else torch.zeros
    dg = make(p.g.shape, dtype=p.g.dtype, device=dev) if need_g else None
    dh0 = None
    if p.h0 is not None and (need_g or need_h0):
        dh0 = torch.empty_like(p.h0)
    need = lib.prnn_linear_attention_backward_workspace_size(c, int(need_g))
    ws = _workspace(need, dev) if need else None
    rc = _enqueue(lib.prnn_linear_attention_backward, dev, c, ctypes.byref(_view(go)), _at(gs),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _at(dg), _at(dh0), _at(ws), need)
    _lib.check(rc, "linear_attention backward")
    return dq, dk, dv, dg, dh0


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, h0, packed, scale, want_state):
        p = _Problem(q, k, v, g, h0, None, packed, scale)
        _, _, heads, dk, dv = p.dims
        state = q.new_empty(p.sequences, heads, dk, dv, dtype=torch.float32) if want_state else None
        out = _forward(p, state, None)
        ctx.save_for_backward(q, k, v, g, h0)
        ctx.call = p.forget()
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @_once
    def backward(ctx, go, gs):
        q, k, v, g, h0 = ctx.saved_tensors
        if go is None and gs is None:
            return (None,) * 8
        p = ctx.call.again(q, k, v, g, h0)
        if go is None:
            go = q.new_zeros(1).expand(*p.dims[:3], p.dims[4])
        if go.dtype != q.dtype:
            go = go.to(q.dtype)
        need = ctx.needs_input_grad
        dq, dk, dv, dg, dh0 = _backward(p, go, gs, need[3], need[4])
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dg,
                dh0 if need[4] else None, None, None, None)


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, *,
                     scale: float | None = None, h0: Tensor | None = None,
                     cu_seqlens: Tensor | PackedSequences | None = None,
                     block_table: Tensor | None = None, state_out: Tensor | None = None,
                     state_table: Tensor | None = None,
                     return_state: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """Linear attention over whole sequences; ``(B, T, H, Dv)`` in ``q``'s type.

    ``log_decay``: ``(H,)``, fixed per head, or ``(B, T, H)``, per token; at most zero in use
    (``-inf`` forgets the state), float32 or ``q``'s type.  ``scale`` defaults to ``Dk ** -0.5``.
    ``h0`` ``(B, H, Dk, Dv)`` float32: the states to go on from (zeros without).

    ``cu_seqlens`` packs ``S`` sequences into ``(1, N, ...)``; every one starts from its own
    ``h0`` row.  A tensor is checked at each call (a copy from the device); a
    :class:`PackedSequences` was checked when it was made.

    ``return_state=True`` also returns the final states ``(sequences, H, Dk, Dv)``.  Gradients of
    the output and of the returned states flow to ``q``, ``k``, ``v``, ``log_decay`` and ``h0``.

    Serving: with ``block_table`` ``(sequences,)`` ``h0`` is a pool ``(C, H, Dk, Dv)`` and
    sequence ``s`` starts from row ``block_table[s]`` (an entry that is no row, -1: from zeros).
    ``state_out`` takes the final states: ``(sequences, H, Dk, Dv)``, or with a table a pool whose
    named rows are overwritten: those of ``state_table`` where given, or of ``block_table``.  A pool
    row keeps its last session's state, so a new session's prompt goes without ``h0``
    (``block_table=slots, state_out=pool``: zeros in, the final state to its slot), and next to
    others that go on (``h0=pool``) has -1 in ``block_table`` and its slot in ``state_table``.
    ``state_out`` may be ``h0`` itself if no row that one sequence writes is read or written by
    another.  None of these has a gradient.
    """
    _no_tangents("linear_attention", q, k, v, log_decay, h0)
    packed = cu_seqlens
    if packed is not None and not isinstance(packed, PackedSequences):
        packed = PackedSequences(packed)
    grads = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, log_decay, h0))
    if block_table is not None and h0 is None and (state_out is None or state_table is not None):
        raise ValueError("block_table needs h0, or without a state_table state_out, as a pool "
                         "(C, ...)")
    if state_table is not None and state_out is None:
        raise ValueError("state_table needs state_out as a pool (C, ...)")
    if grads and block_table is None and state_out is None:
        out, state = _LinearAttention.apply(q, k, v, log_decay, h0, packed, scale, return_state)
        return (out, state) if return_state else out
    if grads:
        raise RuntimeError("linear_attention: block_table and state_out are inference-only; call "
                           "it under torch.no_grad()")
    p = _Problem(q, k, v, log_decay, h0, None if h0 is None else block_table, packed, scale)
    dest, table = p.destination(block_table, state_out, state_table, return_state)
    out = _forward(p, dest, table)
    return (out, dest) if return_state else out


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                          scale: float | None = None, block_table: Tensor | None = None,
                          out: Tensor | None = None) -> Tensor:
    """One token for every row; ``state`` ``(B, H, Dk, Dv)`` float32 advances in place.

    ``q`` ``(B, Hq, Dk)``, ``k`` ``(B, Hk, Dk)``, ``v`` ``(B, Hv, Dv)`` (a time axis of 1 after
    ``B`` is allowed on all of them), ``log_decay`` ``(H,)`` or ``(B, H)``.  Returns
    ``(B, H, Dv)`` in ``q``'s type (with the time axis if ``q`` has it), in ``out`` where given.
    With ``block_table`` ``(B,)`` ``state`` is a pool ``(C, H, Dk, Dv)`` and row ``b`` works on
    slot ``block_table[b]``; a slot outside the pool (-1) is an idle row: it starts from zeros and
    nothing is kept.  No two rows may name one slot.  No autograd.  With contiguous operands and
    ``out=`` it allocates nothing and can be captured in a HIP graph.
    """
    what = "linear_attention_step"
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or log_decay.requires_grad or state.requires_grad):
        raise RuntimeError(f"{what} has no autograd; call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _no_tangents(what, q, k, v, log_decay, state)
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
    g_code = _decay_code(what, log_decay, q)
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
    dev = q.device
    _check_state(what, "state", state, q, (heads, dk, dv), None if block_table is not None
                 else batch)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous (it is advanced in place)")
    table = None if block_table is None else _check_table(what, "block_table", block_table, batch, dev)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if out is None:
        res = q.new_empty(batch, heads, dv)
    else:
        if out.shape != ((batch, 1, heads, dv) if timed else (batch, heads, dv)):
            raise ValueError(f"{what}: out {tuple(out.shape)} != {(batch, heads, dv)}")
        if out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
            raise ValueError(f"{what}: out must be contiguous, of q's type and on its device")
        res = out
    if out is None:
        _writes(what, state)
    else:
        _writes(what, state, out)
    rc = _enqueue(
        _lib.load().prnn_linear_attention_step, dev,
        q.data_ptr(), q.stride(0), q.stride(1), hq, k.data_ptr(), k.stride(0), k.stride(1), hk,
        v.data_ptr(), v.stride(0), v.stride(1), hv, log_decay.data_ptr(), g_sb, g_sh, g_code,
        state.data_ptr(), None if table is None else table.data_ptr(), state.shape[0],
        res.data_ptr(), batch, heads, dk, dv, dk ** -0.5 if scale is None else scale, code)
    _lib.check(rc, what)
    if out is not None:
        return out
    return res[:, None] if timed else res
