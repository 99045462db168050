"""Group norm, channels last, with an activation or a gate: the norm behind a token mixer.

    z = weight * (x - mean) * rstd + bias        y = act(z)     or     y = z * act(gate)

per group of consecutive channels of ``x`` ``(..., C)``; the statistics run over one token's group
(``over="token"``, what a causal model uses) or over all tokens of a sample (``over="sample"``: all
dimensions between the first and the last).  float32, bfloat16 and float16; arithmetic, statistics
and the parameters' gradient sums are float32, each result is rounded once.  Sums run in a fixed
order.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor

from pararnn_amd import _lib
from pararnn_amd.attention import _at, _enqueue, _no_tangents, _once
from pararnn_amd.ops import _DTYPES, _validate, _workspace

_ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}


def _shape(x: Tensor, over: str) -> tuple[int, int, int]:
    """(N, L, C): L tokens share their statistics."""
    c = x.shape[-1]
    if over == "token":
        return x.numel() // c, 1, c
    n = x.shape[0] if x.dim() > 1 else 1
    return n, (x.numel() // (n * c) if n else 0), c


def _flat(t: Tensor | None) -> Tensor | None:
    """As the kernels read it: contiguous, from a 16-byte boundary."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n: int, length: int, c: int, groups: int, code: int, backward: int) -> int:
    # 2: all arrays here lie on 16-byte boundaries
    return _lib.load().prnn_group_norm_workspace_size(n, length, c, groups, code, backward | 2)


def _codes(x, weight, bias, groups, eps, act, over) -> tuple:
    """The C entries' numbers: N, L, C, groups, eps, act and the types of w and x."""
    code = _DTYPES[x.dtype]
    w = bias if weight is None else weight
    return (*_shape(x, over), groups, eps, act, code if w is None else _DTYPES[w.dtype], code)


def _forward(x, weight, bias, gate, codes):
    n, length, c, groups, _, _, _, code = codes
    y = torch.empty_like(x)
    need = _workspace_bytes(n, length, c, groups, code, 0)
    ws = stats = None
    if need:  # statistics per sample, or groups too wide for a wave
        ws = _workspace(need, x.device)
        stats = torch.empty(n, groups, 2, dtype=torch.float32, device=x.device)
    rc = _enqueue(_lib.load().prnn_group_norm, x.device, x.data_ptr(), _at(weight), _at(bias),
                  _at(gate), y.data_ptr(), _at(stats), *codes, _at(ws), need)
    _lib.check(rc, "group_norm")
    return y, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, codes):
        y, stats = _forward(x, weight, bias, gate, codes)
        ctx.save_for_backward(x, weight, bias, gate, stats)
        ctx.codes = codes
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, weight, bias, gate, stats = ctx.saved_tensors
        codes = ctx.codes
        n, length, c, groups, _, _, _, code = codes
        dev = x.device
        if gy.dtype != x.dtype:
            gy = gy.to(x.dtype)
        gy = gy.contiguous()
        if gy.data_ptr() % 16:
            gy = gy.clone()
        dx = torch.empty_like(x)
        dgate = None if gate is None else torch.empty_like(x)
        dw = None if weight is None else torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        need = _workspace_bytes(n, length, c, groups, code, 1)
        ws = _workspace(need, dev)
        rc = _enqueue(_lib.load().prnn_group_norm_backward, dev, gy.data_ptr(), x.data_ptr(),
                      _at(weight), _at(bias), _at(gate), _at(stats), dx.data_ptr(), _at(dw),
                      _at(db), _at(dgate), *codes, ws.data_ptr(), ws.numel())
        _lib.check(rc, "group_norm backward")
        return dx if ctx.needs_input_grad[0] else None, dw, db, dgate, None


def group_norm(x: Tensor, num_groups: int, weight: Tensor | None = None,
               bias: Tensor | None = None, *, gate: Tensor | None = None,
               activation: str | None = None, over: str = "token", eps: float = 1e-5) -> Tensor:
    """Group norm of ``x`` ``(..., C)``, channels last, in ``x``'s type.

    ``num_groups`` divides ``C``.  ``weight`` and ``bias`` ``(C,)``: float32 or ``x``'s type (ones
    and zeros without).  ``activation``: ``None``, ``"silu"`` or ``"sigmoid"``, applied to the
    normalised values, or, where ``gate`` (like ``x``) is given, to the gate that multiplies them.
    ``over``: ``"token"`` or ``"sample"`` (``x`` ``(N, ..., C)``).  Differentiable in all tensors.
    """
    what = "group_norm"
    # the quick look first: calls of small sizes are bound by the host
    if not (x.is_cuda and x.dtype in _DTYPES
            and (gate is None or (gate.dtype is x.dtype and gate.device == x.device))):
        _validate(what, x, gate)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be (..., C), got {tuple(x.shape)}")
    c = x.shape[-1]
    if num_groups < 1 or c % num_groups:
        raise ValueError(f"{what}: {num_groups} groups do not divide C={c}")
    if gate is not None and gate.shape != x.shape:
        raise ValueError(f"{what}: gate {tuple(gate.shape)} != x {tuple(x.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None, 'silu' or 'sigmoid', got "
                         f"{activation!r}")
    if over not in ("token", "sample"):
        raise ValueError(f"{what}: over must be 'token' or 'sample', got {over!r}")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must be >= 0, got {eps!r}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError(f"{what}: tensors on different devices ({t.device} vs {x.device})")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"{what}: {name} must be float32 or {x.dtype}, got {t.dtype}")
        if t.shape != (c,):
            raise ValueError(f"{what}: {name} shape {tuple(t.shape)} != {(c,)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{what}: dtype mismatch {weight.dtype} vs {bias.dtype}")
    if x.numel() // c >= 1 << 31 or c >= 1 << 31:
        raise ValueError(f"{what}: x has {x.numel() // c} tokens of {c} channels, more than 2^31 - 1")

    _no_tangents(what, x, weight, bias, gate)
    x, gate = _flat(x), _flat(gate)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    codes = _codes(x, weight, bias, int(num_groups), float(eps), _ACTIVATIONS[activation], over)
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        return _GroupNorm.apply(x, weight, bias, gate, codes)
    return _forward(x, weight, bias, gate, codes)[0]
