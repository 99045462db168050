"""Beam search's selection: the best continuations over beams and vocabulary.

``beam_select`` chooses, ``reorder_pages`` lets the sessions' states follow their beams.  Both work on
the current stream and leave their answers on the device, so a decoding step with them waits for
nothing and can be captured in a HIP graph.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor
from torch.autograd import forward_ad

from pararnn_amd import _lib
from pararnn_amd.attention import _at, _enqueue, _no_tangents
from pararnn_amd.ops import _DTYPES, _validate, _workspace


@functools.lru_cache(maxsize=256)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.load().prnn_beam_select_workspace_size(*sizes)


def beam_select(logits: Tensor, scores: Tensor, *, beams: int | None = None,
                ended: Tensor | None = None, pad: int = 0) -> tuple[Tensor, Tensor, Tensor]:
    """The best of ``scores + log_softmax(logits)`` over the beams and tokens of every search.

    ``logits`` ``(B, K, V)`` float32, bfloat16 or float16, ``scores`` ``(B, K)`` float32, the beams'
    totals so far (``-inf``: a beam that is not there, as all but the first at a search's start).
    Returns ``(scores, parents, tokens)``, each ``(B, beams)`` (``K`` of them by default, at most 128),
    the largest total first, float32, int32 and int32.  Totals are formed and compared in float64, an
    exponential to 2^-51 of its row's largest, and do not depend on where a row lies in memory; ties go to
    the lowest beam, in a beam to the larger logit, then to the lowest token.  Where fewer candidates are
    left, the rest are ``-inf``, -1 and -1.  A logit of ``-inf`` is masked; a beam whose logits hold NaN or
    ``+inf`` proposes nothing.

    ``ended`` ``(B, K)`` bool: beams that are finished and compete with their score as it is; they
    propose the token ``pad`` alone, whatever their logits.  No autograd.
    """
    what = "beam_select"
    code = _DTYPES.get(logits.dtype) if logits.is_cuda else None
    if code is None:
        _validate(what, logits)
    if logits.dim() != 3:
        raise ValueError(f"{what}: logits must be (B, K, V), got {tuple(logits.shape)}")
    searches, given, vocab = logits.shape
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError(f"{what} has no autograd; call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _no_tangents(what, logits, scores)
    if scores.device != logits.device or (ended is not None and ended.device != logits.device):
        raise RuntimeError(f"{what}: tensors on different devices")
    if scores.dtype != torch.float32:
        raise TypeError(f"{what}: scores must be float32, got {scores.dtype}")
    if scores.shape != (searches, given):
        raise ValueError(f"{what}: scores {tuple(scores.shape)} != {(searches, given)}")
    if given < 1 or vocab < 1:
        raise ValueError(f"{what}: {given} beams of {vocab} tokens")
    wanted = given if beams is None else int(beams)
    if not 1 <= wanted <= 128:
        raise ValueError(f"{what}: beams must be in 1 .. 128, got {wanted}")
    if given * vocab >= 1 << 31 or searches * given >= 1 << 31:
        raise ValueError(f"{what}: {searches} x {given} beams of {vocab} tokens are more than 2^31 - 1")
    if ended is not None:
        if ended.dtype != torch.bool:
            raise TypeError(f"{what}: ended must be bool, got {ended.dtype}")
        if ended.shape != scores.shape:
            raise ValueError(f"{what}: ended {tuple(ended.shape)} != {(searches, given)}")
        if not 0 <= pad < vocab:
            raise ValueError(f"{what}: pad={pad} is no token of {vocab}")
        ended = ended.contiguous()
    if logits.stride(-1) != 1 and vocab > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    dev = logits.device
    best = torch.empty(searches, wanted, dtype=torch.float32, device=dev)
    both = torch.empty(2, searches, wanted, dtype=torch.int32, device=dev)
    need = _workspace_bytes(searches, given, vocab, wanted)
    ws = _workspace(need, dev)
    rc = _enqueue(_lib.load().prnn_beam_select, dev, logits.data_ptr(), logits.stride(0), logits.stride(1),
                  scores.data_ptr(), _at(ended), int(pad), best.data_ptr(), both.data_ptr(),
                  both.data_ptr() + 4 * searches * wanted, searches, given, vocab, wanted, code,
                  ws.data_ptr(), need)
    _lib.check(rc, what)
    return best, *both.unbind()
