"""What the linear attention's C entries refuse, with made-up addresses: no GPU needed, none used."""

import ctypes
import os

import pytest
import torch

from pararnn_amd import _lib

pytestmark = [
    pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: without a device only"),
    pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")]


def _view(st=16, sb=128, sh=8, heads=2):
    return _lib.LaView(4096, sb, st, sh, heads)


def _problem(q=None, k=None, v=None, g_st=2, B=1, T=8):
    """Two heads of (8, 8) in float32."""
    return _lib.LaProblem(q or _view(), k or _view(), v or _view(), 4096, 16, g_st, 1, None, None, None,
                          0, 0, B, T, 2, 8, 8, 0, 0, 1.0)


def _forward(p, out=None):
    ws = _lib.load().prnn_linear_attention_workspace_size(ctypes.byref(p))
    return _lib.load().prnn_linear_attention(ctypes.byref(p), ctypes.byref(out or _view()), None, None,
                                             0, 4096, max(ws, 256), None)


def _backward(p, go=None):
    lib = _lib.load()
    ws = lib.prnn_linear_attention_backward_workspace_size(ctypes.byref(p), 1)
    return lib.prnn_linear_attention_backward(ctypes.byref(p), ctypes.byref(go or _view()), None, 4096,
                                              4096, 4096, 4096, None, 4096, max(ws, 256), None)


def test_tokens_in_descending_order_are_refused():
    """The walks read rows by unsigned offsets from a chunk's lowest one."""
    lib = _lib.load()
    down = _view(st=-16)
    for p in (_problem(q=down), _problem(k=down), _problem(v=down), _problem(g_st=-2)):
        assert lib.prnn_linear_attention_workspace_size(ctypes.byref(p)) == 0
        for call in (_forward, _backward):
            assert call(p) == _lib.PRNN_ERR_VALUE
            assert b"apart" in lib.prnn_last_error()
    for call in (_forward, _backward):
        assert call(_problem(), down) == _lib.PRNN_ERR_VALUE
        assert b"apart" in lib.prnn_last_error()
    # a problem like these, but ascending, is not refused (what fails then is the missing device)
    for call in (_forward, _backward):
        assert call(_problem()) == _lib.PRNN_ERR_RUNTIME


def test_an_only_tokens_stride_does_not_matter():
    far = 1 << 40
    p = _problem(_view(st=far), _view(st=-far), _view(st=far), g_st=far, B=3, T=1)
    for call in (_forward, _backward):
        assert call(p, _view(st=far)) == _lib.PRNN_ERR_RUNTIME  # not refused: no device
