"""What the delta-rule block's operators refuse without a GPU, and their definitions: made-up addresses
in the C entries, none of which is used."""

import ctypes
import os

import pytest
import torch

import pararnn_amd as P
from oracle import delta_rule as O
from oracle import linear_attention as L
from pararnn_amd import _lib

built = pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: without a device only")


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_cpu_tensors_are_refused():
    q, g, b = torch.zeros(1, 4, 2, 8), torch.zeros(2), torch.zeros(1, 4, 2)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.delta_rule(q, q, q, g, b)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g, b[:, 0], torch.zeros(1, 2, 8, 8))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.reorder_pages(torch.zeros(4, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_oracle_rule():
    """Packed is each sequence alone; orthonormal keys at a rate of 1 without decay are the linear
    attention; a key written twice holds its last value; the chunks' formulas give the recurrence."""
    q, k, v = _r(1, 9, 2, 4, seed=1), _r(1, 9, 2, 4, seed=2), _r(1, 9, 2, 3, seed=3)
    g, b = -_r(1, 9, 2, seed=4).abs(), _r(1, 9, 2, seed=5).sigmoid()
    out, state = O.delta_rule(q, k, v, g, b, cu=[0, 4, 4, 9])
    one, s = O.delta_rule(*(t[:, 4:] for t in (q, k, v, g, b)))
    assert torch.equal(out[:, 4:], one) and torch.equal(state[2:], s)
    assert torch.equal(state[1], torch.zeros(2, 4, 3, dtype=torch.float64))
    unit = torch.eye(4, dtype=torch.float64)[None, :, None].expand(1, 4, 2, 4)
    ones, none = torch.ones(1, 4, 2, dtype=torch.float64), torch.zeros(2, dtype=torch.float64)
    out, state = O.delta_rule(q[:, :4], unit, v[:, :4], none, ones)
    want, last = L.linear_attention(q[:, :4], unit, v[:, :4], none)
    assert torch.allclose(out, want, atol=1e-14) and torch.allclose(state, last, atol=1e-14)
    twice = unit[:, [0, 1, 0]]
    _, state = O.delta_rule(q[:, :3], twice, v[:, :3], none, ones[:, :3])
    assert torch.allclose(state[0, :, 0], v[0, 2], atol=1e-14)
    # one chunk: (1 + N diag(b)) e = v - exp(G) K S, o and S' from e
    h0 = _r(1, 2, 4, 3, seed=6)
    out, state = O.delta_rule(q, k, v, g, b, h0=h0, scale=0.7)
    for h in range(2):
        K, Q, V, S = k[0, :, h], q[0, :, h], v[0, :, h], h0[0, h]
        G, B = g[0, :, h].cumsum(0), b[0, :, h]
        w = (G[:, None] - G).exp().tril()
        M = torch.eye(9, dtype=torch.float64) + ((K @ K.T) * w).tril(-1) * B
        u = B[:, None] * torch.linalg.solve(M, V - G.exp()[:, None] * (K @ S))
        o = 0.7 * (G.exp()[:, None] * (Q @ S) + ((Q @ K.T) * w) @ u)
        assert torch.allclose(out[0, :, h], o, atol=1e-12)
        assert torch.allclose(state[0, h], G[-1].exp() * S + ((G[-1] - G).exp()[:, None] * K).T @ u, atol=1e-12)


def test_oracle_norm_and_beams():
    x, y = _r(3, 16, seed=1), _r(3, 16, seed=2)
    h, z = O.residual_norm(x, y, post_norm=True, norm="layer", scale=0.5)
    want = x + 0.5 * torch.nn.functional.layer_norm(y, (16,), eps=1e-6)
    assert torch.allclose(h, want) and torch.allclose(z, torch.nn.functional.layer_norm(h, (16,), eps=1e-6))
    h, z = O.residual_norm(x, y)
    assert torch.equal(h, x + y)
    assert torch.allclose(z, torch.nn.functional.rms_norm(h, (16,), eps=1e-6))
    logits, scores = _r(2, 3, 11, seed=3), _r(2, 3, seed=4)
    found = O.beam_select(logits, scores, 5)
    total = (scores[..., None] + torch.log_softmax(logits, -1)).flatten(1)
    top = total.topk(5)
    for b in range(2):
        assert [k * 11 + t for _, k, t in found[b]] == top.indices[b].tolist()
    new, copies = O.reorder_pages([7, 3, 9], [2, 2, 0])
    assert new == [9, 3, 7] and copies == {3: 9}


def _view(st=16, sb=128, sh=8, heads=2, p=4096):
    return _lib.LaView(p, sb, st, sh, heads)


def _problem(q=None, k=None, v=None, g_st=2, B=1, T=8, dtype=0, b=4096, b_dtype=0, Dk=8, H=2, h0=None,
             table=None):
    """Two heads of (8, 8) in float32."""
    la = _lib.LaProblem(q or _view(), k or _view(), v or _view(), 4096, 16, g_st, 1, h0, table, None,
                        1 if h0 else 0, 0, B, T, H, Dk, 8, dtype, dtype, 1.0)
    return _lib.DeltaProblem(la, b, 16, 2, 1, b_dtype)


def _forward(p, out=None, ws=4096, size=1 << 30, kept=None):
    return _lib.load().prnn_delta_rule(ctypes.byref(p), ctypes.byref(out or _view()), None, None, 0, kept,
                                       ws, size, None)


def _backward(p, go=None, ws=4096, size=1 << 30, kept=4096, dq=4096):
    return _lib.load().prnn_delta_rule_backward(ctypes.byref(p), ctypes.byref(go or _view()), None, kept,
                                                dq, 4096, 4096, 4096, 4096, None, ws, size, None)


CALLS = (_forward, _backward)
VALUE, TYPE, RUNTIME = _lib.PRNN_ERR_VALUE, _lib.PRNN_ERR_TYPE, _lib.PRNN_ERR_RUNTIME


def _said(what):
    return what in _lib.load().prnn_last_error()


@built
@no_device
def test_rule_entries_refuse():
    lib = _lib.load()
    down = _view(st=-16)
    for p in (_problem(q=down), _problem(k=down), _problem(v=down), _problem(g_st=-2)):
        assert lib.prnn_delta_rule_workspace_size(ctypes.byref(p), 0) == 0
        assert lib.prnn_delta_rule_kept_size(ctypes.byref(p)) == 0
        assert lib.prnn_delta_rule_backward_workspace_size(ctypes.byref(p), 1) == 0
        for call in CALLS:
            assert call(p) == VALUE and _said(b"apart")
    for call in CALLS:
        assert call(_problem(), down) == VALUE and _said(b"apart")
        assert call(_problem(b=None)) == VALUE and _said(b"beta")
        assert call(_problem(b_dtype=1)) == TYPE and _said(b"beta")
        assert call(_problem(dtype=9)) == TYPE
        assert call(_problem(Dk=257)) == VALUE and _said(b"257")
        assert call(_problem(H=3)) == VALUE
        assert call(_problem(), _view(p=None)) == VALUE and _said(b"non-null")
        assert call(_problem(), ws=None) == VALUE and _said(b"workspace")
        assert call(_problem(), ws=4097) == VALUE and _said(b"workspace")
        assert call(_problem(), size=255) == VALUE and _said(b"workspace")
        # rows of bfloat16 off a 16-byte boundary, or on top of each other
        for bad in (_view(p=4098), _view(st=12), _view(st=0, sh=0), _view(sh=4)):
            for p, other in ((_problem(q=bad, dtype=1), None), (_problem(k=bad, dtype=1), None),
                             (_problem(v=bad, dtype=1), None), (_problem(dtype=1), bad)):
                assert call(p, other) == VALUE and _said(b"16-byte")
        # nothing of these: what fails then is the missing device
        assert call(_problem()) == RUNTIME
        assert call(_problem(dtype=1)) == RUNTIME
    assert _forward(_problem(), kept=4097) == VALUE and _said(b"boundary")
    assert _backward(_problem(), kept=None) == VALUE and _said(b"kept")
    assert _backward(_problem(), dq=None) == VALUE and _said(b"non-null")
    assert _backward(_problem(dtype=1), dq=4104) == VALUE and _said(b"16-byte")
    assert _backward(_problem(h0=4096, table=4096)) == VALUE and _said(b"block table")
    assert _backward(_problem(h0=4096, B=2)) == VALUE and _said(b"h0")
    assert lib.prnn_delta_rule(None, ctypes.byref(_view()), None, None, 0, None, None, 0, None) == VALUE


@built
@no_device
def test_rule_workspaces():
    """What a forward pass keeps is not in its workspace; both are whole for no tokens at all; a grid
    beyond what a launch takes is refused."""
    lib = _lib.load()
    size = lambda p, kept: lib.prnn_delta_rule_workspace_size(ctypes.byref(p), kept)  # noqa: E731
    p = _problem(T=1000)
    assert size(p, 0) > size(p, 1) and lib.prnn_delta_rule_kept_size(ctypes.byref(p)) > size(p, 0) - size(p, 1)
    for empty in (_problem(B=0), _problem(T=0)):
        assert size(empty, 0) >= 0
    many = _problem(B=1 << 20, T=1, q=_view(heads=64), k=_view(heads=64), v=_view(heads=64), H=64)
    assert _forward(many, size=1 << 62) == VALUE and _said(b"too many for a launch")
    far = 1 << 40
    one = _problem(_view(st=far), _view(st=-far), _view(st=far), g_st=far, B=3, T=1)
    for call in CALLS:
        assert call(one, _view(st=far)) == RUNTIME  # an only token's stride does not matter


@built
@no_device
def test_step_entry_refuses():
    args = dict(q=(4096, 8, 8, 2), k=(4096, 8, 8, 2), v=(4096, 8, 8, 2), g=(4096, 2, 1, 0), b=(4096, 2, 1, 0),
                state=4096, B=1, H=2, Dk=8, Dv=8, dtype=0)

    def call(**kw):
        a = {**args, **kw}
        return _lib.load().prnn_delta_rule_step(*a["q"], *a["k"], *a["v"], *a["g"], *a["b"], a["state"],
                                                None, 1, 4096, a["B"], a["H"], a["Dk"], a["Dv"], 1.0,
                                                a["dtype"], None)

    for bad in (dict(q=(None, 8, 8, 2)), dict(k=(4096, 8, 8, 3)), dict(v=(4096, 8, 8, 0)), dict(b=(None, 2, 1, 0)),
                dict(state=None), dict(B=-1), dict(B=65536), dict(H=0), dict(Dk=0), dict(Dv=257)):
        assert call(**bad) == VALUE, bad
    for bad in (dict(dtype=7), dict(g=(4096, 2, 1, 1)), dict(b=(4096, 2, 1, 2))):
        assert call(**bad) == TYPE, bad
    assert call(B=0) == _lib.PRNN_OK and call() == RUNTIME


@built
@no_device
def test_norm_entries_refuse():
    lib = _lib.load()

    def forward(x=4096, y=4096, h=4096, z=4096, N=4, C=8, eps=1e-6, act=0, w_dtype=0, dtype=0):
        return lib.prnn_residual_norm(x, y, None, None, None, None, None, 1.0, h, z, N, C, eps, 0, 0, act,
                                      w_dtype, dtype, None)

    def backward(gh=4096, gz=4096, x=4096, dw=None, N=4, C=8, ws=4096, size=1 << 30):
        return lib.prnn_residual_norm_backward(gh, gz, x, 4096, None, None, None, None, 1.0, 4096, 4096, dw,
                                               None, None, None, None, N, C, 1e-6, 0, 0, 0, 0, 0, ws, size,
                                               None)

    for bad in (dict(x=None), dict(z=None), dict(h=None), dict(N=-1), dict(C=0), dict(C=16385), dict(eps=-1.0),
                dict(eps=float("nan")), dict(act=3)):
        assert forward(**bad) == VALUE, bad
    for bad in (dict(dtype=5), dict(w_dtype=1), dict(dtype=1, w_dtype=2)):
        assert forward(**bad) == TYPE, bad
    for bad in (dict(gh=None, gz=None), dict(x=None), dict(dw=4096, ws=None), dict(dw=4096, size=4)):
        assert backward(**bad) == VALUE, bad
    assert forward(N=0) == backward(N=0) == _lib.PRNN_OK
    assert forward() == backward() == backward(dw=4096) == RUNTIME
    assert lib.prnn_residual_norm_backward_workspace_size(0, 8) == 0
    assert lib.prnn_residual_norm_backward_workspace_size(4, 8) > 0


@built
@no_device
def test_beam_entries_refuse():
    lib = _lib.load()

    def select(logits=4096, ended=None, pad=0, out=4096, B=1, K=2, V=9, M=2, dtype=0, ws=4096, size=1 << 40):
        return lib.prnn_beam_select(logits, K * V, V, 4096, ended, pad, out, 4096, 4096, B, K, V, M, dtype,
                                    ws, size, None)

    for bad in (dict(logits=None), dict(out=None), dict(B=-1), dict(K=0), dict(V=0), dict(M=0), dict(M=129),
                dict(ended=4096, pad=9), dict(ended=4096, pad=-1), dict(ws=None), dict(ws=4100), dict(size=64),
                dict(K=1 << 16, V=1 << 15), dict(B=1 << 30, K=2)):
        assert select(**bad) == VALUE, bad
    assert select(B=1 << 23, size=1 << 62) == VALUE and _said(b"too many for a launch")
    assert select(dtype=3) == TYPE
    assert select(B=0) == _lib.PRNN_OK and select() == RUNTIME

    def reorder(slots=4, pool=4096, size=64, table=4096, parents=4096, scratch=4096, B=1, K=2, n=1):
        pools = (_lib.Pool * 1)(_lib.Pool(pool, size))
        return lib.prnn_pages_reorder(slots, pools, n, table, parents, B, K, scratch, None)

    for bad in (dict(table=None), dict(parents=None), dict(scratch=None), dict(B=-1), dict(K=0), dict(K=1025),
                dict(slots=-1), dict(pool=None), dict(B=1 << 21, K=1024)):
        assert reorder(**bad) == VALUE, bad
    assert reorder(B=0) == _lib.PRNN_OK and reorder() == RUNTIME
