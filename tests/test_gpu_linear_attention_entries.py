"""The linear attention's C entries on arrays that the Python call never passes: 16-bit values off every
16-byte boundary."""

import ctypes

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _off(t, shift):
    """A dense copy that starts ``shift`` elements behind a 256-byte boundary."""
    base = torch.empty(t.numel() + shift, dtype=t.dtype, device=DEV)[shift:].view(t.shape)
    return base.copy_(t)


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("which", ["q", "out", "go", "dq", "dk", "dv"])
def test_arrays_off_16_bytes(which, shift):
    """Each array in turn; bfloat16 tolerances as everywhere (3.9e-3, 8e-3 for the decays' gradient)."""
    from pararnn_amd import _lib

    print(f"case entries off 16 bytes {which} {shift}", flush=True)
    lib, (B, T, H, D) = _lib.load(), (2, 90, 2, 64)
    r = torch.Generator().manual_seed(4)
    q, k, v, go = (torch.randn(B, T, H, D, generator=r).to(torch.bfloat16) for _ in range(4))
    k = (k / 8).to(torch.bfloat16)
    g = -torch.rand(B, T, H, generator=r)
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g)]
    o64, _ = O.linear_attention(*exact)
    want = dict(zip(("dq", "dk", "dv", "dg"), torch.autograd.grad(o64, exact, go.double())), out=o64)

    a = {n: _off(t, shift if n == which else 0) for n, t in dict(q=q, k=k, v=v, go=go, out=q, dq=q, dk=k,
                                                                dv=v).items()}
    g = g.to(DEV)
    dg = torch.empty_like(g)

    def view(t):
        return _lib.LaView(t.data_ptr(), T * H * D, H * D, D, H)

    p = _lib.LaProblem(view(a["q"]), view(a["k"]), view(a["v"]), g.data_ptr(), T * H, H, 1, None, None,
                       None, 0, 0, B, T, H, D, D, 0, 1, D ** -0.5, 0)
    c, stream = ctypes.byref(p), torch.cuda.current_stream().cuda_stream
    need = max(lib.prnn_linear_attention_workspace_size(c),
               lib.prnn_linear_attention_backward_workspace_size(c, 1), 256)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    out, go_view = view(a["out"]), view(a["go"])
    _lib.check(lib.prnn_linear_attention(c, ctypes.byref(out), None, None, 0, ws.data_ptr(), need,
                                         stream), "forward")
    _lib.check(lib.prnn_linear_attention_backward(
        c, ctypes.byref(go_view), None, a["dq"].data_ptr(), a["dk"].data_ptr(), a["dv"].data_ptr(),
        dg.data_ptr(), None, ws.data_ptr(), need, stream), "backward")
    torch.cuda.synchronize()
    for name, e in want.items():
        got = (dg if name == "dg" else a[name]).double().cpu()
        off = float((got - e.detach()).norm() / e.detach().norm())
        assert off <= (8e-3 if name == "dg" else 3.9e-3), (name, off)
