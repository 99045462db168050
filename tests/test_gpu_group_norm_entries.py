"""The group norm's C entries where a caller may do what the Python call does not: arrays that lie
differently in the forward and the backward call."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rel(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("dtype,C,groups,shift", [
    (torch.bfloat16, 1000, 1, 2), (torch.bfloat16, 1200, 2, 1), (torch.float16, 2048, 2, 1),
    (torch.float32, 600, 1, 1)])
def test_backward_arrays_lie_differently(dtype, C, groups, shift):
    """The forward call's rows are aligned, and it takes whole groups into registers; the backward call's
    gradient is ``shift`` elements off, and it works from the statistics.  One rounding of the results,
    2^-8 (bfloat16) or 2^-11 (float16) at most; float32 as the norm's other tests: 1e-5."""
    from pararnn_amd import _lib

    print(f"case entries {dtype} {C} {groups} {shift}", flush=True)
    lib, n = _lib.load(), 5
    r = torch.Generator().manual_seed(C)
    x, gy = torch.randn(n, C, generator=r).to(dtype), torch.randn(n, C, generator=r).to(dtype)
    w, b = (1 + 0.2 * torch.randn(C, generator=r)).to(dtype), torch.randn(C, generator=r).to(dtype)
    exact = [t.double().requires_grad_(True) for t in (x, w, b)]
    y64 = O.group_norm(exact[0], groups, exact[1], exact[2], None, "silu")
    want = torch.autograd.grad(y64, exact, gy.double())

    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    mine = [t.to(DEV) for t in (x, w, b)]
    off = torch.empty(n * C + shift, dtype=dtype, device=DEV)[shift:].view(n, C)
    off.copy_(gy)
    y, dx, dw, db = (torch.empty_like(t) for t in (mine[0], *mine))
    stats = torch.full((n, groups, 2), float("nan"), device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    tail = (n, 1, C, groups, 1e-5, 1, code, code)
    need = [lib.prnn_group_norm_workspace_size(n, 1, C, groups, code, k) for k in (0, 1)]
    ws = torch.empty(max(*need, 256), dtype=torch.uint8, device=DEV)
    p = [t.data_ptr() for t in mine]
    _lib.check(lib.prnn_group_norm(*p, None, y.data_ptr(), stats.data_ptr(), *tail, ws.data_ptr(),
                                   ws.numel(), stream), "forward")
    _lib.check(lib.prnn_group_norm_backward(
        off.data_ptr(), *p, None, stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), None,
        *tail, ws.data_ptr(), ws.numel(), stream), "backward")
    torch.cuda.synchronize()
    tol = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for name, got, e in zip(("y", "dx", "dw", "db"), (y, dx, dw, db), (y64.detach(), *want)):
        assert _rel(got, e) <= tol, name
