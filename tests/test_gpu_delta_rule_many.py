"""The gated delta rule where sequences are many: workgroups of four waves, waves of 32 columns, cut
sequences among them.  Sequences do not depend on each other, so some are checked against 64 bits."""

import pytest
import torch
from test_gpu_delta_rule import BF16, DEV, F32, NAMES, _inputs, _rel, _tol

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu


def _check(dtype, names, got, want, what):
    errs = {n: _rel(x, y) for n, x, y in zip(names, got, want)}
    print(f"  {what}", {n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    for n, e in errs.items():
        assert e <= _tol(n, dtype), (what, n, e)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [(40, 130, 4, 64, 64), (520, 130, 4, 64, 64), (300, 70, 4, 128, 128),
                                  (300, 70, 8, 32, 96), (700, 65, 4, 24, 16), (150, 66, 8, 200, 72)],
                         ids=lambda c: f"B{c[0]}T{c[1]}D{c[3]}x{c[4]}")
def test_many_sequences(case, dtype):
    from pararnn_amd import delta_rule

    B, T, H, Dk, Dv = case
    print(f"case many {case} {dtype}", flush=True)
    given = _inputs(B, T, (H, H, H), Dk, Dv, dtype, "token", seed=B)
    go, gs = given[6:]
    mine = [t.to(DEV).requires_grad_(True) for t in given[:6]]
    out, state = delta_rule(*mine[:5], h0=mine[5], return_state=True)
    grads = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    with torch.no_grad():  # without what a backward pass needs
        again, last = delta_rule(*mine[:5], h0=mine[5], return_state=True)
    assert torch.equal(again, out) and torch.equal(last, state)
    for b in (0, B // 2, B - 1):
        exact = [t[b:b + 1].double().requires_grad_(True) for t in given[:6]]
        o64, s64 = O.delta_rule(*exact)
        want = torch.autograd.grad([o64, s64], exact, [go[b:b + 1].double(), gs[b:b + 1].double()])
        _check(dtype, ("out", "state", *NAMES), [t[b:b + 1] for t in (out, state, *grads)],
               (o64, s64, *want), f"sequence {b}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(4, 64, 64), (4, 128, 72), (2, 48, 130)], ids=lambda s: f"D{s[1]}x{s[2]}")
def test_a_long_sequence_among_short_ones(shape, dtype):
    from pararnn_amd import PackedSequences, delta_rule

    H, Dk, Dv = shape
    lens = [3] * 250 + [2100] + [2] * 250
    cu = [0, *torch.tensor(lens).cumsum(0).tolist()]
    print(f"case long among short {shape} {dtype}", flush=True)
    given = _inputs(1, cu[-1], (H, 1, H), Dk, Dv, dtype, "token", seed=5, seqs=len(lens))
    go, gs = given[6:]
    mine = [t.to(DEV).requires_grad_(True) for t in given[:6]]
    out, state = delta_rule(*mine[:5], h0=mine[5], return_state=True,
                            cu_seqlens=PackedSequences(torch.tensor(cu)))
    grads = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    for s in (0, 249, 250, 251, 500):
        rows = slice(cu[s], cu[s + 1])
        exact = [t[:, rows].double().requires_grad_(True) for t in given[:5]]
        exact.append(given[5][s:s + 1].double().requires_grad_(True))
        o64, s64 = O.delta_rule(*exact)
        want = torch.autograd.grad([o64, s64], exact, [go[:, rows].double(), gs[s:s + 1].double()])
        got = [out[:, rows], state[s:s + 1], *(t[:, rows] for t in grads[:5]), grads[5][s:s + 1]]
        _check(dtype, ("out", "state", *NAMES), got, (o64, s64, *want), f"sequence {s}")
