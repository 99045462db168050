"""bfloat16 calls of the delta rule compute in 24 bits and round once: their results are those of 64 bits,
rounded, but for the few that lie next to a border.

A value that is off by d before it is rounded falls to the other side of a border with probability d /
step and is then a step off: its square on average is d step, and a step is at most 2^-7 of a value, so
results off by d (relative 2-norm) differ from the rounded exact ones by sqrt(d 2^-7).  d: a chunk's sums
have some 100 additions on their way (products with the state and the pairs, the system, the state's own
update), each off by 2^-25 in the mean square at most, and a state remembers some ten chunks: sqrt(1000)
2^-25 = 9.4e-7, below 1e-6.  With operands of 16 bits d is 2^-18 or more, and the difference 1.3e-4.
Gradients pass two such chains: twice d; the decays' and rates' are small differences of such sums: 16."""

import pytest
import torch
from test_gpu_delta_rule import BF16, DEV, _inputs, _rel

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

D = 1e-6
NAMES = ("dq", "dk", "dv", "dg", "dbeta")


def _border(d):
    return (d * 2.0 ** -7) ** 0.5


CASES = [  # B, T, heads, Dk, Dv
    (2, 600, (2, 2, 2), 64, 64),
    (1, 1500, (2, 1, 2), 128, 128),
    (1, 400, (2, 2, 2), 256, 64),
    (520, 70, (4, 4, 4), 32, 96),
    (300, 70, (4, 4, 4), 64, 64),
    (300, 70, (4, 4, 4), 128, 128),
]


@pytest.mark.parametrize("case", CASES, ids=[f"B{c[0]}T{c[1]}D{c[3]}x{c[4]}" for c in CASES])
def test_results_are_the_rounded_exact_ones(case):
    from pararnn_amd import delta_rule

    B, T, heads, Dk, Dv = case
    print(f"case bits {case}", flush=True)
    *given, go, gs = _inputs(B, T, heads, Dk, Dv, BF16, "token", seed=T + Dk)
    mine = [t.to(DEV).requires_grad_(True) for t in given]
    out, state = delta_rule(*mine[:5], h0=mine[5], return_state=True)
    got = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    with torch.no_grad():
        alone = delta_rule(*mine[:5], h0=mine[5])
    some = slice(0, min(B, 6))  # (sequences do not depend on each other)
    exact = [t[some].double().to(DEV).requires_grad_(True) for t in given]
    o64, s64 = O.delta_rule(*exact)
    want = torch.autograd.grad([o64, s64], exact, [go[some].double().to(DEV), gs[some].double().to(DEV)])
    errs = dict(out=_rel(out[some], o64.to(BF16)), alone=_rel(alone[some], o64.to(BF16)))
    tols = dict(out=_border(D), alone=_border(D))
    for name, x, y in zip(NAMES, got, want):
        errs[name] = _rel(x[some], y.to(BF16))
        tols[name] = _border((16 if name in ("dg", "dbeta") else 2) * D)
    errs.update(state=_rel(state[some], s64), dh0=_rel(got[5][some], want[5]))
    tols.update(state=D, dh0=2 * D)
    print("  ", {n: f"{e:.1e} ({tols[n]:.1e})" for n, e in errs.items()}, flush=True)
    for name, e in errs.items():
        assert e <= tols[name], (name, e)
