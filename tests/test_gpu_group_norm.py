"""Group norm against its sums in float64: values and all gradients over types, group widths (even,
odd, wider than a wave's registers), gates, activations and both kinds of statistics.

Tolerances (relative 2-norm): float32: sums of n values of one sign lose at most sqrt(n) 2^-24,
in any order no more than n; at the largest n here (2^17) a tree of partial sums stays below
64 2^-24 = 3.8e-6, and the input gradient cancels two such sums: 1e-5.  16 bits: one rounding of
the result, at most half a unit in the last of 8 (bfloat16) or 11 (float16) places: 2^-8, 2^-11."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 1e-5, BF16: 2.0 ** -8, F16: 2.0 ** -11}

CASES = [
    # shape, groups, activation, gate, over
    ((1, 8), 1, None, False, "token"),
    ((5, 16), 16, "silu", True, "token"),
    ((3, 7, 64), 4, "silu", True, "token"),
    ((300, 1024), 16, "silu", True, "token"),
    ((33, 50), 1, "sigmoid", False, "token"),
    ((20, 150), 3, "silu", True, "token"),
    ((9, 96), 8, None, True, "token"),
    ((6, 7), 7, "silu", False, "token"),
    ((4, 2000), 1, "silu", True, "token"),
    ((3, 5000), 1, "silu", False, "token"),
    ((2, 6006), 2, "sigmoid", True, "token"),
    ((3, 50, 64), 8, "silu", False, "sample"),
    ((2, 8, 9, 96), 3, None, True, "sample"),
    ((1, 2047, 24), 4, "silu", True, "sample"),
    ((5, 1, 30), 2, "silu", False, "sample"),
    ((2, 130, 3000), 2, "silu", False, "sample"),
    ((2, 20, 2600), 1, "sigmoid", True, "sample"),
    ((400, 3, 10), 5, None, False, "sample"),
]


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    n = want.norm()
    return float((got - want).norm() / n) if n > 0 else float((got - want).norm())


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_values_and_gradients(case, dtype):
    from pararnn_amd import group_norm

    shape, groups, act, gated, over = case
    print(f"case group norm {case} {dtype}", flush=True)
    r = torch.Generator().manual_seed(len(shape) + shape[-1])
    x = (torch.randn(shape, generator=r) * 2 + 0.5).to(dtype)
    C = shape[-1]
    w_dtype = F32 if groups % 2 else dtype  # float32 parameters of 16-bit values too
    w = (1 + 0.2 * torch.randn(C, generator=r)).to(w_dtype)
    b = (0.2 * torch.randn(C, generator=r)).to(w_dtype)
    gate = torch.randn(shape, generator=r).to(dtype) if gated else None
    gy = torch.randn(shape, generator=r).to(dtype)
    given = [x, w, b] + ([gate] if gated else [])
    # one group of one channel at one token has no deviation: its gradient is zero but for rounding
    exact = [t.double().requires_grad_(True) for t in given]
    y64 = O.group_norm(exact[0], groups, *exact[1:3], exact[3] if gated else None, act, over)
    want = torch.autograd.grad(y64, exact, gy.double())
    mine = [t.to(DEV).requires_grad_(True) for t in given]
    y = group_norm(mine[0], groups, mine[1], mine[2], gate=mine[3] if gated else None,
                   activation=act, over=over)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, mine, gy.to(DEV))
    with torch.no_grad():
        assert torch.equal(group_norm(mine[0], groups, mine[1], mine[2],
                                      gate=mine[3] if gated else None, activation=act, over=over),
                           y)
    errs = dict(y=_rel(y, y64))
    for name, a, e in zip(("dx", "dw", "db", "dgate"), got, want):
        assert a.dtype == dict(dx=dtype, dgate=dtype).get(name, w_dtype)
        if float(e.norm()) > 1e-9 * float(gy.double().norm()):
            errs[name] = _rel(a, e)
        else:
            assert float(a.double().norm()) <= 1e-5 * float(gy.double().norm())
    print("  ", {n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    for name, e in errs.items():
        t = TOL[w_dtype] if name in ("dw", "db") else TOL[dtype]
        assert e <= t, (name, e)


def test_parameters_left_out_and_large_mean():
    """Without weight and bias; and values far from zero: the deviations keep their digits (a mean
    of 1000 deviations costs 1000 2^-24 of one, 6e-5 relative to it)."""
    from pararnn_amd import group_norm

    r = torch.Generator().manual_seed(3)
    for shape, over in (((50, 256), "token"), ((4, 300, 64), "sample")):
        x = torch.randn(shape, generator=r) + 1000
        y = group_norm(x.to(DEV), 4, over=over)
        assert _rel(y, O.group_norm(x.double(), 4, over=over)) <= 1e-4


def test_views_and_misaligned_inputs():
    from pararnn_amd import group_norm

    r = torch.Generator().manual_seed(4)
    for dtype in (F32, BF16):
        base = torch.randn(40 * 64 + 3, generator=r).to(DEV, dtype)
        x = base[3:].view(40, 64)
        y = group_norm(x, 8, activation="silu")
        assert torch.equal(y, group_norm(x.clone(), 8, activation="silu"))
        xt = torch.randn(64, 40, generator=r).to(DEV, dtype).t()
        leaf = xt.detach().requires_grad_(True)
        g = torch.autograd.grad(group_norm(leaf, 8).sum(), leaf)[0]  # an expanded gradient
        dense = xt.contiguous().requires_grad_(True)
        assert torch.equal(g, torch.autograd.grad(group_norm(dense, 8), dense,
                                                  torch.ones_like(dense))[0])


def test_gradient_against_differences():
    """Central differences along random directions, step 2^-5: third order (2^-5)^2 = 1e-3 of the
    slope's scale at most, rounding sqrt(1000) 2^-24 / 2^-5 = 6e-5."""
    from pararnn_amd import group_norm

    r = torch.Generator().manual_seed(5)
    for shape, over in (((12, 40), "token"), ((2, 9, 40), "sample")):
        x, gate, gy = (torch.randn(shape, generator=r).to(DEV) for _ in range(3))
        w, b = (torch.randn(40, generator=r).to(DEV) for _ in range(2))
        leaves = [x, w, b, gate]

        def loss(t):
            y = group_norm(t[0], 4, t[1], t[2], gate=t[3], activation="silu", over=over)
            return (y.double() * gy.double()).sum()

        grads = torch.autograd.grad(loss([t.requires_grad_(True) for t in leaves]), leaves)
        with torch.no_grad():
            for t, g in zip(leaves, grads):
                d = torch.randn(t.shape, generator=r).to(DEV)
                e = 2.0 ** -5 / float(d.norm())
                up, down = ([u + s * e * d if u is t else u for u in leaves] for s in (1, -1))
                slope = float((loss(up) - loss(down)) / (2 * e))
                scale = float(g.double().norm() * d.double().norm())
                assert abs(slope - float((g.double() * d.double()).sum())) <= 2e-3 * scale


def test_nothing_and_other_stream():
    from pararnn_amd import group_norm

    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = group_norm(x, 2, w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))
    assert group_norm(torch.zeros(0, 5, 8, device=DEV), 2, over="sample").shape == (0, 5, 8)
    assert group_norm(torch.zeros(3, 0, 8, device=DEV), 2, over="sample").shape == (3, 0, 8)
    x = torch.randn(64, 128, device=DEV)
    want = group_norm(x, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = group_norm(x, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
