"""The residual norm against its definition in float64: types, widths, options, missing gradients.

Tolerances (relative 2-norm), from the arithmetic.  float32: sums over at most 16384 channels or 3000
rows, each of their roundings 2^-24, like a random walk sqrt(16384) 2^-24 = 7.6e-6 at the very most;
the sums are trees, so 2e-6 bounds them with room.  16 bits: every result is rounded once, at most
half a step of a value (2^-8 in bfloat16, 2^-11 in float16)."""

import pytest
import torch

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 2e-6, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    n = want.norm()
    return float((got - want).norm() / n) if n > 0 else float((got - want).norm())


CASES = [
    # shape, norm, post, post weight, act, gate, scale, weight, bias, parameters in float32
    ((1, 1), "rms", True, True, None, True, "vector", True, True, False),
    ((3, 7), "layer", True, True, "silu", True, "vector", True, True, False),
    ((2, 5, 64), "rms", False, False, "sigmoid", True, 0.5, True, False, True),
    ((33, 1000), "layer", True, False, None, False, "vector", False, True, False),
    ((5, 1024), "rms", True, True, "silu", True, "vector", True, False, False),
    ((1, 2048), "rms", False, False, None, False, None, False, False, False),
    ((3000, 40), "layer", True, True, "silu", True, "vector", True, True, True),
    ((17, 4104), "layer", True, True, "sigmoid", True, "vector", True, True, False),
    ((6, 8191), "rms", True, True, None, True, -1.5, True, True, False),
    ((3, 16384), "layer", True, True, "silu", True, "vector", True, True, False),
]


def _case(case, dtype, seed=0):
    shape, norm, post, pweight, act, gated, scale, weight, bias, wide = case
    r = torch.Generator().manual_seed(seed + shape[-1])
    c, pt = shape[-1], F32 if wide else dtype
    given = dict(x=(torch.randn(*shape, generator=r) * 2 + 0.3).to(dtype),
                 y=(torch.randn(*shape, generator=r) - 0.2).to(dtype))
    if weight:
        given["weight"] = (1 + 0.1 * torch.randn(c, generator=r)).to(pt)
    if bias:
        given["bias"] = (0.1 * torch.randn(c, generator=r)).to(pt)
    if pweight:
        given["post_weight"] = (1 + 0.1 * torch.randn(c, generator=r)).to(pt)
    if gated:
        given["gate"] = torch.randn(*shape, generator=r).to(dtype)
    fixed = dict(post_norm=post, activation=act, norm=norm, eps=1e-6)
    if scale == "vector":
        given["scale"] = torch.randn(c, generator=r).to(pt)
    elif scale is not None:
        fixed["scale"] = scale
    seeds = [torch.randn(*shape, generator=r).to(dtype) for _ in range(2)]
    return given, fixed, seeds


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=["x".join(map(str, c[0])) for c in CASES])
def test_forward_and_gradients(case, dtype):
    from pararnn_amd import residual_norm

    print(f"case residual norm {case} {dtype}", flush=True)
    given, fixed, seeds = _case(case, dtype)
    exact = {n: t.double().requires_grad_(True) for n, t in given.items()}
    want = O.residual_norm(**exact, **fixed)
    gwant = torch.autograd.grad(want, list(exact.values()), [s.double() for s in seeds])
    mine = {n: t.to(DEV).requires_grad_(True) for n, t in given.items()}
    got = residual_norm(**mine, **fixed)
    grads = torch.autograd.grad(got, list(mine.values()), [s.to(DEV) for s in seeds])
    for n, g, w in zip(["h", "z"] + ["d" + n for n in mine], [*got, *grads], [*want, *gwant]):
        e = _rel(g, w)
        # of a single channel norm(t) is 1 or 0 and its gradient cancels: against what goes in
        if case[0][-1] == 1 and n in ("dx", "dy"):
            assert float((g.double().cpu() - w.double()).abs().max()) <= 16 * TOL[g.dtype]
            continue
        assert e <= TOL[g.dtype], (n, e)
    with torch.no_grad():
        again = residual_norm(**mine, **fixed)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_in_front_of_the_first_block(norm):
    from pararnn_amd import residual_norm

    x = torch.randn(40, 320, generator=torch.Generator().manual_seed(2))
    w = torch.randn(320, generator=torch.Generator().manual_seed(3))
    gz = torch.randn(40, 320, generator=torch.Generator().manual_seed(4))
    ex, ew = x.double().requires_grad_(True), w.double().requires_grad_(True)
    _, want = O.residual_norm(ex, None, ew, norm=norm)
    gwant = torch.autograd.grad(want, [ex, ew], gz.double())
    mx, mw = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    h, z = residual_norm(mx, None, mw, norm=norm)
    assert h is mx and _rel(z, want) <= TOL[F32]
    got = torch.autograd.grad(z, [mx, mw], gz.to(DEV))
    assert all(_rel(a, b) <= TOL[F32] for a, b in zip(got, gwant))


@pytest.mark.parametrize("only", [0, 1], ids=["h", "z"])
def test_one_of_the_outputs_has_a_gradient(only):
    from pararnn_amd import residual_norm

    given, fixed, seeds = _case(CASES[4], BF16)
    exact = {n: t.double().requires_grad_(True) for n, t in given.items()}
    want = torch.autograd.grad(O.residual_norm(**exact, **fixed)[only], list(exact.values()),
                               seeds[only].double(), allow_unused=True)
    mine = {n: t.to(DEV).requires_grad_(True) for n, t in given.items()}
    got = torch.autograd.grad(residual_norm(**mine, **fixed)[only], list(mine.values()),
                              seeds[only].to(DEV), allow_unused=True)
    for n, g, w in zip(mine, got, want):
        w = torch.zeros_like(exact[n]) if w is None else w
        assert (g is None and float(w.norm()) == 0) or _rel(g, w) <= TOL[BF16], n


def test_empty_and_strided():
    from pararnn_amd import residual_norm

    x = torch.zeros(0, 96, device=DEV, requires_grad=True)
    w = torch.ones(96, device=DEV, requires_grad=True)
    h, z = residual_norm(x, x * 2, w)
    assert h.shape == z.shape == (0, 96)
    gx, gw = torch.autograd.grad([h, z], [x, w], [torch.zeros_like(h), torch.zeros_like(z)])
    assert gx.shape == (0, 96) and float(gw.abs().sum()) == 0
    big = torch.randn(6, 200, device=DEV)
    a, b = big[:, 3:99], big[:, 101:197]  # off a 16-byte boundary
    got = residual_norm(a, b, w, post_norm=True)
    want = residual_norm(a.contiguous(), b.contiguous(), w, post_norm=True)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
