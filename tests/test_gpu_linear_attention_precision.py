"""How exact the linear attention is beyond a tolerance per type: outputs against their own rounding."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    return float((got - want).norm() / want.norm())


def _inputs(B, T, heads, Dk, Dv, dtype, seed, g=None, g_dtype=None):
    """q, k, v, decays (drawn, or all ``g``), an initial state, gradients of output and state."""
    r = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    H = max(heads)
    q = torch.randn(B, T, hq, Dk, generator=r).to(dtype)
    k = (torch.randn(B, T, hk, Dk, generator=r) / Dk ** 0.5).to(dtype)
    v = torch.randn(B, T, hv, Dv, generator=r).to(dtype)
    a = -torch.nn.functional.softplus(torch.randn(B, T, H, generator=r) - 2)
    a = (a if g is None else torch.full_like(a, g)).to(g_dtype or dtype)
    h0 = torch.randn(B, H, Dk, Dv, generator=r)
    go = torch.randn(B, T, H, Dv, generator=r).to(dtype)
    gs = torch.randn(B, H, Dk, Dv, generator=r)
    return q, k, v, a, h0, go, gs


@pytest.mark.parametrize("B,T,heads,Dk,Dv", [(2, 130, (2, 2, 2), 64, 64), (1, 1500, (2, 1, 2), 128, 128),
                                             (3, 70, (4, 2, 1), 24, 48)])
def test_bf16_outputs_are_sums_rounded_once(B, T, heads, Dk, Dv):
    """Every operand of the products is held to 16 bits at least: what they add to the last rounding's
    error, some 0.4 2^-8 in the mean square, is a few times 2^-17, in the root of the squares' sum less
    than one part in a hundred; a tenth is allowed.  (One operand in 8 bits adds as much as the rounding
    itself: a factor of 1.4 for two.)"""
    from pararnn_amd import linear_attention

    q, k, v, g, h0, _, _ = _inputs(B, T, heads, Dk, Dv, BF16, seed=T)
    o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g, h0)))
    once = _rel(o64.to(BF16), o64)
    with torch.no_grad():
        out, state = linear_attention(*(x.to(DEV) for x in (q, k, v, g)), h0=h0.to(DEV),
                                      return_state=True)
    print(f"case {B, T, heads, Dk, Dv}: {_rel(out, o64):.2e}, rounded once {once:.2e}", flush=True)
    assert _rel(out, o64) <= 1.1 * once
    assert _rel(state, s64) <= 2.7e-6


def _decay_gradient(q, k, v, g, go, scale):
    """dL/dg of one head by its definition in 64 bits, exp(g_t) <S_{t-1}, R_t>: states forwards, adjoints
    backwards, no running sum."""
    q, k, v, g, go = (x[0, :, 0].to(DEV).double() for x in (q, k, v, g[..., None], go))
    T, a = q.shape[0], torch.exp(g[:, 0])
    states = torch.empty(T, q.shape[1], v.shape[1], device=DEV, dtype=torch.float64)
    s = torch.zeros_like(states[0])
    for t in range(T):
        states[t] = s  # before token t
        s = a[t] * s + k[t][:, None] * v[t]
    r, dg = torch.zeros_like(s), torch.empty(T, device=DEV, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        r = r + scale * q[t][:, None] * go[t]
        dg[t] = a[t] * (states[t] * r).sum()
        r = a[t] * r
    return dg


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [512, 8192])
@pytest.mark.parametrize("g", [-4.0, -8.0, -12.0])
def test_decay_gradient_behind_strong_decays(g, T, dtype):
    """The flow behind a decay of exp(-12) is a small part of what a token hands to itself.  The running
    sum's increments are each off by e of their value, two of them a token, and add up like a walk that
    is tied at both ends: sqrt(2 T / 6) e in the mean square, 52 e at 8192 tokens.  fp32 sums of 64
    products, like a walk of 8 roundings: e = 8 2^-24, 2.5e-5.  bf16: operands of 16 bits, each off by
    2^-17 at most, and exponents from sums of up to 64 12 / ln 2 = 1108, off by 2^-14 at most twice, 0.4
    of that in the mean square: e = 3.5e-5, 1.8e-3; the bound of all 16-bit decay gradients is kept."""
    from pararnn_amd import linear_attention

    q, k, v, a, _, go, _ = _inputs(1, T, (1, 1, 1), 64, 64, dtype, seed=T, g=g, g_dtype=F32)
    want = _decay_gradient(q, k, v, a, go, 64 ** -0.5)
    # in several sequences of one batch, that are not cut, too
    for n in (1, 3):
        leaf = a.expand(n, T, 1).contiguous().to(DEV).requires_grad_(True)
        out = linear_attention(*(x.to(DEV).expand(n, T, 1, 64) for x in (q, k, v)), leaf)
        got = torch.autograd.grad(out, leaf, go.to(DEV).expand(n, T, 1, 64))[0]
        assert got.dtype == F32
        for i in range(n):
            e = _rel(got[i, :, 0], want)
            print(f"case decay {g}, {T} tokens, {dtype}, {n} sequences: {e:.1e}", flush=True)
            assert e <= (8e-3 if dtype == BF16 else 2.5e-5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("at", [(0,), (40, 41, 60), (64, 127, 128), tuple(range(0, 300, 7))])
def test_gradients_through_resets(at, dtype):
    """Decays of -inf, several in a chunk, at chunks' and pieces' ends, next to each other: all gradients
    against the definition, and exactly zero for the resets themselves.  Tolerances as everywhere."""
    from pararnn_amd import linear_attention

    T = 300
    q, k, v, g, h0, go, gs = _inputs(2, T, (2, 1, 2), 64, 48, dtype, seed=3, g_dtype=F32)
    g[:, list(at)] = float("-inf")
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g, h0)]
    o64, s64 = O.linear_attention(*exact)
    names = ("dq", "dk", "dv", "dg", "dh0")
    want = dict(zip(names, torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])))
    mine = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, h0)]
    out, state = linear_attention(*mine[:4], h0=mine[4], return_state=True)
    got = dict(zip(names, torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])))
    assert torch.equal(got["dg"][:, list(at)].cpu(), torch.zeros(2, len(at), 2))
    for name, x in got.items():
        assert torch.isfinite(x).all(), name
        if name == "dg":
            tol = 1e-5 if dtype == F32 else 8e-3
        else:
            tol = 2.7e-6 if dtype == F32 or name == "dh0" else 3.9e-3
        e = _rel(x, want[name]) if want[name].any() else float(x.double().norm())
        print(f"case resets {at[:3]} {dtype} {name}: {e:.1e}", flush=True)
        assert e <= tol, (name, e)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [1, 2, 64, 300, 1500])
@pytest.mark.parametrize("g", [-6.0, -10.0, -20.0])
def test_decay_gradient_of_strong_decays_with_states(g, T, dtype):
    """With gradients of the final state: what the last token hands to it is of the order of one, what
    flows through the token's decay exp(g) of that.  The bounds of the test above (2.5e-5 for e of sums
    of 64 in fp32, 8e-3 in bfloat16 operands)."""
    from pararnn_amd import linear_attention

    q, k, v, a, h0, go, gs = _inputs(2, T, (2, 1, 2), 64, 64, dtype, seed=T, g=g, g_dtype=F32)
    exact = [t.double().requires_grad_(True) for t in (q, k, v, a, h0)]
    o64, s64 = O.linear_attention(*exact)
    want = torch.autograd.grad([o64, s64], exact[3], [go.double(), gs.double()])[0]
    mine = [t.to(DEV).requires_grad_(True) for t in (q, k, v, a, h0)]
    out, state = linear_attention(*mine[:4], h0=mine[4], return_state=True)
    got = torch.autograd.grad([out, state], mine[3], [go.to(DEV), gs.to(DEV)])[0]
    e = _rel(got, want)
    print(f"case decay {g}, {T} tokens with states, {dtype}: {e:.1e}", flush=True)
    assert e <= (8e-3 if dtype == BF16 else 2.5e-5)
