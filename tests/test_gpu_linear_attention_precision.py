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
