"""Scales of any sign, float32 decays of 16-bit data, long sequences, infinities and NaN: what the
operators' first tests left out.

Tolerances as there: float32 2.7e-6 (the decays' gradient 1e-5), states likewise; bfloat16 3.9e-3 and
8e-3.  float16 is float32 arithmetic rounded once, 2^-11 of a value at most: 4.9e-4.  What lies below
float32's normal range, 2^-126, may be anything below it (an initial state's gradient behind 600 tokens
of decay, where nothing else adds to it)."""

import pytest
import torch

from oracle import linear_attention as O
from test_gpu_linear_attention_precision import DEV, BF16, F16, F32, _decay_gradient, _inputs

pytestmark = pytest.mark.gpu

TOL = {F32: 2.7e-6, BF16: 3.9e-3, F16: 2.0 ** -11}
TOL_G = {F32: 1e-5, BF16: 8e-3, F16: 2.0 ** -11}
NAN, INF = float("nan"), float("inf")


def _off(got, want, below=2.0 ** -126):
    """Relative 2-norm of the difference, but for ``below`` a value; of what should be zero, the norm
    itself."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    n, least = float(want.norm()), below * want.numel() ** 0.5
    return max(0.0, float((got - want).norm()) - least) / (n if n > 0 else 1.0)


def _check(got, want, dtype, g_dtype):
    for name, x in got.items():
        state = name in ("state", "dh0")
        tol = TOL[F32] if state else TOL_G[dtype] if name == "dg" else TOL[dtype]
        e = _off(x, want[name])
        print(f"  {name} {e:.1e}", flush=True)
        assert x.dtype == (F32 if state else g_dtype if name == "dg" else dtype), name
        assert e <= tol, (name, e)


def _both(inputs, cu=None, scale=None):
    from pararnn_amd import linear_attention

    q, k, v, g, h0, go, gs = inputs
    names = ("dq", "dk", "dv", "dg", "dh0")
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g, h0)]
    o64, s64 = O.linear_attention(*exact, scale=scale, cu=cu)
    want = dict(zip(names, torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])),
                out=o64, state=s64)
    mine = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, h0)]
    out, state = linear_attention(*mine[:4], h0=mine[4], scale=scale, return_state=True,
                                  cu_seqlens=None if cu is None else torch.tensor(cu))
    got = dict(zip(names, torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])),
               out=out, state=state)
    return got, want


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0, 7.5])
def test_scales(scale, dtype):
    for T in (1, 90, 600):
        print(f"case scale {scale} {dtype} {T}", flush=True)
        _check(*_both(_inputs(2, T, (2, 1, 2), 32, 48, dtype, seed=T), scale=scale), dtype, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("cu", [None, [0, 0, 1, 257, 400, 1000]], ids=["batch", "packed"])
def test_float32_decays_of_16_bit_data(cu, dtype):
    B, T = (2, 300) if cu is None else (1, cu[-1])
    print(f"case float32 decays {cu} {dtype}", flush=True)
    q, k, v, g, h0, go, gs = _inputs(B, T, (4, 2, 1), 64, 64, dtype, seed=5, g_dtype=F32)
    if cu is not None:
        r = torch.Generator().manual_seed(6)
        h0, gs = (torch.randn(len(cu) - 1, 4, 64, 64, generator=r) for _ in range(2))
    _check(*_both((q, k, v, g, h0, go, gs), cu=cu), dtype, F32)


def test_a_step_with_scales_and_float32_decays():
    from pararnn_amd import linear_attention_step

    for dtype in (F32, BF16, F16):
        q, k, v, g, h0, _, _ = _inputs(3, 1, (4, 1, 2), 64, 40, dtype, seed=2, g_dtype=F32)
        for scale in (-0.3, 0.0, 2.0):
            o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g, h0)), scale=scale)
            state = h0.to(DEV)
            out = linear_attention_step(*(x[:, 0].to(DEV) for x in (q, k, v, g)), state, scale=scale)
            assert _off(out, o64[:, 0]) <= TOL[dtype] and _off(state, s64) <= TOL[F32]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decay_gradient_of_a_long_sequence(dtype):
    """20000 tokens, horizons of some 40: against the definition, no running sum.  The increments' errors
    add up like a walk tied at the pieces' ends, at most at the sequence's: sqrt(2 20000 / 6) = 82 of
    2^-17 (bfloat16 operands in two parts) and 2^-24 8 (fp32 sums of 64): 6e-4 and 4e-5; float32 decays,
    so nothing is rounded behind that."""
    from pararnn_amd import linear_attention

    q, k, v, g, _, go, _ = _inputs(1, 20000, (1, 1, 1), 64, 64, dtype, seed=8, g_dtype=F32)
    g = g / 5
    want = _decay_gradient(q, k, v, g, go, 64 ** -0.5)
    leaf = g.to(DEV).requires_grad_(True)
    out = linear_attention(*(x.to(DEV) for x in (q, k, v)), leaf)
    e = _off(torch.autograd.grad(out, leaf, go.to(DEV))[0][0, :, 0], want)
    print(f"case long decay gradient {dtype}: {e:.1e}", flush=True)
    assert e <= (4e-5 if dtype == F32 else 6e-4)


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_a_steps_rows_keep_to_themselves(bad):
    """A row's infinity or NaN, in its token or its state, reaches no other row; an idle row and a slot
    that no row names keep theirs; a decay of -inf forgets any finite state."""
    from pararnn_amd import linear_attention_step

    q, k, v, g, h0, _, _ = (t.to(DEV) for t in _inputs(5, 1, (2, 1, 2), 64, 48, BF16, seed=4))
    q, k, v, g = (x[:, 0] for x in (q, k, v, g))
    table = torch.tensor([3, 0, -1, 4, 1], dtype=torch.int32, device=DEV)
    clean = h0.clone()
    want = linear_attention_step(q, k, v, g, clean, block_table=table)
    others, slots = [0, 2, 3, 4], [0, 2, 3, 4]
    for name in ("q", "k", "v", "g", "state", "idle"):
        given, pool = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone()), h0.clone()
        if name == "state":
            pool[0, 0, 3, 5] = bad  # row 1's
        elif name == "idle":
            pool[2] = bad  # nobody's
        else:
            given[name][1] = bad if name != "g" else NAN
        out = linear_attention_step(*given.values(), pool, block_table=table)
        assert torch.equal(out[others], want[others]), name
        keep = [s for s in slots if s != 0 and not (name == "idle" and s == 2)]
        assert torch.equal(pool[keep], clean[keep]), name
        if name == "idle":
            assert torch.equal(out, want) and not torch.isfinite(pool[2]).any()
        elif name == "q":
            assert not torch.isfinite(out[1]).all() and torch.equal(pool, clean)
        else:
            assert not torch.isfinite(out[1]).all() and not torch.isfinite(pool[0]).all()
    g = g.clone()
    g[1] = -INF
    pool = h0.clone()
    out = linear_attention_step(q, k, v, g, pool, block_table=table)
    zero = h0.clone()
    zero[0] = 0
    assert torch.equal(out, linear_attention_step(q, k, v, g, zero, block_table=table))
    assert torch.equal(pool, zero)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("C,groups", [(64, 4), (5000, 2)], ids=["narrow", "wide"])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_a_norms_groups_keep_to_themselves(bad, C, groups, dtype):
    """An infinity or NaN in x reaches its own token's group (sample's group) and nothing else; one in
    the gate its own value."""
    from pararnn_amd import group_norm

    r = torch.Generator().manual_seed(C)
    cg = C // groups
    for shape, over in (((6, C), "token"), ((3, 4, C), "sample")):
        x, gate, gy = (torch.randn(shape, generator=r).to(DEV, dtype) for _ in range(3))
        w = torch.randn(C, generator=r).to(DEV, dtype)

        def run(x, gate):
            leaves = [x.clone().requires_grad_(True), gate.clone().requires_grad_(True)]
            y = group_norm(leaves[0], groups, w, gate=leaves[1], activation="silu", over=over)
            return (y.detach(), *torch.autograd.grad(y, leaves, gy))

        clean = run(x, gate)
        at = (2, 1) if over == "sample" else (2,)
        mine = torch.zeros(shape, dtype=torch.bool, device=DEV)
        mine[2, ..., cg:2 * cg] = True  # the group that shares the statistics
        poisoned = x.clone()
        poisoned[at + (cg + 3,)] = bad
        for got, want in zip(run(poisoned, gate), clean):
            assert torch.equal(got[~mine], want[~mine])
            assert not torch.isfinite(got[mine]).any() or over == "sample"
        y, dx, dgate = run(x, _set(gate, at + (cg + 3,), bad))
        one = torch.zeros_like(mine)
        one[at + (cg + 3,)] = True
        assert torch.equal(y[~one], clean[0][~one]) and not torch.isfinite(y[one]).all()
        assert torch.equal(dgate[~one], clean[2][~one])
        assert torch.equal(dx[~mine], clean[1][~mine])


def _set(t, at, value):
    t = t.clone()
    t[at] = value
    return t


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_large_values_of_the_activations(dtype):
    """Gates far from zero: silu and its derivative tend to 0 and z, without an overflow on the way.
    float16 holds nothing below 2^-24 (sigmoid's derivative at 20)."""
    from pararnn_amd import group_norm

    r = torch.Generator().manual_seed(1)
    x = torch.randn(4, 64, generator=r).to(dtype)
    gate = torch.tensor([-6e4, -300.0, -90.0, -20.0, 20.0, 90.0, 300.0, 6e4]).repeat(8).expand(4, 64)
    gate = gate.to(dtype).contiguous()
    gy = (torch.randn(4, 64, generator=r) * 2.0 ** -10).to(dtype)
    exact = [x.double().requires_grad_(True), gate.double().requires_grad_(True)]
    for act in ("silu", "sigmoid"):
        y64 = O.group_norm(exact[0], 4, None, None, exact[1], act)
        want = (y64, *torch.autograd.grad(y64, exact, gy.double()))
        mine = [x.to(DEV).requires_grad_(True), gate.to(DEV).requires_grad_(True)]
        y = group_norm(mine[0], 4, gate=mine[1], activation=act)
        for got, e in zip((y, *torch.autograd.grad(y, mine, gy.to(DEV))), want):
            finite = e.abs() <= torch.finfo(dtype).max
            assert torch.isfinite(got.cpu()[finite]).all()
            tol = {F32: 1e-5, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
            least = 2.0 ** -24 if dtype == F16 else 2.0 ** -126
            assert _off(got.cpu()[finite], e.detach()[finite], least) <= tol
