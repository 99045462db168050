"""The gated delta rule against the recurrence in float64: outputs, final states and gradients over
types, head layouts, odd widths and lengths, packed sequences, strides, resets, rates at their ends.

Tolerances (relative 2-norm), from the arithmetic.  Keys have unit length and rates lie in (0, 1), so
a token's system shrinks what reaches it and errors do not grow along a sequence.  float32: an element
is a sum of up to Dk products and 64 solved terms a chunk, each rounded to 2^-24, which add up like a
random walk: sqrt(2000) 2^-24 = 2.7e-6 at these sizes; gradients pass two such chains, 1e-5 (the
decays', a double sum over a chunk, among them).  States of bfloat16 inputs: operands of 16 bits (two
parts: 2^-17 of a value at most, 0.4 of that in the mean square) in three products of a chain (key
times state, the system, the state), 2^-17 0.4 sqrt(3) = 5.3e-6; three parts in the last one: 1e-5
bounds both chains.  Results of 16 bits: one rounding, at most 2^-8 = 3.9e-3 of a value, of sums whose
operands have 16 bits at least (the decays' and rates' gradients are small differences of such sums
where keys are few: twice that)."""

import pytest
import torch

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 2.7e-6, BF16: 3.9e-3, F16: 3.9e-3}
TOL_GRAD = {F32: 1e-5, BF16: 3.9e-3, F16: 3.9e-3}
TOL_SUMS = {F32: 1e-5, BF16: 7.8e-3, F16: 7.8e-3}
TOL_STATE = 1e-5


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    n = want.norm()
    return float((got - want).norm() / n) if n > 0 else float((got - want).norm())


def _inputs(B, T, heads, Dk, Dv, dtype, decay, seed, seqs=None, g_dtype=None):
    r = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    H = max(heads)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q = unit(torch.randn(B, T, hq, Dk, generator=r)).to(dtype)
    k = unit(torch.randn(B, T, hk, Dk, generator=r)).to(dtype)
    v = torch.randn(B, T, hv, Dv, generator=r).to(dtype)
    if decay == "token":
        g = -torch.nn.functional.softplus(torch.randn(B, T, H, generator=r) - 2)
        g = g.to(g_dtype or dtype)
    else:
        g = -0.2 * torch.rand(H, generator=r)
    beta = torch.rand(B, T, H, generator=r).to(dtype)
    h0 = torch.randn(seqs or B, H, Dk, Dv, generator=r)
    go = torch.randn(B, T, H, Dv, generator=r).to(dtype)
    gs = torch.randn(seqs or B, H, Dk, Dv, generator=r)
    return q, k, v, g, beta, h0, go, gs


NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dh0")


def _tol(name, dtype):
    if name == "state":
        return TOL[F32] if dtype == F32 else TOL_STATE
    if name == "dh0":
        return TOL_STATE
    if name == "out":
        return TOL[dtype]
    return (TOL_SUMS if name in ("dg", "dbeta") else TOL_GRAD)[dtype]


def _compare(dtype, given, go, gs, cu=None, packed=None):
    from pararnn_amd import delta_rule

    exact = [t.double().requires_grad_(True) for t in given]
    o64, s64 = O.delta_rule(*exact, cu=cu)
    want = torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])
    mine = [t.to(DEV).requires_grad_(True) for t in given]
    out, state = delta_rule(*mine[:5], h0=mine[5] if len(mine) > 5 else None, cu_seqlens=packed,
                            return_state=True)
    assert out.dtype == dtype and state.dtype == F32
    got = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    torch.cuda.synchronize()
    errs = dict(out=_rel(out, o64), state=_rel(state, s64))
    for name, x, y in zip(NAMES, got, want):
        errs[name] = _rel(x, y)
    print("  ", {n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    for name, e in errs.items():
        assert e <= _tol(name, dtype), (name, e)


CASES = [
    # B, T, (heads of q, k, v), Dk, Dv, decay, h0
    (1, 1, (1, 1, 1), 1, 1, "token", True),
    (2, 1, (4, 2, 1), 64, 64, "head", True),
    (3, 5, (2, 1, 2), 3, 7, "token", True),
    (1, 31, (1, 1, 1), 32, 16, "token", False),
    (2, 64, (2, 2, 2), 64, 64, "token", True),
    (2, 65, (4, 2, 1), 48, 72, "token", True),
    (1, 129, (2, 4, 4), 96, 33, "head", False),
    (1, 700, (1, 1, 1), 64, 64, "token", True),
    (1, 1500, (2, 1, 2), 128, 128, "token", False),
    (2, 600, (1, 1, 1), 64, 130, "head", True),
    (1, 300, (1, 1, 1), 256, 200, "token", True),
    (1, 200, (1, 1, 1), 128, 40, "token", True),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=[f"B{c[0]}T{c[1]}D{c[3]}x{c[4]}" for c in CASES])
def test_forward_and_gradients(case, dtype):
    B, T, heads, Dk, Dv, decay, with_h0 = case
    print(f"case delta rule {case} {dtype}", flush=True)
    q, k, v, g, beta, h0, go, gs = _inputs(B, T, heads, Dk, Dv, dtype, decay, seed=T + Dk)
    _compare(dtype, [q, k, v, g, beta] + ([h0] if with_h0 else []), go, gs)


PACKED = [
    ([0, 0, 1, 257, 257, 400, 600, 600], 33, 130, (2, 2, 2)),
    ([0, 513, 768, 1024, 1300], 64, 48, (2, 1, 1)),
    ([0, 1, 2, 3, 67, 131], 64, 64, (4, 4, 4)),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", PACKED, ids=["empty", "long", "short"])
def test_packed(case, dtype):
    from pararnn_amd import PackedSequences

    cu, Dk, Dv, heads = case
    S, N = len(cu) - 1, cu[-1]
    print(f"case packed delta rule {cu} {Dk}x{Dv} {dtype}", flush=True)
    q, k, v, g, beta, h0, go, gs = _inputs(1, N, heads, Dk, Dv, dtype, "token", 3, seqs=S)
    _compare(dtype, [q, k, v, g, beta, h0], go, gs, cu=cu,
             packed=PackedSequences(torch.tensor(cu, device=DEV)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 8, 64, 64), (5, 4, 33, 7), (3, 16, 128, 128), (2, 2, 256, 256),
                                  (300, 4, 48, 72)], ids=lambda c: f"B{c[0]}H{c[1]}D{c[2]}x{c[3]}")
def test_steps_follow_the_prompt(case, dtype):
    """Tokens one at a time, on a pool with an idle row, against the recurrence."""
    from pararnn_amd import delta_rule_step

    B, H, Dk, Dv = case
    print(f"case delta rule steps {case} {dtype}", flush=True)
    q, k, v, g, beta, h0, _, _ = _inputs(B, 4, (H, 1, H), Dk, Dv, dtype, "token", 5)
    o64, s64 = O.delta_rule(*(t.double() for t in (q, k, v, g, beta, h0)))
    table = torch.randperm(B + 3, generator=torch.Generator().manual_seed(1))[:B].to(torch.int32)
    idle = B > 1
    pool = torch.zeros(B + 3, H, Dk, Dv)
    pool[table.long()] = h0
    before = pool.clone()
    if idle:
        spared, table[-1] = int(table[-1]), -1
    pool, table = pool.to(DEV), table.to(DEV)
    q, k, v, g, beta = (t.to(DEV) for t in (q, k, v, g, beta))
    live = B - 1 if idle else B
    with torch.no_grad():
        for t in range(4):
            o = delta_rule_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], pool,
                                block_table=table)
            assert _rel(o[:live], o64[:live, t]) <= TOL[dtype]
    assert _rel(pool[table[:live].long()], s64[:live]) <= TOL[F32]
    if idle:
        assert torch.equal(pool[spared].cpu(), before[spared])
