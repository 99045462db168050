"""How the gated delta rule is called: layouts, pools and tables, streams, graphs, types of decays and
rates, values at their ends, infinities and NaN, differences.  Equal work on equal values in another
layout, stream or graph is equal bits."""

import pytest
import torch
from test_gpu_delta_rule import (
    BF16,
    DEV,
    F16,
    F32,
    TOL,
    TOL_GRAD,
    TOL_STATE,
    TOL_SUMS,
    _compare,
    _inputs,
    _rel,
)

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _on(ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _train(given, go, gs, **kw):
    """(out, state, gradients) of a call on detached copies of `given` in their own layout."""
    from pararnn_amd import delta_rule

    leaves = [t.detach().requires_grad_(True) for t in given]
    out, state = delta_rule(*leaves[:5], h0=leaves[5] if len(leaves) > 5 else None,
                            return_state=True, **kw)
    return (out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, gs]))


def _same(a, b):
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [1, 70, 700])
def test_layouts(T, dtype):
    """Slices of a projection, heads before tokens, off a 16-byte boundary, every other token, shared
    rows by a stride of zero: as contiguous ones."""
    B, H, Dk, Dv = 2, 2, 64, 32
    print(f"case layouts {T} {dtype}", flush=True)
    given = _on(_inputs(B, T, (H, H, H), Dk, Dv, dtype, "token", seed=T))
    q, k, v, g, beta, h0, go, gs = given
    want = _train([q, k, v, g, beta, h0], go, gs)
    wide = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), g, beta], -1)
    ends = [0, H * Dk, 2 * H * Dk, 2 * H * Dk + H * Dv, 2 * H * Dk + H * Dv + H]
    cut = [wide[..., a:b] for a, b in zip(ends, ends[1:] + [wide.shape[-1]])]
    shapes = [(H, Dk), (H, Dk), (H, Dv), (H,), (H,)]
    first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    every = lambda t: t.repeat_interleave(2, dim=1)[:, ::2]  # noqa: E731
    layouts = dict(
        projection=[c.unflatten(-1, s) for c, s in zip(cut, shapes)],
        heads=[first(t) for t in (q, k, v, g, beta)], odd=[odd(t) for t in (q, k, v, g, beta)],
        every=[every(t) for t in (q, k, v, g, beta)])
    for name, (a, b, c, d, e) in layouts.items():
        print(f"  {name}", flush=True)
        _same(_train([a, b, c, d, e, h0], go, gs), want)
        _same(_train([a, b, c, d, e, odd(h0)], every(go), odd(gs)), want)
    ones = torch.ones(1, dtype=dtype, device=DEV)
    _same(_train([q, k, v, g, ones.expand(B, T, H), h0], ones.expand(go.shape), gs),
          _train([q, k, v, g, ones.expand(B, T, H).contiguous(), h0],
                 ones.expand(go.shape).contiguous(), gs))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("cu", [None, [0, 0, 1, 257, 400, 1000]], ids=["batch", "packed"])
def test_float32_decays_and_rates_of_16_bit_data(cu, dtype):
    """Their gradients are float32, sums of the same products as in 16 bits."""
    B, T = (2, 300) if cu is None else (1, cu[-1])
    print(f"case float32 decays {cu} {dtype}", flush=True)
    S = None if cu is None else len(cu) - 1
    q, k, v, g, beta, h0, go, gs = _inputs(B, T, (4, 2, 1), 64, 64, dtype, "token", 5, seqs=S,
                                           g_dtype=F32)
    beta = torch.rand(beta.shape, generator=torch.Generator().manual_seed(2))
    packed = None if cu is None else torch.tensor(cu, device=DEV)
    _compare(dtype, [q, k, v, g, beta, h0], go, gs, cu=cu, packed=packed)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [100, 900])
def test_rates_and_decays_at_their_ends(T, dtype):
    """Rates of 0 (nothing written), 1 (the key's value replaced) and 2 (reflected), decays of 0, far
    down and -inf (the state forgotten): outputs and every gradient.  A decay of -inf has the gradient
    zero, as its factor.  At a rate of 2 a token writes twice its error: twice the tolerances."""
    from pararnn_amd import delta_rule

    print(f"case ends {T} {dtype}", flush=True)
    q, k, v, g, beta, h0, go, gs = _inputs(1, T, (2, 2, 2), 64, 48, dtype, "token", seed=9)
    r = torch.Generator().manual_seed(T)
    beta = torch.randint(0, 3, beta.shape, generator=r).to(dtype)
    pick = torch.randint(0, 40, g.shape, generator=r)
    g = torch.where(pick == 0, -INF, torch.where(pick == 1, -60.0, torch.where(pick < 8, 0.0, g.float())))
    g = g.to(dtype)
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g, beta, h0)]
    o64, s64 = O.delta_rule(*exact)
    want = torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])
    got = _train(_on([q, k, v, g, beta, h0]), go.to(DEV), gs.to(DEV))
    errs = [_rel(x, y) for x, y in zip(got, (o64, s64, *want[:3], torch.nan_to_num(want[3]), *want[4:]))]
    print("  ", [f"{e:.1e}" for e in errs], flush=True)
    tols = [TOL[dtype], TOL_STATE, *[TOL_GRAD[dtype]] * 3, *[TOL_SUMS[dtype]] * 2, TOL_STATE]
    for e, tol in zip(errs, tols):
        assert e <= 2 * tol
    assert (got[5][g.to(DEV) == -INF] == 0).all()
    # nothing is written at a rate of zero: the state only decays
    none = torch.zeros_like(beta).to(DEV)
    with torch.no_grad():
        _, state = delta_rule(*_on([q, k, v]), torch.zeros(2, device=DEV), none, h0=h0.to(DEV),
                              return_state=True)
    assert torch.equal(state.cpu(), h0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lens", [(5, 64, 130), (3000, 1, 700)], ids=["short", "cut"])
def test_pools_in_place(lens, dtype):
    """Prompts that begin from and end in a pool's slots, in place, with idle rows and new sessions, are
    the calls on states of their own; other slots are left as they were."""
    from pararnn_amd import PackedSequences, delta_rule

    print(f"case pools {lens} {dtype}", flush=True)
    S, N, H, Dk, Dv = len(lens), sum(lens), 2, 64, 48
    q, k, v, g, beta, h0, _, _ = _on(_inputs(1, N, (H, 1, H), Dk, Dv, dtype, "token", 3, seqs=S))
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()])
    pool = torch.randn(S + 4, H, Dk, Dv, generator=torch.Generator().manual_seed(1)).to(DEV)
    slots = torch.tensor([4, 0, 5], dtype=torch.int32, device=DEV)
    pool[slots.long()] = h0
    call = dict(cu_seqlens=PackedSequences(cu))
    with torch.no_grad():
        want, last = delta_rule(q, k, v, g, beta, h0=h0, return_state=True, **call)
        zeros, fresh = delta_rule(q, k, v, g, beta, return_state=True, **call)
        # in place
        mine = pool.clone()
        assert torch.equal(delta_rule(q, k, v, g, beta, h0=mine, block_table=slots, state_out=mine, **call), want)
        after = pool.clone()
        after[slots.long()] = last
        assert torch.equal(mine, after)
        # only read
        mine = pool.clone()
        assert torch.equal(delta_rule(q, k, v, g, beta, h0=mine, block_table=slots, **call), want)
        assert torch.equal(mine, pool)
        # new sessions: zeros in, states to their slots
        assert torch.equal(delta_rule(q, k, v, g, beta, block_table=slots, state_out=mine, **call), zeros)
        after[slots.long()] = fresh
        assert torch.equal(mine, after)
        # one that is new, one that keeps no state, one that goes on
        mine = pool.clone()
        begin = torch.tensor([-1, 0, 99], dtype=torch.int32, device=DEV)
        end = torch.tensor([6, -1, 2], dtype=torch.int32, device=DEV)
        out = delta_rule(q, k, v, g, beta, h0=mine, block_table=begin, state_out=mine, state_table=end, **call)
        a, b = lens[0], lens[0] + lens[1]
        assert torch.equal(out[:, :a], zeros[:, :a]) and torch.equal(out[:, a:b], want[:, a:b])
        assert torch.equal(out[:, b:], zeros[:, b:])
        after = pool.clone()
        after[6], after[2] = fresh[0], fresh[2]
        assert torch.equal(mine, after)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_prompts_and_steps_follow_each_other(dtype):
    """A prompt cut anywhere, its pieces and single tokens on one pool: the recurrence's outputs."""
    from pararnn_amd import delta_rule, delta_rule_step

    B, T, H, D = 2, 180, 2, 64
    print(f"case prompts and steps {dtype}", flush=True)
    q, k, v, g, beta, h0, _, _ = _inputs(B, T, (1, 1, H), D, D, dtype, "token", 11)
    o64, s64 = O.delta_rule(*(t.double() for t in (q, k, v, g, beta, h0)))
    given, pool = _on([q, k, v, g, beta]), h0.to(DEV)
    out = torch.empty(B, T, H, D, dtype=dtype, device=DEV)
    with torch.no_grad():
        a = 0
        for n in (100, 1, 1, 13, 64, 1):
            part = [t[:, a:a + n] for t in given]
            if n == 1:
                out[:, a:a + 1] = delta_rule_step(*part, pool)
            else:
                out[:, a:a + n] = delta_rule(*part, h0=pool, state_out=pool)
            a += n
    assert a == T
    assert _rel(out, o64) <= TOL[dtype] and _rel(pool, s64) <= TOL_STATE


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(0, 5), (3, 0), (0, 0)], ids=str)
def test_nothing_to_do(shape, dtype):
    from pararnn_amd import delta_rule, delta_rule_step

    B, T = shape
    given = _on(_inputs(B, T, (2, 2, 2), 16, 8, dtype, "token", 0))
    q, k, v, g, beta, h0, go, gs = given
    for decay in (g, torch.zeros(2, dtype=dtype, device=DEV)):
        out, state, *grads = _train([q, k, v, decay, beta, h0], go, gs)
        assert out.shape == (B, T, 2, 8) and torch.equal(state, h0) and torch.equal(grads[5], gs)
        for got, t in zip(grads, (q, k, v, decay, beta)):
            assert torch.equal(got, torch.zeros_like(t))
    if T == 0:
        packed = torch.zeros(4, dtype=torch.long)
        q, k, v, g, beta, h0, go, gs = _on(_inputs(1, 0, (2, 2, 2), 16, 8, dtype, "token", 0, seqs=3))
        out, state, *grads = _train([q, k, v, g, beta, h0], go, gs, cu_seqlens=packed)
        assert torch.equal(state, h0) and torch.equal(grads[5], gs)
    if B == 0:
        with torch.no_grad():
            x, r = torch.empty(0, 2, 16, device=DEV), torch.empty(0, 2, device=DEV)
            assert delta_rule_step(x, x, x, r, r, torch.empty(0, 2, 16, 16, device=DEV)).shape == (0, 2, 16)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_equal_calls_give_equal_bits(dtype):
    from pararnn_amd import PackedSequences

    print(f"case equal bits {dtype}", flush=True)
    cu = [0, 700, 701, 1500]
    q, k, v, g, beta, h0, go, gs = _on(_inputs(1, 1500, (4, 2, 1), 64, 64, dtype, "token", 1, seqs=3))
    packed = PackedSequences(torch.tensor(cu))
    first = _train([q, k, v, g, beta, h0], go, gs, cu_seqlens=packed)
    for _ in range(3):
        torch.empty(1 << 26, dtype=torch.uint8, device=DEV).fill_(255)  # (other values in what is reused)
        _same(_train([q, k, v, g, beta, h0], go, gs, cu_seqlens=packed), first)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_on_another_stream(dtype):
    from pararnn_amd import delta_rule_step

    given = _on(_inputs(1, 900, (2, 2, 2), 64, 64, dtype, "token", 1))
    q, k, v, g, beta, h0, go, gs = given
    want = _train([q, k, v, g, beta, h0], go, gs)
    pool = h0.clone()
    with torch.no_grad():
        step = delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], pool)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        later = [t * 1 for t in given]  # made on the stream
        got = _train(later[:6], later[6], later[7])
        mine = later[5].clone()
        with torch.no_grad():
            one = delta_rule_step(*(t[:, 0] for t in later[:5]), mine)
    side.synchronize()
    _same(got, want)
    assert torch.equal(one, step) and torch.equal(mine, pool)


def _capture(run):
    """A graph of `run` after a warm-up on the capture's stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = run()
    return graph, result


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_captured_training(dtype):
    """Forward and backward pass in one graph, replayed on other values between eager calls."""
    from pararnn_amd import PackedSequences

    print(f"case captured training {dtype}", flush=True)
    cu = PackedSequences(torch.tensor([0, 600, 600, 900]))
    cu.offsets(torch.device(DEV))
    shape = (1, 900, (2, 1, 2), 64, 48, dtype, "token")
    fixed = _on(_inputs(*shape, 0, seqs=3))
    for t in fixed[:6]:
        t.requires_grad_(True)

    def run():
        from pararnn_amd import delta_rule

        out, state = delta_rule(*fixed[:5], h0=fixed[5], cu_seqlens=cu, return_state=True)
        return out, state, *torch.autograd.grad([out, state], fixed[:6], [fixed[6], fixed[7]])

    graph, result = _capture(run)
    for seed in (1, 2, 3):
        fresh = _on(_inputs(*shape, seed, seqs=3))
        with torch.no_grad():
            for t, x in zip(fixed, fresh):
                t.copy_(x)
        graph.replay()
        got = [t.detach().clone() for t in result]
        want = _train(fresh[:6], fresh[6], fresh[7], cu_seqlens=cu)
        torch.cuda.synchronize()
        _same(got, want)


def test_captured_serving():
    """A prompt and steps on one pool in a graph; two graphs of one pool in turn."""
    from pararnn_amd import delta_rule, delta_rule_step

    B, T, H, D = 3, 200, 2, 64
    fixed = _on(_inputs(B, T, (H, H, H), D, D, BF16, "token", 0)[:5])
    pool = torch.zeros(8, H, D, D, device=DEV)
    slots = torch.tensor([6, 1, 3], dtype=torch.int32, device=DEV)
    out = torch.empty(B, H, D, dtype=BF16, device=DEV)

    def prompt():
        with torch.no_grad():
            return delta_rule(*fixed, h0=pool, block_table=slots, state_out=pool)

    def step():
        with torch.no_grad():
            return delta_rule_step(*(t[:, 0] for t in fixed), pool, block_table=slots, out=out)

    (g1, r1), (g2, r2) = _capture(prompt), _capture(step)
    mine = torch.zeros_like(pool)
    pool.zero_()
    for seed in (1, 2, 3):
        fresh = _on(_inputs(B, T, (H, H, H), D, D, BF16, "token", seed)[:5])
        for t, x in zip(fixed, fresh):
            t.copy_(x)
        g1.replay()
        g2.replay()
        with torch.no_grad():
            want = delta_rule(*fresh, h0=mine, block_table=slots, state_out=mine)
            one = delta_rule_step(*(t[:, 0] for t in fresh), mine, block_table=slots)
        torch.cuda.synchronize()
        assert torch.equal(r1, want) and torch.equal(r2, one) and torch.equal(pool, mine)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_tokens_that_are_not_finite(bad, dtype):
    """One in a token's q, k, v, g or beta reaches no earlier token, no other head and no other
    sequence; one in q only its own output, one in v its own column."""
    from pararnn_amd import PackedSequences, delta_rule

    cu, H, D, at = [0, 50, 950], 2, 32, 500
    print(f"case not finite {bad} {dtype}", flush=True)
    q, k, v, g, beta, _, _, _ = _on(_inputs(1, cu[-1], (H, H, H), D, D, dtype, "token", 4))
    packed = PackedSequences(torch.tensor(cu))
    call = lambda *x: delta_rule(*x, cu_seqlens=packed, return_state=True)  # noqa: E731
    with torch.no_grad():
        want, last = call(q, k, v, g, beta)
        for i, name in enumerate(("q", "k", "v", "g", "beta")):
            given = [q, k, v, g, beta]
            given[i] = given[i].clone()
            if i < 3:
                given[i][0, at, 1, 3] = bad
            else:
                given[i][0, at, 1] = NAN if name == "g" else bad
            out, state = call(*given)
            assert torch.equal(out[:, :, 0], want[:, :, 0]) and torch.equal(state[:, 0], last[:, 0]), name
            assert torch.equal(out[:, :at], want[:, :at]) and torch.equal(state[0], last[0]), name
            if name == "q":
                assert torch.equal(out[:, at + 1:], want[:, at + 1:]) and torch.equal(state, last)
                assert not torch.isfinite(out[0, at, 1]).any()
            elif name == "v":
                others = [c for c in range(D) if c != 3]
                assert torch.equal(out[..., others], want[..., others])
                assert torch.equal(state[..., others], last[..., others])
                assert not torch.isfinite(out[0, at:, 1, 3]).any()
                assert not torch.isfinite(state[1, 1, :, 3]).all()
            else:
                assert not torch.isfinite(out[0, at:, 1]).any(), name
                assert not torch.isfinite(state[1, 1]).any(), name


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_a_steps_rows_keep_to_themselves(bad):
    from pararnn_amd import delta_rule_step

    q, k, v, g, beta, h0, _, _ = _on(_inputs(5, 1, (2, 1, 2), 64, 48, BF16, "token", 4))
    q, k, v, g, beta = (x[:, 0] for x in (q, k, v, g, beta))
    table = torch.tensor([3, 0, -1, 4, 1], dtype=torch.int32, device=DEV)
    others = [0, 2, 3, 4]
    with torch.no_grad():
        clean = h0.clone()
        want = delta_rule_step(q, k, v, g, beta, clean, block_table=table)
        for name in ("q", "k", "v", "g", "beta", "state", "idle"):
            given, pool = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone(), beta=beta.clone()), h0.clone()
            if name == "state":
                pool[0, 0, 3, 5] = bad  # row 1's
            elif name == "idle":
                pool[2] = bad  # nobody's
            else:
                given[name][1] = bad if name != "g" else NAN
            out = delta_rule_step(*given.values(), pool, block_table=table)
            assert torch.equal(out[others], want[others]), name
            keep = [s for s in range(1, 5) if not (name == "idle" and s == 2)]
            assert torch.equal(pool[keep], clean[keep]), name
            if name == "idle":
                assert torch.equal(out, want) and not torch.isfinite(pool[2]).any()
            elif name == "q":
                assert not torch.isfinite(out[1]).all() and torch.equal(pool, clean)
            else:
                assert not torch.isfinite(out[1]).all() and not torch.isfinite(pool[0]).all()
        # a decay of -inf forgets any finite state
        g = g.clone()
        g[1] = -INF
        pool, zero = h0.clone(), h0.clone()
        zero[0] = 0
        out = delta_rule_step(q, k, v, g, beta, pool, block_table=table)
        assert torch.equal(out, delta_rule_step(q, k, v, g, beta, zero, block_table=table))
        assert torch.equal(pool, zero)


@pytest.mark.parametrize("which", range(6), ids=["q", "k", "v", "g", "beta", "h0"])
def test_gradients_against_differences(which):
    """Along the gradient's own direction, five points: the loss moves by |gradient|.  In float32 the
    loss is off by 2.7e-6 |out| |go| at most (as the outputs), 1.5 of that in the quotient's two
    differences, over the step; what the points leave out is of the fourth power of the step over the
    tokens' own sizes (0.05 over sqrt(2 x 150) of a unit), below 1e-6."""
    q, k, v, g, beta, h0, go, gs = _inputs(1, 150, (2, 2, 2), 32, 16, F32, "token", 21)
    g = g - 0.05  # (the steps stay below zero)
    given = _on([q, k, v, g, beta, h0])
    go, gs = go.to(DEV), gs.to(DEV)
    out, state, *grads = _train(given, go, gs)
    size = float(grads[which].double().norm())
    along = grads[which] / size

    def loss(step):
        from pararnn_amd import delta_rule

        moved = list(given)
        moved[which] = moved[which] + step * along
        with torch.no_grad():
            o, s = delta_rule(*moved[:5], h0=moved[5], return_state=True)
        return float((o.double() * go.double()).sum() + (s.double() * gs.double()).sum())

    h = 0.05
    slope = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
    noise = 2.7e-6 * 1.5 / h * (float(out.norm() * go.norm()) + float(state.norm() * gs.norm()))
    print(f"case differences {which}: {slope:.6f} {size:.6f} +- {noise:.1e}", flush=True)
    assert noise < 0.1 * size
    assert abs(slope - size) <= noise + 1e-5 * size


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_some_gradients_only(dtype):
    """Leaves without a gradient, a loss of the states alone, of the outputs alone."""
    from pararnn_amd import delta_rule

    q, k, v, g, beta, h0, go, gs = _on(_inputs(2, 150, (2, 2, 2), 64, 64, dtype, "token", 2))
    all_of = _train([q, k, v, g, beta, h0], go, gs)[2:]
    for i in range(6):
        leaves = [q, k, v, g, beta, h0]
        leaves[i] = leaves[i].detach().requires_grad_(True)
        out, state = delta_rule(*leaves[:5], h0=leaves[5], return_state=True)
        got, = torch.autograd.grad([out, state], [leaves[i]], [go, gs])
        assert torch.equal(got, all_of[i])
    states = _train([q, k, v, g, beta, h0], torch.zeros_like(go), gs)
    outs = _train([q, k, v, g, beta, h0], go, torch.zeros_like(gs))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, g, beta, h0)]
    out, state = delta_rule(*leaves[:5], h0=leaves[5], return_state=True)
    _same(torch.autograd.grad(state, leaves, gs, retain_graph=True), states[2:])
    _same(torch.autograd.grad(out, leaves, go), outs[2:])


def test_offsets_beyond_32_bits():
    """Tokens 8 MiB apart, 600 of them, and the slots of a pool over 4 GiB."""
    from pararnn_amd import PackedSequences, delta_rule, delta_rule_step

    T, H, D = 600, 2, 64
    print("case offsets beyond 32 bits", flush=True)
    given = _on(_inputs(1, T, (H, H, H), D, D, BF16, "token", 2, seqs=2))
    q, k, v, g, beta, h0, go, gs = given
    wide = torch.empty(T, 1 << 22, dtype=BF16, device=DEV)
    n = H * D
    far = []
    for i, t in enumerate((q, k, v, go)):
        wide[:, i * n:(i + 1) * n] = t[0].flatten(1)
        far.append(wide[:, i * n:(i + 1) * n].view(T, H, D)[None])
    for i, t in enumerate((g, beta)):
        at = 4 * n + i * H
        wide[:, at:at + H] = t[0]
        far.append(wide[:, at:at + H][None])
    packed = PackedSequences(torch.tensor([0, 599, 600]))
    want = _train([q, k, v, g, beta, h0], go, gs, cu_seqlens=packed)
    _same(_train([*far[:3], *far[4:], h0], far[3], gs, cu_seqlens=packed), want)
    pool = torch.empty(70000, H, 128, 64, device=DEV)  # 64 KiB a slot: 4.6 GB
    slots = torch.tensor([69999, 3], dtype=torch.int32, device=DEV)
    r = torch.Generator(device=DEV).manual_seed(1)
    x = torch.nn.functional.normalize(torch.randn(1, T, H, 128, generator=r, device=DEV), dim=-1).to(BF16)
    h = torch.randn(2, H, 128, 64, generator=r, device=DEV)
    pool[slots.long()] = h
    with torch.no_grad():
        out, state = delta_rule(x, x, v, g, beta, h0=h, cu_seqlens=packed, return_state=True)
        assert torch.equal(delta_rule(x, x, v, g, beta, h0=pool, block_table=slots, state_out=pool,
                                      cu_seqlens=packed), out)
        assert torch.equal(pool[slots.long()], state)
        tok = [t[0, :2] for t in (x, x, v, g, beta)]
        one = delta_rule_step(*tok, state)
        assert torch.equal(delta_rule_step(*tok, pool, block_table=slots), one)
        assert torch.equal(pool[slots.long()], state)


def _t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda: _t(1, 6, 2)), ValueError),
    (dict(k=lambda: _t(1, 5, 2, 8)), ValueError),
    (dict(k=lambda: _t(1, 6, 2, 9)), ValueError),
    (dict(k=lambda: _t(1, 6, 3, 8)), ValueError),
    (dict(v=lambda: _t(1, 6, 2, 300)), ValueError),
    (dict(v=lambda: _t(1, 6, 2, 8, dtype=BF16)), TypeError),
    (dict(q=lambda: _t(1, 6, 2, 8, dtype=torch.float64)), TypeError),
    (dict(g=lambda: _t(1, 6, 2, dtype=BF16)), TypeError),
    (dict(g=lambda: _t(1, 7, 2)), ValueError),
    (dict(g=lambda: torch.zeros(2)), RuntimeError),
    (dict(beta=lambda: _t(1, 6, 2, dtype=BF16)), TypeError),
    (dict(beta=lambda: _t(1, 7, 2)), ValueError),
    (dict(beta=lambda: _t(2)), ValueError),
    (dict(beta=lambda: torch.zeros(1, 6, 2)), RuntimeError),
    (dict(h0=lambda: _t(2, 2, 8, 8)), ValueError),
    (dict(h0=lambda: _t(1, 2, 8, 8, dtype=BF16)), TypeError),
    (dict(cu_seqlens=lambda: torch.tensor([0, 5])), ValueError),
    (dict(cu_seqlens=lambda: torch.tensor([0, 4, 3, 6])), ValueError),
    (dict(block_table=lambda: torch.tensor([0])), ValueError),
    (dict(state_table=lambda: torch.tensor([0])), ValueError),
    (dict(h0=lambda: _t(4, 2, 8, 8), block_table=lambda: torch.tensor([0, 1])), ValueError),
    (dict(h0=lambda: _t(4, 2, 8, 8), block_table=lambda: torch.tensor([0.0])), TypeError),
    (dict(state_out=lambda: _t(1, 2, 8, 9)), ValueError),
    (dict(state_out=lambda: _t(1, 2, 8, 16)[..., ::2]), ValueError),
    (dict(state_out=lambda: _t(1, 2, 8, 8), return_state=lambda: True), ValueError),
])
def test_refuses(change, error):
    from pararnn_amd import delta_rule

    args = dict(q=_t(1, 6, 2, 8), k=_t(1, 6, 2, 8), v=_t(1, 6, 2, 8), g=_t(1, 6, 2), beta=_t(1, 6, 2))
    args.update({n: f() for n, f in change.items()})
    first = [args.pop(n) for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(error, match="delta_rule|PackedSequences|cu_seqlens"):
        delta_rule(*first, **args)


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda: _t(2, 2, 2, 8)), ValueError),
    (dict(k=lambda: _t(3, 2, 8)), ValueError),
    (dict(v=lambda: _t(2, 3, 8)), ValueError),
    (dict(g=lambda: _t(2, 3)), ValueError),
    (dict(g=lambda: _t(3, 2)), ValueError),
    (dict(beta=lambda: _t(3, 2)), ValueError),
    (dict(beta=lambda: _t(2)), ValueError),
    (dict(beta=lambda: _t(2, 2, dtype=F16)), TypeError),
    (dict(state=lambda: _t(1, 2, 8, 8)), ValueError),
    (dict(state=lambda: _t(2, 2, 8, 8, dtype=BF16)), TypeError),
    (dict(state=lambda: _t(2, 2, 8, 16)[..., ::2]), ValueError),
    (dict(block_table=lambda: torch.tensor([0, 1, 2])), ValueError),
    (dict(out=lambda: _t(2, 2, 9)), ValueError),
    (dict(out=lambda: _t(2, 2, 8, dtype=BF16)), ValueError),
])
def test_step_refuses(change, error):
    from pararnn_amd import delta_rule_step

    args = dict(q=_t(2, 2, 8), k=_t(2, 2, 8), v=_t(2, 2, 8), g=_t(2, 2), beta=_t(2, 2),
                state=_t(2, 2, 8, 8))
    args.update({n: f() for n, f in change.items()})
    first = [args.pop(n) for n in ("q", "k", "v", "g", "beta", "state")]
    with pytest.raises(error, match="delta_rule_step"):
        delta_rule_step(*first, **args)


def test_autograd_is_refused_where_there_is_none():
    from torch.autograd import forward_ad

    from pararnn_amd import delta_rule, delta_rule_step

    q, g, state = _t(2, 6, 2, 32), -_t(2, 6, 2), _t(2, 2, 32, 32)
    b = _t(2, 6, 2)
    first = [q[:, 0], q[:, 0], q[:, 0], g[:, 0], b[:, 0]]
    leaf, rate = q.clone().requires_grad_(True), b.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference"):
        delta_rule(leaf, q, q, g, b, h0=state, block_table=torch.tensor([1, 0]))
    with pytest.raises(RuntimeError, match="inference"):
        delta_rule(q, q, q, g, rate, state_out=state)
    with pytest.raises(RuntimeError, match="autograd"):
        delta_rule_step(*first[:4], rate[:, 0], state)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(b, torch.ones_like(b))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                delta_rule(q, q, q, g, dual)
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                delta_rule_step(*first[:4], dual[:, 0], state)
    out = delta_rule(leaf, q, q, g, rate)
    grad, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grad.sum().backward()
    # states that a graph has saved and a call overwrites
    for call in (lambda: delta_rule(q, q, q, g, b, state_out=state), lambda: delta_rule_step(*first, state)):
        y = delta_rule(leaf, q, q, g, b, h0=state).square().sum()
        with torch.no_grad():
            call()
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    saved = state.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no_grad"):
        delta_rule_step(*first, saved)
    with pytest.raises(RuntimeError, match="inference"):
        delta_rule(q, q, q, g, b, h0=saved, state_out=state)
