"""Linear attention against the recurrence in float64: outputs, final states and gradients over
types, head layouts, odd widths and lengths, packed and cut sequences, strides, resets, non-finite
values, pools, streams and graphs.

Tolerances (relative 2-norm), from the arithmetic.  float32: an element is a sum of up to T + Dk
products, each rounded to 2^-24, whose errors add up like a random walk: at most
sqrt(2000) 2^-24 = 2.7e-6 at these sizes; the decay's gradient runs over the tokens again, 1e-5.
16 bits: one rounding of the result, and in the bfloat16 products one more of the pairs' weights and
one of the state; each is at most 2^-8 (bfloat16) of its value and 0.4 times that in the mean square,
so three independent ones stay below 2^-8 = 3.9e-3; the decay's gradient is a sum of such values:
8e-3.  States are float32 sums of products of the given 16-bit values: the float32 bound."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 2.7e-6, BF16: 3.9e-3, F16: 3.9e-3}
TOL_G = {F32: 1e-5, BF16: 8e-3, F16: 8e-3}


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    n = want.norm()
    return float((got - want).norm() / n) if n > 0 else float((got - want).norm())


def _inputs(B, T, heads, Dk, Dv, dtype, decay, seed, seqs=None, g_dtype=None):
    r = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    H = max(heads)
    q = torch.randn(B, T, hq, Dk, generator=r).to(dtype)
    k = (torch.randn(B, T, hk, Dk, generator=r) / Dk ** 0.5).to(dtype)
    v = torch.randn(B, T, hv, Dv, generator=r).to(dtype)
    if decay == "token":
        g = -torch.nn.functional.softplus(torch.randn(B, T, H, generator=r) - 2)
        g = g.to(g_dtype or dtype)
    else:
        g = -0.2 * torch.rand(H, generator=r)
    h0 = torch.randn(seqs or B, H, Dk, Dv, generator=r)
    go = torch.randn(B, T, H, Dv, generator=r).to(dtype)
    gs = torch.randn(seqs or B, H, Dk, Dv, generator=r)
    return q, k, v, g, h0, go, gs


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
    (1, 520, (1, 1, 1), 256, 200, "token", True),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=[f"B{c[0]}T{c[1]}D{c[3]}x{c[4]}" for c in CASES])
def test_forward_and_gradients(case, dtype):
    from pararnn_amd import linear_attention

    B, T, heads, Dk, Dv, decay, with_h0 = case
    print(f"case linear attention {case} {dtype}", flush=True)
    q, k, v, g, h0, go, gs = _inputs(B, T, heads, Dk, Dv, dtype, decay, seed=T + Dk)
    given = [q, k, v, g] + ([h0] if with_h0 else [])
    exact = [t.double().requires_grad_(True) for t in given]
    o64, s64 = O.linear_attention(*exact)
    want = torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])
    mine = [t.to(DEV).requires_grad_(True) for t in given]
    out, state = linear_attention(*mine[:4], h0=mine[4] if with_h0 else None, return_state=True)
    assert out.dtype == dtype and state.dtype == F32
    got = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    torch.cuda.synchronize()
    errs = dict(out=_rel(out, o64), state=_rel(state, s64))
    for name, x, y in zip(("dq", "dk", "dv", "dg", "dh0"), got, want):
        errs[name] = _rel(x, y)
    print("  ", {n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    for name, e in errs.items():
        tol = TOL[F32] if name in ("state", "dh0") else TOL_G[dtype] if name == "dg" else TOL[dtype]
        assert e <= tol, (name, e)


PACKED = [
    ([0, 0, 1, 257, 257, 400, 600, 600], 33, 130, (2, 2, 2)),
    ([0, 513, 768, 1024, 1300], 64, 48, (2, 1, 1)),
    ([0, 1, 2, 3, 67, 131], 64, 64, (4, 4, 4)),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", PACKED, ids=["empty", "long", "short"])
def test_packed(case, dtype):
    from pararnn_amd import PackedSequences, linear_attention

    cu, Dk, Dv, heads = case
    S, N = len(cu) - 1, cu[-1]
    print(f"case packed linear attention {cu} {Dk}x{Dv} {dtype}", flush=True)
    q, k, v, g, h0, go, gs = _inputs(1, N, heads, Dk, Dv, dtype, "token", 3, seqs=S)
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g, h0)]
    o64, s64 = O.linear_attention(*exact, cu=cu)
    want = torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])
    mine = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, h0)]
    offsets = torch.tensor(cu, device=DEV)
    out, state = linear_attention(*mine[:4], h0=mine[4], cu_seqlens=PackedSequences(offsets),
                                  return_state=True)
    got = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    assert _rel(out, o64) <= TOL[dtype] and _rel(state, s64) <= TOL[F32]
    for name, x, y in zip(("dq", "dk", "dv", "dg", "dh0"), got, want):
        e = _rel(x, y)
        print(f"  {name} {e:.1e}", flush=True)
        assert e <= (TOL[F32] if name == "dh0" else TOL_G[dtype] if name == "dg" else TOL[dtype]), name
    # offsets as a tensor are the same call, and no sequence sees another
    with torch.no_grad():
        again = linear_attention(*mine[:4], h0=mine[4], cu_seqlens=offsets)
        assert torch.equal(again, out)
        poisoned = [t.detach().clone() for t in mine[:4]]
        a, b = cu[-3], cu[-2]
        if b > a:
            for t in poisoned[:3]:
                t[:, a:b] = float("nan")
            other = linear_attention(*poisoned, h0=mine[4], cu_seqlens=offsets)
            keep = torch.ones(N, dtype=torch.bool)
            keep[a:b] = False
            assert torch.equal(other[:, keep.to(DEV)], out[:, keep.to(DEV)])


def test_gradient_against_differences():
    """dL along a random direction by central differences of the float32 kernels' own float64-summed
    loss.  Step 2^-6: the third-order term is about (2^-6)^2 = 2.4e-4 of the slope, the rounding of
    a loss of some 500 terms 500^0.5 2^-24 / 2^-6 = 8.5e-5: together below 1e-3."""
    from pararnn_amd import linear_attention

    q, k, v, g, h0, go, gs = (t.to(DEV) for t in _inputs(2, 70, (2, 1, 2), 24, 40, F32, "token", 5))
    r = torch.Generator().manual_seed(6)
    leaves = [q, k, v, g, h0]
    dirs = [torch.randn(t.shape, generator=r).to(DEV) * (0.1 if t is g else 1.0) for t in leaves]

    def loss(ts):
        o, s = linear_attention(*ts[:4], h0=ts[4], return_state=True)
        return (o.double() * go.double()).sum() + (s.double() * gs.double()).sum()

    grads = torch.autograd.grad(loss([t.requires_grad_(True) for t in leaves]), leaves)
    with torch.no_grad():
        for t, d, x in zip(leaves, dirs, grads):
            e = 2.0 ** -6 / float(d.norm()) * 4
            up, down = [], []
            for s, side in ((1, up), (-1, down)):
                side += [u + s * e * d if u is t else u for u in leaves]
            slope = float((loss(up) - loss(down)) / (2 * e))
            mine = float((x.double() * d.double()).sum())
            scale = float(x.double().norm() * d.double().norm())
            assert abs(slope - mine) <= 1e-3 * scale


def test_strided_views_of_one_projection():
    """Heads as views of one fused projection (aligned or not), an expanded gradient, and a decay
    with its heads first."""
    from pararnn_amd import linear_attention

    for dtype in (F32, BF16):
        for pad in (0, 1):
            B, T, H, D = 2, 80, 3, 40
            r = torch.Generator().manual_seed(8)
            fused = torch.randn(B, T, 3 * H * D + pad, generator=r).to(DEV, dtype)
            at = fused[..., pad:].view(B, T, 3, H, D) if pad == 0 else \
                fused[..., pad:].unflatten(-1, (3, H, D))
            q, k, v = at.unbind(2)
            g = (-torch.rand(H, B, T, generator=r)).to(DEV, dtype).permute(1, 2, 0)
            assert not q.is_contiguous()
            with torch.no_grad():
                a = linear_attention(q, k, v, g)
                b = linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous())
            assert torch.equal(a, b)
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v, g)]
            got = torch.autograd.grad(linear_attention(*leaves).sum(), leaves)
            dense = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v, g)]
            want = torch.autograd.grad(linear_attention(*dense), dense,
                                       torch.ones(B, T, H, D, device=DEV, dtype=dtype))
            for x, y in zip(got, want):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("low", [float("-inf"), "lowest", -1e4])
def test_reset_decay(low, dtype):
    """A decay that forgets everything: what follows is a sequence of its own, exactly."""
    from pararnn_amd import linear_attention

    q, k, v, g, h0, _, _ = _inputs(1, 150, (2, 2, 2), 64, 64, dtype, "token", 11)
    low = torch.finfo(dtype).min if low == "lowest" else low
    for t in (0, 1, 40, 64, 100):
        g2 = g.clone()
        g2[:, t] = low
        a, sa = linear_attention(*(x.to(DEV) for x in (q, k, v, g2)), h0=h0.to(DEV),
                                 return_state=True)
        o64, s64 = O.linear_attention(*(x[:, t:].double() for x in (q, k, v, g)))
        assert _rel(a[:, t:], o64) <= TOL[dtype]
        assert _rel(sa, s64) <= TOL[F32]
        assert torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_tokens_reach_nothing_earlier(bad, dtype):
    from pararnn_amd import linear_attention

    q, k, v, g, _, _, _ = (t.to(DEV) for t in _inputs(1, 140, (1, 1, 1), 64, 48, dtype, "token", 2))
    with torch.no_grad():
        clean = linear_attention(q, k, v, g)
        for t in (3, 17, 63, 64, 100):
            for name, x in (("q", q), ("k", k), ("v", v), ("g", g)):
                y = x.clone()
                y[:, t] = float("nan") if name == "g" else bad
                given = [y if name == n else z for n, z in zip("qkvg", (q, k, v, g))]
                out = linear_attention(*given)
                assert torch.equal(out[:, :t], clean[:, :t]), (name, t)
                if name == "q":
                    assert torch.equal(out[:, t + 1:], clean[:, t + 1:])
                assert not torch.isfinite(out[:, t]).all()


def test_pool_states_and_idle_rows():
    from pararnn_amd import linear_attention

    q, k, v, g, _, _, _ = _inputs(3, 90, (2, 2, 2), 64, 64, BF16, "token", 4)
    r = torch.Generator().manual_seed(1)
    pool = torch.randn(6, 2, 64, 64, generator=r)
    table = torch.tensor([4, -1, 1])
    h0 = torch.stack([pool[4], torch.zeros_like(pool[0]), pool[1]])
    o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g)), h0.double())
    want = pool.double().clone()
    want[4], want[1] = s64[0], s64[2]
    for T in (90, 600):  # whole and cut walks, in place
        if T == 600:
            q, k, v, g = (x.repeat(1, 7, 1, 1)[:, :600] if x.dim() == 4 else
                          x.repeat(1, 7, 1)[:, :600] for x in (q, k, v, g))
            o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g)), h0.double())
            want[4], want[1] = s64[0], s64[2]
        mine = pool.to(DEV)
        out = linear_attention(*(x.to(DEV) for x in (q, k, v, g)), h0=mine, block_table=table,
                               state_out=mine)
        assert _rel(out, o64) <= TOL[BF16]
        assert _rel(mine, want) <= TOL[F32]
        assert torch.equal(mine[[0, 2, 3, 5]].cpu(), pool[[0, 2, 3, 5]])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,heads,Dk,Dv,slots", [
    (1, (1, 1, 1), 1, 1, 0), (3, (4, 2, 1), 64, 64, 0), (5, (2, 1, 2), 33, 37, 9),
    (4, (2, 2, 2), 128, 128, 6), (2, (2, 2, 2), 256, 256, 0), (70, (1, 1, 1), 16, 6, 80)])
def test_step(B, heads, Dk, Dv, slots, dtype):
    from pararnn_amd import linear_attention_step

    q, k, v, g, h0, _, _ = _inputs(B, 1, heads, Dk, Dv, dtype, "token", 7, seqs=slots or B)
    table = torch.randperm(slots, generator=torch.Generator().manual_seed(2))[:B] if slots else None
    if table is not None:
        table[B // 2] = -1
    rows = h0 if table is None else h0[table.clamp(min=0)] * (table >= 0).view(-1, 1, 1, 1)
    o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g)), rows.double())
    want = h0.double().clone()
    if table is None:
        want = s64
    else:
        want[table[table >= 0]] = s64[table >= 0]
    state = h0.to(DEV)
    out = linear_attention_step(*(x[:, 0].to(DEV) for x in (q, k, v, g)), state, block_table=table)
    assert out.dtype == dtype and _rel(out, o64[:, 0]) <= TOL[dtype]
    assert _rel(state, want) <= TOL[F32]
    # with the time axis and a destination: the same bits
    state2, dest = h0.to(DEV), torch.empty(B, 1, max(heads), Dv, device=DEV, dtype=dtype)
    got = linear_attention_step(*(x.to(DEV) for x in (q, k, v, g)), state2, block_table=table,
                                out=dest)
    assert got is dest and torch.equal(dest[:, 0], out) and torch.equal(state2, state)


def test_prompt_then_steps_equals_the_whole():
    """A prompt's final state is what single tokens go on from."""
    from pararnn_amd import linear_attention, linear_attention_step

    q, k, v, g, _, _, _ = (t.to(DEV) for t in _inputs(2, 100, (4, 2, 2), 64, 64, F32, "token", 9))
    with torch.no_grad():
        whole, last = linear_attention(q, k, v, g, return_state=True)
        out, state = linear_attention(q[:, :90], k[:, :90], v[:, :90], g[:, :90], return_state=True)
        outs = [out]
        for t in range(90, 100):
            outs.append(linear_attention_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1],
                                              g[:, t:t + 1], state))
    assert _rel(torch.cat(outs, 1), whole) <= 2 * TOL[F32]
    assert _rel(state, last) <= 2 * TOL[F32]


def test_repeatable_other_stream_and_graph():
    """The same bits at every call, on another stream, and from replays of a captured graph."""
    from pararnn_amd import linear_attention, linear_attention_step

    q, k, v, g, h0, go, _ = (t.to(DEV) for t in _inputs(1, 900, (2, 1, 2), 64, 64, BF16, "token", 9))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, g)]
        out = linear_attention(*leaves, h0=h0)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))

    first = step()
    for x, y in zip(first, step()):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, other):
        assert torch.equal(x, y)
    state, dest = h0.clone(), torch.empty(1, 2, 64, device=DEV, dtype=BF16)

    def tick():
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, out=dest)

    with torch.no_grad():
        with torch.cuda.stream(side):
            tick()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tick()
            whole = linear_attention(q, k, v, g, h0=h0)
        want = h0.clone()
        state.copy_(h0)
        for _ in range(4):
            graph.replay()
            torch.cuda.synchronize()
            ref = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], want)
            assert torch.equal(dest, ref) and torch.equal(state, want)
            assert torch.equal(whole, first[0])


def test_no_tokens_no_rows():
    from pararnn_amd import linear_attention, linear_attention_step

    q, k, v, g, h0, _, gs = _inputs(2, 0, (2, 1, 2), 8, 8, F32, "token", 1)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, h0)]
    out, state = linear_attention(*leaves[:4], h0=leaves[4], return_state=True)
    assert out.shape == (2, 0, 2, 8) and torch.equal(state.detach().cpu(), h0)
    grads = torch.autograd.grad(state, leaves, gs.to(DEV))
    assert torch.equal(grads[4].cpu(), gs)
    empty = torch.empty(0, 2, 8, device=DEV)
    state = torch.empty(0, 2, 8, 8, device=DEV)
    assert linear_attention_step(empty, empty, empty, empty[..., 0], state).shape == (0, 2, 8)
    out = linear_attention(empty[:, None], empty[:, None], empty[:, None], empty[:, None, :, 0])
    assert out.shape == (0, 1, 2, 8)


def test_offsets_beyond_32_bits():
    """A pool and arrays of more than 2^32 bytes: the last slots and tokens are right."""
    from pararnn_amd import linear_attention, linear_attention_step

    slots, H, D = 17000, 4, 128  # 256 KiB a slot, 4.15 GiB
    pool = torch.empty(slots, H, D, D, device=DEV)
    table = torch.tensor([slots - 1, 3, 16385], dtype=torch.int32, device=DEV)
    q, k, v, g, h0, _, _ = _inputs(3, 1, (H, H, H), D, D, BF16, "token", 5)
    pool[table.long()] = h0.to(DEV)
    out = linear_attention_step(*(x[:, 0].to(DEV) for x in (q, k, v, g)), pool, block_table=table)
    o64, s64 = O.linear_attention(*(x.double() for x in (q, k, v, g)), h0.double())
    assert _rel(out, o64[:, 0]) <= TOL[BF16] and _rel(pool[table.long()], s64) <= TOL[F32]
    del pool
    T, H = (1 << 20) + 70, 33  # 2^31 and more elements of q and out
    gen = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(1, T, H, 64, device=DEV, dtype=BF16, generator=gen)
    k, v = (torch.randn(1, T, 1, 64, device=DEV, dtype=BF16, generator=gen) for _ in range(2))
    g = torch.full((1, T, H), -0.1, device=DEV, dtype=BF16)
    g[:, T - 100] = float("-inf")  # what follows stands on its own
    with torch.no_grad():
        out = linear_attention(q, k, v, g)
        tail = [x[:, T - 100:].cpu().double() for x in (q, k, v, g)]
    o64, _ = O.linear_attention(*tail)
    assert _rel(out[:, T - 100:], o64) <= TOL[BF16]


def test_shared_decay_and_lone_strides():
    """A decay expanded over batch and time has the gradient of an expanded tensor; one token whose
    strides are odd; keys expanded over time."""
    from pararnn_amd import linear_attention

    for dtype in (F32, BF16):
        q, k, v, _, _, go, _ = (t.to(DEV) for t in _inputs(2, 70, (2, 2, 2), 64, 64, dtype, "token", 3))
        head = torch.tensor([-0.1, -0.02], device=DEV, dtype=dtype).requires_grad_(True)
        got = torch.autograd.grad(linear_attention(q, k, v, head.expand(2, 70, 2)), head, go)[0]
        leaf = head.detach().double().cpu().requires_grad_(True)
        o64, _ = O.linear_attention(*(x.double().cpu() for x in (q, k, v)), leaf)
        want = torch.autograd.grad(o64, leaf, go.double().cpu())[0]
        # summed over the batch in its own type by autograd: one rounding more in 16 bits
        assert _rel(got, want) <= (TOL_G[dtype] if dtype == F32 else 2 * TOL_G[dtype])
        with torch.no_grad():
            one = torch.randn(2, 3, 2, 64, device=DEV).to(dtype)[:, 1:2]
            a = linear_attention(one, one, one, head)
            b = linear_attention(*(one.contiguous(),) * 3, head)
            assert torch.equal(a, b)
            wide = k[:, :1].expand(2, 70, 2, 64)
            assert torch.equal(linear_attention(q, wide, v, head),
                               linear_attention(q, wide.contiguous(), v, head))



@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cu", [None, [0, 2900, 2901, 2901, 4303, 6000]], ids=["batch", "packed"])
def test_pieces_of_several_parts(cu, dtype):
    """So many narrow heads that pieces are as long as the chip's workgroups ask for, three times
    what the states' contributions are formed for."""
    from pararnn_amd import linear_attention

    B, T, S = (1, cu[-1], len(cu) - 1) if cu else (3, 2000, 3)
    print(f"case pieces of several parts {cu} {dtype}", flush=True)
    q, k, v, g, h0, go, gs = _inputs(B, T, (16, 8, 16), 16, 16, dtype, "token", 11, seqs=S)
    exact = [t.double().requires_grad_(True) for t in (q, k, v, g, h0)]
    o64, s64 = O.linear_attention(*exact, cu=cu)
    want = torch.autograd.grad([o64, s64], exact, [go.double(), gs.double()])
    mine = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, h0)]
    out, state = linear_attention(*mine[:4], h0=mine[4], return_state=True,
                                  cu_seqlens=torch.tensor(cu) if cu else None)
    got = torch.autograd.grad([out, state], mine, [go.to(DEV), gs.to(DEV)])
    assert _rel(out, o64) <= TOL[dtype] and _rel(state, s64) <= TOL[F32]
    for name, x, y in zip(("dq", "dk", "dv", "dg", "dh0"), got, want):
        e = _rel(x, y)
        print(f"  {name} {e:.1e}", flush=True)
        assert e <= (TOL[F32] if name == "dh0" else TOL_G[dtype] if name == "dg" else TOL[dtype]), name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_one_long_sequence_among_short_ones(dtype):
    """Cut for the long one's sake; told or not, the longest length changes no more than the order of
    sums: twice the tolerance between two results that are each within it."""
    from pararnn_amd import PackedSequences, linear_attention

    cu = torch.tensor([0] + [20] * 10 + [1500] + [3] * 7).cumsum(0)
    S, N = cu.numel() - 1, int(cu[-1])
    q, k, v, g, h0, go, gs = _inputs(1, N, (2, 2, 2), 32, 64, dtype, "token", 13, seqs=S)
    o64, s64 = O.linear_attention(*(t.double() for t in (q, k, v, g, h0)), cu=cu.tolist())
    mine = [t.to(DEV) for t in (q, k, v, g)]
    with torch.no_grad():
        packed = PackedSequences(cu)
        assert packed.longest == 1500
        out, state = linear_attention(*mine, h0=h0.to(DEV), cu_seqlens=packed, return_state=True)
        packed.longest = 0  # not known
        other, last = linear_attention(*mine, h0=h0.to(DEV), cu_seqlens=packed, return_state=True)
    assert _rel(out, o64) <= TOL[dtype] and _rel(state, s64) <= TOL[F32]
    assert _rel(other, out) <= 2 * TOL[dtype] and _rel(last, state) <= 2 * TOL[F32]
