"""How beam selection and the pages behind it are called: refusals, streams, graphs, scores at their
ends, large strides and pools."""

import pytest
import torch
from test_gpu_beams import BF16, DEV, F16, F32, INF, _check

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_scores_at_their_ends(dtype):
    """A beam whose score is NaN or -inf proposes nothing, nor does one that has ended with it; the
    type's largest logits and differences over the whole range are sorted like others."""
    r = torch.Generator().manual_seed(3)
    logits = torch.randn(2, 4, 700, generator=r).to(dtype)
    scores = torch.tensor([[NAN, -INF, -1.0, -2.0], [-3.4e38, NAN, NAN, -INF]])
    ended = torch.tensor([[True, True, False, True], [False, True, False, False]])
    _check(logits, scores, 8)
    _check(logits, scores, 8, ended=ended, pad=5)
    top = torch.finfo(dtype).max
    logits[:, :, 100] = top
    logits[:, :, 200:300] = -top
    _check(logits, torch.zeros(2, 4), 8)
    logits[:, 2] = -top
    _check(logits, torch.zeros(2, 4), 8)


def test_zeros_of_either_sign_and_scores_that_swallow_logits():
    """-0.0 and 0.0 are one value: the lowest token; at a score of 1e30 all totals are equal, and a beam's
    larger logits go first, in a slice of its tokens and across them."""
    r = torch.Generator().manual_seed(5)
    zeros = torch.where(torch.rand(1, 3, 20000, generator=r) < 0.5, -0.0, 0.0)
    _check(zeros, torch.zeros(1, 3), 100)
    _check(zeros, torch.tensor([[-0.0, 0.0, -0.0]]), 4, ended=torch.ones(1, 3, dtype=torch.bool))
    logits = torch.randn(1, 3, 20000, generator=r)
    _check(logits, torch.tensor([[-INF, -1e30, -1e30]]), 100)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [8177, 8192, 16384, 16381])
def test_slices_end_where_the_vocabulary_does(V, dtype):
    """Rows off a 16-byte boundary and slices with nothing or little of them; what lies next to a row (an
    infinity here) is not read as its own."""
    r = torch.Generator().manual_seed(V)
    wide = torch.full((2, 3, V + 3), INF).to(dtype)
    for shift in (0, 1, 2, 3):
        logits = wide.clone()[..., shift:shift + V]
        logits.copy_((torch.randn(2, 3, V, generator=r) * 2).to(dtype))
        want = O.beam_select(logits, torch.zeros(2, 3), 5)
        there = wide.to(DEV)[..., shift:shift + V]
        there.copy_(logits)
        from pararnn_amd import beam_select

        _, p, t = beam_select(there, _t(2, 3), beams=5)
        for b in range(2):
            assert list(zip(p[b].tolist(), t[b].tolist())) == [(k, i) for _, k, i in want[b]]


def test_captured_search():
    """Selection and pages in one graph, replayed on other logits: as eager calls."""
    from pararnn_amd import beam_select, reorder_pages

    B, K, V = 3, 4, 9000
    r = torch.Generator().manual_seed(7)
    logits, scores, ended = _t(B, K, V, dtype=BF16), _t(B, K), _t(B, K, dtype=torch.bool)
    pool, table = _t(16, 5, 7), torch.arange(2, 14, dtype=torch.int32, device=DEV).view(B, K)

    def step(logits, scores, pool, table, ended):
        s, p, t = beam_select(logits, scores, ended=ended, pad=1)
        reorder_pages(pool, table, p)
        scores.copy_(s)
        ended.copy_(torch.gather(ended, 1, p.clamp(min=0).long()) | (t == 1))
        return s, p, t

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(logits, scores, pool, table, ended)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step(logits, scores, pool, table, ended)
    table.copy_(torch.arange(2, 14, dtype=torch.int32, device=DEV).view(B, K))
    pool.copy_(torch.randn(16, 5, 7, generator=r))
    scores.copy_(torch.tensor([0.0, -INF, -INF, -INF]).expand(B, K))
    ended.zero_()
    mine = [t.clone() for t in (scores, pool, table, ended)]
    for _ in range(4):
        fresh = (torch.randn(B, K, V, generator=r) * 2).to(BF16).to(DEV)
        logits.copy_(fresh)
        graph.replay()
        got = [t.clone() for t in (*result, scores, pool, table, ended)]
        want = step(fresh, *mine)
        torch.cuda.synchronize()
        for x, y in zip(got, (*want, *mine)):
            assert torch.equal(x, y)


def test_on_another_stream_and_equal_bits():
    from pararnn_amd import beam_select, reorder_pages

    r = torch.Generator().manual_seed(1)
    logits, scores = torch.randn(2, 6, 20000, generator=r).to(DEV), torch.rand(2, 6, generator=r).to(DEV)
    want = beam_select(logits, scores, beams=20)
    for x, y in zip(beam_select(logits, scores, beams=20), want):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = beam_select(logits * 1, scores * 1, beams=20)
        pool = torch.arange(36, device=DEV, dtype=F32).view(12, 3) * 1
        table = torch.arange(12, dtype=torch.int32, device=DEV).view(2, 6)
        reorder_pages(pool, table, torch.zeros_like(table))
        rows = pool[table.long()].clone()
    side.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert (rows[0] == rows[0, 0]).all() and (rows[1] == rows[1, 0]).all() and rows[1, 0, 0] == 18


@pytest.mark.parametrize("dtype", [torch.float64, torch.int8, BF16, torch.complex64], ids=str)
@pytest.mark.parametrize("width", [1, 3, 17, 4096])
def test_reorder_any_rows(width, dtype):
    """Pools of any type and row size, several at once, more than a launch takes; parents of 64 bits."""
    from pararnn_amd import reorder_pages

    r = torch.Generator().manual_seed(width)
    B, K = 4, 6
    pools = [torch.randint(-100, 100, (40, *s), generator=r).to(dtype) for s in ((width,), (2, width), ())]
    pools += [torch.randint(0, 100, (40, 2), generator=r).to(torch.int32) for _ in range(9)]
    table = torch.randperm(40, generator=r)[:B * K].to(torch.int32).view(B, K)
    parents = torch.randint(-1, K + 1, (B, K), generator=r)
    mine = [p.to(DEV) for p in pools]
    names = table.to(DEV)
    assert reorder_pages(mine, names, parents.to(DEV)) is names
    for b in range(B):
        new, copies = O.reorder_pages(table[b].tolist(), parents[b].tolist())
        assert names[b].tolist() == new
        for p in pools:
            before = p.clone()
            for slot, source in copies.items():
                p[slot] = before[source]
    for got, want in zip(mine, pools):
        assert torch.equal(got.cpu(), want)


def test_offsets_beyond_32_bits():
    from pararnn_amd import beam_select, reorder_pages

    print("case beam offsets beyond 32 bits", flush=True)
    far = torch.empty((1 << 31) + 40000, dtype=BF16, device=DEV)
    view = far.as_strided((2, 2, 5000), (1 << 31, 20000, 1))
    near = (torch.randn(2, 2, 5000, generator=torch.Generator().manual_seed(1)) * 2).to(BF16).to(DEV)
    view.copy_(near)
    scores = _t(2, 2)
    for x, y in zip(beam_select(view, scores, beams=7), beam_select(near, scores, beams=7)):
        assert torch.equal(x, y)
    del far, view
    pool = torch.empty(70000, 1 << 14, device=DEV)  # 64 KiB a slot: 4.6 GB
    table = torch.tensor([3, 69999, 69000], dtype=torch.int32, device=DEV)
    pool[table.long()] = torch.arange(3.0, device=DEV)[:, None].expand(3, 1 << 14)
    reorder_pages(pool, table, torch.tensor([1, 1, 0], device=DEV))
    assert table.tolist() == [69999, 69000, 3]
    assert [pool[s].unique().tolist() for s in table.tolist()] == [[1.0], [1.0], [0.0]]


@pytest.mark.parametrize("change,error", [
    (dict(logits=lambda: _t(2, 9)), ValueError),
    (dict(logits=lambda: _t(2, 3, 0)), ValueError),
    (dict(logits=lambda: _t(2, 0, 9), scores=lambda: _t(2, 0)), ValueError),
    (dict(logits=lambda: _t(2, 3, 9, dtype=torch.float64)), TypeError),
    (dict(logits=lambda: torch.zeros(2, 3, 9)), RuntimeError),
    (dict(scores=lambda: _t(2, 4)), ValueError),
    (dict(scores=lambda: _t(2, 3, dtype=BF16)), TypeError),
    (dict(scores=lambda: torch.zeros(2, 3)), RuntimeError),
    (dict(beams=lambda: 0), ValueError),
    (dict(beams=lambda: 129), ValueError),
    (dict(ended=lambda: _t(2, 3)), TypeError),
    (dict(ended=lambda: _t(2, 4, dtype=torch.bool)), ValueError),
    (dict(ended=lambda: torch.zeros(2, 3, dtype=torch.bool)), RuntimeError),
    (dict(ended=lambda: _t(2, 3, dtype=torch.bool), pad=lambda: 9), ValueError),
    (dict(ended=lambda: _t(2, 3, dtype=torch.bool), pad=lambda: -1), ValueError),
    (dict(logits=lambda: _t(1, 1, 1).expand(1, 1 << 16, 1 << 15), scores=lambda: _t(1, 1 << 16),
          beams=lambda: 4), ValueError),
    (dict(logits=lambda: _t(2, 3, 9).requires_grad_(True)), RuntimeError),
    (dict(scores=lambda: _t(2, 3).requires_grad_(True)), RuntimeError),
])
def test_select_refuses(change, error):
    from pararnn_amd import beam_select

    args = dict(logits=_t(2, 3, 9), scores=_t(2, 3))
    args.update({n: f() for n, f in change.items()})
    with pytest.raises(error, match="beam_select"):
        beam_select(args.pop("logits"), args.pop("scores"), **args)


@pytest.mark.parametrize("change,error", [
    (dict(pools=lambda: []), ValueError),
    (dict(pools=lambda: [_t(9, 4), _t(8, 4)]), ValueError),
    (dict(pools=lambda: _t(9, 8)[:, ::2]), ValueError),
    (dict(pools=lambda: torch.zeros(9, 4)), RuntimeError),
    (dict(table=lambda: _t(2, 3)), TypeError),
    (dict(table=lambda: _t(2, 3, dtype=torch.int64)), TypeError),
    (dict(table=lambda: _t(2, 6, dtype=torch.int32)[:, ::2]), ValueError),
    (dict(table=lambda: _t(1, 2, 3, dtype=torch.int32)), ValueError),
    (dict(table=lambda: torch.zeros(2, 3, dtype=torch.int32)), RuntimeError),
    (dict(table=lambda: _t(2, 0, dtype=torch.int32), parents=lambda: _t(2, 0, dtype=torch.int32)), ValueError),
    (dict(table=lambda: _t(1, 1025, dtype=torch.int32), parents=lambda: _t(1, 1025, dtype=torch.int32)),
     ValueError),
    (dict(parents=lambda: _t(2, 4, dtype=torch.int32)), ValueError),
    (dict(parents=lambda: _t(2, 3)), TypeError),
    (dict(parents=lambda: _t(2, 3, dtype=torch.bool)), TypeError),
    (dict(parents=lambda: torch.zeros(2, 3, dtype=torch.int32)), RuntimeError),
    (dict(pools=lambda: _t(9, 4).requires_grad_(True)), RuntimeError),
])
def test_reorder_refuses(change, error):
    from pararnn_amd import reorder_pages

    args = dict(pools=_t(9, 4), table=torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3),
                parents=_t(2, 3, dtype=torch.int32))
    args.update({n: f() for n, f in change.items()})
    with pytest.raises(error):
        reorder_pages(args["pools"], args["table"], args["parents"])


def test_writes_are_seen_by_autograd():
    from pararnn_amd import reorder_pages

    pool = torch.randn(4, 3, device=DEV)
    leaf = torch.randn(4, 3, device=DEV).requires_grad_(True)
    y = (leaf * pool).sum()
    reorder_pages(pool, torch.arange(4, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_no_searches():
    from pararnn_amd import beam_select, reorder_pages

    s, p, t = beam_select(_t(0, 3, 9), _t(0, 3), beams=2)
    assert s.shape == p.shape == t.shape == (0, 2)
    none = _t(0, 3, dtype=torch.int32)
    assert reorder_pages(_t(4, 2), none, none) is none
