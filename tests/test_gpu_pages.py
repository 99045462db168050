"""The state cache's slots against lists on the host: exact, whatever the sizes and orders."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _used(slots, share, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(slots, generator=g) < share).to(torch.int32)


def _pools(slots, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(slots, 3, 5, generator=g), torch.randn(slots, 2, 64, 40, generator=g),
            torch.randint(0, 255, (slots, 7), generator=g, dtype=torch.uint8),
            torch.randn(slots, 9000, generator=g).to(torch.bfloat16)]


@pytest.mark.parametrize("slots,share,n", [
    (1, 0.0, 1), (1, 1.0, 1), (7, 0.5, 0), (64, 0.5, 10), (64, 0.5, 64), (1000, 0.9, 50),
    (5000, 0.99, 80), (9001, 0.0, 9001), (300, 1.0, 3)])
def test_take(slots, share, n):
    from pararnn_amd import take_pages

    used = _used(slots, share, slots + n)
    mine, ref = used.to(DEV), used.tolist()
    want = O.take_pages(ref, n)
    assert take_pages(mine, n).tolist() == want and mine.tolist() == ref


@pytest.mark.parametrize("slots,share,n", [(4, 0.25, 2), (40, 0.5, 30), (600, 0.3, 100),
                                           (1500, 0.2, 1200)])
def test_fork(slots, share, n):
    from pararnn_amd import fork_pages

    print(f"case fork {slots} {share} {n}", flush=True)
    used, pools = _used(slots, share, 3), _pools(slots, 4)
    used[0] = 1
    g = torch.Generator().manual_seed(9)
    live = torch.nonzero(used)[:, 0]
    parents = live[torch.randint(0, live.numel(), (n,), generator=g)]
    parents[n // 2] = -1
    if n > 20:
        parents[7] = slots + 3
    ref, kids = used.tolist(), []
    have = [p for p in parents.tolist() if 0 <= p < slots]
    got = iter(O.take_pages(ref, len(have)))
    kids = [next(got) if 0 <= p < slots else -1 for p in parents.tolist()]
    mine, data = used.to(DEV), [p.to(DEV) for p in pools]
    assert fork_pages(mine, data, parents).tolist() == kids and mine.tolist() == ref
    for p, d in zip(pools, data):
        want = p.clone()
        for k, a in zip(kids, parents.tolist()):
            if k >= 0:
                want[k] = p[a]
        assert torch.equal(d.cpu(), want)


def test_free_and_copy():
    from pararnn_amd import copy_pages, free_pages

    used, pools = torch.ones(50, dtype=torch.int32), _pools(50, 6)
    mine = used.to(DEV)
    gone = torch.tensor([3, 3, -1, 49, 50, 1 << 40, -(1 << 40), 0])
    free_pages(mine, gone)
    used[[3, 49, 0]] = 0
    assert torch.equal(mine.cpu(), used)
    free_pages(mine, torch.empty(0, dtype=torch.int32, device=DEV))
    src, dst = torch.tensor([1, 2, 1, -1, 5, 70]), torch.tensor([10, 11, 12, 13, -1, 3])
    data = [p.to(DEV) for p in pools]
    copy_pages(data, src, dst)
    for p, d in zip(pools, data):
        want = p.clone()
        want[[10, 11, 12]] = p[[1, 2, 1]]
        assert torch.equal(d.cpu(), want)
    one = pools[0].to(DEV)
    copy_pages(one, torch.tensor([4], device=DEV), torch.tensor([8], device=DEV))
    assert torch.equal(one[8].cpu(), pools[0][4])


@pytest.mark.parametrize("slots,share", [(1, 0.0), (1, 1.0), (2, 0.5), (65, 0.5), (700, 0.1),
                                         (700, 0.9), (3000, 0.5), (64, 0.0), (64, 1.0)])
def test_compact(slots, share):
    from pararnn_amd import compact_pages

    print(f"case compact {slots} {share}", flush=True)
    used, pools = _used(slots, share, slots), _pools(slots, 5)
    g = torch.Generator().manual_seed(1)
    tables = [torch.randint(-2, slots + 2, (n,), generator=g, dtype=torch.int32)
              for n in (1, 300, 0)] + [torch.arange(slots, dtype=torch.int32).view(1, -1)]
    ref, lists = used.tolist(), [t.flatten().tolist() for t in tables]
    moves, live = O.compact_pages(ref, lists)
    mine, data, mt = used.to(DEV), [p.to(DEV) for p in pools], [t.to(DEV) for t in tables]
    count = compact_pages(mine, data, mt)
    assert int(count) == live and mine.tolist() == ref
    for t, want in zip(mt, lists):
        assert t.flatten().tolist() == want
    for p, d in zip(pools, data):
        want = p.clone()
        for a, b in moves:
            want[b] = p[a]
        assert torch.equal(d.cpu(), want)
    # again: nothing moves
    compact_pages(mine, data, mt)
    assert mine.tolist() == ref


def test_many_pools_and_tables():
    """More pools and tables than one launch takes."""
    from pararnn_amd import compact_pages, fork_pages

    used = _used(40, 0.4, 2)
    pools = [torch.randn(40, 5, generator=torch.Generator().manual_seed(i)) for i in range(37)]
    tables = [torch.arange(40, dtype=torch.int32) for _ in range(20)]
    ref, lists = used.tolist(), [t.tolist() for t in tables]
    first = ref.index(1)
    kids = O.take_pages(ref, 3)
    for p in pools:
        p_ref = p
        p_ref[kids] = p[first].clone()
    data = [torch.randn(40, 5, generator=torch.Generator().manual_seed(i)).to(DEV)
            for i in range(37)]
    mine = used.to(DEV)
    assert fork_pages(mine, data, torch.full((3,), first)).tolist() == kids
    moves, live = O.compact_pages(ref, lists)
    mt = [t.to(DEV) for t in tables]
    assert int(compact_pages(mine, data, mt)) == live
    for t, want in zip(mt, lists):
        assert t.tolist() == want
    for p, d in zip(pools, data):
        want = p.clone()
        for a, b in moves:
            want[b] = p[a]
        assert torch.equal(d.cpu(), want)


def test_a_serving_step_in_a_graph():
    """Fork, free, take and compact captured once and replayed, against lists on the host."""
    from pararnn_amd import compact_pages, fork_pages, free_pages, take_pages

    slots = 30
    used = _used(slots, 0.4, 8).to(DEV)
    pool = torch.randn(slots, 2, 8, generator=torch.Generator().manual_seed(1)).to(DEV)
    table = torch.nonzero(used)[:, 0].to(torch.int32)
    begin = [t.clone() for t in (used, pool, table)]

    def step():
        kids = fork_pages(used, [pool], table)
        free_pages(used, table)
        table.copy_(kids)
        count = compact_pages(used, [pool], [table])
        new = take_pages(used, 1)
        free_pages(used, new)
        return count, new

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count, new = step()
    for t, b in zip((used, pool, table), begin):
        t.copy_(b)
    want_pool, n = begin[1][begin[2].long()], begin[2].numel()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert int(count) == n and new.tolist() == [n]
        assert used.tolist() == [1] * n + [0] * (slots - n)
        assert sorted(table.tolist()) == list(range(n))
        assert torch.equal(pool[table.long()], want_pool)
        torch.cuda.synchronize()


def test_slots_beyond_32_bits():
    """Pools of more than 2^32 bytes: slots at the far end move and are copied like others."""
    from pararnn_amd import compact_pages, copy_pages, fork_pages

    slots, n = 4200, 1 << 18  # 1 MiB a slot, 4.1 GiB
    pool = torch.empty(slots, n, device=DEV)
    used = torch.zeros(slots, dtype=torch.int32, device=DEV)
    live = torch.tensor([1, 4097, 4199], device=DEV)
    used[live] = 1
    pool[live] = torch.arange(3.0, device=DEV)[:, None] + torch.rand(n, device=DEV)
    want = pool[live].clone()
    copy_pages(pool, live[2:], torch.tensor([4198]))
    assert torch.equal(pool[4198], want[2])
    table = live.to(torch.int32)
    assert fork_pages(used, pool, table[2:]).tolist() == [0]
    assert torch.equal(pool[0], want[2])
    assert int(compact_pages(used, pool, [table])) == 4
    assert table.tolist() == [1, 2, 3] and torch.equal(pool[1:4], want)
