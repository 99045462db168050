"""Calls of the page operators that a program may well make and that once went wrong."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("slots,n", [(4, 2), (40, 30), (3000, 2500)])
def test_free_slots_have_no_children(slots, n):
    """A parent that is free would be handed out as a child itself, and read while it is written."""
    from pararnn_amd import fork_pages

    print(f"case fork of free slots {slots} {n}", flush=True)
    r = torch.Generator().manual_seed(slots)
    used = (torch.rand(slots, generator=r) < 0.4).to(torch.int32)
    used[0] = 1
    parents = torch.randint(-1, slots + 1, (n,), generator=r)
    parents[0], parents[1] = int((used == 0).nonzero()[0]), 0
    pool = torch.randn(slots, 3, 50, generator=r)
    ref = used.tolist()
    live = [p for p in parents.tolist() if 0 <= p < slots and used[p]]
    got = iter(O.take_pages(ref, len(live)))
    kids = [next(got) if 0 <= p < slots and used[p] else -1 for p in parents.tolist()]
    mine, data = used.to(DEV), pool.to(DEV)
    assert fork_pages(mine, data, parents).tolist() == kids and mine.tolist() == ref
    want = pool.clone()
    for k, p in zip(kids, parents.tolist()):
        if k >= 0:
            want[k] = pool[p]
    assert torch.equal(data.cpu(), want)


def test_one_table_of_several_layers():
    """The same table for every layer is renamed once; tables that share a part are refused."""
    from pararnn_amd import compact_pages

    used = torch.tensor([0, 1, 0, 1, 1, 0], dtype=torch.int32, device=DEV)
    pool = torch.arange(6.0, device=DEV)[:, None].repeat(1, 8)
    table = torch.tensor([4, 1, 3], dtype=torch.int32, device=DEV)
    assert int(compact_pages(used, pool, [table, table, table.view(3, 1)])) == 3
    assert sorted(table.tolist()) == [0, 1, 2]
    assert pool[table.long(), 0].tolist() == [4.0, 1.0, 3.0]
    both = torch.tensor([0, 1, 2, 2], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        compact_pages(used, pool, [both[:3], both[2:]])
    compact_pages(used, pool, [both[:2], both[2:], both[:0]])
    assert both.tolist() == [0, 1, 2, 2]
