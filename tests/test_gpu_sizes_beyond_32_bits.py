"""Counts that 32 bits cannot hold are refused, not cut to what is left of them (2^32 + 5 tokens would be
5).  Most tensors here are expanded or never written: no call reaches a kernel."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
MANY = (1 << 32) + 5


def _wide(*shape, dtype=torch.bfloat16):
    return torch.zeros((1,) * len(shape), dtype=dtype, device=DEV).expand(shape)


def test_tokens_and_rows():
    from pararnn_amd import linear_attention, linear_attention_step

    g = torch.zeros(1, device=DEV)
    q = _wide(1, MANY, 1, 1)
    with torch.no_grad():
        with pytest.raises(ValueError, match="2\\^30"):
            linear_attention(q, q, q, g)
        one = _wide(1, 1, 1, 1)
        pool = torch.empty(MANY, 1, 1, 1, device=DEV)
        with pytest.raises(ValueError, match="rows"):
            linear_attention(one, one, one, g, h0=pool, block_table=torch.tensor([7]))
        with pytest.raises(ValueError, match="rows"):
            linear_attention(one, one, one, g, block_table=torch.tensor([7]), state_out=pool)
        with pytest.raises(ValueError, match="rows"):
            linear_attention_step(one[0], one[0], one[0], g, pool, block_table=torch.tensor([7]))
        many = _wide(1 << 16, 1, 1)
        with pytest.raises(ValueError, match="65535"):
            linear_attention_step(many, many, many, g, pool[:1 << 16])


def test_slots_and_lists():
    from pararnn_amd import compact_pages, copy_pages, fork_pages, free_pages, take_pages

    used = torch.empty(MANY, dtype=torch.int32, device=DEV)
    few, one = torch.zeros(5, dtype=torch.int32, device=DEV), torch.tensor([0])
    pool = torch.zeros(5, 4, device=DEV)
    for call in (lambda: take_pages(used, 1), lambda: free_pages(used, one),
                 lambda: take_pages(few, MANY), lambda: free_pages(few, used),
                 lambda: fork_pages(few, pool, used), lambda: copy_pages(pool, used, used),
                 lambda: copy_pages(used, one, one + 1), lambda: compact_pages(few, pool, [used])):
        with pytest.raises(ValueError, match="2\\^30"):
            call()
    assert few.tolist() == [0] * 5


def test_channels():
    from pararnn_amd import group_norm

    with pytest.raises(ValueError, match="2\\^31"):
        group_norm(_wide(1, MANY), 1)
    with pytest.raises(ValueError, match="2\\^31"):
        group_norm(_wide(MANY, 1), 1)
