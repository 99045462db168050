"""Slots of a state cache: taking, forking, freeing, reordering and compacting them on the GPU.

A serving program keeps its sessions' recurrent states in pools ``(slots, ...)``: a linear
attention's ``(slots, H, Dk, Dv)``, a cell's ``(slots, 4, d)`` or ``(slots, d)``, one per layer;
slot ``s`` is row ``s`` of all of them, a session's ``block_table`` entry names it, and ``used``
``(slots,)`` int32 says which are taken.  A recurrent state changes with every token, so a fork
copies it at once: there is nothing to share.

Every call works on the current stream and leaves its answer on the device; none waits for the
host, so a serving step with them can be captured in a HIP graph (lists int32, contiguous and on
the pools' device then).  Which slots are chosen depends on ``used`` alone: always the lowest ones.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch
from torch import Tensor

from pararnn_amd import _lib
from pararnn_amd.attention import _enqueue, _slots, _writes


def _used(what: str, used: Tensor) -> Tensor:
    if used.device.type != "cuda":
        raise RuntimeError(f"{what} requires a ROCm GPU tensor, got {used.device}")
    if used.dtype != torch.int32:
        raise TypeError(f"{what}: used must be int32, got {used.dtype}")
    if used.dim() != 1 or not used.is_contiguous():
        raise ValueError(f"{what}: used must be (slots,) and contiguous, got {tuple(used.shape)}")
    if used.shape[0] > 1 << 30:
        raise ValueError(f"{what}: {used.shape[0]} slots are more than 2^30")
    return used


def _pools(what: str, pools: Sequence[Tensor] | Tensor, slots: int | None, dev):
    pools = [pools] if isinstance(pools, Tensor) else list(pools)
    for p in pools:
        if p.device.type != "cuda":
            raise RuntimeError(f"{what} requires a ROCm GPU tensor, got {p.device}")
        if dev is not None and p.device != dev:
            raise RuntimeError(f"{what}: tensors on different devices ({p.device} vs {dev})")
        if p.dim() < 1 or not p.is_contiguous():
            raise ValueError(f"{what}: pools must be contiguous (slots, ...), got "
                             f"{tuple(p.shape)}")
        if slots is not None and p.shape[0] != slots:
            raise ValueError(f"{what}: a pool has {p.shape[0]} slots, not {slots}")
        dev, slots = p.device, p.shape[0]
        if slots > 1 << 30:
            raise ValueError(f"{what}: {slots} slots are more than 2^30")
    rows = (_lib.Pool * max(1, len(pools)))(*(
        _lib.Pool(p.data_ptr(), p.numel() // p.shape[0] * p.element_size() if p.shape[0] else 0)
        for p in pools))
    return pools, rows, slots, dev


def take_pages(used: Tensor, n: int) -> Tensor:
    """The ``n`` lowest free slots, now used, ``(n,)`` int32; -1 where none is left.  The pools are
    not touched: a slot's rows still hold what its last session left, so a new session's prompt
    starts without them (``linear_attention`` without ``h0``), and one that starts with a single
    token clears them first."""
    dev = _used("take_pages", used).device
    if not 0 <= n <= 1 << 30:
        raise ValueError(f"take_pages: n must be in 0 .. 2^30, got {n!r}")
    out = torch.empty(n, dtype=torch.int32, device=dev)
    _writes("take_pages", used)
    rc = _enqueue(_lib.load().prnn_pages_take, dev, used.data_ptr(), used.shape[0],
                  out.data_ptr(), n)
    _lib.check(rc, "take_pages")
    return out


def fork_pages(used: Tensor, pools: Sequence[Tensor] | Tensor, parents: Tensor) -> Tensor:
    """For every entry of ``parents`` ``(n,)`` a free slot of its own, lowest first, holding a copy
    of the parent's row in every pool; ``(n,)`` int32.  An entry that is no slot in use (-1, a free
    one), and one for which no slot is left, gets -1."""
    dev = _used("fork_pages", used).device
    pools, rows, _, _ = _pools("fork_pages", pools, used.shape[0], dev)
    parents = _slots("fork_pages", "parents", parents, dev)
    _writes("fork_pages", used, *pools)
    n = parents.shape[0]
    both = torch.empty(2, n, dtype=torch.int32, device=dev)
    rc = _enqueue(_lib.load().prnn_pages_fork, dev, used.data_ptr(), used.shape[0], rows, len(pools),
                  parents.data_ptr(), both.data_ptr(), n, both.data_ptr() + 4 * n)
    _lib.check(rc, "fork_pages")
    return both[0]


def free_pages(used: Tensor, slots: Tensor) -> None:
    """Gives ``slots`` ``(n,)`` back; entries that are no slots are passed over."""
    dev = _used("free_pages", used).device
    slots = _slots("free_pages", "slots", slots, dev)
    _writes("free_pages", used)
    rc = _enqueue(_lib.load().prnn_pages_free, dev, used.data_ptr(), used.shape[0],
                  slots.data_ptr(), slots.shape[0])
    _lib.check(rc, "free_pages")


def copy_pages(pools: Sequence[Tensor] | Tensor, src: Tensor, dst: Tensor) -> None:
    """Row ``dst[i]`` of every pool gets row ``src[i]``.  No ``dst`` may be another entry's ``src``
    or ``dst``; an entry with either outside the pool is passed over."""
    pools, rows, slots, dev = _pools("copy_pages", pools, None, None)
    if dev is None:
        raise ValueError("copy_pages needs a pool")
    src = _slots("copy_pages", "src", src, dev)
    dst = _slots("copy_pages", "dst", dst, dev)
    if src.shape != dst.shape:
        raise ValueError(f"copy_pages: src {tuple(src.shape)} != dst {tuple(dst.shape)}")
    _writes("copy_pages", *pools)
    rc = _enqueue(_lib.load().prnn_pages_copy, dev, slots, rows, len(pools), src.data_ptr(),
                  dst.data_ptr(), src.shape[0])
    _lib.check(rc, "copy_pages")


def reorder_pages(pools: Sequence[Tensor] | Tensor, table: Tensor, parents: Tensor) -> Tensor:
    """Lets the beams' states follow a selection: ``table`` ``(B, K)`` (or ``(K,)``) int32 names the
    slots of the beams of ``B`` searches, ``parents`` of the same shape each child's beam of its own
    search (:func:`beam_select`'s); ``table``, rewritten in place and returned, then names a slot for
    every child that holds its parent's rows in every pool.

    A beam's first child keeps its slot; the other children, in order, take the slots of the beams
    without children, in order, so a search keeps its slots and only what they hold is copied, once
    for every beam without a child.  A child without a parent (an entry outside ``0 .. K - 1``, -1) or
    of a beam whose slot is outside the pool gets a slot that is not written.  ``K`` at most 1024,
    ``B`` below 2^22; no two entries of ``table`` may name one slot."""
    what = "reorder_pages"
    pools, rows, slots, dev = _pools(what, pools, None, None)
    if dev is None:
        raise ValueError(f"{what} needs a pool")
    if table.device != dev or parents.device != dev:
        raise RuntimeError(f"{what}: tensors on different devices ({table.device}, "
                           f"{parents.device} vs {dev})")
    if table.dtype != torch.int32:
        raise TypeError(f"{what}: table must be int32, got {table.dtype}")
    if table.dim() not in (1, 2) or not table.is_contiguous():
        raise ValueError(f"{what}: table must be (B, K) or (K,) and contiguous (it is changed in "
                         f"place), got {tuple(table.shape)}")
    if parents.shape != table.shape:
        raise ValueError(f"{what}: parents {tuple(parents.shape)} != table {tuple(table.shape)}")
    beams = table.shape[-1]
    if not 1 <= beams <= 1024 or table.numel() > 1 << 30:
        raise ValueError(f"{what}: K={beams} beams are not in 1 .. 1024")
    parents = _slots(what, "parents", parents.reshape(-1), dev)
    _writes(what, table, *pools)
    searches = table.numel() // beams
    scratch = torch.empty(2 * table.numel(), dtype=torch.int32, device=dev)
    rc = _enqueue(_lib.load().prnn_pages_reorder, dev, slots, rows, len(pools), table.data_ptr(),
                  parents.data_ptr(), searches, beams, scratch.data_ptr())
    _lib.check(rc, what)
    return table


def compact_pages(used: Tensor, pools: Sequence[Tensor] | Tensor,
                  tables: Sequence[Tensor] = ()) -> Tensor:
    """Moves the used slots into the lowest ones and returns their number (one int32 on the
    device).  Only as many rows move as there are free slots below that number: the lowest of those
    gets the lowest used slot above it, and so on.  The entries of ``tables`` (int32, contiguous;
    changed in place) follow; an entry that named a free slot becomes -1, one that named no slot
    stays."""
    what = "compact_pages"
    dev = _used(what, used).device
    pools, rows, _, _ = _pools(what, pools, used.shape[0], dev)
    tables = [tables] if isinstance(tables, Tensor) else list(tables)
    for t in tables:
        if t.device != dev:
            raise RuntimeError(f"{what}: tensors on different devices ({t.device} vs {dev})")
        if t.dtype != torch.int32:
            raise TypeError(f"{what}: tables must be int32, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{what}: tables must be contiguous (they are changed in place)")
        if t.numel() > 1 << 30:
            raise ValueError(f"{what}: a table has {t.numel()} entries, more than 2^30")
    # a table given twice is one table: renamed twice, its moved entries would name free slots
    spans = sorted({(t.data_ptr(), t.numel()) for t in tables if t.numel()})
    if any(a + 4 * n > b for (a, n), (b, _) in zip(spans, spans[1:])):
        raise ValueError(f"{what}: tables must not overlap")
    _writes(what, used, *pools, *tables)
    n = len(spans)
    scratch = torch.empty(2 + 2 * used.shape[0], dtype=torch.int32, device=dev)
    ptrs = (ctypes.c_void_p * max(1, n))(*(p for p, _ in spans))
    lens = (ctypes.c_int * max(1, n))(*(k for _, k in spans))
    rc = _enqueue(_lib.load().prnn_pages_compact, dev, used.data_ptr(), used.shape[0], rows,
                  len(pools), ptrs, lens, n, scratch.data_ptr(), scratch.data_ptr() + 4)
    _lib.check(rc, what)
    return scratch[0]
