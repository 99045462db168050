"""Cases for timing the linear-attention layer's operators: the decayed linear attention itself
(prompts, training steps, single tokens on a paged state), the group norm with a gate or an
activation that follows it, and the pages of the state cache that it is served from.

``run`` does one pass of a case.  With ``own`` false it computes the operator from elementary torch
operations in 32 bits, rounded once at the end; with ``own`` true it calls this package's operator.
``exact`` gives the same outputs in 64 bits from the definition.

The operators, for one head with state ``S`` (Dk x Dv) and log decay ``g_t <= 0``:

* linear attention: ``S_t = exp(g_t) S_{t-1} + k_t v_t^T`` and ``o_t = scale q_t^T S_t``;
* group norm: ``z = w (x - mean) rstd + b`` per group of channels, then ``act(z)`` or
  ``z act(gate)``;
* pages: a slot of the pools per session; taking, forking, freeing and compacting slots.
"""

from __future__ import annotations

import heapq
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64  # tokens of the plain form's chunks


def _package():
    """This repository's package (not installed: it lies in a folder of the repository)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "pararnn-torch_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pararnn_amd

    return pararnn_amd


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # one session's next token through one small layer: latency alone
        dict(name="step_one", kind="step", dtype="bf16", B=1, H=8, Hkv=8, Dk=64, Dv=64,
             decay="head", slots=0),
        # the next token of 256 sessions whose states lie in a pool of 384 slots: the state is
        # read and written once
        dict(name="step_paged", kind="step", dtype="bf16", B=256, H=16, Hkv=16, Dk=128, Dv=128,
             decay="token", slots=384),
        # one long document and few heads: rows are scarce, the sequence is long
        dict(name="prompt_long", kind="prompt", dtype="bf16", B=1, T=16384, H=8, Hkv=8, Dk=128,
             Dv=128, decay="token", h0=False),
        # a packed batch of ragged prompts, grouped heads, states read from and written to a pool
        dict(name="prompt_packed", kind="packed", dtype="bf16", N=20011, seqs=37, H=16, Hkv=4,
             Dk=64, Dv=64, decay="head"),
        # a batch of short turns that go on from kept states, float16
        dict(name="prompt_short_f16", kind="prompt", dtype="f16", B=32, T=100, H=8, Hkv=8, Dk=64,
             Dv=64, decay="token", h0=True),
        # an ordinary bf16 training step of the mixer
        dict(name="train_bf16", kind="train", dtype="bf16", B=8, T=2048, H=16, Hkv=16, Dk=64,
             Dv=64, decay="token", h0=False),
        # float32 training on odd sizes, the state carried over from the batch before
        dict(name="train_f32_odd", kind="train", dtype="f32", B=3, T=1001, H=6, Hkv=3, Dk=48,
             Dv=72, decay="token", h0=True),
        # the gated norm after the mixer in training, forward and backward
        dict(name="norm_gate_train", kind="norm", dtype="bf16", N=16384, L=1, C=1024, G=16,
             act="silu", gate=True, train=True),
        # the same norm at one token for each of 32 sessions
        dict(name="norm_gate_step", kind="norm", dtype="bf16", N=32, L=1, C=1024, G=16,
             act="silu", gate=True, train=False),
        # statistics over whole samples, channels last, float32 training
        dict(name="norm_sample_train", kind="norm", dtype="f32", N=8, L=2047, C=256, G=32,
             act="silu", gate=False, train=True),
        # a beam search's step over 8 beams: children take the states of their parents
        dict(name="pages_beams", kind="beams", beams=8, slots=64, H=8, Dk=64, Dv=64),
        # sessions end and others begin: their slots are freed, the pool is compacted, new ones
        # are taken
        dict(name="pages_turnover", kind="turnover", live=1500, ended=300, slots=2048, H=8, Dk=128,
             Dv=128),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng, most: int) -> dict:
    h = _log(rng, 1, most)
    return dict(H=h, Hkv=rng.choice([d for d in range(1, h + 1) if h % d == 0]))


def _dims(rng) -> dict:
    return dict(Dk=rng.choice([16, 32, 48, 64, 64, 96, 128]),
                Dv=rng.choice([16, 32, 64, 64, 72, 96, 128]))


def draw(rng) -> dict:
    kind = rng.choice(["step", "step", "prompt", "prompt", "packed", "train", "train", "norm",
                       "norm", "beams", "turnover"])
    if kind == "step":
        b = _log(rng, 1, 256)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), B=b, **_heads(rng, 16),
                    **_dims(rng), decay=rng.choice(["head", "token"]),
                    slots=rng.choice([0, b + rng.randint(0, 100)]))
    if kind in ("prompt", "train"):
        dtype = rng.choice(["bf16", "bf16", "f32", "f32" if kind == "train" else "f16"])
        heads, dims = _heads(rng, 16), _dims(rng)
        # head-tokens, so that no case outweighs the listed training step
        most = (1 << (17 if dtype != "bf16" else 18)) // max(1, dims["Dk"] * dims["Dv"] >> 12)
        t = _log(rng, 1 if kind == "prompt" else 16, min(16384, most // heads["H"]))
        return dict(kind=kind, dtype=dtype, B=_log(rng, 1, min(32, most // (heads["H"] * t))), T=t,
                    **heads, **dims, decay=rng.choice(["head", "token"]),
                    h0=rng.random() < 0.5)
    if kind == "packed":
        heads, dims = _heads(rng, 16), _dims(rng)
        most = (1 << 18) // max(1, dims["Dk"] * dims["Dv"] >> 12)
        n = _log(rng, 256, min(32768, most // heads["H"]))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), N=n,
                    seqs=_log(rng, max(2, n // 2048), max(3, n // 64)), **heads, **dims,
                    decay=rng.choice(["head", "token"]))
    if kind == "norm":
        g = rng.choice([1, 4, 8, 16, 32])
        c = g * rng.choice([8, 12, 32, 50, 64, 128])
        sample = rng.random() < 0.4
        n = _log(rng, 1, 16) if sample else _log(rng, 1, min(1 << 16, (1 << 23) // c))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32", "f16"]), N=n,
                    L=_log(rng, 2, max(2, (1 << 22) // (n * c))) if sample else 1, C=c, G=g,
                    act=rng.choice(["silu", "sigmoid", "none"]), gate=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    d = dict(H=rng.choice([1, 4, 8]), Dk=rng.choice([32, 64]), Dv=rng.choice([48, 64, 128]))
    if kind == "beams":
        n = _log(rng, 1, 256)
        return dict(kind=kind, beams=n, slots=2 * n + rng.randint(0, 300), **d)
    live = _log(rng, 8, 1500)
    return dict(kind=kind, live=live, ended=rng.randint(1, max(1, live // 3)),
                slots=live + rng.randint(0, 500), **d)


# ---------------------------------------------------------------------------
# What a user's program holds
# ---------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 11)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _decay(case, g, *lead):
    """Log decays.  ``head``: fixed, horizons from 32 tokens up, doubling from head to head (at
    most 4096); ``token``: from the input, -softplus, most of them short of one."""
    h = case["H"]
    if case["decay"] == "head":
        n = torch.arange(h, device=DEVICE, dtype=torch.float32)
        return torch.log1p(-torch.exp2(-5.0 - 7.0 * n / max(1, h - 1)))
    x = _randn(g, *lead, h) - 3.0
    return (-torch.nn.functional.softplus(x)).to(DTYPES[case["dtype"]])


def _qkv(case, g, *lead):
    """Projected heads as a layer hands them over: keys of about unit length, queries and values
    N(0, 1)."""
    dt, hkv = DTYPES[case["dtype"]], case["Hkv"]
    q = _randn(g, *lead, case["H"], case["Dk"])
    k = _randn(g, *lead, hkv, case["Dk"]) / math.sqrt(case["Dk"])
    v = _randn(g, *lead, hkv, case["Dv"])
    return q.to(dt), k.to(dt), v.to(dt)


def _lengths(case, seed) -> list[int]:
    """Uneven lengths, at least one token each, that add up to N."""
    import random

    r = random.Random(int(seed) * 31 + 7)
    n, s = case["N"], case["seqs"]
    w = [math.exp(r.gauss(0.0, 0.6)) for _ in range(s)]
    left = n - s
    got = [1 + int(left * x / sum(w)) for x in w]
    got[-1] += n - sum(got)
    return got


def prepare(case: dict, seed: int) -> dict:
    g, kind = _gen(seed), case["kind"]
    st = dict(case=case)
    if kind in ("step", "prompt", "packed", "train"):
        H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
        st["scale"] = Dk ** -0.5
        if kind == "step":
            B = case["B"]
            st["q"], st["k"], st["v"] = _qkv(case, g, B)
            st["g"] = _decay(case, g, B)
            st["state"] = _randn(g, case["slots"] or B, H, Dk, Dv)
            if case["slots"]:
                st["table"] = torch.randperm(case["slots"], generator=g,
                                             device=DEVICE)[:B].to(torch.int32)
        elif kind == "packed":
            lens = _lengths(case, seed)
            st["q"], st["k"], st["v"] = _qkv(case, g, 1, case["N"])
            st["g"] = _decay(case, g, 1, case["N"])
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + n)
            S = case["seqs"]
            st["pool"] = _randn(g, S + 5, H, Dk, Dv)
            st["pool_out"] = torch.zeros_like(st["pool"])
            st["table"] = torch.randperm(S + 5, generator=g, device=DEVICE)[:S].to(torch.int32)
            st["cu"] = torch.tensor(cu, device=DEVICE, dtype=torch.int32)
            st["longest"] = max(lens)
            if own:  # the batch's offsets, checked once: the handle of all layers and steps
                st["packed"] = _package().PackedSequences(st["cu"])
        else:
            B, T = case["B"], case["T"]
            st["q"], st["k"], st["v"] = _qkv(case, g, B, T)
            st["g"] = _decay(case, g, B, T)
            st["h0"] = _randn(g, B, H, Dk, Dv) if case["h0"] else None
            if kind == "train":
                st["go"] = _randn(g, B, T, H, Dv).to(DTYPES[case["dtype"]])
                st["gs"] = _randn(g, B, H, Dk, Dv) if case["h0"] else None
                for n in ("q", "k", "v", "g", "h0"):
                    if st[n] is not None and not (n == "g" and case["decay"] == "head"):
                        st[n].requires_grad_(True)
    elif kind == "norm":
        N, L, C, dt = case["N"], case["L"], case["C"], DTYPES[case["dtype"]]
        shape = (N, C) if L == 1 else (N, L, C)
        st["x"] = (_randn(g, *shape) * 1.5 + 0.3).to(dt)
        st["w"] = (1 + 0.1 * _randn(g, C)).to(dt)
        st["b"] = (0.1 * _randn(g, C)).to(dt)
        st["gate"] = _randn(g, *shape).to(dt) if case["gate"] else None
        if case["train"]:
            st["gy"] = _randn(g, *shape).to(dt)
            for n in ("x", "w", "b", "gate"):
                if st[n] is not None:
                    st[n].requires_grad_(True)
    else:
        C = case["slots"]
        st["pool"] = _randn(g, C, case["H"], case["Dk"], case["Dv"])
        n = case["beams"] if kind == "beams" else case["live"]
        st["used"] = torch.zeros(C, dtype=torch.int32, device=DEVICE)
        # beams lie anywhere, sessions in the lowest slots (the pool was compacted before)
        st["table"] = torch.randperm(C if kind == "beams" else n, generator=g,
                                     device=DEVICE)[:n].to(torch.int32)
        st["used"][st["table"].long()] = 1
        if kind == "beams":
            # the survivors: some beams have several children, some none
            st["parents"] = torch.randint(0, n, (n,), generator=g, device=DEVICE)
        else:
            st["order"] = torch.randperm(n, generator=g, device=DEVICE)
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(st: dict):
    kind = st["case"]["kind"]
    if kind == "step":
        return _step_own(st) if own else _step_plain(st)
    if kind == "prompt":
        with torch.no_grad():
            return _mix(st, st["h0"])
    if kind == "packed":
        with torch.no_grad():
            return _packed_own(st) if own else _packed_plain(st)
    if kind == "train":
        return _train(st)
    if kind == "norm":
        return _norm(st)
    if kind == "beams":
        return _beams(st)
    return _turnover(st)


# -- linear attention --------------------------------------------------------


def _spread(x, heads: int):
    """Shared heads for every head that uses them."""
    n = heads // x.shape[-2]
    return x if n == 1 else x.repeat_interleave(n, dim=-2)


def _step_plain(st):
    c, state = st["case"], st["state"]
    dt = st["q"].dtype
    q, k, v = (_spread(st[n].float(), c["H"]) for n in ("q", "k", "v"))
    rows = st["table"].long() if c["slots"] else None
    s = state if rows is None else state[rows]
    s = torch.exp(st["g"].float())[..., None, None] * s + k[..., :, None] * v[..., None, :]
    o = (q[..., :, None] * s).sum(-2) * st["scale"]
    if rows is None:
        state.copy_(s)
    else:
        state[rows] = s
    return dict(o=o.to(dt), state=state)


def _step_own(st):
    p = _package()
    o = p.linear_attention_step(st["q"], st["k"], st["v"], st["g"], st["state"],
                                scale=st["scale"], block_table=st.get("table"))
    return dict(o=o, state=st["state"])


def _chunked(q, k, v, g, h0, scale):
    """The chunked form in 32 bits: q, k, v (B, T, H, D), g (B, T, H), h0 (B, H, Dk, Dv) or
    None.  Inside a chunk the masked product, between chunks the states at their starts, all
    at once through the matrix of the decays from chunk to chunk."""
    B, T, H, Dk = q.shape
    n = -(-T // CHUNK)
    pad = n * CHUNK - T

    def split(x):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad))
        return x.view(B, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v, G = split(q), split(k), split(v), split(g[..., None])[..., 0].cumsum(-1)
    last = G[..., -1]
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    pair = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf))
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * pair, v)
    U = torch.matmul((k * torch.exp(last[..., None] - G)[..., None]).transpose(-1, -2), v)
    # S[c] = state before chunk c (c = n: the final one) = sum_{c' < c} exp(A_c - A_{c'+1}) U_c'
    A = torch.nn.functional.pad(last.cumsum(-1), (1, 0))
    before = torch.ones(n + 1, n, dtype=torch.bool, device=q.device).tril(-1)
    M = torch.exp((A[..., :, None] - A[..., None, 1:]).masked_fill(~before, -math.inf))
    S = torch.matmul(M, U.reshape(B, H, n, -1)).view(B, H, n + 1, Dk, -1)
    if h0 is not None:
        S = S + torch.exp(A)[..., None, None] * h0[:, :, None]
    o = o + torch.exp(G)[..., None] * torch.matmul(q, S[:, :, :-1])
    o = (o * scale).permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, -1)[:, :T]
    return o, S[:, :, -1]


def _attend_plain(q, k, v, g, h0, scale):
    H, dt = max(q.shape[-2], k.shape[-2]), q.dtype
    g = g.float()
    if g.dim() == 1:
        g = g.expand(q.shape[0], q.shape[1], H)
    o, s = _chunked(_spread(q.float(), H), _spread(k.float(), H), _spread(v.float(), H), g, h0,
                    scale)
    return o.to(dt), s


def _mix(st, h0):
    if own:
        o, s = _package().linear_attention(st["q"], st["k"], st["v"], st["g"], h0=h0,
                                           scale=st["scale"], return_state=True)
    else:
        o, s = _attend_plain(st["q"], st["k"], st["v"], st["g"], h0, st["scale"])
    return dict(o=o, state=s)


def _packed_own(st):
    o = _package().linear_attention(st["q"], st["k"], st["v"], st["g"], h0=st["pool"],
                                    scale=st["scale"], cu_seqlens=st["packed"],
                                    block_table=st["table"], state_out=st["pool_out"])
    return dict(o=o, pool=st["pool_out"])


def _packed_plain(st):
    """As a padded rectangle: zero keys and no decay behind a sequence's end."""
    cu, T = st["cu"].long(), st["longest"]
    t = torch.arange(T, device=cu.device)
    live = t[None] < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + t[None]) * live
    q, k, v = st["q"][0][at], st["k"][0][at] * live[..., None, None], st["v"][0][at]
    g = st["g"].expand(1, st["case"]["N"], -1)[0][at].float() * live[..., None]
    rows = st["table"].long()
    o, s = _attend_plain(q, k, v, g, st["pool"][rows], st["scale"])
    out = o.new_empty(1, st["case"]["N"], *o.shape[2:])
    out[0, at[live]] = o[live]
    st["pool_out"][rows] = s
    return dict(o=out, pool=st["pool_out"])


def _train(st):
    leaves = {n: st[n] for n in ("q", "k", "v", "g", "h0")
              if st[n] is not None and st[n].requires_grad}
    out = _mix(st, st["h0"])
    ends, seeds = [out["o"]], [st["go"]]
    if st["gs"] is not None:
        ends, seeds = ends + [out["state"]], seeds + [st["gs"]]
    grads = torch.autograd.grad(ends, list(leaves.values()), seeds)
    got = {"d" + n: x for n, x in zip(leaves, grads)}
    got["o"] = out["o"].detach()
    if st["gs"] is not None:
        got["state"] = out["state"].detach()
    return got


# -- group norm --------------------------------------------------------------


def _act(z, act: str):
    return z if act == "none" else torch.sigmoid(z) * (z if act == "silu" else 1.0)


def _norm_plain(x, w, b, gate, case):
    dt = x.dtype
    x = x.float()
    y = x.reshape(case["N"], case["L"], case["G"], -1)
    mean = y.mean(dim=(1, 3), keepdim=True)
    d = y - mean
    y = d * torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + 1e-5)
    z = y.reshape(x.shape) * w.float() + b.float()
    z = _act(z, case["act"]) if gate is None else z * _act(gate.float(), case["act"])
    return z.to(dt)


def _norm(st):
    c = st["case"]
    with torch.set_grad_enabled(c["train"]):
        if own:
            y = _package().group_norm(st["x"], c["G"], st["w"], st["b"], gate=st["gate"],
                                      activation=None if c["act"] == "none" else c["act"],
                                      over="token" if c["L"] == 1 else "sample")
        else:
            y = _norm_plain(st["x"], st["w"], st["b"], st["gate"], c)
    if not c["train"]:
        return dict(y=y)
    leaves = {n: st[n] for n in ("x", "w", "b", "gate") if st[n] is not None}
    grads = torch.autograd.grad(y, list(leaves.values()), st["gy"])
    return dict({"d" + n: x for n, x in zip(leaves, grads)}, y=y.detach())


# -- pages -------------------------------------------------------------------


def _free_slots(used, n: int):
    """The n lowest free slots."""
    return torch.nonzero(used == 0)[:n, 0]


def _beams(st):
    """Every child takes a copy of its parent's state in a slot of its own, then the old ones go."""
    used, pool, table = st["used"], st["pool"], st["table"]
    parents = table[st["parents"]]
    if own:
        p = _package()
        kids = p.fork_pages(used, [pool], parents)
        p.free_pages(used, table)
    else:
        kids = _free_slots(used, parents.numel())
        used[kids] = 1
        pool[kids] = pool[parents.long()]
        used[table.long()] = 0
    table.copy_(kids)
    return dict(table=table, used=used, pool=pool)


def _turnover(st):
    """The sessions of the first rows end, the pool closes up, as many new ones begin."""
    used, pool, m = st["used"], st["pool"], st["case"]["ended"]
    table = st["table"][st["order"]]
    if own:
        p = _package()
        p.free_pages(used, table[:m])
        p.compact_pages(used, [pool], [table[m:]])
        table[:m] = p.take_pages(used, m)
    else:
        used[table[:m].long()] = 0
        rest = table[m:].long()
        live = int(used.sum())
        holes = torch.nonzero(used[:live] == 0)[:, 0]
        high = torch.nonzero(used[live:])[:, 0] + live
        pool[holes] = pool[high]
        to = torch.arange(used.numel(), device=used.device)
        to[high] = holes
        used.copy_(torch.arange(used.numel(), device=used.device) < live)
        table[m:] = to[rest].to(torch.int32)
        new = _free_slots(used, m)
        used[new] = 1
        table[:m] = new.to(torch.int32)
    st["table"].copy_(table)
    return dict(table=table, used=used, pool=pool)


# ---------------------------------------------------------------------------
# Work that cannot be done without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind in ("beams", "turnover"):
        page = 4 * case["H"] * case["Dk"] * case["Dv"]
        if kind == "beams":
            return dict(bytes=2 * page * case["beams"] + 8 * case["slots"], flops=0)
        # of the m ended among n live ones, those below slot n - m leave holes that are filled
        m, n = case["ended"], case["live"]
        moved = m * (1 - m / n)
        return dict(bytes=2 * page * moved + 8 * case["slots"], flops=0)
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        n = case["N"] * case["L"] * case["C"]
        # forward: x, gate, y; backward: gy, x, gate, gx, ggate
        arrays = (3 if case["gate"] else 2) + (0 if not case["train"] else 5 if case["gate"] else 3)
        return dict(bytes=arrays * n * size, flops=n * (12 if not case["train"] else 40))
    H, Hkv, Dk, Dv = case["H"], case["Hkv"], case["Dk"], case["Dv"]
    tokens = case["N"] if kind == "packed" else case["B"] * case.get("T", 1)
    seqs = case["seqs"] if kind == "packed" else case["B"]
    io = tokens * (H * (Dk + Dv) + Hkv * (Dk + Dv)) * size
    if case["decay"] == "token":
        io += tokens * H * size
    state = seqs * H * Dk * Dv * 4
    if kind == "step":
        return dict(bytes=io + 2 * state, flops=6 * tokens * H * Dk * Dv)
    first = kind == "packed" or case["h0"]
    # per token: the state's update, its product with q, and the causal half of a chunk's pairs
    flops = tokens * H * (4 * Dk * Dv + CHUNK * (Dk + Dv))
    if kind != "train":
        return dict(bytes=io + (2 if first else 1) * state, flops=flops)
    # forward, then q, k, v, go read and the gradients written
    return dict(bytes=io + 2 * io + (4 if first else 0) * state, flops=3 * flops)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------


def exact(case: dict, seed: int):
    kind = case["kind"]
    st = prepare(case, seed)
    with torch.no_grad():
        if kind in ("step", "prompt", "packed", "train"):
            return _exact_mixer(case, st)
        if kind == "norm":
            return _exact_norm(case, st)
        return _exact_pages(case, st)


def _recur(q, k, v, a, s, scale):
    """o and the last state by the recurrence; (B, T, H, D) in 64 bits, a = exp(g)."""
    out = torch.empty(*q.shape[:3], v.shape[-1], dtype=torch.float64, device=q.device)
    for t in range(q.shape[1]):
        s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, None, :] @ s)[..., 0, :]
    return out, s


def _exact_mixer(case, st):
    H, Dk, Dv, kind, scale = case["H"], case["Dk"], case["Dv"], case["kind"], st["scale"]

    def each(x):
        return x.detach().double().repeat_interleave(H // x.shape[-2], dim=-2)

    q, k, v = each(st["q"]), each(st["k"]), each(st["v"])
    g = st["g"].detach().double()
    if g.dim() == 1:
        g = g.expand(*q.shape[:-1])
    a = torch.exp(g)
    if kind == "step":
        pool = st["state"].double()
        rows = st["table"].long() if case["slots"] else torch.arange(case["B"], device=q.device)
        o, s = _recur(q[:, None], k[:, None], v[:, None], a[:, None], pool[rows], scale)
        pool[rows] = s
        return dict(o=o[:, 0], state=pool)
    if kind == "packed":
        cu, rows = st["cu"].tolist(), st["table"].tolist()
        pool = torch.zeros_like(st["pool"]).double()
        # sequences side by side, each cut where it ends
        order = sorted(range(case["seqs"]), key=lambda i: cu[i] - cu[i + 1])
        s = torch.stack([st["pool"][rows[i]] for i in order]).double()
        start = torch.tensor([cu[i] for i in order], device=q.device)
        lens = [cu[i + 1] - cu[i] for i in order]
        out = torch.empty(1, case["N"], H, Dv, dtype=torch.float64, device=q.device)
        n = len(order)
        for t in range(lens[0]):
            while lens[n - 1] <= t:
                n -= 1
            at = start[:n] + t
            kv = k[0, at][..., :, None] * v[0, at][..., None, :]
            s[:n] = a[0, at][..., None, None] * s[:n] + kv
            out[0, at] = scale * (q[0, at][..., None, :] @ s[:n])[..., 0, :]
        for j, i in enumerate(order):
            pool[rows[i]] = s[j]
        return dict(o=out, pool=pool)
    B, T = case["B"], case["T"]
    s0 = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=q.device) if st["h0"] is None \
        else st["h0"].detach().double()
    if kind == "prompt":
        o, s = _recur(q, k, v, a, s0, scale)
        return dict(o=o, state=s)
    # training: the adjoint R_t = dL/dS_t runs backwards,
    #   R_t = exp(g_{t+1}) R_{t+1} + scale q_t go_t^T,
    # with dq = scale S go, dk = R v, dv = R^T k, and S_t, R_t both decayed forms of one flow:
    #   exp(g_t) <S_{t-1}, R_t> = <S_t, R_t> - k_t . dk_t, the gradient of g_t
    go = st["go"].double()
    o, dq, s = torch.empty_like(go), torch.empty_like(q), s0
    for t in range(T):
        s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * (q[:, t, :, None, :] @ s)[..., 0, :]
        dq[:, t] = scale * (s @ go[:, t, :, :, None])[..., 0]
    last = s
    r = torch.zeros_like(s0) if st["gs"] is None else st["gs"].double()
    flow = (last * r).sum((-1, -2))  # <S_T, dL/dS_T> of the state that is handed out
    dk, dv, dg = torch.empty_like(k), torch.empty_like(v), torch.empty_like(g)
    for t in range(T - 1, -1, -1):
        r = r + scale * q[:, t, :, :, None] * go[:, t, :, None, :]
        dk[:, t] = (r @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ r)[..., 0, :]
        flow = flow + (q[:, t] * dq[:, t]).sum(-1) - (k[:, t] * dk[:, t]).sum(-1)
        dg[:, t] = flow
        r = a[:, t, :, None, None] * r

    def shared(x, n):
        return x.view(B, T, n, H // n, -1).sum(3)

    got = dict(o=o, dq=dq, dk=shared(dk, case["Hkv"]), dv=shared(dv, case["Hkv"]))
    if case["decay"] == "token":
        got["dg"] = dg
    if st["gs"] is not None:
        got.update(state=last, dh0=r)
    return got


def _exact_norm(case, st):
    N, L, C, G = case["N"], case["L"], case["C"], case["G"]
    x = st["x"].detach().double().view(N, L, G, C // G)
    w, b = (st[n].detach().double().view(G, C // G) for n in ("w", "b"))
    count = L * (C // G)
    mean = x.sum((1, 3), keepdim=True) / count
    var = (x - mean).pow(2).sum((1, 3), keepdim=True) / count
    r = (var + 1e-5) ** -0.5
    h = (x - mean) * r
    z = h * w + b
    t = z if st["gate"] is None else st["gate"].detach().double().view(x.shape)
    sig = 1 / (1 + torch.exp(-t))
    f, df = {"silu": (t * sig, sig * (1 + t * (1 - sig))), "sigmoid": (sig, sig * (1 - sig)),
             "none": (t, torch.ones_like(t))}[case["act"]]
    shape = st["x"].shape
    y = f if st["gate"] is None else z * f
    if not case["train"]:
        return dict(y=y.reshape(shape))
    gy = st["gy"].double().view(x.shape)
    dz = gy * (df if st["gate"] is None else f)
    dh = dz * w
    m1 = dh.sum((1, 3), keepdim=True) / count
    m2 = (dh * h).sum((1, 3), keepdim=True) / count
    got = dict(y=y.reshape(shape), dx=(r * (dh - m1 - h * m2)).reshape(shape),
               dw=(dz * h).sum((0, 1)).reshape(C), db=dz.sum((0, 1)).reshape(C))
    if st["gate"] is not None:
        got["dgate"] = (gy * z * df).reshape(shape)
    return got


def _exact_pages(case, st):
    """Slot by slot, with lists on the host."""
    pool, table = st["pool"], st["table"].tolist()
    state = {s: s for s in range(case["slots"])}  # slot -> whose state it holds
    free = sorted(set(range(case["slots"])) - set(table))
    if case["kind"] == "beams":
        heapq.heapify(free)
        kids = []
        for i in st["parents"].tolist():
            kids.append(heapq.heappop(free))
            state[kids[-1]] = table[i]
    else:
        live = sorted(table[i] for i in st["order"].tolist()[case["ended"]:])
        holes = [s for s in range(len(live)) if s not in set(live)]
        for hole, s in zip(holes, [s for s in live if s >= len(live)]):
            state[hole] = s
    who = torch.tensor([state[s] for s in range(case["slots"])], device=pool.device)
    return dict(pool=pool.double()[who])
