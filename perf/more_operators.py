"""Cases for timing the operators of a gated delta-rule block: the delta rule itself (prompts,
training steps, single tokens on a paged state), the norms before and after a block with its gate
and residual scale, and a beam search's step over the sessions that such a layer serves (selection
over beams and vocabulary, states following their beams).

``run`` does one pass of a case.  With ``own`` false it computes the operator from elementary torch
operations in 32 bits (64 where ties are decided), rounded once at the end; with ``own`` true it
calls this package's operator.  ``exact`` gives the same outputs in 64 bits from the definition.

The operators, for one head with state ``S`` (Dk x Dv), log decay ``g_t <= 0`` and rate ``b_t``:

* delta rule: ``u_t = b_t (v_t - exp(g_t) S_{t-1}^T k_t)``, ``S_t = exp(g_t) S_{t-1} + k_t u_t^T``,
  ``o_t = scale S_t^T q_t``;
* residual norm: ``h = x + scale act(gate) norm(y)`` and ``z = norm(h)``, both norms over channels;
* beam step: the best of ``score + log_softmax(logits)`` over beams and vocabulary, ties to the
  lowest index; a beam's first child keeps its slot of the state pool, the other children take
  copies in the slots of beams that have none.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64  # tokens of the plain form's chunks
EPS = 1e-6


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
        dict(name="step_one", kind="step", dtype="bf16", B=1, H=8, Hk=8, Dk=64, Dv=64,
             decay="token", slots=0),
        # the next token of 256 sessions whose states lie in a pool of 384 slots: the state is
        # read and written once
        dict(name="step_paged", kind="step", dtype="bf16", B=256, H=16, Hk=16, Dk=128, Dv=128,
             decay="token", slots=384),
        # one long document and few heads: rows are scarce, the sequence is long
        dict(name="prompt_long", kind="prompt", dtype="bf16", B=1, T=16384, H=8, Hk=8, Dk=128,
             Dv=128, decay="token", h0=False),
        # a packed batch of ragged prompts, keys shared by heads, states from and to a pool
        dict(name="prompt_packed", kind="packed", dtype="bf16", N=20011, seqs=37, H=16, Hk=4,
             Dk=64, Dv=64, decay="token"),
        # an ordinary bf16 training step of the mixer
        dict(name="train_bf16", kind="train", dtype="bf16", B=8, T=2048, H=16, Hk=16, Dk=64,
             Dv=64, decay="token", h0=False),
        # float32 training on odd sizes, the state carried over from the batch before
        dict(name="train_f32_odd", kind="train", dtype="f32", B=3, T=1001, H=6, Hk=3, Dk=48,
             Dv=72, decay="token", h0=True),
        # between two blocks in training: norm behind the one, gate, residual, norm before the next
        dict(name="norm_train", kind="norm", dtype="bf16", N=16384, C=1024, norm="rms", post=True,
             act="silu", gate=True, scale="vector", train=True),
        # the same for one token of each of 32 sessions
        dict(name="norm_step", kind="norm", dtype="bf16", N=32, C=1024, norm="rms", post=True,
             act="silu", gate=True, scale="vector", train=False),
        # a layer norm behind a plain residual, float32 training, an odd width
        dict(name="norm_layer_odd", kind="norm", dtype="f32", N=4099, C=1001, norm="layer",
             post=False, act="none", gate=False, scale="number", train=True),
        # one search of 4 beams
        dict(name="beams_one", kind="beams", dtype="f32", B=1, K=4, V=32000, H=8, Dk=64, Dv=64),
        # 32 searches of 8 beams over a large vocabulary
        dict(name="beams_many", kind="beams", dtype="bf16", B=32, K=8, V=50257, H=8, Dk=64, Dv=64),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng, most: int) -> dict:
    h = _log(rng, 1, most)
    return dict(H=h, Hk=rng.choice([d for d in range(1, h + 1) if h % d == 0]))


def _dims(rng) -> dict:
    return dict(Dk=rng.choice([16, 32, 48, 64, 64, 96, 128]),
                Dv=rng.choice([16, 32, 64, 64, 72, 96, 128]))


def draw(rng) -> dict:
    kind = rng.choice(["step", "prompt", "packed", "train", "train", "norm", "norm", "beams",
                       "beams"])
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
        c = _log(rng, 48, 8192)
        gate = rng.random() < 0.5
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32", "f16"]),
                    N=_log(rng, 1, min(1 << 16, (1 << 23) // c)), C=c,
                    norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.5,
                    act=rng.choice(["silu", "sigmoid", "none"]) if gate else "none", gate=gate,
                    scale=rng.choice(["vector", "number"]), train=rng.random() < 0.6)
    k = _log(rng, 1, 16)
    v = _log(rng, 500, 128000)
    return dict(kind=kind, dtype=rng.choice(["bf16", "f32", "f16"]),
                B=_log(rng, 1, max(1, min(64, 12_000_000 // (k * v)))), K=k, V=v,
                H=rng.choice([1, 4, 8]), Dk=rng.choice([32, 64]), Dv=rng.choice([48, 64, 128]))


# ---------------------------------------------------------------------------
# What a user's program holds
# ---------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 6271 + 5)


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


def _mixer_inputs(case, g, st, *lead):
    """Projected heads as a layer hands them over: keys and queries of unit length, values
    N(0, 1), rates in (0, 1)."""
    dt = DTYPES[case["dtype"]]
    for n in ("q", "k"):
        x = _randn(g, *lead, case["Hk"], case["Dk"])
        st[n] = (x / x.norm(dim=-1, keepdim=True)).to(dt)
    st["v"] = _randn(g, *lead, case["H"], case["Dv"]).to(dt)
    st["g"] = _decay(case, g, *lead)
    st["b"] = torch.sigmoid(_randn(g, *lead, case["H"])).to(dt)


def _lengths(case, seed) -> list[int]:
    """Uneven lengths, at least one token each, that add up to N."""
    import random

    r = random.Random(int(seed) * 37 + 3)
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
            _mixer_inputs(case, g, st, B)
            st["state"] = _randn(g, case["slots"] or B, H, Dk, Dv)
            if case["slots"]:
                st["table"] = torch.randperm(case["slots"], generator=g,
                                             device=DEVICE)[:B].to(torch.int32)
        elif kind == "packed":
            lens = _lengths(case, seed)
            _mixer_inputs(case, g, st, 1, case["N"])
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
            _mixer_inputs(case, g, st, B, T)
            st["h0"] = _randn(g, B, H, Dk, Dv) if case["h0"] else None
            if kind == "train":
                st["go"] = _randn(g, B, T, H, Dv).to(DTYPES[case["dtype"]])
                st["gs"] = _randn(g, B, H, Dk, Dv) if case["h0"] else None
                for n in ("q", "k", "v", "g", "b", "h0"):
                    if st[n] is not None and not (n == "g" and case["decay"] == "head"):
                        st[n].requires_grad_(True)
    elif kind == "norm":
        N, C, dt = case["N"], case["C"], DTYPES[case["dtype"]]
        st["x"] = (_randn(g, N, C) * 2.0 + 0.2).to(dt)
        st["y"] = (_randn(g, N, C) * 0.7 - 0.1).to(dt)
        st["w"] = (1 + 0.1 * _randn(g, C)).to(dt)
        st["bias"] = (0.1 * _randn(g, C)).to(dt) if case["norm"] == "layer" else None
        st["pw"] = (1 + 0.1 * _randn(g, C)).to(dt) if case["post"] else None
        st["gate"] = _randn(g, N, C).to(dt) if case["gate"] else None
        st["scale"] = (0.3 + 0.1 * _randn(g, C)).to(dt) if case["scale"] == "vector" else 0.5
        if case["train"]:
            st["gh"] = _randn(g, N, C).to(dt)
            st["gz"] = _randn(g, N, C).to(dt)
            for n in _norm_leaves(st):
                st[n].requires_grad_(True)
    else:
        B, K, V = case["B"], case["K"], case["V"]
        # a few likely continuations stand out of a long tail
        st["logits"] = (_randn(g, B, K, V) * 2.5).to(DTYPES[case["dtype"]])
        st["scores"] = -20.0 + 1.5 * _randn(g, B, K)
        slots = B * K + 7
        st["pool"] = _randn(g, slots, case["H"], case["Dk"], case["Dv"])
        st["table"] = torch.randperm(slots, generator=g,
                                     device=DEVICE)[:B * K].to(torch.int32).view(B, K)
    return st


def _norm_leaves(st):
    return [n for n in ("x", "y", "w", "bias", "pw", "gate", "scale")
            if isinstance(st[n], torch.Tensor)]


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
    return _beams_own(st) if own else _beams_plain(st)


# -- delta rule --------------------------------------------------------------


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
    s = torch.exp(st["g"].float())[..., None, None] * s
    u = st["b"].float()[..., None] * (v - (k[..., :, None] * s).sum(-2))
    s = s + k[..., :, None] * u[..., None, :]
    o = (q[..., :, None] * s).sum(-2) * st["scale"]
    if rows is None:
        state.copy_(s)
    else:
        state[rows] = s
    return dict(o=o.to(dt), state=state)


def _step_own(st):
    p = _package()
    o = p.delta_rule_step(st["q"], st["k"], st["v"], st["g"], st["b"], st["state"],
                          scale=st["scale"], block_table=st.get("table"))
    return dict(o=o, state=st["state"])


def _chunked(q, k, v, g, b, h0, scale):
    """The chunked form in 32 bits: q, k, v (B, T, H, D), g and b (B, T, H), h0 (B, H, Dk, Dv) or
    None.  Inside a chunk what the tokens write solves a unit triangular system, whose inverse is
    the product of (1 + N^2^i) with N = -(its strictly lower part); the state goes from chunk to
    chunk, the one order in which it exists."""
    B, T, H, Dk = q.shape
    n = -(-T // CHUNK)
    pad = n * CHUNK - T

    def split(x):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad))
        return x.view(B, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v, b = split(q), split(k), split(v), split(b[..., None])
    G = split(g[..., None])[..., 0].cumsum(-1)
    last = G[..., -1]
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    pair = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf))
    kt = k.transpose(-1, -2)
    power = -b * torch.matmul(k, kt) * pair.tril(-1)
    inverse = torch.eye(CHUNK, device=q.device) + power
    for _ in range((CHUNK - 1).bit_length() - 1):
        power = torch.matmul(power, power)
        inverse = inverse + torch.matmul(inverse, power)
    e = torch.exp(G)[..., None]
    own_part = torch.matmul(inverse, b * v)
    through = torch.matmul(inverse, b * e * k)
    into = (k * torch.exp(last[..., None] - G)[..., None]).transpose(-1, -2)
    s = q.new_zeros(B, H, Dk, v.shape[-1]) if h0 is None else h0
    states, wrote = [], []
    for c in range(n):
        u = own_part[:, :, c] - torch.matmul(through[:, :, c], s)
        states.append(s)
        wrote.append(u)
        s = torch.exp(last[:, :, c])[..., None, None] * s + torch.matmul(into[:, :, c], u)
    o = torch.matmul(torch.matmul(q, kt) * pair, torch.stack(wrote, 2))
    o = o + e * torch.matmul(q, torch.stack(states, 2))
    o = (o * scale).permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, -1)[:, :T]
    return o, s


def _mix_plain(q, k, v, g, b, h0, scale):
    H, dt = v.shape[-2], q.dtype
    g = g.float()
    if g.dim() == 1:
        g = g.expand(q.shape[0], q.shape[1], H)
    o, s = _chunked(_spread(q.float(), H), _spread(k.float(), H), v.float(), g, b.float(), h0,
                    scale)
    return o.to(dt), s


def _mix(st, h0):
    if own:
        o, s = _package().delta_rule(st["q"], st["k"], st["v"], st["g"], st["b"], h0=h0,
                                     scale=st["scale"], return_state=True)
    else:
        o, s = _mix_plain(st["q"], st["k"], st["v"], st["g"], st["b"], h0, st["scale"])
    return dict(o=o, state=s)


def _packed_own(st):
    o = _package().delta_rule(st["q"], st["k"], st["v"], st["g"], st["b"], h0=st["pool"],
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
    o, s = _mix_plain(q, k, v, g, st["b"][0][at], st["pool"][rows], st["scale"])
    out = o.new_empty(1, st["case"]["N"], *o.shape[2:])
    out[0, at[live]] = o[live]
    st["pool_out"][rows] = s
    return dict(o=out, pool=st["pool_out"])


def _train(st):
    leaves = {n: st[n] for n in ("q", "k", "v", "g", "b", "h0")
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


# -- residual norm -----------------------------------------------------------


def _normed(x, kind: str):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _norm_plain(st):
    c, dt = st["case"], st["x"].dtype
    f = st["y"].float()
    if c["post"]:
        f = _normed(f, c["norm"]) * st["pw"].float()
    if c["gate"]:
        gate = st["gate"].float()
        sig = torch.sigmoid(gate)
        f = f * {"silu": gate * sig, "sigmoid": sig, "none": gate}[c["act"]]
    scale = st["scale"]
    h = st["x"].float() + f * (scale if isinstance(scale, float) else scale.float())
    z = _normed(h, c["norm"]) * st["w"].float()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    return h.to(dt), z.to(dt)


def _norm(st):
    c = st["case"]
    with torch.set_grad_enabled(c["train"]):
        if own:
            h, z = _package().residual_norm(
                st["x"], st["y"], st["w"], st["bias"], post_norm=c["post"], post_weight=st["pw"],
                gate=st["gate"], activation=None if c["act"] == "none" else c["act"],
                scale=st["scale"], norm=c["norm"], eps=EPS)
        else:
            h, z = _norm_plain(st)
    if not c["train"]:
        return dict(h=h, z=z)
    names = _norm_leaves(st)
    grads = torch.autograd.grad([h, z], [st[n] for n in names], [st["gh"], st["gz"]])
    return dict({"d" + n: x for n, x in zip(names, grads)}, h=h.detach(), z=z.detach())


# -- beams -------------------------------------------------------------------


def _beams_own(st):
    p = _package()
    scores, parents, tokens = p.beam_select(st["logits"], st["scores"])
    p.reorder_pages([st["pool"]], st["table"], parents)
    return dict(scores=scores, parents=parents, tokens=tokens, table=st["table"], pool=st["pool"])


def _beams_plain(st):
    """The sums and the selection in 64 bits: candidates of two beams may be next to each other."""
    logits, table, pool = st["logits"].double(), st["table"], st["pool"]
    B, K, V = logits.shape
    top = logits.amax(-1, keepdim=True)
    logp = logits - top - torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    total = (logp + st["scores"].double()[..., None]).view(B, K * V)
    order = torch.sort(total, dim=-1, descending=True, stable=True)
    at = order.indices[:, :K]
    parents, tokens = at // V, at % V
    # the first child of a beam keeps its slot
    same = parents[:, :, None] == parents[:, None, :]
    first = ~same.tril(-1).any(-1)
    kept = torch.zeros(B, K, dtype=torch.bool, device=at.device).scatter_(1, parents, True)
    old = table.gather(1, parents)
    # the others, in order, the slots of the beams without children, in order
    spare = torch.sort(kept.to(torch.int32), dim=-1, stable=True).indices
    rank = torch.cumsum(~first, -1) - 1
    new = torch.where(first, old, table.gather(1, spare.gather(1, rank.clamp(min=0))))
    pool[new[~first].long()] = pool[old[~first].long()]
    table.copy_(new)
    return dict(scores=order.values[:, :K].float(), parents=parents.to(torch.int32),
                tokens=tokens.to(torch.int32), table=table, pool=pool)


# ---------------------------------------------------------------------------
# Work that cannot be done without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        n = case["N"] * case["C"]
        more = 1 if case["gate"] else 0
        # forward: x, y, gate, h, z; backward: gh, gz, x, y, gate, dx, dy, dgate
        arrays = 4 + more + ((6 + 2 * more) if case["train"] else 0)
        return dict(bytes=arrays * n * size, flops=n * (40 if case["train"] else 14))
    if kind == "beams":
        B, K, V = case["B"], case["K"], case["V"]
        page = 4 * case["H"] * case["Dk"] * case["Dv"]
        # about 0.4 of the beams are left without a child
        return dict(bytes=B * K * V * size + 2 * page * (0.4 * B * K if K > 1 else 0),
                    flops=4 * B * K * V)
    H, Hk, Dk, Dv = case["H"], case["Hk"], case["Dk"], case["Dv"]
    tokens = case["N"] if kind == "packed" else case["B"] * case.get("T", 1)
    seqs = case["seqs"] if kind == "packed" else case["B"]
    io = tokens * (2 * H * Dv + 2 * Hk * Dk + H) * size
    if case["decay"] == "token":
        io += tokens * H * size
    state = seqs * H * Dk * Dv * 4
    if kind == "step":
        return dict(bytes=io + 2 * state, flops=8 * tokens * H * Dk * Dv)
    first = kind == "packed" or case["h0"]
    # per token: the state read by k and by q and written; the causal halves of a chunk's pairs
    # (k with k, q with k, what is written solved from and read by them)
    flops = tokens * H * (6 * Dk * Dv + 2 * CHUNK * (Dk + Dv))
    if kind != "train":
        return dict(bytes=io + (2 if first else 1) * state, flops=flops)
    # forward, then q, k, v, go, rates and decays read and their gradients written
    return dict(bytes=3 * io + (4 if first else 0) * state, flops=3 * flops)


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
        return _exact_beams(case, st)


def _advance(s, q, k, v, a, b, scale):
    """One token: (the state, the output, what was missing); (..., D) in 64 bits, a = exp(g)."""
    s = a[..., None, None] * s
    miss = v - (k[..., None, :] @ s)[..., 0, :]
    s = s + k[..., :, None] * (b[..., None] * miss)[..., None, :]
    return s, scale * (q[..., None, :] @ s)[..., 0, :], miss


def _exact_mixer(case, st):
    H, Dk, Dv, kind, scale = case["H"], case["Dk"], case["Dv"], case["kind"], st["scale"]

    def each(x):
        return x.detach().double().repeat_interleave(H // x.shape[-2], dim=-2)

    q, k, v, b = each(st["q"]), each(st["k"]), each(st["v"]), st["b"].detach().double()
    g = st["g"].detach().double()
    if g.dim() == 1:
        g = g.expand(*b.shape)
    a = torch.exp(g)
    if kind == "step":
        pool = st["state"].double()
        rows = st["table"].long() if case["slots"] else torch.arange(case["B"], device=q.device)
        pool[rows], o, _ = _advance(pool[rows], q, k, v, a, b, scale)
        return dict(o=o, state=pool)
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
            s[:n], out[0, at], _ = _advance(s[:n], *(x[0, at] for x in (q, k, v, a, b)), scale)
        for j, i in enumerate(order):
            pool[rows[i]] = s[j]
        return dict(o=out, pool=pool)
    B, T = case["B"], case["T"]
    s = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=q.device) if st["h0"] is None \
        else st["h0"].detach().double()
    train = kind == "train"
    if train and B * T * H * Dk * Dv * 8 > 40e9:  # all states are kept
        return None
    o, before, missed = torch.empty_like(v), [], []
    for t in range(T):
        if train:
            before.append(s)
        s, o[:, t], miss = _advance(s, q[:, t], k[:, t], v[:, t], a[:, t], b[:, t], scale)
        missed.append(miss)
    if not train:
        return dict(o=o, state=s)
    # r = dL/dS_t.  Through u_t = b_t miss_t: du = r^T k, dv = b du, and what the state before is
    # read for, a S k, takes -dv
    go, last = st["go"].double(), s
    r = torch.zeros_like(s) if st["gs"] is None else st["gs"].double()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, db = torch.empty_like(g), torch.empty_like(b)
    for t in range(T - 1, -1, -1):
        kt, bt, at = k[:, t], b[:, t, :, None], a[:, t, :, None, None]
        held = at * before[t]
        now = held + kt[..., :, None] * (bt * missed[t])[..., None, :]
        dq[:, t] = scale * (now @ go[:, t, :, :, None])[..., 0]
        r = r + scale * q[:, t, :, :, None] * go[:, t, :, None, :]
        du = (kt[..., None, :] @ r)[..., 0, :]
        dv[:, t] = bt * du
        db[:, t] = (du * missed[t]).sum(-1)
        dk[:, t] = (r @ (bt * missed[t])[..., None] - held @ (bt * du)[..., None])[..., 0]
        r = r - kt[..., :, None] * (bt * du)[..., None, :]
        dg[:, t] = (held * r).sum((-1, -2))
        r = at * r

    def shared(x):
        return x.view(B, T, case["Hk"], H // case["Hk"], -1).sum(3)

    got = dict(o=o, dq=shared(dq), dk=shared(dk), dv=dv, db=db)
    if case["decay"] == "token":
        got["dg"] = dg
    if st["gs"] is not None:
        got.update(state=last, dh0=r)
    return got


def _exact_norm(case, st):
    C, layer = case["C"], case["norm"] == "layer"

    def wide(n):
        return None if st[n] is None else st[n].detach().double() \
            if isinstance(st[n], torch.Tensor) else torch.full((), st[n], dtype=torch.float64,
                                                               device=DEVICE)

    x, y, w, bias, pw, gate, scale = (wide(n) for n in ("x", "y", "w", "bias", "pw", "gate",
                                                        "scale"))

    def forward(t):
        d = t - t.sum(-1, keepdim=True) / C if layer else t
        r = ((d * d).sum(-1, keepdim=True) / C + EPS) ** -0.5
        return d * r, r

    def backward(dn, n, r):
        m = (dn * n).sum(-1, keepdim=True) / C
        shift = dn.sum(-1, keepdim=True) / C if layer else 0.0
        return r * (dn - shift - n * m)

    n1, r1 = forward(y) if case["post"] else (y, None)
    f = n1 * pw if case["post"] else n1
    act = dact = torch.ones((), dtype=torch.float64, device=DEVICE)
    if case["gate"]:
        sig = 1 / (1 + torch.exp(-gate))
        act, dact = {"silu": (gate * sig, sig * (1 + gate * (1 - sig))),
                     "sigmoid": (sig, sig * (1 - sig)),
                     "none": (gate, torch.ones_like(gate))}[case["act"]]
    h = x + scale * act * f
    n2, r2 = forward(h)
    z = n2 * w + (0.0 if bias is None else bias)
    if not case["train"]:
        return dict(h=h, z=z)
    gh, gz = st["gh"].double(), st["gz"].double()
    dh = gh + backward(gz * w, n2, r2)
    df = dh * scale * act
    got = dict(h=h, z=z, dx=dh, dw=(gz * n2).sum(0),
               dy=backward(df * pw, n1, r1) if case["post"] else df)
    if bias is not None:
        got["dbias"] = gz.sum(0)
    if case["post"]:
        got["dpw"] = (df * n1).sum(0)
    if case["gate"]:
        got["dgate"] = dh * scale * f * dact
    if scale.dim():
        got["dscale"] = (dh * act * f).sum(0)
    return got


def _exact_beams(case, st):
    """Row by row from the sorted candidates; the pool slot by slot, with lists on the host."""
    B, K = case["B"], case["K"]
    logits, table = st["logits"].double(), st["table"].tolist()
    logp = logits - torch.logsumexp(logits, -1, keepdim=True) + st["scores"].double()[..., None]
    best, at = logp.topk(min(K, case["V"]), dim=-1)  # no beam gives more than K
    who = list(range(st["pool"].shape[0]))
    scores = []
    for b in range(B):
        rows = [(-s, k, t) for k in range(K) for s, t in zip(best[b, k].tolist(), at[b, k].tolist())]
        chosen = sorted(rows)[:K]
        scores.append([-s for s, _, _ in chosen])
        parents = [k for _, k, _ in chosen]
        spare = [table[b][k] for k in range(K) if k not in parents]
        seen = set()
        for k in parents:
            if k in seen:
                who[spare.pop(0)] = table[b][k]
            seen.add(k)
    pool = st["pool"].double()[torch.tensor(who, device=DEVICE)]
    return dict(scores=torch.tensor(scores, dtype=torch.float64, device=DEVICE), pool=pool)
