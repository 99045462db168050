"""The linear-attention layer's operators from their definitions, on the CPU: the recurrence token
by token, the group norm from its sums, the cache's slots one after another.  Plain torch in the
inputs' own type (float64 in the tests), differentiable by autograd."""

from __future__ import annotations

import torch


def linear_attention(q, k, v, log_decay, h0=None, scale=None, cu=None):
    """(out (B, T, H, Dv), final states (sequences, H, Dk, Dv)); ``cu``: offsets as a list."""
    H = max(q.shape[2], k.shape[2], v.shape[2], log_decay.shape[-1])
    q, k, v = (x.repeat_interleave(H // x.shape[2], dim=2) for x in (q, k, v))
    B, T, _, Dk = q.shape
    scale = Dk ** -0.5 if scale is None else scale
    a = torch.exp(log_decay).expand(B, T, H)
    S = B if cu is None else len(cu) - 1
    if h0 is None:
        h0 = q.new_zeros(S, H, Dk, v.shape[-1])

    def walk(q, k, v, a, s):
        out = []
        for t in range(q.shape[1]):
            s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
            out.append(scale * (q[:, t, :, :, None] * s).sum(-2))
        return (torch.stack(out, 1) if out else v[:, :0]), s

    if cu is None:
        return walk(q, k, v, a, h0)
    parts = [walk(*(x[:, cu[i]:cu[i + 1]] for x in (q, k, v, a)), h0[i:i + 1]) for i in range(S)]
    return torch.cat([o for o, _ in parts], 1), torch.cat([s for _, s in parts])


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, over="token",
               eps=1e-5):
    C = x.shape[-1]
    n = x.numel() // C if over == "token" else x.shape[0]
    y = x.reshape(n, -1, groups, C // groups)
    mean = y.mean((1, 3), keepdim=True)
    var = ((y - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((y - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    z = z if weight is None else z * weight
    z = z if bias is None else z + bias
    act = {None: lambda t: t, "sigmoid": torch.sigmoid,
           "silu": lambda t: t * torch.sigmoid(t)}[activation]
    return act(z) if gate is None else z * act(gate)


def take_pages(used: list[int], n: int) -> list[int]:
    free = [s for s, u in enumerate(used) if not u][:n]
    for s in free:
        used[s] = 1
    return free + [-1] * (n - len(free))


def compact_pages(used: list[int], tables: list[list[int]]):
    """(moves as (from, to), the number of live slots); used and tables change in place."""
    live = sum(1 for u in used if u)
    holes = [s for s in range(live) if not used[s]]
    high = [s for s in range(live, len(used)) if used[s]]
    to = {s: s for s in range(live) if used[s]}
    to.update(zip(high, holes))
    for t in tables:
        t[:] = [to.get(s, -1) if 0 <= s < len(used) else s for s in t]
    used[:] = [int(s < live) for s in range(len(used))]
    return list(zip(high, holes)), live
