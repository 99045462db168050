"""The delta-rule block's operators from their definitions, on the CPU: the rule token by token, the
residual norm from its sums, a beam step candidate by candidate.  Plain torch in the inputs' own type
(float64 in the tests), the first two differentiable by autograd."""

from __future__ import annotations

import torch


def delta_rule(q, k, v, log_decay, beta, h0=None, scale=None, cu=None):
    """(out (B, T, H, Dv), final states (sequences, H, Dk, Dv)); ``cu``: offsets as a list."""
    H = max(q.shape[2], k.shape[2], v.shape[2], log_decay.shape[-1])
    q, k, v = (x.repeat_interleave(H // x.shape[2], dim=2) for x in (q, k, v))
    B, T, _, Dk = q.shape
    scale = Dk ** -0.5 if scale is None else scale
    a = torch.exp(log_decay).expand(B, T, H)
    S = B if cu is None else len(cu) - 1
    if h0 is None:
        h0 = q.new_zeros(S, H, Dk, v.shape[-1])

    def walk(q, k, v, a, b, s):
        out = []
        for t in range(q.shape[1]):
            s = a[:, t, :, None, None] * s
            u = b[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * s).sum(-2))
            s = s + k[:, t, :, :, None] * u[:, :, None, :]
            out.append(scale * (q[:, t, :, :, None] * s).sum(-2))
        return (torch.stack(out, 1) if out else v[:, :0]), s

    if cu is None:
        return walk(q, k, v, a, beta, h0)
    parts = [walk(*(x[:, cu[i]:cu[i + 1]] for x in (q, k, v, a, beta)), h0[i:i + 1])
             for i in range(S)]
    return torch.cat([o for o, _ in parts], 1), torch.cat([s for _, s in parts])


def residual_norm(x, y, weight=None, bias=None, post_norm=False, post_weight=None, gate=None,
                  activation=None, scale=1.0, norm="rms", eps=1e-6):
    """(h, z) of one token after another's channels."""

    def normed(t):
        if norm == "layer":
            t = t - t.mean(-1, keepdim=True)
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)

    h = x
    if y is not None:
        f = normed(y) if post_norm else y
        f = f if post_weight is None else f * post_weight
        if gate is not None:
            f = f * {None: lambda t: t, "sigmoid": torch.sigmoid,
                     "silu": lambda t: t * torch.sigmoid(t)}[activation](gate)
        h = x + scale * f
    z = normed(h)
    z = z if weight is None else z * weight
    return h, z if bias is None else z + bias


def beam_select(logits, scores, beams, ended=None, pad=0):
    """Lists (score, parent, token) per search, candidate by candidate in float64; equal totals go to the
    lowest beam, the larger logit, the lowest token."""
    B, K, V = logits.shape
    found = []
    for b in range(B):
        rows = []
        for k in range(K):
            s = float(scores[b, k])
            if ended is not None and ended[b, k]:
                rows.append((-s, k, 0.0, pad))
                continue
            x = logits[b, k].double()
            if bool(torch.isnan(x).any() | (x == float("inf")).any()):
                continue
            p = s + torch.log_softmax(x, -1) if bool((x > float("-inf")).any()) else x
            rows += [(-float(p[t]), k, -float(x[t]), t)
                     for t in torch.nonzero(p > float("-inf"))[:, 0].tolist()]
        rows = sorted(r for r in rows if r[0] < float("inf"))[:beams]
        found.append([(-s, k, t) for s, k, _, t in rows])
    return found


def reorder_pages(table, parents):
    """(the new table, {slot: the slot whose rows it takes}) of one search; lists."""
    K, kept, copies, new = len(table), set(), {}, [None] * len(table)
    for i, p in enumerate(parents):
        if 0 <= p < K and p not in kept:
            kept.add(p)
            new[i] = table[p]
    spare = [table[k] for k in range(K) if k not in kept]
    for i, p in enumerate(parents):
        if new[i] is None:
            new[i] = spare.pop(0)
            if 0 <= p < K:
                copies[new[i]] = table[p]
    return new, copies
