"""A model of gated delta-rule blocks, trained and then searched with beams, on this package's operators.

    python examples/delta_rule.py

* training: ``residual_norm``, ``delta_rule`` and ``group_norm`` under autograd on recall (pairs of a
  key and a value, then keys again, whose values are to be given), packed ragged sequences;
* serving: beam search. Ragged prompts in one call, their final states in the first beams' slots of a
  state pool per block; then a token a beam with ``delta_rule_step``, ``beam_select`` over beams and
  vocabulary, and ``reorder_pages``, which lets the states follow the beams. The totals that the search
  ends with are checked against one pass over the sequences it found.
"""

from __future__ import annotations

import os
import sys

import torch
from torch import Tensor, nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "pararnn-torch_amd"))

from pararnn_amd import (  # noqa: E402
    PackedSequences,
    beam_select,
    delta_rule,
    delta_rule_step,
    group_norm,
    reorder_pages,
    residual_norm,
    take_pages,
)


class DeltaBlock(nn.Module):
    """q, k, v, two gates, a log decay and a rate per head from the input; the rule over keys of unit
    length, a norm per head that the first gate multiplies, a projection back.  The second gate, the
    norm of what the block gives and its scale belong to the residual stream."""

    def __init__(self, width: int, heads: int, d_key: int, d_value: int):
        super().__init__()
        self.heads, self.d_key, self.d_value = heads, d_key, d_value
        self.split = (heads * d_key, heads * d_key, heads * d_value, heads * d_value, width, heads, heads)
        self.inp = nn.Linear(width, sum(self.split))
        self.weight = nn.Parameter(torch.ones(heads * d_value))
        self.out = nn.Linear(heads * d_value, width, bias=False)
        # of the residual stream in front of the block and behind it
        self.norm = nn.Parameter(torch.ones(width))
        self.post = nn.Parameter(torch.ones(width))
        self.scale = nn.Parameter(torch.full((width,), 0.5))

    def project(self, x: Tensor):
        q, k, v, gate, back, decay, rate = self.inp(x).split(self.split, dim=-1)
        h, unit = self.heads, nn.functional.normalize
        q, k = unit(q.unflatten(-1, (h, self.d_key)), dim=-1), unit(k.unflatten(-1, (h, self.d_key)), dim=-1)
        return ((q, k, v.unflatten(-1, (h, self.d_value)), nn.functional.logsigmoid(decay + 4),
                 rate.sigmoid()), gate, back)

    def finish(self, o: Tensor, gate: Tensor) -> Tensor:
        return self.out(group_norm(o.flatten(-2), self.heads, self.weight, gate=gate, activation="silu"))


class Model(nn.Module):
    def __init__(self, tokens: int, width: int, blocks: int, heads: int, d_key: int, d_value: int):
        super().__init__()
        self.embed = nn.Embedding(tokens, width)
        self.blocks = nn.ModuleList(DeltaBlock(width, heads, d_key, d_value) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(width))
        self.head = nn.Linear(width, tokens)

    def _run(self, ids: Tensor, mix) -> Tensor:
        """``mix(i, block, *projected)``: block ``i``'s outputs of the rule."""
        h, z = residual_norm(self.embed(ids), None, self.blocks[0].norm)
        for i, block in enumerate(self.blocks):
            projected, gate, back = block.project(z)
            y = block.finish(mix(i, *projected), gate)
            after = self.blocks[i + 1].norm if i + 1 < len(self.blocks) else self.norm
            h, z = residual_norm(h, y, after, post_norm=True, post_weight=block.post, gate=back,
                                 activation="sigmoid", scale=block.scale)
        return self.head(z)

    def forward(self, ids: Tensor, packed: PackedSequences | None = None,
                pools: list[Tensor] | None = None, table: Tensor | None = None) -> Tensor:
        """With ``pools``: new sessions, whose states go to the slots of ``table``."""
        def mix(i, *projected):
            into = {} if pools is None else dict(block_table=table, state_out=pools[i])
            return delta_rule(*projected, cu_seqlens=packed, **into)
        return self._run(ids, mix)

    def step(self, ids: Tensor, pools: list[Tensor], table: Tensor) -> Tensor:
        return self._run(ids, lambda i, *projected: delta_rule_step(*projected, pools[i],
                                                                    block_table=table))


def recall(tokens: int, lens: list[int], gen: torch.Generator) -> tuple[Tensor, Tensor]:
    """Sequences of pairs, keys from the lower half of the tokens, values from the upper; a key that
    comes again has its first value.  Ids, and where a value follows a key that was seen."""
    ids, known = [], []
    for n in lens:
        values, at = {}, 0
        while at < n:
            key = int(torch.randint(0, tokens // 2, (), generator=gen))
            seen = key in values
            value = values.setdefault(key, int(torch.randint(tokens // 2, tokens, (), generator=gen)))
            pair = [key, value][:n - at]
            ids += pair
            known += [False, seen][:len(pair)]
            at += len(pair)
    return torch.tensor(ids), torch.tensor(known)


def train(model: Model, tokens: int, steps: int, device: str, seed: int = 0) -> list[float]:
    gen = torch.Generator().manual_seed(seed)
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    lens = [64, 1, 100, 91]
    packed = PackedSequences(torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()]))
    losses = []
    for _ in range(steps):
        ids, known = recall(tokens, lens, gen)
        logits = model(ids[None].to(device), packed)[0]
        at = known.nonzero()[:, 0]  # never a sequence's first token
        loss = nn.functional.cross_entropy(logits[at.to(device) - 1].float(), ids[at].to(device))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def search(model: Model, prompts: list[Tensor], beams: int, new: int, end: int, device: str):
    """Beam search: (totals, the tokens of every beam, -1 behind its end), the best beam first."""
    B, K = len(prompts), beams
    slots = B * K + 3
    used = torch.zeros(slots, dtype=torch.int32, device=device)
    pools = [torch.zeros(slots, b.heads, b.d_key, b.d_value, device=device) for b in model.blocks]
    table = take_pages(used, B * K).view(B, K)
    cu = torch.tensor([0, *torch.tensor([len(p) for p in prompts]).cumsum(0).tolist()])
    logits = model(torch.cat(prompts)[None].to(device), PackedSequences(cu), pools, table[:, 0].contiguous())
    last = logits[0, cu[1:].to(device) - 1][:, None].expand(B, K, -1)
    scores = torch.full((B, K), float("-inf"), device=device)
    scores[:, 0] = 0.0  # one beam at first
    ended = torch.zeros(B, K, dtype=torch.bool, device=device)
    text = torch.empty(B, K, 0, dtype=torch.int32, device=device)
    for _ in range(new):
        scores, parents, tokens = beam_select(last, scores, ended=ended, pad=end)
        reorder_pages(pools, table, parents)
        kin = parents.clamp(min=0).long()
        ended = ended.gather(1, kin)
        tokens = torch.where(ended, -1, tokens)
        text = torch.cat([text.gather(1, kin[..., None].expand(-1, -1, text.shape[2])), tokens[..., None]], -1)
        ended = ended | (tokens == end)
        last = model.step(tokens.clamp(min=0).flatten(), pools, table.flatten()).view(B, K, -1)
    return scores, text


@torch.no_grad()
def totals(model: Model, prompt: Tensor, text: Tensor, device: str) -> float:
    """A found sequence's total from one pass over it."""
    text = text[text >= 0].long()
    whole = torch.cat([prompt, text])
    p = torch.log_softmax(model(whole[None].to(device))[0].double(), -1)
    at = torch.arange(len(prompt) - 1, len(whole) - 1)
    return float(p[at.to(device), text.to(device)].sum())


def main(device: str = "cuda", steps: int = 200) -> tuple[list[float], float]:
    torch.manual_seed(0)
    tokens = 16
    model = Model(tokens, width=64, blocks=2, heads=4, d_key=32, d_value=16).to(device)
    losses = train(model, tokens, steps, device)
    print(f"training: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps")
    gen = torch.Generator().manual_seed(1)
    prompts = [recall(tokens, [n], gen)[0] for n in (33, 1, 70)]
    scores, text = search(model, prompts, beams=4, new=9, end=3, device=device)
    off = max(abs(float(s) - totals(model, prompt, row, device))
              for prompt, found, total in zip(prompts, text.cpu(), scores)
              for row, s in zip(found, total))
    print(f"search: {text.shape[0]} x {text.shape[1]} sequences, totals within {off:.1e} of one pass")
    return losses, off


if __name__ == "__main__":
    main()
