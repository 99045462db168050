"""A gated linear-attention layer, trained and then served, on this package's operators.

    python examples/linear_attention.py

* training: ``linear_attention`` and ``group_norm`` under autograd on a copy task (a token comes
  back a fixed number of steps later), packed ragged sequences;
* serving: ragged prompts in one call, their final states written to the slots of a state pool,
  then a token at a time with ``linear_attention_step``; a session is forked, others end and their
  slots are freed, the pool is compacted, a new session takes one of the slots, and the served tokens
  are checked against one pass over the whole sequences.
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
    compact_pages,
    fork_pages,
    free_pages,
    group_norm,
    linear_attention,
    linear_attention_step,
    take_pages,
)


class GatedLinearAttention(nn.Module):
    """q, k, v, a gate and a log decay per head from the input, the recurrence, a norm per head that
    the gate multiplies, a projection back."""

    def __init__(self, width: int, heads: int, d_key: int, d_value: int):
        super().__init__()
        self.heads, self.d_key, self.d_value = heads, d_key, d_value
        self.split = (heads * d_key, heads * d_key, heads * d_value, heads * d_value, heads)
        self.inp = nn.Linear(width, sum(self.split))
        self.weight = nn.Parameter(torch.ones(heads * d_value))
        self.bias = nn.Parameter(torch.zeros(heads * d_value))
        self.out = nn.Linear(heads * d_value, width, bias=False)

    def _project(self, x: Tensor):
        q, k, v, gate, decay = self.inp(x).split(self.split, dim=-1)
        h = self.heads
        # views of one projection: the operators read them as they are
        return (q.unflatten(-1, (h, self.d_key)), k.unflatten(-1, (h, self.d_key)),
                v.unflatten(-1, (h, self.d_value)), gate, nn.functional.logsigmoid(decay + 4))

    def _finish(self, o: Tensor, gate: Tensor) -> Tensor:
        y = group_norm(o.flatten(-2), self.heads, self.weight, self.bias, gate=gate.contiguous(),
                       activation="silu")
        return self.out(y)

    def forward(self, x: Tensor, packed: PackedSequences | None = None, **state) -> Tensor:
        q, k, v, gate, decay = self._project(x)
        return self._finish(linear_attention(q, k, v, decay, cu_seqlens=packed, **state), gate)

    def step(self, x: Tensor, pool: Tensor, table: Tensor) -> Tensor:
        q, k, v, gate, decay = self._project(x)
        return self._finish(linear_attention_step(q, k, v, decay, pool, block_table=table), gate)


class Model(nn.Module):
    def __init__(self, tokens: int, width: int, heads: int, d_key: int, d_value: int):
        super().__init__()
        self.embed = nn.Embedding(tokens, width)
        self.mix = GatedLinearAttention(width, heads, d_key, d_value)
        self.norm = nn.LayerNorm(width)
        self.head = nn.Linear(width, tokens)

    def forward(self, ids: Tensor, packed: PackedSequences | None = None, **state) -> Tensor:
        x = self.embed(ids)
        return self.head(self.norm(x + self.mix(x, packed, **state)))

    def step(self, ids: Tensor, pool: Tensor, table: Tensor) -> Tensor:
        x = self.embed(ids)
        return self.head(self.norm(x + self.mix.step(x, pool, table)))


def train(model: Model, tokens: int, steps: int, device: str, seed: int = 0) -> tuple[float, float]:
    """First and last loss of the copy task: the token of two steps before."""
    gen = torch.Generator().manual_seed(seed)
    opt = torch.optim.Adam(model.parameters(), lr=1e-2)
    cu = torch.tensor([0, 40, 41, 130, 256])
    packed, losses = PackedSequences(cu), []
    for _ in range(steps):
        ids = torch.randint(0, tokens, (1, 256), generator=gen)
        want = ids.roll(2, dims=1)
        known = torch.ones(256, dtype=torch.bool)
        for a in cu[:-1].tolist():  # nothing to copy yet
            known[a:a + 2] = False
        logits = model(ids.to(device), packed)
        loss = nn.functional.cross_entropy(logits[0, known.to(device)].float(),
                                           want[0, known].to(device))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses[0], losses[-1]


@torch.no_grad()
def serve(model: Model, tokens: int, device: str, seed: int = 1, new: int = 12) -> float:
    """Serves four ragged prompts for ``new`` tokens; the largest difference of its logits from
    those of one pass over the whole sequences, relative to their size."""
    gen = torch.Generator().manual_seed(seed)
    lens = [17, 1, 64, 30]
    prompts = [torch.randint(0, tokens, (n,), generator=gen) for n in lens]
    m, slots = model.mix, 16
    pool = torch.zeros(slots, m.heads, m.d_key, m.d_value, device=device)
    used = torch.zeros(slots, dtype=torch.int32, device=device)

    table = take_pages(used, len(lens))
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()])
    # new sessions start from zeros, whatever their slots hold, and leave their states there
    logits = model(torch.cat(prompts)[None].to(device), PackedSequences(cu), block_table=table,
                   state_out=pool)
    last = logits[0, cu[1:].to(device) - 1]
    texts, seen = [p.tolist() for p in prompts], [[] for _ in lens]
    for step in range(new):
        if step == 4:  # a second continuation of the third session
            kid = fork_pages(used, [pool], table[2:3])
            table = torch.cat([table, kid])
            texts.append(list(texts[2]))
            seen.append(list(seen[2]))
            last = torch.cat([last, last[2:3]])
        if step == 7:  # the first two end; the others' slots move up
            free_pages(used, table[:2])
            table = table[2:].contiguous()
            live = compact_pages(used, [pool], [table])
            assert int(live) == table.numel() and int(table.max()) < table.numel()
            texts, seen, last = texts[2:], seen[2:], last[2:]
        if step == 9:  # another session begins, on a slot that one of those has left
            prompt = torch.randint(0, tokens, (23,), generator=gen)
            slot = take_pages(used, 1)
            logits = model(prompt[None].to(device), block_table=slot, state_out=pool)
            table, last = torch.cat([table, slot]), torch.cat([last, logits[:, -1]])
            texts.append(prompt.tolist())
            seen.append([])
        ids = last.argmax(-1)
        if step == 4:
            ids[-1] = (ids[-1] + 1) % tokens  # the fork goes its own way
        for text, row, i, out in zip(texts, seen, ids.tolist(), last):
            text.append(i)
            row.append(out)
        last = model.step(ids, pool, table)
    worst = 0.0
    for text, row in zip(texts, seen):
        whole = model(torch.tensor(text, device=device)[None])[0]
        at = len(text) - len(row) - 1
        got, want = torch.stack(row).float(), whole[at:at + len(row)].float()
        worst = max(worst, float((got - want).abs().max() / want.abs().max()))
    return worst


def main(device: str = "cuda", steps: int = 150) -> tuple[float, float, float]:
    torch.manual_seed(0)
    tokens = 24
    model = Model(tokens, width=64, heads=4, d_key=32, d_value=32).to(device)
    first, last = train(model, tokens, steps, device)
    print(f"training: loss {first:.3f} -> {last:.3f} in {steps} steps")
    off = serve(model, tokens, device)
    print(f"serving: logits of single tokens within {off:.1e} of one pass over the whole sequences")
    return first, last, off


if __name__ == "__main__":
    main()
