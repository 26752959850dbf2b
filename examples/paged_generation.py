"""Several continuations of one prompt, generated over a paged key-value cache.

    python examples/paged_generation.py [--samples 8] [--steps 32] [--prompt 200]

The prompt runs once; its pages are shared by all samples, which copy a page only when they write into it. Every sample
punishes repetition in its own way, so they part, and the choice of a token stays on the device. When half of the samples are
dropped, their pages come free, and what is left is moved to the front of the pool.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import chroma_b200  # noqa: E402
from chroma_b200 import models  # noqa: E402


class PagedModel:
    """A ``models.Transformer`` on the GPU with a paged cache for up to ``slots`` sequences."""

    def __init__(self, model: models.Transformer, *, slots: int, pages: int, page: int = 16, width: int = 64) -> None:
        self.model = model.cuda()
        first = model.block[0].attn
        shape = (len(model.block), pages, page, first.num_key_value_heads, first.head_dim)
        kind = first.qkv.weight.dtype
        self.keys, self.values = (torch.empty(shape, dtype=kind, device="cuda") for _ in range(2))
        self.table = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(slots, dtype=torch.int32, device="cuda")

    def reserve(self, parents: Tensor, counts: Tensor) -> Tensor:
        """Slot s goes on from slot ``parents[s]`` with ``counts[s]`` new rows; returns [pages free, short, copied]."""
        self.table, self.lengths, info = chroma_b200.step_pages(self.table, self.lengths, parents, counts, self.keys,
                                                                self.values, cut=False)
        return info

    def compact(self) -> Tensor:
        self.table, info = chroma_b200.compact_pages(self.table, self.lengths, self.keys, self.values)
        return info

    @torch.no_grad()
    def forward(self, tokens: Tensor, starts: Tensor | None = None) -> Tensor:
        """Logits of every slot's last token. ``tokens`` are the rows reserved last: one per slot, or slot b's at
        ``starts[b] : starts[b + 1]``."""
        model, slots = self.model, self.lengths.shape[0]
        if starts is None:
            positions, last = self.lengths - 1, torch.arange(slots, device="cuda")
        else:
            owner = torch.searchsorted(starts[1:], torch.arange(len(tokens), device="cuda"), right=True)
            positions = self.lengths[owner] - starts[owner + 1] + torch.arange(len(tokens), device="cuda")
            last = (starts[1:] - 1).clamp(min=0).long()
        with torch.device("cuda"):
            x = model.embedding(tokens)
            for layer, block in enumerate(model.block):
                attn = block.attn
                q, k, v = attn.project(x, positions.float())
                chroma_b200.paged_append(self.keys[layer], self.values[layer], k, v, self.table, self.lengths, starts)
                o = chroma_b200.paged_attention(
                    q.flatten(1, 2), self.keys[layer], self.values[layer], self.table, self.lengths, starts,
                    scale=attn.sm_scale, window=attn.sliding_window, sinks=attn.sinks)
                x = block.mlp(x + attn.out(o.flatten(1)))
            return model.unembedding(model.norm(x[last]))


def generate(model: models.Transformer, prompt: Tensor, samples: int, steps: int, *, repetition: Tensor,
             page: int = 16) -> tuple[Tensor, dict[str, list[int]]]:
    """Greedy continuations [samples, steps] of ``prompt``, one per entry of ``repetition``; and what became of pages."""
    total = len(prompt) + steps
    width = -(-total // page) + 1
    paged = PagedModel(model, slots=samples, pages=width * samples, page=page, width=width)

    def ints(values: list[int]) -> Tensor:
        return torch.tensor(values, dtype=torch.int32).cuda()

    # The prompt goes through slot 0 alone, then every slot goes on from it.
    own, none = ints(list(range(samples))), [0] * (samples - 1)
    paged.reserve(own, ints([len(prompt), *none]))
    logits = paged.forward(prompt.cuda(), ints([0, *([len(prompt)] * samples)]))[:1].expand(samples, -1).contiguous()
    history = torch.zeros(samples, total, dtype=torch.int32, device="cuda")
    history[:, : len(prompt)] = prompt.cuda()
    seen, said = ints([len(prompt)] * samples), ints([len(prompt)] * samples)
    seen_pages: dict[str, list[int]] = {}
    parents, ones = ints([0] * samples), ints([1] * samples)
    for step in range(steps):
        logits, ids = chroma_b200.process_logits(logits, history=history, lengths=seen, prompts=said,
                                                 repetition=repetition, argmax=True)
        history[:, len(prompt) + step] = ids
        seen += 1
        if step + 1 == steps:
            break
        info = paged.reserve(parents, ones)
        if step == 0:
            seen_pages["after the fork: free, short, copied"] = info.tolist()
        parents = own
        logits = paged.forward(ids)
    keep = ints([s if s % 2 == 0 else -1 for s in range(samples)])
    seen_pages["every other sample dropped: free, short, copied"] = paged.reserve(keep, ints([0] * samples)).tolist()
    seen_pages["compacted: held, moved"] = paged.compact().tolist()
    return history[:, len(prompt) :].long().cpu(), seen_pages


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--samples", type=int, default=8)
    parser.add_argument("--steps", type=int, default=32)
    parser.add_argument("--prompt", type=int, default=200)
    args = parser.parse_args()
    model = models.make_dev_model(0)
    prompt = torch.randint(models.dev.vocab_size, (args.prompt,), generator=torch.Generator().manual_seed(1))
    repetition = torch.linspace(1.0, 1.5, args.samples).cuda()
    ids, pages = generate(model, prompt, args.samples, args.steps, repetition=repetition)
    for what, counts in pages.items():
        print(f"{what}: {counts}")
    for row, penalty in zip(ids.tolist(), repetition.tolist()):
        print(f"repetition {penalty:.2f}: {row[:12]}{' ...' if len(row) > 12 else ''}")


if __name__ == "__main__":
    main()
