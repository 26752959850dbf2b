"""The operators together, as examples/paged_generation.py uses them, against the model's own forward pass."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import chroma_b200
from chroma_b200 import models
from examples.paged_generation import PagedModel, generate

pytestmark = pytest.mark.gpu


def small(dtype=torch.float32, **more):  # type: ignore[no-untyped-def]
    config = dataclasses.replace(models.dev, num_hidden_layers=3, vocab_size=3000, sliding_window=9, **more)
    return models.random_transformer(config, seed=4, std=0.06, dtype=dtype)


def greedy(model, prompt, steps):  # type: ignore[no-untyped-def]
    tokens = prompt.tolist()
    with torch.no_grad():
        for _ in range(steps):
            tokens.append(int(model(torch.tensor(tokens))[-1].float().argmax()))
    return tokens[len(prompt) :]


def test_samples_follow_the_model(gpu: None) -> None:
    prompt = torch.randint(3000, (37,), generator=torch.Generator().manual_seed(2))
    want = greedy(small(), prompt, 12)
    repetition = torch.tensor([1.0, 1.3, 1.0, 1.1], device="cuda")
    ids, pages = generate(small(), prompt, 4, 12, repetition=repetition, page=8)
    assert ids[0].tolist() == want and ids[2].tolist() == want
    # 37 rows are 5 pages; three of four samples copy the fifth when they first write into it.
    assert pages["after the fork: free, short, copied"] == [4 * 8 - 5 - 3, 0, 3]
    # two samples of 37 + 11 rows: 4 whole pages in common, 2 each of their own
    assert pages["every other sample dropped: free, short, copied"] == [4 * 8 - 8, 0, 0]
    assert pages["compacted: held, moved"][0] == 8


def test_logits_of_ragged_chunks_match_the_forward_pass(gpu: None) -> None:
    model, g = small(), torch.Generator().manual_seed(6)
    rows = [torch.randint(3000, (n,), generator=g) for n in (40, 3, 17)]
    with torch.no_grad():
        want = [model(r) for r in rows]
    paged = PagedModel(model, slots=3, pages=40, page=4, width=12)
    own = torch.arange(3, dtype=torch.int32).cuda()
    cuts = [(0, 25, 30, 39, 40), (0, 1, 1, 2, 3), (0, 9, 16, 16, 17)]
    for part in range(4):
        counts = [c[part + 1] - c[part] for c in cuts]
        assert paged.reserve(own, torch.tensor(counts, dtype=torch.int32).cuda()).tolist()[1:] == [0, 0]
        tokens = torch.cat([r[c[part] : c[part + 1]] for r, c in zip(rows, cuts)]).cuda()
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()
        logits = paged.forward(tokens, starts).cpu()
        for b, c in enumerate(cuts):
            if counts[b]:
                np.testing.assert_allclose(logits[b], want[b][c[part + 1] - 1], rtol=1e-4, atol=1e-4)
    chroma_b200.check_operators()


def test_bf16_model(gpu: None) -> None:
    # 64-wide heads in bf16 take the tensor-core kernels; the plain forward pass rounds at the same places but one (its
    # softmax weights are rounded once more), so logits agree to a few units of bf16 at their own scale.
    model = small(torch.bfloat16, head_dim=64, num_attention_heads=16, num_key_value_heads=2)
    rows = torch.randint(3000, (150,), generator=torch.Generator().manual_seed(3))
    paged = PagedModel(model, slots=1, pages=20, page=16, width=12)
    own = torch.zeros(1, dtype=torch.int32).cuda()
    paged.reserve(own, own + 149)
    first = paged.forward(rows[:149].cuda(), torch.tensor([0, 149], dtype=torch.int32).cuda())
    paged.reserve(own, own + 1)
    second = paged.forward(rows[149:].cuda())
    with torch.no_grad(), torch.device("cuda"):
        want = model(rows.cuda())[148:].float()
    got = torch.cat([first, second]).float()
    scale = float(want.abs().max())
    assert float((got - want).abs().max()) <= 0.04 * scale
