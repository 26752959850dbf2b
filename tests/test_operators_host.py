"""What the operators on CUDA tensors refuse before anything reaches a GPU (their binding loads without one)."""

from __future__ import annotations

import subprocess

import pytest
import torch

import chroma_b200
from chroma_b200 import build


def cache():  # type: ignore[no-untyped-def]
    pool = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    return pool, pool.clone(), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


def test_tensors_must_be_on_a_cuda_device() -> None:
    keys, values, table, lengths = cache()
    q = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
    calls = [lambda: chroma_b200.paged_attention(q, keys, values, table, lengths),
             lambda: chroma_b200.paged_append(keys, values, q[:, :2], q[:, :2], table, lengths),
             lambda: chroma_b200.step_pages(table, lengths, lengths, lengths, keys, values),
             lambda: chroma_b200.compact_pages(table, lengths, keys, values),
             lambda: chroma_b200.process_logits(torch.zeros(2, 5))]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_what_is_no_tensor_is_a_type_error() -> None:
    keys, values, table, lengths = cache()
    with pytest.raises(TypeError, match="q must be a tensor, not list"):
        chroma_b200.paged_attention([1], keys, values, table, lengths)
    with pytest.raises(TypeError, match="table must be a tensor"):
        chroma_b200.step_pages(None, lengths, lengths, lengths, keys, values)
    with pytest.raises(TypeError, match="mask must be a tensor"):
        chroma_b200.process_logits(torch.zeros(2, 5), mask=3)
    with pytest.raises(TypeError):
        chroma_b200.process_logits(torch.zeros(2, 5), masks=None)


def test_the_binding_shares_the_c_plus_plus_runtime_of_the_process() -> None:
    # A copy of the runtime inside the module crashes as soon as a message is put together.
    needed = subprocess.run(["readelf", "-d", str(build.TENSORS)], capture_output=True, text=True).stdout
    assert "libstdc++.so" in needed and "libtorch_python.so" in needed
