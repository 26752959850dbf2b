"""The paged-cache operators where a cache, a table or an argument ends, against the plain forms in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import chroma_b200
from tests import paged_reference as ref
from tests.test_gpu_paged import B16, F32, cache, check, queries, sink_values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,page,lengths,window,first,sinks", [
    (8, 1, 16, [16, 31, 32, 33, 500], 0, 0, True), (32, 2, 64, [3000, 1, 64], 0, 0, False),
    (3, 3, 5, [40, 41], 0, 0, True), (8, 2, 32, [700, 96], 100, 20, False),
])
def test_rows_of_32_values_at_the_end_of_the_pool(gpu, heads, kv, page, lengths, window, first, sinks) -> None:  # type: ignore[no-untyped-def]
    # Every page of the pool is in use, the last row of it too. Both pools are the first halves of larger tensors.
    k, v, table, n = cache(lengths, dtype=B16, kv=kv, dim=32, page=page, spare=0, poison=False)
    halves = [torch.full((2 * len(x), *x.shape[1:]), float("nan"), dtype=B16, device="cuda") for x in (k, v)]
    for half, x in zip(halves, (k, v)):
        half[: len(x)] = x
    q = queries(len(lengths), heads, 32, B16)
    s = sink_values(heads, B16) if sinks else None
    want = ref.attention(q, k, v, table, n, scale=32**-0.5, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, halves[0][: len(k)], halves[1][: len(v)], table, n, window=window, first=first,
                                            sinks=s, lse=True)
    check(got, want, dtype=B16, dim=32, lse=logs)
