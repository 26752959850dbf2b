"""The paged-cache operators where a cache, a table or an argument ends, against the plain forms in 64 bits."""

from __future__ import annotations

import ctypes

import pytest
import torch

import chroma_b200
from chroma_b200._src import native as nat
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


class Pages(ctypes.Structure):  # chroma_b200_pages
    _fields_ = [(x, ctypes.c_void_p) for x in ("keys", "values", "table", "lengths")] + [
        ("key_strides", ctypes.c_int64 * 4), ("value_strides", ctypes.c_int64 * 4), ("table_stride", ctypes.c_int64)] + [
        (x, ctypes.c_int32) for x in ("storage", "layers", "pages", "page_rows", "kv_heads", "head_dim", "slots", "width")]


class Attention(ctypes.Structure):  # chroma_b200_attention
    _fields_ = [(x, ctypes.c_void_p) for x in ("q", "out", "lse", "sinks", "starts", "workspace")] + [
        ("workspace_bytes", ctypes.c_int64), ("q_strides", ctypes.c_int64 * 2), ("out_strides", ctypes.c_int64 * 2)] + [
        (x, ctypes.c_int32) for x in ("tokens", "heads", "sinks_fp32", "window", "first")] + [("scale", ctypes.c_float)]


def pages_struct(keys, values, table, lengths):  # type: ignore[no-untyped-def]
    strides = [(ctypes.c_int64 * 4)(*([0] * (5 - x.dim())), *x.stride()[:-1]) for x in (keys, values)]
    return Pages(keys.data_ptr(), values.data_ptr(), table.data_ptr(), lengths.data_ptr(), *strides, table.stride(0),
                 int(keys.dtype is B16), *([1] * (5 - keys.dim())), *keys.shape, *table.shape)


def test_falling_starts_stay_within_the_workspace(gpu) -> None:  # type: ignore[no-untyped-def]
    # Rows that are given to many slots at once: more tiles than the workspace has room for. Their results mean nothing,
    # but nothing outside of the call's memory is written.
    slots, tokens, page, width = 40, 2560, 64, 20
    k, v, table, n = cache([200] * slots, dtype=B16, kv=1, dim=64, page=page, width=width)
    starts = torch.tensor([0, tokens] * (slots // 2) + [0], dtype=torch.int32).cuda()
    q = queries(tokens, 1, 64, B16)
    out = torch.zeros_like(q)
    p = pages_struct(k, v, table, n)
    g = Attention(q.data_ptr(), out.data_ptr(), None, None, starts.data_ptr(), None, 0, (ctypes.c_int64 * 2)(64, 64),
                  (ctypes.c_int64 * 2)(64, 64), tokens, 1, 0, 0, 0, 0.125)
    g.workspace_bytes = need = nat.lib().chroma_b200_attention_workspace(ctypes.byref(p), ctypes.byref(g))
    assert need > 0
    room = torch.full((need + (64 << 20),), 123, dtype=torch.uint8, device="cuda")
    g.workspace = room.data_ptr()
    nat.call("chroma_b200_paged_attention", ctypes.byref(p), ctypes.byref(g), torch.cuda.current_stream().cuda_stream)
    assert bool((room[need:] == 123).all())
    chroma_b200.check_operators()
    # the same rows, each with one slot
    starts = torch.tensor([0] + [tokens] * slots, dtype=torch.int32).cuda()
    n[0] = 1270
    chroma_b200.paged_attention(q, k, v, table, n, starts)
    rise = torch.arange(slots + 1, dtype=torch.int32).cuda() * (tokens // slots)
    want = ref.attention(q, k, v, table, n, rise, scale=0.125)
    check(chroma_b200.paged_attention(q, k, v, table, n, rise), want, dtype=B16, dim=64)
