"""The paged-cache operators on the GPU against plain forms in 64 bits (``tests/paged_reference.py``)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import chroma_b200
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

F32, B16 = torch.float32, torch.bfloat16


def cache(lengths, *, dtype, kv, dim, page, width=None, spare=3, seed=0, poison=True, layers=None):  # type: ignore[no-untyped-def]
    """A pool with pages in random order. Rows and pages that no sequence holds are NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    width = width or max(max(held), 1) + 1
    shape = (pages, page, kv, dim) if layers is None else (layers, pages, page, kv, dim)
    keys, values = (torch.randn(*shape, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table = np.full((len(lengths), width), -1, np.int64)
    at, used = 0, torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for m in range(held[b]):
            table[b, m] = order[at]
            used[order[at], : min(page, n - m * page)] = True
            at += 1
        table[b, held[b] :] = 2**30 if b % 2 else -1  # what lies past the held pages names no page
    if poison:
        gone = ~used.cuda()
        for pool in (keys, values):
            (pool if layers is None else pool.movedim(0, 2))[gone] = float("nan")
    return keys, values, torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


def check(got, want, *, dtype, dim, lse=None):  # type: ignore[no-untyped-def]
    out, logs, most_value, most_score = want
    a, r, e = ref.attention_tolerance(dtype, dim, most_value, most_score)
    np.testing.assert_allclose(got.double().cpu().numpy(), out.numpy(), atol=a, rtol=r)
    if lse is not None:
        np.testing.assert_allclose(lse.double().cpu().numpy(), logs.numpy(), atol=e, rtol=2.0**-20)


def queries(tokens, heads, dim, dtype, seed=1):  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g, device="cuda") * 1.5).to(dtype)


def sink_values(heads, dtype):  # type: ignore[no-untyped-def]
    return torch.linspace(-2, 3, heads, device="cuda").to(dtype)


DECODE = [
    # dtype, heads, kv, dim, page, lengths, window, first, sinks
    (F32, 8, 1, 16, 16, [160], 0, 0, True),
    (F32, 8, 1, 16, 4, [1, 0, 3, 4, 5, 16, 17], 0, 0, False),
    (F32, 6, 2, 20, 7, [64, 63, 65, 0, 1, 200], 10, 2, True),
    (F32, 12, 3, 128, 32, [300, 31, 32, 33], 0, 0, False),
    (F32, 40, 1, 64, 48, [97, 1000], 100, 0, True),
    (B16, 64, 8, 64, 64, [1, 63, 64, 65, 129, 1000], 0, 0, True),
    (B16, 8, 1, 16, 16, [0, 1, 15, 16, 17, 33], 0, 0, False),
    (B16, 32, 8, 128, 32, [2000, 31, 5], 0, 0, True),
    (B16, 5, 5, 80, 24, [77, 24, 25, 500], 0, 0, True),
    (B16, 21, 3, 64, 5, [100, 1, 0, 401], 0, 0, False),
    (B16, 64, 8, 64, 16, [500, 128, 127, 129, 130, 3], 128, 0, True),
    (B16, 16, 2, 128, 16, [900, 20, 21, 4], 17, 4, False),
    (B16, 24, 1, 64, 128, [300, 5], 1, 3, True),
    (B16, 64, 1, 128, 1, [150, 3], 50, 60, False),
    (B16, 4, 4, 8, 16, [40], 0, 0, True),
    (B16, 8, 2, 104, 16, [333, 2], 100, 9, True),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,lengths,window,first,sinks", DECODE)
def test_single_tokens(gpu, dtype, heads, kv, dim, page, lengths, window, first, sinks) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    q = queries(len(lengths), heads, dim, dtype)
    s = sink_values(heads, dtype) if sinks else None
    want = ref.attention(q, k, v, table, n, scale=dim**-0.5, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=dtype, dim=dim, lse=logs)
    again = chroma_b200.paged_attention(q, k, v, table, n, scale=dim**-0.5, window=window, first=first, sinks=s)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype,heads,kv,dim,page,window,first", [
    (B16, 32, 4, 64, 64, 0, 0), (B16, 16, 8, 128, 48, 0, 0), (B16, 64, 8, 64, 16, 4097, 5), (B16, 8, 1, 128, 16, 0, 0),
    (F32, 8, 1, 16, 16, 0, 0), (F32, 16, 2, 64, 32, 3000, 4),
])
def test_long_caches_are_split_and_joined(gpu, dtype, heads, kv, dim, page, window, first) -> None:  # type: ignore[no-untyped-def]
    lengths = [20011, 1, 4096, 0, 7777]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    q = queries(len(lengths), heads, dim, dtype)
    s = sink_values(heads, F32)
    want = ref.attention(q, k, v, table, n, scale=0.2, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, scale=0.2, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=dtype, dim=dim, lse=logs)
    assert torch.equal(chroma_b200.paged_attention(q, k, v, table, n, scale=0.2, window=window, first=first, sinks=s), got)


def test_many_sequences(gpu) -> None:  # type: ignore[no-untyped-def]
    lengths = [(i * 37) % 90 for i in range(700)]
    k, v, table, n = cache(lengths, dtype=B16, kv=2, dim=64, page=16)
    q = queries(len(lengths), 6, 64, B16)
    want = ref.attention(q, k, v, table, n, scale=0.125)
    check(chroma_b200.paged_attention(q, k, v, table, n), want, dtype=B16, dim=64)


PROMPT = [
    # dtype, heads, kv, dim, page, new rows, prior rows, window, first, sinks
    (F32, 8, 1, 16, 16, [61, 5, 30], [37, 37, 37], 0, 0, True),
    (F32, 6, 2, 20, 7, [1, 0, 64, 65, 130], [0, 9, 200, 0, 3], 10, 2, True),
    (F32, 4, 1, 128, 32, [200, 3], [0, 100], 0, 0, False),
    (B16, 64, 8, 64, 64, [128, 127, 1, 0, 130], [0, 0, 500, 3, 64], 0, 0, True),
    (B16, 8, 1, 16, 16, [300, 1], [0, 0], 0, 0, True),
    (B16, 32, 8, 128, 32, [260, 33], [0, 1000], 0, 0, False),
    (B16, 5, 5, 80, 24, [150, 2, 129], [0, 77, 1], 0, 0, True),
    (B16, 21, 3, 64, 5, [100, 1, 257], [401, 0, 30], 0, 0, False),
    (B16, 64, 8, 64, 16, [500, 40], [0, 300], 128, 0, True),
    (B16, 16, 2, 128, 16, [700, 9], [33, 900], 100, 4, False),
    (B16, 24, 1, 64, 128, [300, 5], [0, 0], 1, 3, True),
    (B16, 8, 8, 64, 1, [70], [130], 50, 60, False),
    (B16, 4, 4, 8, 16, [40, 41], [0, 500], 0, 0, True),
    (B16, 3, 1, 64, 64, [400], [1500], 333, 200, True),
    (B16, 200, 1, 64, 64, [9, 30], [100, 0], 0, 0, True),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,new,prior,window,first,sinks", PROMPT)
def test_prompts(gpu, dtype, heads, kv, dim, page, new, prior, window, first, sinks) -> None:  # type: ignore[no-untyped-def]
    lengths = [a + b for a, b in zip(new, prior)]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    q = queries(sum(new), heads, dim, dtype)
    s = sink_values(heads, dtype) if sinks else None
    want = ref.attention(q, k, v, table, n, starts, scale=dim**-0.5, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=dtype, dim=dim, lse=logs)
    assert torch.equal(chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s), got)


@pytest.mark.parametrize("dtype", [F32, B16])
def test_short_chunk_after_a_long_cache(gpu, dtype) -> None:  # type: ignore[no-untyped-def]
    new, prior = [4, 17], [9000, 21000]
    k, v, table, n = cache([a + b for a, b in zip(new, prior)], dtype=dtype, kv=2, dim=64, page=32)
    starts = torch.tensor([0, 4, 21], dtype=torch.int32).cuda()
    q = queries(21, 16, 64, dtype)
    want = ref.attention(q, k, v, table, n, starts, scale=0.125)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, lse=True)
    check(got, want, dtype=dtype, dim=64, lse=logs)


@pytest.mark.parametrize("heads,kv,dim,page,window,first,sinks", [
    (8, 1, 64, 16, 0, 0, True), (8, 2, 128, 48, 0, 0, False), (6, 2, 80, 5, 3000, 300, True), (16, 1, 64, 64, 200, 0, False),
])
def test_split_prompts(gpu, heads, kv, dim, page, window, first, sinks) -> None:  # type: ignore[no-untyped-def]
    # Few rows and many keys: the keys are split. Slots without new rows, with nothing held before, and with nothing to see.
    new, prior = [5, 0, 40, 1], [7001, 300, 2500, 0]
    k, v, table, n = cache([a + b for a, b in zip(new, prior)], dtype=B16, kv=kv, dim=dim, page=page)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    q = queries(sum(new), heads, dim, B16)
    s = sink_values(heads, F32) if sinks else None
    n[3] = 0  # a token that is at no position
    want = ref.attention(q, k, v, table, n, starts, scale=dim**-0.5, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=B16, dim=dim, lse=logs)
    assert torch.equal(chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s), got)
    # a value that is not finite where only the later of a tile's tokens see it
    k[table[2, 2520 // page].item(), 2520 % page] = float("nan")
    again = chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s)
    assert torch.equal(again[:25], got[:25]) and bool(again[25].isnan().any())


@pytest.mark.parametrize("dtype,heads,kv,dim", [(F32, 4, 2, 16), (B16, 8, 2, 64), (B16, 4, 1, 128)])
def test_non_finite_rows_reach_only_those_who_see_them(gpu, dtype, heads, kv, dim) -> None:  # type: ignore[no-untyped-def]
    new, prior, page = 150, 20, 16
    k, v, table, n = cache([new + prior], dtype=dtype, kv=kv, dim=dim, page=page)
    starts = torch.tensor([0, new], dtype=torch.int32).cuda()
    bad = {40: float("inf"), 101: float("nan")}  # positions; the first with a window that loses sight of it
    clean = [x.clone() for x in (k, v)]
    for p, x in bad.items():
        k[table[0, p // page].item(), p % page] = x
        v[table[0, p // page].item(), p % page] = -x
    q = queries(new, heads, dim, dtype)
    want = ref.attention(q, *clean, table, n, starts, scale=dim**-0.5, window=30)
    got = chroma_b200.paged_attention(q, k, v, table, n, starts, window=30).double().cpu()
    seen = torch.zeros(new, dtype=torch.bool)
    for p in bad:
        at = torch.arange(new) + prior
        seen |= (at >= p) & (at - p < 30)
    a, r, _ = ref.attention_tolerance(dtype, dim, want[2], want[3])
    np.testing.assert_allclose(got[~seen].numpy(), want[0][~seen].numpy(), atol=a, rtol=r)
    # single tokens after the rows have left the window
    n2 = torch.tensor([140], dtype=torch.int32).cuda()
    want = ref.attention(q[:1], *clean, table, n2, scale=dim**-0.5, window=30)
    check(chroma_b200.paged_attention(q[:1], k, v, table, n2, window=30), want, dtype=dtype, dim=dim)


@pytest.mark.parametrize("dtype", [F32, B16])
@pytest.mark.parametrize("prompt", [False, True])
def test_strided_pools_and_queries(gpu, dtype, prompt) -> None:  # type: ignore[no-untyped-def]
    kv, dim, page, lengths = 4, 64, 16, [50, 17, 3]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    both = torch.stack([k, v], 1).transpose(2, 3).contiguous().transpose(2, 3)  # [pages, 2, page, kv, dim], heads first
    wide = torch.zeros(3, 9, device="cuda", dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    starts = torch.tensor([0, 10, 11, 14], dtype=torch.int32).cuda() if prompt else None
    rows = 14 if prompt else 3
    qkv = queries(rows, 8 + 2 * kv, dim, dtype)
    q = qkv[:, :8]
    want = ref.attention(q, k, v, table, n, starts, scale=0.125)
    check(chroma_b200.paged_attention(q, both[:, 0], both[:, 1], wide[:, : table.shape[1]], n, starts), want,
          dtype=dtype, dim=dim)
    # rows that start at any element, heads in another order, an output that is part of a larger one
    odd = torch.empty(rows * 8 * dim + 1, device="cuda", dtype=dtype)[1:].view(rows, 8, dim).copy_(q)
    out = torch.full((rows, 9, dim + 3), 7.0, device="cuda", dtype=dtype)
    got = chroma_b200.paged_attention(odd, both[:, 0], both[:, 1], wide[:, : table.shape[1]], n, starts, out=out[:, :8, 1 : dim + 1])
    check(got, want, dtype=dtype, dim=dim)
    assert bool((out[:, 8] == 7).all()) and bool((out[:, :, 0] == 7).all()) and bool((out[:, :, dim + 1 :] == 7).all())
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    check(chroma_b200.paged_attention(turned, k, v, table, n, starts), want, dtype=dtype, dim=dim)


def test_pages_beyond_32_bit_offsets(gpu) -> None:  # type: ignore[no-untyped-def]
    # 2.3e9 elements per pool: the last pages lie past 2^31 elements and 2^32 bytes.
    kv, dim, page, pages = 8, 64, 64, 70000
    k = torch.empty(pages, page, kv, dim, dtype=B16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[69999, 1, 68000], [69998, 69997, -1]], dtype=torch.int32).cuda()
    n = torch.tensor([140, 100], dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    starts = torch.tensor([0, 140, 240], dtype=torch.int32).cuda()
    new = [torch.randn(240, kv, dim, generator=g, device="cuda", dtype=B16) for _ in range(2)]
    chroma_b200.paged_append(k, v, *new, table, n, starts)
    order = torch.tensor([69999, 1, 68000, 69998, 69997]).cuda()
    small = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32).cuda()
    ks, vs = k[order], v[order]
    q = queries(240, 16, dim, B16)
    want = ref.attention(q[:2], ks, vs, small, n, scale=0.125)
    check(chroma_b200.paged_attention(q[:2].contiguous(), k, v, table, n), want, dtype=B16, dim=dim)
    want = ref.attention(q, ks, vs, small, n, starts, scale=0.125)
    check(chroma_b200.paged_attention(q, k, v, table, n, starts), want, dtype=B16, dim=dim)
    parents, counts = torch.tensor([0, 0], dtype=torch.int32).cuda(), torch.tensor([1, 1], dtype=torch.int32).cuda()
    moved, _, info = chroma_b200.step_pages(table, n, parents, counts, k, v)
    assert info.tolist() == [pages - 4, 0, 1] and moved.tolist() == [[69999, 1, 68000], [69999, 1, 0]]
    assert torch.equal(k[0, :12], k[68000, :12]) and torch.equal(v[0, :12], v[68000, :12])
    packed, info = chroma_b200.compact_pages(table, n, k, v)
    assert info.tolist() == [5, 4] and packed.tolist() == [[4, 1, 0], [3, 2, -1]]
    assert torch.equal(k[4], ks[0]) and torch.equal(v[3, :36], vs[3, :36])


@pytest.mark.parametrize("dtype,kv,dim,page", [(B16, 8, 64, 64), (F32, 1, 16, 5), (B16, 3, 8, 1), (F32, 2, 100, 16)])
def test_append(gpu, dtype, kv, dim, page) -> None:  # type: ignore[no-untyped-def]
    new, prior = [3, 0, 1, 70, 16], [0, 5, 15, 9, 16]
    lengths = [a + b for a, b in zip(new, prior)]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    table[3, 1] = -1  # a page that is not there: its rows are dropped
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = torch.randn(sum(new), 2 * kv, dim, generator=g, device="cuda").to(dtype)
    unaligned = torch.empty(rows.numel() + 1, device="cuda", dtype=dtype)[1:].view(rows.shape).copy_(rows)
    for source in (rows, unaligned):
        nk, nv = source[:, :kv], source[:, kv:]
        want_k, want_v = k.clone(), v.clone()
        for b in range(len(new)):
            for i in range(new[b]):
                p = prior[b] + i
                id = int(table[b, p // page])
                if id >= 0:
                    want_k[id, p % page], want_v[id, p % page] = nk[int(starts[b]) + i], nv[int(starts[b]) + i]
        got_k, got_v = k.clone(), v.clone()
        chroma_b200.paged_append(got_k, got_v, nk, nv, table, n, starts)
        assert torch.equal(got_k.nan_to_num(9), want_k.nan_to_num(9))
        assert torch.equal(got_v.nan_to_num(9), want_v.nan_to_num(9))
    # one row per slot; a slot that holds nothing drops its row
    n[1] = 0
    nk, nv = rows[:5, :kv], rows[:5, kv:]
    want_k = k.clone()
    for b in range(5):
        p = int(n[b]) - 1
        if p >= 0 and int(table[b, p // page]) >= 0:
            want_k[int(table[b, p // page]), p % page] = nk[b]
    chroma_b200.paged_append(k, v, nk, nv, table, n)
    assert torch.equal(k.nan_to_num(9), want_k.nan_to_num(9))


def pools(layers, pages, page, kv, dim, dtype, seed):  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(layers, pages, page, kv, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]


def moved(pool, copies):  # type: ignore[no-untyped-def]
    want = pool.clone()
    for a, b, rows in copies:
        want[:, b, :rows] = pool[:, a, :rows]
    return want


@pytest.mark.parametrize("slots,width,pages,page,layers,seed", [
    (1, 1, 1, 1, 1, 0), (2, 3, 7, 4, 2, 1), (9, 12, 60, 16, 3, 2), (33, 40, 900, 5, 1, 3), (300, 9, 1500, 64, 1, 4),
    (1100, 3, 5000, 2, 1, 5), (64, 300, 9000, 16, 1, 6),
])
def test_steps_of_sequences(gpu, slots, width, pages, page, layers, seed) -> None:  # type: ignore[no-untyped-def]
    rng = np.random.default_rng(seed)
    k, v = pools(layers, pages, page, 2, 16, B16, seed)
    table = torch.full((slots, width), -1, dtype=torch.int32).cuda()
    lengths = torch.zeros(slots, dtype=torch.int32).cuda()
    parents = np.arange(slots)
    seen_copies = seen_short = 0
    for turn in range(12):
        counts = rng.integers(0, max(2, width * page // 6), slots) * (rng.random(slots) < 0.7)
        if turn:
            parents = np.where(rng.random(slots) < 0.6, np.arange(slots), rng.integers(-1, slots + 1, slots))
        if turn == 8:
            counts[0] = width * page + 100  # cut at the table's end
        t, n = table.cpu().numpy(), lengths.cpu().numpy()
        want, want_n, info, copies = ref.step(t, n, parents, counts, pages, page)
        wk, wv = moved(k, copies), moved(v, copies)
        args = [torch.tensor(x, dtype=torch.int32).cuda() for x in (parents, counts)]
        before = table.clone()
        new_table, new_lengths, got = chroma_b200.step_pages(table, lengths, *args, k, v)
        assert got.tolist() == info
        assert torch.equal(table, before)
        np.testing.assert_array_equal(new_lengths.cpu().numpy(), want_n)
        np.testing.assert_array_equal(new_table.cpu().numpy(), want)
        assert torch.equal(k, wk) and torch.equal(v, wv)
        seen_copies, seen_short = seen_copies + info[2], seen_short + info[1]
        if info[1]:
            parents = np.where(np.arange(slots) % 2, -1, np.arange(slots))  # tried again with half of them
            args = [torch.tensor(x, dtype=torch.int32).cuda() for x in (parents, counts * 0)]
            new_table, new_lengths, got = chroma_b200.step_pages(table, lengths, *args, k, v)
            assert got.tolist()[1:] == [0, 0]
        table, lengths = new_table, new_lengths
        if turn % 4 == 3:
            want, info, copies = ref.compact(table.cpu().numpy(), lengths.cpu().numpy(), pages, page)
            wk, wv = moved(k, copies), moved(v, copies)
            table, got = chroma_b200.compact_pages(table, lengths, k, v)
            assert got.tolist() == info
            np.testing.assert_array_equal(table.cpu().numpy(), want)
            assert torch.equal(k, wk) and torch.equal(v, wv)
    if slots >= 9:
        assert seen_copies


def test_pages_of_strided_pools(gpu) -> None:  # type: ignore[no-untyped-def]
    both = torch.randn(3, 10, 2, 4, 16, 24, device="cuda")  # layers, pages, k/v, heads, rows, dim
    k, v = both[:, :, 0].transpose(2, 3), both[:, :, 1].transpose(2, 3)
    table = torch.tensor([[7, 3], [9, 77]], dtype=torch.int32).cuda()
    lengths = torch.tensor([20, 16], dtype=torch.int32).cuda()
    parents, counts = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 0], [1, 2]))
    before = both.clone()
    new, n, info = chroma_b200.step_pages(table, lengths, parents, counts, k, v)
    assert new.tolist() == [[7, 3], [7, 0]] and n.tolist() == [21, 22] and info.tolist() == [7, 0, 1]
    before[:, 0, :, :, :4] = before[:, 3, :, :, :4]
    assert torch.equal(both, before)
    new, info = chroma_b200.compact_pages(table, lengths, k, v)
    assert new.tolist() == [[1, 0], [2, -1]] and info.tolist() == [3, 3]  # 3, 7, 9 to 0, 1, 2
    assert all(torch.equal(both[:, b], before[:, a]) for a, b in ((3, 0), (7, 1), (9, 2)))


def test_calls_follow_the_current_stream(gpu) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([3000, 200], dtype=B16, kv=2, dim=64, page=16)
    q = queries(2, 8, 64, B16)
    want = ref.attention(q, k, v, table, n, scale=0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        got = chroma_b200.paged_attention(late, k, v, table, n)
    side.synchronize()
    check(got, want, dtype=B16, dim=64)


def test_calls_can_be_captured(gpu) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([3000, 200, 0], dtype=B16, kv=2, dim=64, page=16)
    q = queries(3, 8, 64, B16)
    chroma_b200.paged_attention(q, k, v, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chroma_b200.paged_attention(q, k, v, table, n)
        tables = chroma_b200.compact_pages(table, n, k.unsqueeze(0), v.unsqueeze(0))
    q.copy_(queries(3, 8, 64, B16, seed=9))
    n.copy_(torch.tensor([100, 201, 0], dtype=torch.int32))
    want = ref.attention(q, k, v, table, n, scale=0.125)
    graph.replay()
    torch.cuda.synchronize()
    assert tables[1].tolist()[0] == 20
    check(out[0], (want[0][0], *want[1:]), dtype=B16, dim=64)


def test_refusals(gpu) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([20, 3], dtype=B16, kv=2, dim=64, page=16)
    q = queries(2, 8, 64, B16)
    call = chroma_b200.paged_attention
    starts = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    bad = [
        lambda: call(q.float(), k, v, table, n),
        lambda: call(q[:, :7], k, v, table, n),
        lambda: call(q[:1], k, v, table, n),
        lambda: call(q[..., :32], k, v, table, n),
        lambda: call(q, k, v.float(), table, n),
        lambda: call(q, k, v[:-1], table, n),
        lambda: call(q, k, v, table.long(), n),
        lambda: call(q, k, v, table, n.long()),
        lambda: call(q, k, v, table, n[:1]),
        lambda: call(q, k, v, table.t(), n),
        lambda: call(q, k.cpu(), v, table, n),
        lambda: call(q.cpu(), k, v, table, n),
        lambda: call(q, k, v, table, n, starts[:2]),
        lambda: call(q, k, v, table, n, window=-1),
        lambda: call(q, k, v, table, n, first=-1),
        lambda: call(q, k, v, table, n, sinks=torch.zeros(7, device="cuda")),
        lambda: call(q, k, v, table, n, out=torch.empty(2, 8, 64, device="cuda")),
        lambda: call(q.half(), k.half(), v.half(), table, n),
        lambda: call(q[..., ::2], k[..., ::2], v[..., ::2], table, n),
        lambda: call(q[..., :12].contiguous(), k[..., :12].contiguous(), v[..., :12].contiguous(), table, n),
        lambda: call(q[..., :60], k[..., 1:61], v[..., 1:61], table, n),
        lambda: call(torch.cat([q] * 3, 2), torch.cat([k] * 3, 3), torch.cat([v] * 3, 3), table, n),
        lambda: chroma_b200.paged_append(k, v, q[:, :2].float(), q[:, :2], table, n),
        lambda: chroma_b200.paged_append(k, v, q[:, :3], q[:, :3], table, n),
        lambda: chroma_b200.paged_append(k, v, q[:1, :2], q[:1, :2], table, n),
        lambda: chroma_b200.step_pages(table, n, n[:1], n, k, v),
        lambda: chroma_b200.step_pages(table, n, n, n.float(), k, v),
        lambda: chroma_b200.step_pages(table, n[:1], n, n, k, v),
        lambda: chroma_b200.compact_pages(table, n, k, v[:, :8]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was not refused")
    with pytest.raises(TypeError):
        call(q, k, v, table.tolist(), n)
    # no rows is no error
    empty = call(q[:0], k, v, table, n, torch.zeros(3, dtype=torch.int32).cuda())
    assert empty.shape == (0, 8, 64)
    check(call(q, k, v, table, n), ref.attention(q, k, v, table, n, scale=0.125), dtype=B16, dim=64)


@pytest.mark.parametrize("heads,kv,dim,page,window,first,sinks", [
    (8, 1, 64, 16, 0, 0, True), (8, 2, 128, 48, 0, 0, False), (6, 2, 80, 5, 3000, 300, True), (16, 1, 16, 64, 200, 0, False),
    (3, 1, 20, 32, 0, 0, True),
])
def test_shared_items_of_fp32_prompts(gpu, heads, kv, dim, page, window, first, sinks) -> None:  # type: ignore[no-untyped-def]
    # Few rows and many keys: CTAs of a cluster share each item. Items with tokens of several slots among them.
    new, prior = [5, 0, 10, 1], [7001, 300, 2500, 0]
    k, v, table, n = cache([a + b for a, b in zip(new, prior)], dtype=F32, kv=kv, dim=dim, page=page)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
    q = queries(sum(new), heads, dim, F32)
    s = sink_values(heads, F32) if sinks else None
    n[3] = 0  # a token that is at no position
    want = ref.attention(q, k, v, table, n, starts, scale=dim**-0.5, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=F32, dim=dim, lse=logs)
    assert torch.equal(chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=first, sinks=s), got)
