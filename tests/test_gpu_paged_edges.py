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


# ---- lengths past the end of the table: such positions have no page, and move no other

@pytest.mark.parametrize("dtype,kv,dim,page", [(B16, 8, 64, 64), (F32, 1, 16, 5), (B16, 3, 8, 1)])
@pytest.mark.parametrize("slots", [6, 300])
def test_rows_past_the_table_are_dropped(gpu, dtype, kv, dim, page, slots) -> None:  # type: ignore[no-untyped-def]
    end = 2 * page  # positions of a slot
    k, v, table, _ = cache([end] * slots, dtype=dtype, kv=kv, dim=dim, page=page, width=2, spare=0)
    new = [(2, 1, 3, 0, 1, 4)[s % 6] for s in range(slots)]
    lengths = [(end, end + 1, end + 2, end + 9, 2**31 - 1, end + 5)[s % 6] for s in range(slots)]
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    starts = torch.tensor([sum(new[:s]) for s in range(slots + 1)], dtype=torch.int32).cuda()
    rows = torch.randn(sum(new), 2 * kv, dim, device="cuda").to(dtype)
    for given in (starts, None):
        nk, nv = (rows[:, :kv], rows[:, kv:]) if given is not None else (rows[:slots, :kv], rows[:slots, kv:])
        want_k, want_v = k.clone(), v.clone()
        at = 0
        for s in range(slots):
            count = new[s] if given is not None else 1
            for i in range(count):
                p = lengths[s] - count + i
                if p < end:
                    want_k[table[s, p // page], p % page], want_v[table[s, p // page], p % page] = nk[at + i], nv[at + i]
            at += count
        got_k, got_v = k.clone(), v.clone()
        chroma_b200.paged_append(got_k, got_v, nk, nv, table, n, given)
        assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [
    (F32, 8, 1, 16, 7), (F32, 4, 2, 64, 16), (B16, 16, 2, 64, 16), (B16, 8, 8, 128, 48), (B16, 6, 2, 80, 24),
    (B16, 4, 1, 32, 5), (B16, 64, 8, 64, 64),
])
@pytest.mark.parametrize("window,first", [(0, 0), (10, 0), (40, 3), (40, 500), (3, 20)])
@pytest.mark.parametrize("prompt", [False, True])
def test_tokens_past_the_table_are_at_their_positions(gpu, dtype, heads, kv, dim, page, window, first, prompt) -> None:  # type: ignore[no-untyped-def]
    end = 4 * page
    k, v, table, _ = cache([end] * 6, dtype=dtype, kv=kv, dim=dim, page=page, width=4, spare=0)
    lengths, new = [end + 3, end - 1, end + 30, end + 12, end + 700, end], [5, 3, 70, 12, 1, 9]
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    starts = torch.tensor([sum(new[:s]) for s in range(7)], dtype=torch.int32).cuda() if prompt else None
    q = queries(sum(new) if prompt else 6, heads, dim, dtype)
    s = sink_values(heads, F32)
    # the same in a table that is wide enough to name those positions, and names no page there
    wide = torch.cat([table, torch.full((6, 700 // page + 1), -1, dtype=torch.int32, device="cuda")], 1)
    want = ref.attention(q, k, v, wide, n, starts, scale=0.2, window=window, first=first, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, scale=0.2, window=window, first=first, sinks=s, lse=True)
    check(got, want, dtype=dtype, dim=dim, lse=logs)
    # a length as large as there are: what is left is the first tokens, or everything where there is no window
    n.fill_(2**31 - 1)
    seen = torch.full_like(n, min(first, end) if window else end)
    want = ref.attention(q[:6], k, v, table, seen, scale=0.2, sinks=s)
    far = torch.arange(7, dtype=torch.int32).cuda() if prompt else None
    got = chroma_b200.paged_attention(q[:6], k, v, table, n, far, scale=0.2, window=window, first=first, sinks=s)
    check(got, want, dtype=dtype, dim=dim)


def test_long_caches_past_the_table(gpu) -> None:  # type: ignore[no-untyped-def]
    # Cut and joined, or split; the tokens lie in the window's reach behind the end.
    for dtype, dim, heads in ((B16, 64, 16), (B16, 128, 8), (F32, 64, 8)):
        k, v, table, _ = cache([4096, 4096], dtype=dtype, kv=2, dim=dim, page=16, width=256)
        wide = torch.cat([table, torch.full((2, 64), -1, dtype=torch.int32, device="cuda")], 1)
        n = torch.tensor([4096 + 500, 4096 + 20], dtype=torch.int32).cuda()
        for starts in (None, torch.tensor([0, 3, 23], dtype=torch.int32).cuda()):
            q = queries(23 if starts is not None else 2, heads, dim, dtype)
            for window in (0, 3000, 400):
                want = ref.attention(q, k, v, wide, n, starts, scale=0.2, window=window, first=window // 300)
                got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, scale=0.2, window=window, first=window // 300, lse=True)
                check(got, want, dtype=dtype, dim=dim, lse=logs)


@pytest.mark.parametrize("slots,width,page", [(4, 3, 4), (70, 1000, 2)])  # decided by one CTA, and by several launches
def test_steps_past_the_table_write_over_nothing(gpu, slots, width, page) -> None:  # type: ignore[no-untyped-def]
    end = width * page
    lengths = [end, end - 1, 0, 2] + [0] * (slots - 4)
    k, v, table, n = cache(lengths, dtype=F32, kv=1, dim=16, page=page, width=width, spare=9, poison=False)
    ints = lambda x: torch.tensor(x + [-1] * (slots - len(x)), dtype=torch.int32).cuda()  # noqa: E731
    # A full sequence is forked, one that is full but for a row goes on by three.
    parents, counts = ints([0, 1, 0, 3]), ints([1, 3, 2, 1])
    want, _, info, copies = ref.step(table.cpu().numpy(), n.cpu().numpy(), parents.tolist(), counts.tolist(), len(k), page)
    before = k.clone()
    new, length, got = chroma_b200.step_pages(table, n, parents, counts, k[None], v[None], cut=False)
    assert new.tolist() == want.tolist() and got.tolist() == info
    assert length.tolist() == [end + 1, end + 2, end + 2, 3] + [0] * (slots - 4)
    for a, b, rows in copies:
        before[b, :rows] = before[a, :rows]
    starts = torch.tensor([0, 1, 4, 6] + [7] * (slots - 3), dtype=torch.int32).cuda()
    rows = torch.randn(7, 1, 16, device="cuda")
    chroma_b200.paged_append(k, v, rows, rows, new, length, starts)
    before[new[1, width - 1], page - 1] = rows[1]
    before[new[3, 2 // page], 2 % page] = rows[6]
    assert torch.equal(k, before)
    # once more, from there; a length stays below 2^31
    new, length, got = chroma_b200.step_pages(new, length, ints([0, 0, 2, 3]), ints([5, 2**31 - 1, 0, 0]), k[None], v[None], cut=False)
    assert length.tolist() == [end + 6, 2**31 - 1, end + 2, 3] + [0] * (slots - 4) and got.tolist()[1:] == [0, 0]
    assert torch.equal(k, before)
    # cut at the end, as without the argument
    for more in ({}, {"cut": True}):
        assert chroma_b200.step_pages(new, length, ints([0, 1, 2, 3]), ints([5, 0, 0, 1]), k[None], v[None], **more)[1].tolist()[:4] == [end, end, end, 4]


# ---- values that are not finite

def agree(got, want, *, dtype, dim, scale_of):  # type: ignore[no-untyped-def]
    """Entries are finite where the 64-bit form's are, and then near them; ``scale_of``: the same without the bad values."""
    got, out = got.double().cpu(), want[0]
    fine = torch.isfinite(out)
    assert torch.equal(torch.isfinite(got), fine)
    a, r, _ = ref.attention_tolerance(dtype, dim, scale_of[2], scale_of[3])
    assert bool(((got - out)[fine].abs() <= a + r * out[fine].abs()).all())


BAD = [("k", 40, slice(None), float("nan")), ("v", 40, slice(None), float("nan")), ("v", 101, 3, float("inf")),
       ("v", 101, 9, float("nan")), ("v", 33, 3, float("-inf")), ("k", 130, slice(2, 5), float("inf")), ("v", 0, 1, float("nan"))]


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [(F32, 4, 2, 16, 16), (B16, 8, 2, 64, 16), (B16, 4, 1, 128, 24), (B16, 3, 1, 80, 5)])
@pytest.mark.parametrize("window,first", [(0, 0), (30, 0), (25, 2)])
@pytest.mark.parametrize("bad", [BAD[:1], BAD[1:2], BAD[2:3], BAD[2:5], BAD[5:], BAD], ids=range(6))
def test_rows_that_see_values_that_are_not_finite(gpu, dtype, heads, kv, dim, page, window, first, bad) -> None:  # type: ignore[no-untyped-def]
    new, prior = 150, 20
    k, v, table, n = cache([new + prior], dtype=dtype, kv=kv, dim=dim, page=page)
    starts = torch.tensor([0, new], dtype=torch.int32).cuda()
    q = queries(new, heads, dim, dtype)
    clean = ref.attention(q, k, v, table, n, starts, scale=0.2, window=window, first=first)
    for pool, p, d, x in bad:
        (k if pool == "k" else v)[table[0, p // page].item(), p % page, 0, d] = x
    want = ref.attention(q, k, v, table, n, starts, scale=0.2, window=window, first=first)
    got = chroma_b200.paged_attention(q, k, v, table, n, starts, scale=0.2, window=window, first=first)
    agree(got, want, dtype=dtype, dim=dim, scale_of=clean)
    for length in (35, 41, 103, 170):  # single tokens
        n[0] = length
        want = ref.attention(q[:1], k, v, table, n, scale=0.2, window=window, first=first)
        agree(chroma_b200.paged_attention(q[:1], k, v, table, n, scale=0.2, window=window, first=first), want, dtype=dtype, dim=dim, scale_of=clean)


@pytest.mark.parametrize("what", ["key", "value", "one entry", "late value"])
@pytest.mark.parametrize("heads,kv,dim,new", [(16, 8, 64, 600), (16, 8, 128, 600), (16, 2, 64, 20)])  # the last: keys are split
def test_bad_values_in_a_long_cache(gpu, what, heads, kv, dim, new) -> None:  # type: ignore[no-untyped-def]
    """Rows that see them are not finite, the others are as without them, and the call takes about as long."""
    prior, page, dtype = 6000, 16, B16
    k, v, table, n = cache([prior + new, new + 5], dtype=dtype, kv=kv, dim=dim, page=page)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda()
    q = queries(2 * new, heads, dim, dtype)

    def timed():  # type: ignore[no-untyped-def]
        times = []
        for _ in range(3):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            out = chroma_b200.paged_attention(q, k, v, table, n, starts)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return out, min(times)

    clean, usual = timed()
    p = 5 if what != "late value" else prior + new // 2
    entries = slice(None) if what in ("key", "value") else 7
    (k if what == "key" else v)[table[0, p // page], p % page, :, entries] = float("nan")
    got, longer = timed()
    chroma_b200.check_operators()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[max(0, p - prior) : new, :, entries] = True
    assert torch.equal(torch.isnan(got), hit)
    # rows that shared a tile with a bad value but do not see it were computed another way
    away = torch.ones_like(hit)
    if what == "late value":
        away[:new] = False
        near = ~hit[:new]
        assert float((got[:new] - clean[:new])[near].float().abs().max()) <= 2.0**-7 * float(clean.float().abs().max())
    assert torch.equal(got[away & ~hit], clean[away & ~hit])
    # 20 times and 5 ms: what is looked at again costs a pass over the values, not one over the cache for every row
    assert longer <= 20 * usual + 5


# ---- many slots, many tiles, tables far wider than what is held

@pytest.mark.parametrize("heads,kv,dim,page,slots,window", [
    (8, 1, 64, 16, 90, 0),      # more than 64 sequences of a tile or two, one of many: the keys are not split
    (16, 1, 128, 16, 90, 20), (40, 2, 64, 24, 70, 0), (3, 3, 80, 7, 130, 9),
])
def test_prompts_of_many_sequences(gpu, heads, kv, dim, page, slots, window) -> None:  # type: ignore[no-untyped-def]
    new = [(s * 7) % 40 if s != 11 else 500 for s in range(slots)]
    prior = [(s * 13) % 50 if s % 3 else 0 for s in range(slots)]
    k, v, table, n = cache([a + b for a, b in zip(new, prior)], dtype=B16, kv=kv, dim=dim, page=page)
    starts = torch.tensor([sum(new[:s]) for s in range(slots + 1)], dtype=torch.int32).cuda()
    q = queries(sum(new), heads, dim, B16)
    s = sink_values(heads, B16)
    want = ref.attention(q, k, v, table, n, starts, scale=dim**-0.5, window=window, first=window // 5, sinks=s)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, window=window, first=window // 5, sinks=s, lse=True)
    check(got, want, dtype=B16, dim=dim, lse=logs)


def test_prompts_of_more_than_1024_tiles(gpu) -> None:  # type: ignore[no-untyped-def]
    # 128 heads to a key-value head: two tokens a tile pair, 1,030 pairs in two sequences.
    new, prior = [2000, 60], [0, 100]
    k, v, table, n = cache([a + b for a, b in zip(new, prior)], dtype=B16, kv=1, dim=64, page=64)
    starts = torch.tensor([0, 2000, 2060], dtype=torch.int32).cuda()
    q = queries(2060, 128, 64, B16)
    got, logs = chroma_b200.paged_attention(q, k, v, table, n, starts, window=50, first=3, lse=True)
    for rows, positions in ((slice(0, 30), 0), (slice(990, 1020), 990), (slice(1970, 2000), 1970)):  # of the first sequence
        part = torch.tensor([0, 30], dtype=torch.int32).cuda()
        want = ref.attention(q[rows], k, v, table[:1], n[:1] * 0 + positions + 30, part, scale=0.125, window=50, first=3)
        check(got[rows], want, dtype=B16, dim=64, lse=logs[rows])
    want = ref.attention(q[2000:], k, v, table[1:], n[1:], torch.tensor([0, 60], dtype=torch.int32).cuda(), scale=0.125, window=50, first=3)
    check(got[2000:], want, dtype=B16, dim=64, lse=logs[2000:])


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [
    (F32, 8, 1, 16, 16), (F32, 8, 2, 64, 32), (B16, 64, 8, 64, 64), (B16, 8, 2, 128, 16), (B16, 8, 1, 32, 16), (B16, 6, 2, 80, 5),
])
@pytest.mark.parametrize("window,first", [(0, 0), (100, 4)])
def test_wide_tables(gpu, dtype, heads, kv, dim, page, window, first) -> None:  # type: ignore[no-untyped-def]
    """What is seen of short sequences does not depend on how many positions their table could name."""
    new, lengths = [5, 61, 0, 1, 30], [160, 98, 7, 1, 30]
    k, v, table, n = cache(lengths, dtype=dtype, kv=kv, dim=dim, page=page)
    wide = torch.full((5, 131072 // page), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    s = sink_values(heads, F32)
    for starts in (None, torch.tensor([0, 5, 66, 66, 67, 97], dtype=torch.int32).cuda()):
        q = queries(sum(new) if starts is not None else 5, heads, dim, dtype)
        want = ref.attention(q, k, v, table, n, starts, scale=0.2, window=window, first=first, sinks=s)
        got, logs = chroma_b200.paged_attention(q, k, v, wide, n, starts, scale=0.2, window=window, first=first, sinks=s, lse=True)
        check(got, want, dtype=dtype, dim=dim, lse=logs)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv,dim,new,prior", [(16, 8, 64, 600, 3000), (8, 4, 128, 20, 6000)])
def test_nothing_but_bad_values(gpu, bad, heads, kv, dim, new, prior) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([prior + new, new], dtype=B16, kv=kv, dim=dim, page=16, poison=False)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda()
    q = queries(2 * new, heads, dim, B16)
    clean = chroma_b200.paged_attention(q, k, v, table, n, starts)
    v[table[0, : -(-(prior + new) // 16)].long()] = bad  # the first sequence's
    got = chroma_b200.paged_attention(q, k, v, table, n, starts)
    chroma_b200.check_operators()
    assert torch.equal(got[new:], clean[new:])
    assert bool((got[:new] == bad).all()) if bad == bad else bool(got[:new].isnan().all())


@pytest.mark.parametrize("dtype,heads,kv,dim,new,prior", [
    (B16, 16, 8, 64, 600, 300), (B16, 8, 2, 128, 20, 3000), (B16, 200, 1, 64, 40, 30), (F32, 8, 2, 64, 90, 30), (F32, 8, 1, 16, 5, 4000),
])
def test_results_over_their_queries(gpu, dtype, heads, kv, dim, new, prior) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([prior + new, new], dtype=dtype, kv=kv, dim=dim, page=16, poison=False)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda()
    for bad in (False, True):
        if bad:
            p = prior + new // 2
            v[table[0, p // 16], p % 16, :, 3] = float("nan")
        for s, rows in ((starts, 2 * new), (None, 2)):
            for parts in (1, 3):  # queries of their own, and the first of what a projection gave
                q = queries(rows, parts * heads, dim, dtype)[:, :heads]
                want, logs = chroma_b200.paged_attention(q, k, v, table, n, s, lse=True)
                got, again = chroma_b200.paged_attention(q, k, v, table, n, s, lse=True, out=q)
                assert got.data_ptr() == q.data_ptr()
                assert torch.equal(got.nan_to_num(9), want.nan_to_num(9)) and torch.equal(again, logs)
    chroma_b200.check_operators()


def test_results_over_their_queries_through_the_c_entry(gpu) -> None:  # type: ignore[no-untyped-def]
    new, prior = 600, 300
    k, v, table, n = cache([prior + new, new], dtype=B16, kv=8, dim=64, page=16, poison=False)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda()
    q = queries(2 * new, 16, 64, B16)
    p = prior + new // 2
    v[table[0, p // 16], p % 16, :, 3] = float("nan")
    want = chroma_b200.paged_attention(q, k, v, table, n, starts)
    pages = pages_struct(k, v, table, n)
    g = Attention(q.data_ptr(), q.data_ptr(), None, None, starts.data_ptr(), None, 0, (ctypes.c_int64 * 2)(1024, 64),
                  (ctypes.c_int64 * 2)(1024, 64), 2 * new, 16, 0, 0, 0, 0.125)
    g.workspace_bytes = nat.lib().chroma_b200_attention_workspace(ctypes.byref(pages), ctypes.byref(g))
    room = torch.empty(max(1, g.workspace_bytes), dtype=torch.uint8, device="cuda")
    g.workspace = room.data_ptr()
    nat.call("chroma_b200_paged_attention", ctypes.byref(pages), ctypes.byref(g), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(q.nan_to_num(9), want.nan_to_num(9))
