"""Operators over a paged key-value cache, on CUDA tensors (no reference counterpart: the reference's cache is one
contiguous block per Program, chroma/_src/decoder.py:44-152).

A cache is two pools ``keys`` and ``values`` of pages, ``[pages, page_rows, kv_heads, head_dim]`` (with a leading
``layers`` for the page operators), in float32 or bfloat16; an int32 ``table [slots, width]`` with the pages of each
sequence (below 0: none); and int32 ``lengths [slots]``, the rows that each holds. Position ``p`` of slot ``s`` is row
``p % page_rows`` of page ``table[s, p // page_rows]``. A step of a program that serves from it::

    table, lengths, info = step_pages(table, lengths, parents, counts, keys, values)   # fork, empty, reserve
    for layer in range(layers):
        ...
        paged_append(keys[layer], values[layer], k, v, table, lengths, starts)
        o = paged_attention(q, keys[layer], values[layer], table, lengths, starts, scale=..., sinks=...)

Pools may have any strides that are multiples of 16 bytes (a layer of a larger pool, keys and values side by side); a
head's row is contiguous and a multiple of 16 bytes. Everything is queued on the current stream of the tensors' device;
nothing waits for the device or reads it from the host. Wrong arguments raise ``ValueError`` (``TypeError`` for what is
not a tensor).
"""

from __future__ import annotations

import struct
from typing import Any

import torch
from torch import Tensor

from chroma_b200._src import native as nat

_STORAGE = {torch.float32: nat.FP32, torch.bfloat16: nat.BF16}
_PAGES = struct.Struct("=4Q9q8i")  # chroma_b200_pages
_ATTENTION = struct.Struct("=6Q5q5if")  # chroma_b200_attention
_NEW_STRIDES = struct.Struct("=4q")


def _device(first: Any, *others: Any) -> int:
    """The one CUDA device of these tensors (None among them is passed over)."""
    try:
        index = first.get_device()
        if index < 0:
            raise ValueError("tensors must be on a CUDA device")
        for t in others:
            if t is not None and t.get_device() != index:
                raise ValueError("tensors on different devices")
    except AttributeError:
        raise TypeError("not a tensor among the arguments that have to be tensors") from None
    return index


def _ints(t: Tensor, shape: tuple[int, ...], name: str) -> int:
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def _pages(keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor, layered: bool) -> bytes:
    """The packed chroma_b200_pages of a cache."""
    shape, ks, vs = keys.shape, keys.stride(), values.stride()
    storage = _STORAGE.get(keys.dtype)
    if storage is None or values.dtype is not keys.dtype:
        raise ValueError(f"pools are both float32 or both bfloat16, got {keys.dtype} and {values.dtype}")
    rank = len(shape)
    if values.shape != shape or (rank != 4 and not (layered and rank == 5)):
        raise ValueError(f"pools must be [{'layers, ' if layered else ''}pages, rows, heads, dim], alike, got "
                         f"{list(shape)} and {list(values.shape)}")
    if ks[-1] != 1 or vs[-1] != 1:
        raise ValueError("a head's row must be contiguous")
    table_shape, ts = table.shape, table.stride()
    if table.dtype is not torch.int32 or len(ts) != 2 or ts[1] != 1:
        raise ValueError("table must be int32 [slots, width] with contiguous rows")
    slots, width = table_shape
    pointers = keys.data_ptr(), values.data_ptr(), table.data_ptr(), _ints(lengths, (slots,), "lengths")
    if rank == 4:
        return _PAGES.pack(*pointers, 0, ks[0], ks[1], ks[2], 0, vs[0], vs[1], vs[2], ts[0], storage, 1, *shape, slots, width)
    return _PAGES.pack(*pointers, *ks[:4], *vs[:4], ts[0], storage, *shape, slots, width)


def _launch(index: int, name: str, *args: Any) -> None:
    """Calls the native operator on the device's current stream; ``args`` end before the stream."""
    if index == torch._C._cuda_getDevice():
        nat.call_op(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            nat.call_op(name, *args, torch._C._cuda_getCurrentRawStream(index))


def paged_append(keys: Tensor, values: Tensor, new_keys: Tensor, new_values: Tensor, table: Tensor, lengths: Tensor,
                 starts: Tensor | None = None) -> None:
    """Writes new rows ``[tokens, kv_heads, head_dim]`` into the pages of their sequences, in place.

    Rows ``starts[b] : starts[b + 1]`` are slot b's (``starts`` int32 ``[slots + 1]``, from 0 to ``tokens``; without it
    there is one row per slot). ``lengths`` counts them already: the last is written at ``lengths[b] - 1``. The pages
    must belong to the slot alone from there on (``step_pages`` sees to it); rows without a page are dropped.
    """
    index = _device(keys, values, new_keys, new_values, table, lengths, starts)
    pages = _pages(keys, values, table, lengths, False)
    tokens = new_keys.shape[0]
    want = (tokens, keys.shape[2], keys.shape[3])
    if new_keys.shape != want or new_values.shape != want or new_keys.dtype is not keys.dtype \
            or new_values.dtype is not keys.dtype:
        raise ValueError(f"new rows must be {list(want)} {keys.dtype}, got {list(new_keys.shape)} {new_keys.dtype} "
                         f"and {list(new_values.shape)} {new_values.dtype}")
    ns, vs = new_keys.stride(), new_values.stride()
    if ns[2] != 1 or vs[2] != 1:
        raise ValueError("a head's row must be contiguous")
    _launch(index, "chroma_b200_paged_append", pages, new_keys.data_ptr(), new_values.data_ptr(),
            _NEW_STRIDES.pack(ns[0], ns[1], vs[0], vs[1]),
            None if starts is None else _ints(starts, (table.shape[0] + 1,), "starts"), tokens)


def paged_attention(q: Tensor, keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor,
                    starts: Tensor | None = None, *, scale: float | None = None, window: int = 0, first: int = 0,
                    sinks: Tensor | None = None, lse: bool = False, out: Tensor | None = None) -> Any:
    """Attention of ``q [tokens, heads, head_dim]`` over the pages of each token's sequence, ``heads / kv_heads``
    query heads to a key-value head: ``softmax(scale * q @ k.T) @ v`` over the positions that the token sees.

    Without ``starts`` there is one token per slot, at position ``lengths[b] - 1``. With it (int32 ``[slots + 1]``,
    from 0 to ``tokens``) rows ``starts[b] : starts[b + 1]`` are slot b's last positions: a prompt, or a chunk of one
    after what the cache holds already. A token at position p sees position j iff ``j <= p``, j has a page, and
    ``p - j < window`` or ``j < first`` (``window`` 0: no window): a sliding window that keeps the first tokens in
    sight. ``sinks [heads]`` are learned logits that join the softmax's sum without a value
    (chroma/models/gpt_oss.py:133-151). ``scale`` is ``head_dim ** -0.5`` unless given.

    Returns the output in q's type, and with ``lse`` the fp32 ``[tokens, heads]`` logarithms of the sums, by which parts
    of an attention can be joined. A token that sees nothing gives zeros and its sink (or -inf). Non-finite values in
    rows that a token does not see do not reach it.
    """
    index = _device(q, keys, values, table, lengths, starts, sinks, out)
    pages = _pages(keys, values, table, lengths, False)
    tokens, heads, dim = q.shape
    if q.dtype is not keys.dtype or dim != keys.shape[3]:
        raise ValueError(f"q must be [tokens, heads, {keys.shape[3]}] {keys.dtype}, got {list(q.shape)} {q.dtype}")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype:
        raise ValueError(f"out must be {list(q.shape)} {q.dtype}, got {list(out.shape)} {out.dtype}")
    qs, os = q.stride(), out.stride()
    if qs[2] != 1 or os[2] != 1:
        raise ValueError("a head's row must be contiguous")
    logs = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if lse else None
    fp32 = 0
    if sinks is not None:
        if sinks.shape != (heads,) or not sinks.is_contiguous() or sinks.dtype not in (q.dtype, torch.float32):
            raise ValueError(f"sinks must be [{heads}] {q.dtype} or float32, got {list(sinks.shape)} {sinks.dtype}")
        fp32 = int(sinks.dtype is torch.float32)
    if window < 0 or first < 0:
        raise ValueError(f"window and first must be nonnegative, got {window} and {first}")
    fields = (
        q.data_ptr(), out.data_ptr(), 0 if logs is None else logs.data_ptr(), 0 if sinks is None else sinks.data_ptr(),
        0 if starts is None else _ints(starts, (table.shape[0] + 1,), "starts"))
    more = (qs[0], qs[1], os[0], os[1], tokens, heads, fp32, window, first, dim**-0.5 if scale is None else scale)
    args = _ATTENTION.pack(*fields, 0, 0, *more)
    size = nat.lib().chroma_b200_attention_workspace(pages, args)
    if size > 0:
        room = torch.empty(size, dtype=torch.uint8, device=q.device)
        args = _ATTENTION.pack(*fields, room.data_ptr(), size, *more)
    _launch(index, "chroma_b200_paged_attention", pages, args)
    return out if logs is None else (out, logs)


def step_pages(table: Tensor, lengths: Tensor, parents: Tensor, counts: Tensor, keys: Tensor,
               values: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """One step of a set of sequences: returns the new ``(table, lengths, info)`` and leaves the given ones as they are.

    Slot s continues slot ``parents[s]`` (int32 ``[slots]``: s itself, another that several slots may continue, or -1,
    which empties s), and ``counts[s]`` more rows are reserved for it. Pages are shared between slots that hold the
    same rows; one that a slot will write into while another holds it too is copied first (its rows so far, every
    layer of the pools), except for the holder with the most rows in it, the lowest slot among equals. A page that no
    slot holds is free; free pages are given out from the lowest number to slots from the lowest. ``info`` (int32,
    on the device) is [pages left free, pages short, pages copied]; where pages are short, entries stay -1, nothing is
    copied, and the step can be tried again from the old table.
    """
    index = _device(keys, values, table, lengths, parents, counts)
    pages = _pages(keys, values, table, lengths, True)
    slots, width = table.shape
    new_table, new_lengths = table.new_empty((slots, width)), torch.empty_like(lengths)
    size = nat.lib().chroma_b200_pages_workspace(keys.shape[-4], slots)
    room = lengths.new_empty(3 + size // 4)  # info, and the native code's workspace behind it
    at = room.data_ptr()
    _launch(index, "chroma_b200_step_pages", pages, _ints(parents, (slots,), "parents"),
            _ints(counts, (slots,), "counts"), new_table.data_ptr(), new_lengths.data_ptr(), at, at + 12, size)
    return new_table, new_lengths, room[:3]


def compact_pages(table: Tensor, lengths: Tensor, keys: Tensor, values: Tensor) -> tuple[Tensor, Tensor]:
    """Moves the n pages that slots hold to the first n of the pools, so that the rest can be given up: the i-th held
    page from n up goes to the i-th free page below n. Returns the new table and ``info`` (int32, on the device):
    [n, pages moved]."""
    index = _device(keys, values, table, lengths)
    pages = _pages(keys, values, table, lengths, True)
    slots, width = table.shape
    new_table = table.new_empty((slots, width))
    size = nat.lib().chroma_b200_pages_workspace(keys.shape[-4], slots)
    room = lengths.new_empty(2 + size // 4)  # info, and the native code's workspace behind it
    at = room.data_ptr()
    _launch(index, "chroma_b200_compact_pages", pages, new_table.data_ptr(), at, at + 8, size)
    return new_table, room[:2]
