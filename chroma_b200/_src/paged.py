"""Operators over a paged key-value cache, on CUDA tensors (no reference counterpart: the reference's cache is one
contiguous block per Program, chroma/_src/decoder.py:44-152).

A cache is two pools ``keys`` and ``values`` of pages, ``[pages, page_rows, kv_heads, head_dim]`` (with a leading
``layers`` for the page operators), in float32 or bfloat16; an int32 ``table [slots, width]`` with the pages of each
sequence (below 0: none); and int32 ``lengths [slots]``, the rows that each holds. Position ``p`` of slot ``s`` is row
``p % page_rows`` of page ``table[s, p // page_rows]``. A step of a program that serves from it::

    # fork, empty, reserve
    table, lengths, info = step_pages(table, lengths, parents, counts, keys, values, cut=False)
    for layer in range(layers):
        ...
        paged_append(keys[layer], values[layer], k, v, table, lengths, starts)
        o = paged_attention(q, keys[layer], values[layer], table, lengths, starts, scale=..., sinks=...)

Pools may have any strides that are multiples of 16 bytes (a layer of a larger pool, keys and values side by side); a
head's row is contiguous and a multiple of 16 bytes. Everything is queued on the current stream of the tensors' device;
nothing waits for the device or reads it from the host (``check_operators`` does). No operator has a gradient: an output of
tensors that want one raises when it is differentiated, and nothing passes through the cache. Wrong arguments raise ``ValueError``
(``TypeError`` for what is not a tensor). The binding is ``chroma_b200/csrc/tensors.cpp``.
"""

from __future__ import annotations

import ctypes
import sysconfig
from typing import Any

import torch
from torch import Tensor

from chroma_b200._src import native as nat

_ENTRIES = ("paged_append", "paged_attention", "attention_workspace", "step_pages", "step_pages_uncut", "compact_pages",
            "pages_workspace", "process_logits", "logits_workspace")


def _module() -> Any:
    """The binding of the operators (chroma_b200/csrc/tensors.cpp), given the entry points of the native library."""
    assert torch.version.cuda, "the operators need a Torch that was built with CUDA"
    lib = nat.lib()
    tag = f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"
    try:
        from chroma_b200._src import _tensors

        if _tensors.built_for != tag:
            raise ImportError(f"it is built for {_tensors.built_for}, this is {tag}")
    except ImportError as error:
        raise RuntimeError(f"the operators' binding is not built for this Torch ({error}); build it with "
                           "`python -m chroma_b200.build --force`") from error
    _tensors.bind(*(ctypes.cast(getattr(lib, f"chroma_b200_{name}"), ctypes.c_void_p).value for name in _ENTRIES))
    return _tensors


ops = _module()


def paged_append(keys: Tensor, values: Tensor, new_keys: Tensor, new_values: Tensor, table: Tensor, lengths: Tensor,
                 starts: Tensor | None = None) -> None:
    """Writes new rows ``[tokens, kv_heads, head_dim]`` into the pages of their sequences, in place.

    Rows ``starts[b] : starts[b + 1]`` are slot b's (``starts`` int32 ``[slots + 1]``, from 0 to ``tokens``; without it
    there is one row per slot). ``lengths`` counts them already: the last is written at ``lengths[b] - 1``. The pages
    must belong to the slot alone from there on (``step_pages`` sees to it); rows without a page, those past the end of
    the table among them, are dropped.
    """
    ops.paged_append(keys, values, new_keys, new_values, table, lengths, starts)


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
    of an attention can be joined. ``out`` may be ``q`` itself. A token that sees nothing gives zeros and its sink (or -inf). Non-finite values in
    rows that a token does not see do not reach it. A token past the end of the table sees what has pages.

    In float32 everything is held in 32 bits. In bfloat16 so are scores, sums and the running maximum, but the softmax's
    weights go into the product with the values as bfloat16, as the tensor cores take them: against 64 bits the relative
    error of a result is about 2.2e-3, where rounding the result alone costs 1.7e-3.
    """
    return ops.paged_attention(q, keys, values, table, lengths, starts, scale, window, first, sinks, lse, out)


def step_pages(table: Tensor, lengths: Tensor, parents: Tensor, counts: Tensor, keys: Tensor, values: Tensor, *,
               cut: bool = True) -> tuple[Tensor, Tensor, Tensor]:
    """One step of a set of sequences: returns the new ``(table, lengths, info)`` and leaves the given ones as they are.

    Slot s continues slot ``parents[s]`` (int32 ``[slots]``: s itself, another that several slots may continue, or -1,
    which empties s), and ``counts[s]`` more rows are reserved for it. Pages are shared between slots that hold the
    same rows; one that a slot will write into while another holds it too is copied first (its rows so far, every
    layer of the pools), except for the holder with the most rows in it, the lowest slot among equals. A page that no
    slot holds is free; free pages are given out from the lowest number to slots from the lowest. ``info`` (int32,
    on the device) is [pages left free, pages short, pages copied]; where pages are short, entries stay -1, nothing is
    copied, and the step can be tried again from the old table.

    A sequence may ask for rows past the end of its row of the table, ``width * page_rows`` positions. With ``cut`` its
    length ends there, and the caller must not append the rows that were cut off: ``paged_append`` counts back from the
    length, so it would put them over the last rows before the end. With ``cut=False`` lengths count every row that was
    asked for; ``paged_append`` drops those past the end, ``paged_attention`` sees what has pages, and a length above
    ``width * page_rows`` says that the sequence has outgrown its table.
    """
    return ops.step_pages(table, lengths, parents, counts, keys, values, cut)


def compact_pages(table: Tensor, lengths: Tensor, keys: Tensor, values: Tensor) -> tuple[Tensor, Tensor]:
    """Moves the n pages that slots hold to the first n of the pools, so that the rest can be given up: the i-th held
    page from n up goes to the i-th free page below n. Returns the new table and ``info`` (int32, on the device):
    [n, pages moved]."""
    return ops.compact_pages(table, lengths, keys, values)


def check_operators(device: Any = None) -> None:
    """Waits for the current stream of ``device`` (the current one unless given), and raises ``RuntimeError`` if since the
    last check there a kernel of the operators gave up on a bounded wait inside itself: its outputs are incomplete. A program
    calls it where it synchronises anyway."""
    with torch.cuda.device(device):
        nat.call("chroma_b200_operators_check", torch.cuda.current_stream().cuda_stream)
