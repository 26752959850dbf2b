"""What is done to logits before a token is chosen: penalties for tokens that occurred, biases, temperature, the mask
of a grammar, the greedy choice (no reference counterpart: the reference returns logits, chroma/_src/decoder.py:96-139).
"""

from __future__ import annotations

import struct
from typing import Any

import torch
from torch import Tensor

from chroma_b200._src import native as nat
from chroma_b200._src.paged import _STORAGE, _device, _ints, _launch

_LOGITS = struct.Struct("=14Q7q5i4x")  # chroma_b200_logits


def _floats(t: Tensor | None, rows: int, name: str) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 [{rows}], got {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def _matrix(t: Tensor, dtype: torch.dtype, rows: int, cols: int | None, name: str) -> int:
    """The row stride of a matrix whose rows are contiguous (rows that are all one row, stride 0, are fine)."""
    if t.dtype is not dtype or t.dim() != 2 or t.shape[0] != rows or (cols is not None and t.shape[1] != cols) \
            or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be {dtype} [{rows}, {'n' if cols is None else cols}] with contiguous rows, got "
                         f"{t.dtype} {list(t.shape)}")
    return t.stride(0)


def process_logits(logits: Tensor, *, history: Tensor | None = None, lengths: Tensor | None = None,
                   prompts: Tensor | None = None, repetition: Tensor | None = None, presence: Tensor | None = None,
                   frequency: Tensor | None = None, bias_ids: Tensor | None = None, bias: Tensor | None = None,
                   mask: Tensor | None = None, temperature: Tensor | None = None, out: Tensor | None = None,
                   argmax: bool = False) -> Any:
    """Processed logits ``[rows, vocab]`` in the type of ``logits`` (float32 or bfloat16), and with ``argmax`` the int64
    ``[rows]`` index of each row's largest, the lowest among equals.

    In this order, in 32 bits, rounded once at the end:

    * of a token that occurs in the row's ``history`` (int32 ``[rows, n]`` ids, the first ``lengths[row]`` of them):
      ``l / repetition`` where ``l > 0``, else ``l * repetition``;
    * ``l -= frequency * c``, and ``l -= presence`` where ``c > 0``: c counts the token after the first
      ``prompts[row]`` entries of the history (without ``prompts``: in all of it);
    * ``l += bias`` of the row's ``bias_ids`` (int32 and float32 ``[rows, m]``; ids below 0 are passed over, an id that
      is listed more than once adds up in list order);
    * ``l /= temperature`` (a row whose temperature is 0 is left as it is);
    * -inf where the row's ``mask`` (int32 ``[rows, ceil(vocab / 32)]``, bit ``v % 32`` of word ``v // 32``) is 0.

    ``repetition``, ``presence``, ``frequency``, ``temperature``: float32 ``[rows]``. ``out`` may be ``logits`` itself.
    Ids outside the vocabulary are passed over.
    """
    index = _device(logits, history, lengths, prompts, repetition, presence, frequency, bias_ids, bias, mask,
                    temperature, out)
    storage = _STORAGE.get(logits.dtype)
    if storage is None or logits.dim() != 2 or not logits.shape[1] or logits.stride(1) != 1:
        raise ValueError(f"logits must be float32 or bfloat16 [rows, vocab] with contiguous rows, got {logits.dtype} "
                         f"{list(logits.shape)}")
    rows, vocab = logits.shape
    if out is None:
        out = logits.new_empty((rows, vocab))
    elif out.shape != logits.shape or out.dtype is not logits.dtype or out.stride(1) != 1 \
            or (out.stride(0) < vocab and rows > 1):
        raise ValueError(f"out must be {list(logits.shape)} {logits.dtype} with contiguous rows")
    pointers, strides, width, biases = [0, 0, 0], [0, 0, 0, 0], 0, 0
    if history is not None:
        if lengths is None:
            raise ValueError("a history needs its lengths")
        strides[0], width = _matrix(history, torch.int32, rows, None, "history"), history.shape[1]
        pointers = [history.data_ptr(), _ints(lengths, (rows,), "lengths"),
                    0 if prompts is None else _ints(prompts, (rows,), "prompts")]
    elif repetition is not None or presence is not None or frequency is not None:
        raise ValueError("penalties need a history")
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias_ids is not None and bias is not None:
        biases = bias_ids.shape[-1]
        strides[1] = _matrix(bias_ids, torch.int32, rows, None, "bias_ids")
        strides[2] = _matrix(bias, torch.float32, rows, biases, "bias")
    if mask is not None:
        strides[3] = _matrix(mask, torch.int32, rows, (vocab + 31) // 32, "mask")
    best, room, size = None, 0, 0
    if argmax:
        size = nat.lib().chroma_b200_logits_workspace(rows, vocab)
        whole = torch.empty(rows + size // 8, dtype=torch.int64, device=logits.device)  # and the workspace behind the ids
        best, room = whole[:rows], whole.data_ptr() + 8 * rows
    args = _LOGITS.pack(
        logits.data_ptr(), out.data_ptr(), 0 if best is None else best.data_ptr(), *pointers,
        _floats(repetition, rows, "repetition"), _floats(presence, rows, "presence"),
        _floats(frequency, rows, "frequency"), _floats(temperature, rows, "temperature"),
        0 if bias_ids is None else bias_ids.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if mask is None else mask.data_ptr(), room, logits.stride(0), out.stride(0),
        *strides, size, storage, rows, vocab, width, biases)
    _launch(index, "chroma_b200_process_logits", args)
    return out if best is None else (out, best)
