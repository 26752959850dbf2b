"""What is done to logits before a token is chosen: penalties for tokens that occurred, biases, temperature, the mask
of a grammar, the greedy choice (no reference counterpart: the reference returns logits, chroma/_src/decoder.py:96-139).
"""

from __future__ import annotations

from typing import Any

from torch import Tensor

from chroma_b200._src.paged import ops


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
    return ops.process_logits(logits, history, lengths, prompts, repetition, presence, frequency, bias_ids, bias, mask,
                              temperature, out, argmax)
