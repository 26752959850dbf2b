"""chroma_b200: a B200-native (sm_100a) CUDA backend for Chroma's compiled GPT-OSS-style programs.

Public surface, as in the reference (chroma/__init__.py:14-26): ``compile``, ``Program``, ``Decoder``; plus
``BatchDecoder`` for device-resident batched decoding. Loading and running artefacts needs NumPy only; ``compile``
imports Torch on first use.

Operators for serving over a paged key-value cache, on CUDA tensors: ``paged_append``, ``paged_attention``,
``step_pages``, ``compact_pages``, and ``process_logits`` for the logits that follow; ``check_operators``. They import Torch
when they are first named, so ``from chroma_b200 import *`` leaves them out.
"""

from __future__ import annotations

from pathlib import Path
from typing import Any

from chroma_b200._src.decoder import BatchDecoder, Decoder
from chroma_b200._src.experts import ExpertGroup
from chroma_b200._src.program import Program


def compile(input: Any, output: str | Path, *, blas: bool = True, backend: str = "cuda") -> Program:
    """Compile an ``ExportedProgram`` (or a saved ``.pt2`` path) into ``output`` and load it."""
    from chroma_b200._src.compiler import compile_for_backend

    return compile_for_backend(input, output, blas=blas, backend=backend)


def compile_model(model: Any, output: str | Path, *, steps: int, context: int | None = None, last: bool = False,
                  experts: ExpertGroup | None = None) -> Program:
    """Compile a ``chroma_b200.models.Transformer`` straight from its parameters (no ``torch.export``): a forward
    over ``steps`` tokens, or with ``context`` a KV-cached step of ``steps`` rows (the prefill/decode programs).
    With ``experts`` (an ``ExpertGroup``), this rank's share of the experts only, bound to the group."""
    from chroma_b200._src.compiler import compile_model as _compile_model

    return _compile_model(model, output, steps=steps, context=context, last=last, experts=experts)


# Operators on CUDA tensors of the caller (a paged key-value cache, its attention, logits): Torch is imported by the
# caller, who has the tensors. Not in __all__, which a star import names one by one.
_OPERATORS = {"paged_append": "paged", "paged_attention": "paged", "step_pages": "paged", "compact_pages": "paged",
              "check_operators": "paged", "process_logits": "logits"}


def __getattr__(name: str) -> Any:
    if name in _OPERATORS:
        from importlib import import_module

        value = getattr(import_module(f"chroma_b200._src.{_OPERATORS[name]}"), name)
        globals()[name] = value
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


__all__ = ["BatchDecoder", "Decoder", "ExpertGroup", "Program", "compile", "compile_model"]


def __dir__() -> list[str]:
    return sorted({*globals(), *_OPERATORS})
