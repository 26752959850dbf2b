"""The operators through the C ABI from several host threads at once, each with a stream and sizes of its own."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from chroma_b200._src import native as nat
from tests.test_gpu_paged_edges import B16, pages_struct

pytestmark = pytest.mark.gpu


class Logits(ctypes.Structure):  # chroma_b200_logits
    _fields_ = [(x, ctypes.c_void_p) for x in ("logits", "out", "argmax", "history", "lengths", "prompts", "repetition", "presence", "frequency",
                                               "temperature", "bias_ids", "bias", "mask", "workspace")] + [
        (x, ctypes.c_int64) for x in ("stride", "out_stride", "history_stride", "bias_ids_stride", "bias_stride", "mask_stride", "workspace_bytes")] + [
        (x, ctypes.c_int32) for x in ("storage", "rows", "vocab", "width", "biases")]


def together(calls, times):  # type: ignore[no-untyped-def]
    """Every call ``times`` times in a thread of its own; what they raised."""
    errors = []

    def work(call):  # type: ignore[no-untyped-def]
        try:
            stream = torch.cuda.Stream()
            for i in range(times):
                call(stream.cuda_stream)
                if i % 64 == 63:
                    stream.synchronize()
            stream.synchronize()
        except Exception as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors


def test_steps_and_compaction_of_pools_of_different_sizes(gpu) -> None:  # type: ignore[no-untyped-def]
    kept = []  # what the calls point to

    def stepping(pages):  # type: ignore[no-untyped-def]
        k, v = (torch.zeros(pages, 1, 1, 8, dtype=B16, device="cuda") for _ in range(2))
        table, (lengths, parents, counts) = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
        p = pages_struct(k, v, table, lengths)
        room = torch.empty(nat.lib().chroma_b200_pages_workspace(pages, 2), dtype=torch.uint8, device="cuda")
        new, n, info = torch.empty_like(table), torch.empty_like(lengths), torch.empty(3, dtype=torch.int32, device="cuda")
        kept.append((k, v, table, lengths, parents, counts, p, room, new, n, info))

        def call(stream):  # type: ignore[no-untyped-def]
            nat.call("chroma_b200_step_pages", ctypes.byref(p), parents.data_ptr(), counts.data_ptr(), new.data_ptr(), n.data_ptr(), info.data_ptr(),
                     room.data_ptr(), room.numel(), stream)
            nat.call("chroma_b200_compact_pages", ctypes.byref(p), new.data_ptr(), info.data_ptr(), room.data_ptr(), room.numel(), stream)

        return call

    calls = [stepping(pages) for pages in (30000, 9000, 20000, 100)]
    torch.cuda.synchronize()
    assert not together(calls, 3000)
    assert all(x[-1].tolist()[:2] == [0, 0] for x in kept)


@pytest.mark.parametrize("dtype", [torch.float32, B16])
def test_logits_of_vocabularies_of_different_sizes(gpu, dtype) -> None:  # type: ignore[no-untyped-def]
    kept = []

    def processing(vocab, rows=64):  # type: ignore[no-untyped-def]
        x, out = torch.randn(rows, vocab, device="cuda").to(dtype), torch.empty(rows, vocab, dtype=dtype, device="cuda")
        history, lengths = torch.zeros(rows, 4, dtype=torch.int32, device="cuda"), torch.full((rows,), 4, dtype=torch.int32, device="cuda")
        penalty = torch.full((rows,), 2.0, device="cuda")
        room = torch.empty(nat.lib().chroma_b200_logits_workspace(rows, vocab), dtype=torch.uint8, device="cuda")
        g = Logits(logits=x.data_ptr(), out=out.data_ptr(), history=history.data_ptr(), lengths=lengths.data_ptr(), presence=penalty.data_ptr(),
                   workspace=room.data_ptr(), stride=vocab, out_stride=vocab, history_stride=4, workspace_bytes=room.numel(),
                   storage=int(dtype is B16), rows=rows, vocab=vocab, width=4)
        kept.append((x, out, history, lengths, penalty, room, g))
        return lambda stream: nat.call("chroma_b200_process_logits", ctypes.byref(g), stream)

    calls = [processing(vocab) for vocab in (201088, 32003)]
    torch.cuda.synchronize()
    assert not together(calls, 3000)
    for x, out, *_ in kept:
        assert torch.equal(out[:, 1:], x[:, 1:]) and torch.equal(out[:, 0].float(), (x[:, 0].float() - 2).to(dtype).float())
