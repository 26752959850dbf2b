"""The operators as Torch sees them: gradients that there are none of, versions of what is written in place, odd arguments."""

from __future__ import annotations

import pytest
import torch

import chroma_b200
from tests.test_gpu_paged import B16, F32, cache, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, B16])
@pytest.mark.parametrize("which", ["q", "keys", "values", "sinks"])
def test_a_gradient_of_attention_is_refused_when_it_is_asked_for(gpu, dtype, which) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([40, 3], dtype=dtype, kv=2, dim=64, page=16)
    q, s = queries(2, 8, 64, dtype), torch.zeros(8, device="cuda")
    plain, logs = chroma_b200.paged_attention(q, k, v, table, n, sinks=s, lse=True)
    assert not plain.requires_grad and not logs.requires_grad
    {"q": q, "keys": k, "values": v, "sinks": s}[which].requires_grad_()
    got = chroma_b200.paged_attention(q, k, v, table, n, sinks=s, lse=True)
    for x, same in zip(got, (plain, logs)):
        assert x.requires_grad and torch.equal(x, same)
        with pytest.raises(RuntimeError, match="paged_attention"):
            x.sum().backward()
    with pytest.raises(ValueError, match="no_grad"):
        chroma_b200.paged_attention(q, k, v, table, n, sinks=s, out=torch.empty_like(plain))
    with torch.no_grad():
        out = torch.empty_like(plain)
        got = chroma_b200.paged_attention(q, k, v, table, n, sinks=s, out=out)
        assert not got.requires_grad and torch.equal(out, plain)


def test_a_gradient_of_logits_is_refused_when_it_is_asked_for(gpu) -> None:  # type: ignore[no-untyped-def]
    x, t = torch.randn(2, 100, device="cuda"), torch.full((2,), 0.5, device="cuda")
    for wants in (x, t):
        wants.requires_grad_()
        got, best = chroma_b200.process_logits(x, temperature=t, argmax=True)
        assert torch.equal(got.detach(), x.detach() / 0.5) and not best.requires_grad
        with pytest.raises(RuntimeError, match="process_logits"):
            got.sum().backward()
        with pytest.raises(ValueError, match="no_grad"):
            chroma_b200.process_logits(x, temperature=t, out=torch.empty_like(x))
        wants.requires_grad_(False)
    assert not chroma_b200.process_logits(x, temperature=t).requires_grad


def test_what_is_written_counts_its_version(gpu) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([20, 3], dtype=B16, kv=2, dim=64, page=16, layers=2)
    q = queries(2, 8, 64, B16)
    same = torch.arange(2, dtype=torch.int32, device="cuda")

    def counted(call, *written):  # type: ignore[no-untyped-def]
        before = [x._version for x in written]
        call()
        assert all(x._version > b for x, b in zip(written, before))

    counted(lambda: chroma_b200.paged_append(k[0], v[0], q[:, :2], q[:, 2:4], table, n), k, v)
    counted(lambda: chroma_b200.step_pages(table, n, same, same, k, v), k, v)
    counted(lambda: chroma_b200.compact_pages(table, n, k, v), k, v)
    out, x = torch.empty_like(q), torch.randn(2, 100, device="cuda")
    counted(lambda: chroma_b200.paged_attention(q, k[0], v[0], table, n, out=out), out)
    counted(lambda: chroma_b200.process_logits(x, out=x), x)
    before = k._version
    chroma_b200.paged_attention(q, k[0], v[0], table, n)
    assert k._version == before
    with torch.inference_mode():
        pool = torch.zeros(3, 16, 2, 64, device="cuda", dtype=B16)
        chroma_b200.paged_append(pool, pool.clone(), q[:, :2], q[:, :2], table, n)
    chroma_b200.paged_append(pool, pool.clone(), q[:, :2], q[:, :2], table, n)


def test_flags_that_are_neither_true_nor_false(gpu) -> None:  # type: ignore[no-untyped-def]
    k, v, table, n = cache([20, 3], dtype=B16, kv=2, dim=64, page=16)
    flag = torch.ones(2, dtype=torch.bool)
    with pytest.raises(RuntimeError, match="ambiguous"):
        chroma_b200.paged_attention(queries(2, 8, 64, B16), k, v, table, n, lse=flag)
    with pytest.raises(RuntimeError, match="ambiguous"):
        chroma_b200.process_logits(torch.randn(2, 100, device="cuda"), argmax=flag)
    with pytest.raises(RuntimeError, match="ambiguous"):
        chroma_b200.step_pages(table, n, n, n, k, v, cut=flag)
    with pytest.raises(ValueError, match="below 2"):
        chroma_b200.paged_attention(queries(2, 8, 64, B16), k, v, table, n, window=2**31)
