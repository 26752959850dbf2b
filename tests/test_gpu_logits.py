"""``process_logits`` on the GPU against a plain form in 64 bits (``tests/paged_reference.py``).

Tolerance: each of the at most six operations on an entry rounds once in fp32 (2^-24 of its result, whose magnitude is
at most the largest value on the way), then the result is rounded to its type (2^-8 relative in bf16,
whose significand has 8 bits).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import chroma_b200
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def case(rows, vocab, width, biases, dtype, seed):  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    lengths = (rand(rows) * (width + 1)).to(torch.int32).clamp(max=width)
    lengths[0] = width
    return torch.randn(rows, vocab, generator=g, device="cuda").mul(3).to(dtype), {
        "history": (rand(rows, width) ** 3 * (vocab + 2)).to(torch.int32) - 1,  # a few ids outside the vocabulary
        "lengths": lengths, "prompts": (rand(rows) * width).to(torch.int32), "repetition": 1 + rand(rows),
        "presence": rand(rows), "frequency": rand(rows), "temperature": rand(rows).add(0.5),
        "bias_ids": (rand(rows, biases) * (vocab + 2)).to(torch.int32) - 1, "bias": rand(rows, biases) * 8 - 4,
        "mask": torch.randint(-(2**31), 2**31, (rows, -(-vocab // 32)), generator=g, device="cuda").to(torch.int32),
    }


def check(got, want, dtype, scale):  # type: ignore[no-untyped-def]
    half = 2.0**-8 if dtype is torch.bfloat16 else 0.0
    np.testing.assert_array_equal(np.isneginf(got.float().cpu().numpy()), np.isneginf(want))
    np.testing.assert_allclose(got.double().cpu().numpy(), want, atol=6 * 2.0**-23 * scale, rtol=half + 2.0**-22)


def largest(got):  # type: ignore[no-untyped-def]
    return np.argmax(got.float().cpu().numpy(), -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,width,biases", [
    (1, 1, 1, 1), (3, 31, 5, 2), (2, 33, 40, 64), (5, 1000, 300, 7), (4, 32003, 64, 300), (1, 201088, 500, 20),
    (7, 50257, 2000, 33), (17, 4096, 1, 1), (2, 70000, 33000, 5),
])
def test_processed_logits(gpu, dtype, rows, vocab, width, biases) -> None:  # type: ignore[no-untyped-def]
    x, more = case(rows, vocab, width, biases, dtype, vocab + width)
    want = ref.logits(x, **more)
    before = x.clone()
    got, ids = chroma_b200.process_logits(x, argmax=True, **more)
    # on the way: |x| r, less c frequency, each bias, over 0.5
    scale = float(x.float().abs().max()) * 2 + width + 4 * biases + 2
    check(got, want, dtype, 2 * scale)
    assert torch.equal(x, before) and got.dtype is dtype
    np.testing.assert_array_equal(ids.cpu().numpy(), largest(got))
    again = x.clone()
    assert chroma_b200.process_logits(again, out=again, **more) is again
    assert torch.equal(again, got)


@pytest.mark.parametrize("left", ["history", "bias", "mask", "temperature", "repetition", "frequency", "presence", "prompts", "all"])
def test_any_part_may_be_missing(gpu, left) -> None:  # type: ignore[no-untyped-def]
    x, more = case(3, 5000, 60, 9, torch.float32, 11)
    gone = {"history": ["history", "lengths", "prompts", "repetition", "presence", "frequency"],
            "bias": ["bias", "bias_ids"], "all": list(more)}.get(left, [left])
    more = {k: v for k, v in more.items() if k not in gone}
    got = chroma_b200.process_logits(x, **more)
    check(got, ref.logits(x, **more), torch.float32, 200.0)
    if left == "all":
        assert torch.equal(got, x)


def test_rows_at_any_address(gpu) -> None:  # type: ignore[no-untyped-def]
    x, more = case(4, 1003, 30, 5, torch.bfloat16, 3)
    wide = torch.zeros(4, 1010, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 3:1006]
    view.copy_(x)
    out = torch.full((4, 1011), 5.0, dtype=torch.bfloat16, device="cuda")
    one = {"mask": more["mask"][:1].expand(4, -1), "bias_ids": more["bias_ids"][:1].expand(4, -1),
           "bias": more["bias"][:1].expand(4, -1)}
    got = chroma_b200.process_logits(view, out=out[:, 1:1004], **{**more, **one})
    check(got, ref.logits(x, **{**more, **one}), torch.bfloat16, 400.0)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1004:] == 5).all())


def test_infinities_ties_and_rows_with_nothing_allowed(gpu) -> None:  # type: ignore[no-untyped-def]
    x = torch.zeros(5, 9000, device="cuda")
    x[0, 100] = x[0, 5000] = 2.0          # a tie over two segments
    x[1] = -float("inf")                   # nothing is allowed already
    x[2, 7] = torch.finfo(torch.float32).min
    x[3, 4000], x[3, 4001] = float("inf"), -float("inf")
    x[4] = -0.0
    x[4, 8000] = 0.0                       # equal to -0
    mask = torch.full((5, 282), -1, dtype=torch.int32, device="cuda")
    got, ids = chroma_b200.process_logits(x, mask=mask, argmax=True, temperature=torch.tensor([0.5, 1, 2, 0, 0], device="cuda"))
    assert ids.tolist() == [100, 0, 0, 4000, 0]
    assert float(got[0, 100]) == 4.0 and float(got[2, 7]) == float(torch.finfo(torch.float32).min) / 2
    assert bool(torch.isneginf(got[1]).all()) and torch.equal(got[3], x[3])
    mask.zero_()
    got, ids = chroma_b200.process_logits(x, mask=mask, argmax=True)
    assert bool(torch.isneginf(got).all()) and ids.tolist() == [0] * 5
    ban = torch.tensor([[100, 5000]], dtype=torch.int32, device="cuda").expand(5, -1)
    got, ids = chroma_b200.process_logits(x, bias_ids=ban, bias=torch.full((5, 2), -float("inf"), device="cuda"), argmax=True)
    assert ids.tolist()[0] == 0 and bool(torch.isneginf(got[:, [100, 5000]]).all())


def test_temperatures_divide(gpu) -> None:  # type: ignore[no-untyped-def]
    # l / temperature is the correctly rounded quotient, bit for bit, of ordinary values and of extreme ones.
    g = torch.Generator(device="cuda").manual_seed(8)
    bits = torch.randint(-(2**31), 2**31, (40, 40000), generator=g, device="cuda").to(torch.int32)
    x = bits.view(torch.float32).clone()
    x[:20] = torch.randn(20, 40000, generator=g, device="cuda") * 5
    x[x.isnan()] = 0.0
    t = torch.rand(40, generator=g, device="cuda") + 0.3
    t[5], t[6], t[25], t[26] = 1e-20, 3e25, 1e-38, 1e30
    got = chroma_b200.process_logits(x, temperature=t)
    assert torch.equal(got, x / t[:, None])


def test_biases_add_up_in_list_order(gpu) -> None:  # type: ignore[no-untyped-def]
    x = torch.zeros(1, 300, device="cuda")
    values = torch.tensor([[1e8, 1.0, -1e8, 1.0] * 20], device="cuda")
    ids = torch.full((1, 80), 7, dtype=torch.int32, device="cuda")
    want = np.float32(0)
    for w in values[0].cpu().numpy():
        want = np.float32(want + w)
    assert float(chroma_b200.process_logits(x, bias_ids=ids, bias=values)[0, 7]) == float(want)


def test_refusals(gpu) -> None:  # type: ignore[no-untyped-def]
    x, more = case(2, 100, 6, 3, torch.float32, 1)
    call = chroma_b200.process_logits
    bad = [
        lambda: call(x.half()),
        lambda: call(x[0]),
        lambda: call(x.t()),
        lambda: call(x.cpu()),
        lambda: call(x, history=more["history"]),
        lambda: call(x, history=more["history"].long(), lengths=more["lengths"]),
        lambda: call(x, history=more["history"], lengths=more["lengths"][:1]),
        lambda: call(x, repetition=more["repetition"]),
        lambda: call(x, bias=more["bias"]),
        lambda: call(x, bias_ids=more["bias_ids"], bias=more["bias"][:, :2]),
        lambda: call(x, bias_ids=more["bias_ids"], bias=more["bias"].double()),
        lambda: call(x, mask=more["mask"][:, :3]),
        lambda: call(x, temperature=more["temperature"].double()),
        lambda: call(x, out=x.bfloat16()),
        lambda: call(x, out=x[:1].expand(2, -1)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was not refused")
    with pytest.raises(TypeError):
        call(x.tolist())
    assert call(x[:0]).shape == (0, 100)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,width,biases", [
    (300, 33, 40, 3), (160, 4097, 7000, 300), (80, 20011, 300, 9), (75, 16384, 6000, 400), (300, 1, 2, 1), (40, 70000, 9000, 7),
])
def test_many_rows(gpu, dtype, rows, vocab, width, biases) -> None:  # type: ignore[no-untyped-def]
    # So many that the entries that occurred and the others are processed by launches of their own.
    x, more = case(rows, vocab, width, biases, dtype, vocab + rows)
    want = ref.logits(x, **more)
    before = x.clone()
    got, ids = chroma_b200.process_logits(x, argmax=True, **more)
    scale = float(x.float().abs().max()) * 2 + width + 4 * biases + 2
    check(got, want, dtype, 2 * scale)
    assert torch.equal(x, before)
    np.testing.assert_array_equal(ids.cpu().numpy(), largest(got))
    again = x.clone()
    assert chroma_b200.process_logits(again, out=again, **more) is again
    assert torch.equal(again, got)
    # Rows at any address, in place.
    wide = torch.zeros(rows, vocab + 9, dtype=dtype, device="cuda")
    view = wide[:, 3 : 3 + vocab]
    view.copy_(x)
    _, same = chroma_b200.process_logits(view, out=view, argmax=True, **more)
    assert torch.equal(view, got) and torch.equal(same, ids)
    assert not wide[:, :3].any() and not wide[:, 3 + vocab :].any()


@pytest.mark.parametrize("left", ["history", "bias", "mask", "temperature", "repetition", "frequency", "presence", "prompts", "all"])
def test_any_part_may_be_missing_of_many_rows(gpu, left) -> None:  # type: ignore[no-untyped-def]
    x, more = case(200, 5000, 60, 9, torch.float32, 12)
    gone = {"history": ["history", "lengths", "prompts", "repetition", "presence", "frequency"],
            "bias": ["bias", "bias_ids"], "all": list(more)}.get(left, [left])
    more = {k: v for k, v in more.items() if k not in gone}
    got, ids = chroma_b200.process_logits(x, argmax=True, **more)
    check(got, ref.logits(x, **more), torch.float32, 200.0)
    np.testing.assert_array_equal(ids.cpu().numpy(), largest(got))
    assert torch.equal(chroma_b200.process_logits(x, **more), got)


def test_infinities_ties_and_nan_in_many_rows(gpu) -> None:  # type: ignore[no-untyped-def]
    x = torch.zeros(600, 9000, device="cuda").reshape(100, 6, 9000)
    x[:, 0, 100] = x[:, 0, 5000] = 2.0
    x[:, 1] = -float("inf")
    x[:, 2, 300] = x[:, 2, 8999] = float("nan")
    x[:, 3, 4000], x[:, 3, 4001] = float("inf"), -float("inf")
    x[:, 4] = -0.0
    x[:, 4, 8000] = 0.0
    x[:, 5, 4095], x[:, 5, 4096] = 1.0, 1.0
    x = x.reshape(600, 9000)
    got, ids = chroma_b200.process_logits(x, argmax=True)
    assert ids.reshape(100, 6).tolist() == [[100, 0, 300, 4000, 0, 4095]] * 100
    assert torch.equal(got.nan_to_num(7.0), x.nan_to_num(7.0))
    # The first of the equals has a bias of nothing; then the largest goes to an entry that occurred, and ties with it.
    listed = torch.tensor([[100, 4095, 300]], dtype=torch.int32, device="cuda").expand(600, -1)
    _, ids = chroma_b200.process_logits(x, bias_ids=listed, bias=torch.zeros(600, 3, device="cuda"), argmax=True)
    assert ids.reshape(100, 6).tolist() == [[100, 0, 300, 4000, 0, 4095]] * 100
    _, ids = chroma_b200.process_logits(x, bias_ids=listed, bias=torch.full((600, 3), -1.0, device="cuda"), argmax=True)
    assert ids.reshape(100, 6).tolist() == [[5000, 0, 300, 4000, 0, 4096]] * 100
    mask = torch.zeros(600, 282, dtype=torch.int32, device="cuda")
    got, ids = chroma_b200.process_logits(x, mask=mask, bias_ids=listed, bias=torch.zeros(600, 3, device="cuda"), argmax=True)
    assert bool(torch.isneginf(got).all()) and not ids.any()


def test_biases_of_many_rows_add_up_in_list_order(gpu) -> None:  # type: ignore[no-untyped-def]
    x = torch.zeros(300, 300, device="cuda")
    values = torch.tensor([[1e8, 1.0, -1e8, 1.0] * 100], device="cuda").expand(300, -1)
    for n in (80, 400):  # more than are kept in shared memory
        want = np.float32(0)
        for w in values[0, :n].cpu().numpy():
            want = np.float32(want + w)
        got = chroma_b200.process_logits(x, bias_ids=torch.full((300, n), 7, dtype=torch.int32, device="cuda"), bias=values[:, :n])
        assert torch.equal(got[:, 7], torch.full((300,), float(want), device="cuda")) and not got[:, 8:].any()
