"""Measured cases of the paged-cache operators: attention over pages (one new token, and prompts), the write of new
rows, the page operators, and the processing of logits.

``run`` with ``own`` false computes an operator in elementary torch operations in 32 bits; with ``own`` true it calls
``chroma_b200``. ``exact`` computes the floating outputs in 64 bits, one sequence after another.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# -- cases ----------------------------------------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # One user of the dev model (8 heads, 1 key-value head, width 16, fp32) with a short conversation: latency.
        {"name": "decode dev one user", "op": "decode", "type": "float32", "batch": 1, "heads": 8, "kv": 1, "dim": 16,
         "low": 160, "high": 160, "page": 16, "window": 0, "first": 0, "sinks": True, "lse": False},
        # The 120B-shaped model's decode batch: 128 sequences of up to 4,096 tokens, learned sinks.
        {"name": "decode batch 128", "op": "decode", "type": "bfloat16", "batch": 128, "heads": 64, "kv": 8, "dim": 64,
         "low": 1024, "high": 4096, "page": 64, "window": 0, "first": 0, "sinks": True, "lse": False},
        # Two long documents of uneven length: few rows, a long cache, odd lengths; the log-sum is wanted too.
        {"name": "decode long documents", "op": "decode", "type": "bfloat16", "batch": 2, "heads": 32, "kv": 8,
         "dim": 128, "low": 40001, "high": 131071, "page": 32, "window": 0, "first": 0, "sinks": False, "lse": True},
        # Short prompts of the dev model, each after a few tokens it already holds.
        {"name": "prompt dev ragged", "op": "prompt", "type": "float32", "batch": 3, "heads": 8, "kv": 1, "dim": 16,
         "low": 5, "high": 61, "prior": 37, "page": 16, "window": 0, "first": 0, "sinks": True, "lse": False},
        # The 20B-shaped model's prefill: four prompts of 2,048 tokens.
        {"name": "prompt 4 x 2048", "op": "prompt", "type": "bfloat16", "batch": 4, "heads": 64, "kv": 8, "dim": 64,
         "low": 2048, "high": 2048, "prior": 0, "page": 64, "window": 0, "first": 0, "sinks": True, "lse": False},
        # A chunk of a long stream that keeps its first 4 tokens and a window of 4,096 in sight.
        {"name": "prompt chunk, window", "op": "prompt", "type": "bfloat16", "batch": 1, "heads": 32, "kv": 8,
         "dim": 128, "low": 8192, "high": 8192, "prior": 8001, "page": 32, "window": 4096, "first": 4, "sinks": False,
         "lse": True},
        # New rows of one decode step of 128 sequences.
        {"name": "append step of 128", "op": "append", "type": "bfloat16", "batch": 128, "kv": 8, "dim": 64, "low": 1,
         "high": 1, "prior": 1000, "page": 64},
        # New rows of ragged prompts, about 16 thousand tokens.
        {"name": "append prompts", "op": "append", "type": "bfloat16", "batch": 16, "kv": 8, "dim": 64, "low": 63,
         "high": 2047, "prior": 129, "page": 64},
        # 128 slots of parallel samples: half continue, the others are forked anew from them, one row each.
        {"name": "pages fork step", "op": "step", "type": "bfloat16", "batch": 128, "kv": 8, "dim": 64, "layers": 4,
         "low": 100, "high": 2000, "rows": 1, "page": 64, "pages": 4096},
        # After many sequences have ended, half of the pool is empty: the rest moves to its front.
        {"name": "pages compact", "op": "compact", "type": "bfloat16", "batch": 64, "kv": 8, "dim": 64, "layers": 4,
         "low": 500, "high": 2500, "page": 64, "pages": 4096},
        # One user's logits over the vocabulary, 500 tokens behind them.
        {"name": "logits one user", "op": "logits", "type": "float32", "batch": 1, "vocab": 201088, "low": 500,
         "high": 500, "biases": 20},
        # A batch with histories of up to 4,096 tokens.
        {"name": "logits batch 64", "op": "logits", "type": "float32", "batch": 64, "vocab": 201088, "low": 50,
         "high": 4096, "biases": 50},
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng: random.Random) -> dict:
    kind = rng.choice(["float32", "bfloat16", "bfloat16", "bfloat16"])
    kv = rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([16, 64, 128] if kind == "float32" else [16, 64, 64, 80, 128, 128])
    return {"type": kind, "heads": kv * rng.choice([1, 3, 4, 7, 8]), "kv": kv, "dim": dim}


def draw(rng: random.Random) -> dict:
    op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "step", "compact", "logits", "logits"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "decode":
        case = {"op": op, **_heads(rng), "batch": _log(rng, 1, 256)}
        size = 4 if case["type"] == "float32" else 2
        most = min(131072, 1_000_000_000 // (case["batch"] * case["kv"] * case["dim"] * size * 2))
        high = _log(rng, 40, most)
        window = rng.choice([0, 0, 128, 1000])
        return {**case, "low": _log(rng, 1, high), "high": high, "page": page, "window": window,
                "first": rng.choice([0, 4, 17]) if window else 0, "sinks": rng.random() < 0.5,
                "lse": rng.random() < 0.5}
    if op == "prompt":
        case = {"op": op, **_heads(rng), "batch": _log(rng, 1, 8)}
        high = _log(rng, 16, 4096 // case["batch"])
        prior = rng.choice([0, _log(rng, 1, 4096 // case["batch"])])
        window = rng.choice([0, 0, 128, 1000])
        return {**case, "low": _log(rng, 1, high), "high": high, "prior": prior, "page": page, "window": window,
                "first": rng.choice([0, 4, 17]) if window else 0, "sinks": rng.random() < 0.5,
                "lse": rng.random() < 0.5}
    if op == "append":
        case = {"op": op, **_heads(rng), "batch": _log(rng, 1, 256)}
        del case["heads"]
        high = _log(rng, 1, max(1, 16384 // case["batch"]))
        return {**case, "low": _log(rng, 1, high), "high": high, "prior": _log(rng, 1, 1000), "page": page}
    if op in ("step", "compact"):
        heads = _heads(rng)
        batch, high = _log(rng, 2, 256), _log(rng, 20, 4000)
        need = batch * (-(-high // page) + 2)
        size = (4 if heads["type"] == "float32" else 2) * page * heads["kv"] * heads["dim"]
        layers = rng.choice([1, 2, 4])
        while need * layers * size > 700_000_000 and layers > 1:
            layers -= 1
        while need * layers * size > 700_000_000:
            high = max(20, high // 2)
            batch = max(2, batch // 2)
            need = batch * (-(-high // page) + 2)
        case = {"op": op, "type": heads["type"], "batch": batch, "kv": heads["kv"], "dim": heads["dim"],
                "layers": layers, "low": _log(rng, 1, high), "high": high, "page": page,
                "pages": need + _log(rng, 1, need)}
        return {**case, "rows": rng.choice([1, 1, 5, 33])} if op == "step" else case
    batch, vocab = _log(rng, 1, 64), rng.choice([4096, 32003, 50257, 128256, 201088])
    high = _log(rng, 1, 4096)
    return {"op": "logits", "type": rng.choice(["float32", "bfloat16"]), "batch": batch, "vocab": vocab,
            "low": _log(rng, 1, high), "high": high, "biases": _log(rng, 1, 300)}


def _spread(case: dict, low: str = "low", high: str = "high") -> list[int]:
    """One number per sequence, spread over [low, high] in a fixed order; the first is the largest."""
    a, b = case[low], case[high]
    return [b - int((b - a) * ((i * 0.6180339887498949) % 1.0)) for i in range(case["batch"])]


def _visible(p: int, window: int, first: int) -> int:
    """How many positions a query at position p sees."""
    if window <= 0 or p < window:
        return p + 1
    return window + min(first, p + 1 - window)


def work(case: dict) -> dict:
    size = 2 if case["type"] == "bfloat16" else 4
    op = case["op"]
    if op in ("decode", "prompt"):
        heads, kv, dim = case["heads"], case["kv"], case["dim"]
        pairs = keys = tokens = 0
        for n in _spread(case):
            if op == "decode":
                seen = _visible(n - 1, case["window"], case["first"])
                pairs, keys, tokens = pairs + seen, keys + seen, tokens + 1
                continue
            total, w, f = n + case["prior"], case["window"], case["first"]
            pairs += sum(_visible(p, w, f) for p in range(case["prior"], total))
            start = max(0, case["prior"] - w + 1) if w > 0 else 0
            keys, tokens = keys + total - start + min(f, start), tokens + n
        return {"bytes": 2 * keys * kv * dim * size + 2 * tokens * heads * dim * size, "flops": 4 * pairs * heads * dim}
    if op == "append":
        return {"bytes": 4 * sum(_spread(case)) * case["kv"] * case["dim"] * size, "flops": 0}
    if op == "logits":
        b, v = case["batch"], case["vocab"]
        return {"bytes": 2 * b * v * size + b * v // 8 + 4 * sum(_spread(case)), "flops": 6 * b * v}
    row = case["kv"] * case["dim"] * size * case["layers"] * 2
    lengths, page = _spread(case), case["page"]
    width = _width(case)
    tables = 2 * case["batch"] * width * 4
    if op == "step":
        kept = lengths[: (case["batch"] + 1) // 2]
        forked = [kept[i % len(kept)] for i in range(case["batch"] - len(kept))]
        return {"bytes": tables + 2 * sum(n % page for n in forked) * row, "flops": 0}
    held = sum(-(-n // page) for n in lengths)
    moved = held * (case["pages"] - held) // case["pages"]  # expected for pages spread over the whole pool
    return {"bytes": tables + 2 * moved * page * row, "flops": 0}


# -- inputs ---------------------------------------------------------------------------------------------------------


def _width(case: dict) -> int:
    """Table entries per sequence."""
    most = case["high"] + case.get("prior", 0) + case.get("rows", 0)
    return -(-most // case["page"]) + 1


def _device(values: list[int]) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32).cuda()


def _table(lengths: list[int], page: int, width: int, pages: int, g: torch.Generator) -> torch.Tensor:
    """Each sequence's pages, scattered over the pool; -1 past the last."""
    held = torch.tensor([-(-n // page) for n in lengths], device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < held[:, None]
    order = torch.randperm(pages, generator=g, device="cuda")[: int(held.sum())]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    table[at] = order.to(torch.int32)
    return table


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, op = _TYPES[case["type"]], case["op"]

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device="cuda", dtype=kind)

    def uniform(low: float, high: float, *shape: int) -> torch.Tensor:
        return low + (high - low) * torch.rand(*shape, generator=g, device="cuda")

    state = {"case": case}
    if op == "logits":
        b, v = case["batch"], case["vocab"]
        lengths = _spread(case)
        state |= {
            "logits": (normal(b, v) * 3).to(kind), "lengths": _device(lengths),
            "prompts": _device([n // 3 for n in lengths]),
            # Token ids follow a steep distribution, as text does, so many occur often.
            "history": (v * torch.rand(b, max(lengths), generator=g, device="cuda") ** 6).to(torch.int32),
            "repetition": uniform(1.0, 1.3, b), "presence": uniform(0.0, 0.6, b), "frequency": uniform(0.0, 0.4, b),
            "temperature": uniform(0.6, 1.2, b),
            "bias_ids": ((torch.randint(v, (b, 1), generator=g, device="cuda")
                          + torch.arange(case["biases"], device="cuda") * 13) % v).to(torch.int32),
            "bias": uniform(-4.0, 4.0, b, case["biases"]),
            "mask": torch.randint(-(2**31), 2**31, (b, -(-v // 32)), generator=g, device="cuda").to(torch.int32),
        }
        return state
    counts = _spread(case)
    prior, page, width = case.get("prior", 0), case["page"], _width(case)
    lengths = [n + prior for n in counts]
    held = sum(-(-n // page) for n in lengths)
    pages = case.get("pages", held + 7)
    pool = (case["layers"], pages) if "layers" in case else (pages,)
    state |= {
        "keys": normal(*pool, page, case["kv"], case["dim"]), "values": normal(*pool, page, case["kv"], case["dim"]),
        "table": _table(lengths, page, width, pages, g), "lengths": _device(lengths),
    }
    if op == "step":
        kept = (case["batch"] + 1) // 2
        state["parents"] = _device([i if i < kept else (i - kept) % kept for i in range(case["batch"])])
        state["counts"] = _device([case["rows"]] * case["batch"])
    if op in ("prompt", "append"):
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        state["starts"], tokens = _device(offsets), offsets[-1]
    if op == "append":
        state |= {"new_keys": normal(tokens, case["kv"], case["dim"]),
                  "new_values": normal(tokens, case["kv"], case["dim"])}
    if op in ("decode", "prompt"):
        tokens = case["batch"] if op == "decode" else tokens
        state["q"] = (normal(tokens, case["heads"], case["dim"]) * 1.5).to(kind)
        state["scale"] = case["dim"] ** -0.5
        state["sinks"] = normal(case["heads"]) if case["sinks"] else None
    return state


# -- the operators --------------------------------------------------------------------------------------------------


def run(state: dict):
    return _own(state) if own else _plain(state)


def _own(s: dict):
    import chroma_b200

    case = s["case"]
    op = case["op"]
    if op in ("decode", "prompt"):
        return chroma_b200.paged_attention(
            s["q"], s["keys"], s["values"], s["table"], s["lengths"], s.get("starts"), scale=s["scale"],
            window=case["window"], first=case["first"], sinks=s["sinks"], lse=case["lse"])
    if op == "append":
        chroma_b200.paged_append(s["keys"], s["values"], s["new_keys"], s["new_values"], s["table"], s["lengths"],
                                 s["starts"])
        return s["keys"], s["values"]
    if op == "step":
        table, lengths, info = chroma_b200.step_pages(s["table"], s["lengths"], s["parents"], s["counts"], s["keys"],
                                                      s["values"])
        return table, lengths, info, s["keys"], s["values"]
    if op == "compact":
        table, info = chroma_b200.compact_pages(s["table"], s["lengths"], s["keys"], s["values"])
        return table, info, s["keys"], s["values"]
    return chroma_b200.process_logits(
        s["logits"], history=s["history"], lengths=s["lengths"], prompts=s["prompts"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"],
        temperature=s["temperature"], argmax=True)


def _plain(s: dict):
    op = s["case"]["op"]
    if op in ("decode", "prompt"):
        return _attention(s)
    if op == "append":
        return _append(s)
    if op == "step":
        return _step(s)
    if op == "compact":
        return _compact(s)
    return _logits(s)


def _owners(starts: torch.Tensor, tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequence of each row and its number within it."""
    rows = torch.arange(tokens, device="cuda")
    owner = torch.searchsorted(starts, rows, right=True) - 1
    return owner, rows - starts[owner]


def _attention(s: dict):
    case, q, table, lengths = s["case"], s["q"], s["table"], s["lengths"]
    kv, dim, page = case["kv"], case["dim"], case["page"]
    group, batch, tokens = case["heads"] // kv, table.shape[0], q.shape[0]
    if case["op"] == "decode":
        owner, number, most = torch.arange(batch, device="cuda"), torch.zeros_like(lengths), 1
        new = torch.ones_like(lengths)
    else:
        owner, number = _owners(s["starts"], tokens)
        new, most = s["starts"].diff(), case["high"]
    at = torch.arange(table.shape[1] * page, device="cuda")
    ids = table[:, at // page].long()
    there = (ids >= 0) & (at < lengths[:, None])
    # [batch, kv, rows, dim] in 32 bits; rows that are not there are zero.
    k, v = (torch.where(there[..., None, None], x[ids.clamp(min=0), at % page].float(), 0.0).transpose(1, 2)
            for x in (s["keys"], s["values"]))
    rows = torch.zeros(batch, most, kv, group, dim, device="cuda")
    rows[owner, number] = q.float().view(tokens, kv, group, dim)
    rows = rows.permute(0, 2, 3, 1, 4).reshape(batch, kv, group * most, dim)
    scores = (rows @ k.transpose(2, 3)).view(batch, kv, group, most, -1) * s["scale"]
    p = (lengths - new)[:, None] + torch.arange(most, device="cuda")
    seen = there[:, None, :] & (at <= p[..., None])
    if case["window"] > 0:
        seen &= (at > p[..., None] - case["window"]) | (at < case["first"])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sinks = s["sinks"].float().view(1, kv, group, 1, 1)
        top = torch.maximum(top, sinks)
    top = top.clamp(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sinks - top).exp()
    out = (weights.view(batch, kv, group * most, -1) @ v).view(batch, kv, group, most, dim)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4)[owner, number].reshape(tokens, kv * group, dim).to(q.dtype)
    if not case["lse"]:
        return out
    lse = (total.log() + top).squeeze(-1)
    return out, lse.permute(0, 3, 1, 2)[owner, number].reshape(tokens, kv * group)


def _append(s: dict):
    page, starts = s["case"]["page"], s["starts"]
    owner, number = _owners(starts, s["new_keys"].shape[0])
    p = s["lengths"][owner] - starts.diff()[owner] + number
    ids = s["table"][owner, p // page].long()
    s["keys"][ids, p % page] = s["new_keys"]
    s["values"][ids, p % page] = s["new_values"]
    return s["keys"], s["values"]


def _step(s: dict):
    page, pages = s["case"]["page"], s["keys"].shape[1]
    parents, counts = s["parents"].long(), s["counts"]
    slots, width = s["table"].shape
    at = torch.arange(width, device="cuda")
    old = torch.where(parents >= 0, s["lengths"][parents.clamp(min=0)], 0)
    lengths = old + torch.where(parents >= 0, counts, 0)
    held, need = -(-old // page), -(-lengths // page)
    table = torch.where(at < held[:, None], s["table"][parents.clamp(min=0)], -1)
    # The holder of a page with the most rows in it, the lowest slot among equals.
    used = (old[:, None] - at * page).clamp(0, page)
    slot = torch.arange(slots, device="cuda")
    rank = used * slots + (slots - 1 - slot)[:, None]
    place = torch.where(table >= 0, table, pages).long()
    keeper = torch.full((pages + 1,), -1, device="cuda").scatter_reduce_(0, place.view(-1), rank.view(-1), "amax")
    last = (held - 1).clamp(min=0).long()[:, None]
    mine = rank.gather(1, last)[:, 0]
    shared = keeper[place.gather(1, last)[:, 0]] != mine
    copy = (old % page != 0) & (lengths > old) & shared
    free = torch.argsort((keeper[:pages] >= 0).int(), stable=True).to(torch.int32)
    left = (keeper[:pages] < 0).sum()
    takes = copy + (need - held)
    base = takes.cumsum(0) - takes
    fresh = (at >= held[:, None]) & (at < need[:, None])
    index = base[:, None] + copy[:, None] + at - held[:, None]
    source = table.gather(1, last)[:, 0]
    table = torch.where(fresh, free[index.clamp(0, pages - 1)], table)
    target = torch.where(copy, free[base.clamp(0, pages - 1)], source)
    table.scatter_(1, last, target[:, None])
    moved = torch.nonzero(copy)[:, 0]
    rows = torch.arange(page, device="cuda") < (old[moved] % page)[:, None]
    a, b = source[moved].long(), target[moved].long()
    for pool in (s["keys"], s["values"]):
        pool[:, b] = torch.where(rows[None, :, :, None, None], pool[:, a], pool[:, b])
    info = torch.stack([left - takes.sum(), torch.zeros_like(left), copy.sum()]).to(torch.int32)
    return table, lengths, info, s["keys"], s["values"]


def _compact(s: dict):
    page, pages = s["case"]["page"], s["keys"].shape[1]
    at = torch.arange(s["table"].shape[1], device="cuda")
    there = (at < -(-s["lengths"] // page)[:, None]) & (s["table"] >= 0)
    held = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    held[torch.where(there, s["table"], pages).view(-1).long()] = True
    held = held[:pages]
    count = held.sum()
    place = torch.arange(pages, device="cuda")
    source = torch.nonzero(held & (place >= count))[:, 0]
    target = torch.nonzero(~held & (place < count))[:, 0]
    to = place.clone()
    to[source] = target
    for pool in (s["keys"], s["values"]):
        pool[:, target] = pool[:, source]
    table = torch.where(there, to[s["table"].clamp(min=0).long()].to(torch.int32), -1)
    return table, torch.stack([count, torch.full_like(count, source.numel())]).to(torch.int32), s["keys"], s["values"]


def _logits(s: dict):
    batch, vocab = s["logits"].shape
    place = torch.arange(s["history"].shape[1], device="cuda")
    there = (place < s["lengths"][:, None]).int()
    ids = s["history"].long()
    seen = torch.zeros(batch, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, there)
    made = there * (place >= s["prompts"][:, None])
    count = torch.zeros(batch, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, made)
    x = s["logits"].float()
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0)
    x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), s["bias"])
    x = x / s["temperature"][:, None]
    v = torch.arange(vocab, device="cuda")
    allowed = ((s["mask"][:, v // 32] >> (v % 32).int()) & 1) != 0
    x = torch.where(allowed, x, -math.inf).to(s["logits"].dtype)
    # The lowest index among equals.
    best = torch.where(x == x.amax(1, keepdim=True), v, vocab).amin(1)
    return x, best


# -- in 64 bits -----------------------------------------------------------------------------------------------------


def exact(case: dict, seed: int):
    op = case["op"]
    if op == "logits":
        return _exact_logits(prepare(case, seed))
    if op not in ("decode", "prompt"):
        return None  # rows and page numbers: nothing is computed
    s = prepare(case, seed)
    counts = [1] * case["batch"] if op == "decode" else _spread(case)
    totals = [n + case.get("prior", 0) for n in _spread(case)]
    group, page = case["heads"] // case["kv"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    begin = 0
    for b, (new, total) in enumerate(zip(counts, totals)):
        pages = s["table"][b, : -(-total // page)].long()
        p = torch.arange(total - new, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None, :]
        hidden = j > p
        if case["window"] > 0:
            hidden = hidden | ((p - j >= case["window"]) & (j >= case["first"]))
        for h in range(case["heads"]):
            k = s["keys"][pages, :, h // group].reshape(-1, case["dim"])[:total].double()
            v = s["values"][pages, :, h // group].reshape(-1, case["dim"])[:total].double()
            x = torch.einsum("qd,kd->qk", s["q"][begin : begin + new, h].double(), k) / math.sqrt(case["dim"])
            x[hidden] = -math.inf
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(new, 1)], dim=1)
            lse[begin : begin + new, h] = torch.logsumexp(x, dim=1)
            out[begin : begin + new, h] = torch.softmax(x, dim=1)[:, :total] @ v
        begin += new
    return (out, lse) if case["lse"] else out


def _exact_logits(s: dict):
    rows = []
    for b, (n, p) in enumerate(zip(s["lengths"].tolist(), s["prompts"].tolist())):
        x = s["logits"][b].double()
        tokens = s["history"][b, :n].long()
        r = float(s["repetition"][b])
        heard = tokens.unique()
        x[heard] *= torch.where(x[heard] > 0, 1 / r, r).double()
        times = torch.bincount(tokens[p:], minlength=x.numel()).double()
        x -= float(s["frequency"][b]) * times + float(s["presence"][b]) * times.clamp(max=1)
        x[s["bias_ids"][b].long()] += s["bias"][b].double()
        x /= float(s["temperature"][b])
        bits = (s["mask"][b][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x[bits.view(-1)[: x.numel()] == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows), None
