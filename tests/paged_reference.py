"""Plain forms of the paged-cache operators and of logits processing: 64 bits, one sequence, one token after another."""

from __future__ import annotations

import numpy as np
import torch


def attention(q, keys, values, table, lengths, starts=None, *, scale, window=0, first=0, sinks=None):  # type: ignore[no-untyped-def]
    """(output, log of the sums), in float64 on the CPU; and the largest value magnitude and score error scale seen."""
    q, keys, values = q.double().cpu(), keys.double().cpu(), values.double().cpu()
    table, lengths = table.cpu().tolist(), lengths.cpu().tolist()
    begins = list(range(len(lengths) + 1)) if starts is None else starts.cpu().tolist()
    tokens, heads, dim = q.shape
    pages, page, kv, _ = keys.shape
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((tokens, heads), -float("inf"), dtype=torch.float64)
    most_value = most_score = 0.0
    sink = None if sinks is None else sinks.double().cpu()
    for b, n in enumerate(lengths):
        n = min(max(n, 0), len(table[b]) * page)
        have = [j for j in range(n) if 0 <= table[b][j // page] < pages]
        at = torch.tensor(have, dtype=torch.int64)
        ids = torch.tensor([table[b][j // page] for j in have], dtype=torch.int64)
        k, v = keys[ids, at % page], values[ids, at % page]  # [n, kv, dim]
        for t in range(begins[b], begins[b + 1]):
            p = n - begins[b + 1] + t
            seen = (at <= p) & ((at > p - window) | (at < first) if window > 0 else torch.ones_like(at, dtype=torch.bool))
            ks, vs = k[seen].repeat_interleave(heads // kv, 1), v[seen].repeat_interleave(heads // kv, 1)
            s = torch.einsum("hd,nhd->hn", q[t], ks) * scale
            if ks.numel():
                most_value = max(most_value, float(vs.abs().max()))
                most_score = max(most_score, abs(scale) * float(q[t].norm(dim=-1).max() * ks.norm(dim=-1).max()))
            joined = s if sink is None else torch.cat([s, sink[:, None]], 1)
            if joined.shape[1] == 0:
                continue
            lse[t] = torch.logsumexp(joined, 1)
            if ks.numel():
                out[t] = torch.einsum("hn,nhd->hd", torch.exp(s - lse[t][:, None]), vs)
    return out, lse, most_value, most_score


def attention_tolerance(dtype, dim, most_value, most_score):  # type: ignore[no-untyped-def]
    """(absolute, relative) tolerance of an output, and the absolute one of a log-sum.

    A score is a sum of ``dim`` products in fp32: four standard deviations of its rounding are 4 sqrt(dim) 2^-24 of
    |scale| |q| |k|. A relative error e of every weight moves the quotient by at most 2 e max|v|. The special-function
    unit's 2^x and the order of the sums add 2^-20. In bf16 the weights are rounded to 8 bits before the product with
    the values (2^-8 each at most; they are independent, and half of that is allowed for their sum), and so is the
    result (2^-8).
    """
    score = 4 * dim**0.5 * 2.0**-24 * most_score
    weight = 2 * score + 2.0**-20
    unit = 2.0**-8 if dtype is torch.bfloat16 else 0.0
    return (weight + unit / 2) * max(most_value, 1.0), unit + 2.0**-22, score + 2.0**-20


def step(table, lengths, parents, counts, pages, page):  # type: ignore[no-untyped-def]
    """(table, lengths, info, copies) of one step, copies as (source, target, rows)."""
    slots, width = table.shape
    new = np.full((slots, width), -1, np.int64)
    old = np.zeros(slots, np.int64)
    rows = np.zeros(slots, np.int64)
    for s, p in enumerate(parents):
        if not 0 <= p < slots:
            continue
        old[s] = min(max(lengths[p], 0), width * page)
        rows[s] = min(old[s] + max(counts[s], 0), width * page)
        for m in range(-(-old[s] // page)):
            new[s, m] = table[p, m] if 0 <= table[p, m] < pages else -1
    holders: dict[int, list[tuple[int, int]]] = {}
    for s in range(slots):
        for m in range(width):
            if new[s, m] >= 0:
                holders.setdefault(int(new[s, m]), []).append((int(min(page, old[s] - m * page)), -s))
    free = [p for p in range(pages) if p not in holders]
    have, taken, copies = len(free), 0, []

    def give() -> int:
        nonlocal taken
        taken += 1
        return free[taken - 1] if taken <= have else -1

    result = new.copy()
    for s in range(slots):
        part, last = int(old[s] % page), int(-(-old[s] // page)) - 1
        if part and rows[s] > old[s] and new[s, last] >= 0 and max(holders[int(new[s, last])]) != (part, -s):
            result[s, last] = give()
            copies.append((int(new[s, last]), int(result[s, last]), part))
        for m in range(last + 1, int(-(-rows[s] // page))):
            result[s, m] = give()
    short = max(0, taken - have)
    copies = [] if short else copies
    return result, rows, [max(0, have - taken), short, len(copies)], copies


def compact(table, lengths, pages, page):  # type: ignore[no-untyped-def]
    slots, width = table.shape
    there = np.zeros((slots, width), bool)
    for s in range(slots):
        for m in range(-(-min(max(int(lengths[s]), 0), width * page) // page)):
            there[s, m] = 0 <= table[s, m] < pages
    held = sorted(set(int(x) for x in table[there]))
    n = len(held)
    holes = [p for p in range(n) if p not in set(held)]
    moves = dict(zip([p for p in held if p >= n], holes))
    new = np.full((slots, width), -1, np.int64)
    for s, m in zip(*np.nonzero(there)):
        new[s, m] = moves.get(int(table[s, m]), int(table[s, m]))
    return new, [n, len(moves)], [(a, b, page) for a, b in moves.items()]


def logits(x, *, history=None, lengths=None, prompts=None, repetition=None, presence=None, frequency=None,  # type: ignore[no-untyped-def]
           bias_ids=None, bias=None, mask=None, temperature=None):
    """float64 results, before they are rounded to the type of ``x``."""
    x = x.double().cpu().numpy().copy()
    get = lambda t, b, d: d if t is None else float(t[b])  # noqa: E731
    for b in range(x.shape[0]):
        heard: set[int] = set()
        times: dict[int, int] = {}
        if history is not None:
            for i, t in enumerate(history[b].tolist()[: max(0, int(lengths[b]))]):
                if 0 <= t < x.shape[1]:
                    heard.add(t)
                    if prompts is None or i >= int(prompts[b]):
                        times[t] = times.get(t, 0) + 1
        r = get(repetition, b, 1.0)
        for t in heard:
            x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
        for t, c in times.items():
            x[b, t] -= get(frequency, b, 0.0) * c + get(presence, b, 0.0)
        if bias_ids is not None:
            for t, w in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= t < x.shape[1]:
                    x[b, t] += w
        if get(temperature, b, 0.0) != 0:
            x[b] /= get(temperature, b, 0.0)
        if mask is not None:
            words = mask[b].cpu().numpy().astype(np.int64) & 0xFFFFFFFF
            v = np.arange(x.shape[1])
            x[b, ((words[v // 32] >> (v % 32)) & 1) == 0] = -np.inf
    return x
