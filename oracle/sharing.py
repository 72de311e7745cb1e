"""Requests that share a prompt, by the operators' definitions: on the CPU, in 64 bits.

Plain loops over requests, heads and tokens: linear attention, forked, freed and
compacted pages, adjusted logits.  Test infrastructure only.
"""

from __future__ import annotations

import torch


def linear_attention(q, k, v, log_decay, cu, scale, state=None):
    """(out, size, state, state size) of packed requests, token by token.

    ``state`` [requests, H, Dk, Dv] or None.  The sizes are the same sums over magnitudes.
    """
    q, k, v = q.double(), k.double(), v.double()
    total, h, dv = v.shape
    dk = q.shape[2]
    q = q.repeat_interleave(h // q.shape[1], dim=1) * scale
    k = k.repeat_interleave(h // k.shape[1], dim=1)
    g = log_decay.double().clamp_max(0.0).expand(total, h)
    out, size = torch.zeros_like(v), torch.zeros_like(v)
    n = len(cu) - 1
    start = torch.zeros(n, h, dk, dv) if state is None else state
    ends, weights = start.double().clone(), start.double().abs()
    for b in range(n):
        s, a = ends[b], weights[b]
        for t in range(cu[b], cu[b + 1]):
            keep = g[t].exp()[:, None, None]
            s = s * keep + k[t][:, :, None] * v[t][:, None, :]
            a = a * keep + (k[t][:, :, None] * v[t][:, None, :]).abs()
            out[t] = torch.einsum("hk,hkv->hv", q[t], s)
            size[t] = torch.einsum("hk,hkv->hv", q[t].abs(), a)
        ends[b], weights[b] = s, a
    return out, size, ends, weights


def pages_of(tokens, page_size):
    return -(-tokens // page_size)


def fork(context, table, sources, targets, free, head, page_size):
    """(context, table, copy_from, copy_to, copy_rows, head, missing) as Python lists."""
    context, table = list(context), [list(row) for row in table]
    width, n, missing = len(table[0]), len(context), 0
    named = [(s, t) for s, t in zip(sources, targets) if 0 <= s < n and 0 <= t < n]
    froms = {s for s, _ in named}
    seen, lists = set(), ([], [], [])
    old_context, old_table = list(context), [list(row) for row in table]
    for s, t in zip(sources, targets):
        move = (-1, -1, 0)
        if 0 <= s < n and 0 <= t < n and t not in froms and t not in seen:
            full, part = divmod(old_context[s], page_size)
            row, length = [-1] * width, 0
            if pages_of(old_context[s], page_size) > width or (part and head >= len(free)):
                missing += 1
            else:
                row[:full], length = old_table[s][:full], old_context[s]
                if part:
                    row[full] = free[head]
                    move = (old_table[s][full], free[head], part)
                    head += 1
            table[t], context[t] = row, length
        if 0 <= s < n and 0 <= t < n:
            seen.add(t)
        for out, x in zip(lists, move):
            out.append(x)
    return (context, table, *lists, head, missing)


def free(table, reserved, keep, listed, head, page_size):
    """(free list, head): the pages that come back stand in front of the old head."""
    kept, gone = set(), set()
    for row, have, stay in zip(table, reserved, keep):
        have = max(have, 0)
        stay = pages_of(min(max(stay, 0), have), page_size)
        kept |= set(row[:stay])
        gone |= set(row[stay:min(pages_of(have, page_size), len(row))])
    back = sorted(p for p in gone - kept if p >= 0)
    listed = list(listed)
    back = back[max(0, len(back) - head):]
    listed[head - len(back):head] = back
    return listed, head - len(back)


def compact(table, reserved, listed, head, page_size):
    """(table, free list, head, moves)."""
    held = [row[:pages_of(max(n, 0), page_size)] for row, n in zip(table, reserved)]
    used = {p for row in held for p in row if p >= 0}
    spare = {p for p in listed[head:] if p >= 0} - used
    low = set(sorted(used | spare)[:len(used)])
    moves = list(zip(sorted(used - low), sorted(spare & low)))
    to = dict(moves)
    width = len(table[0])
    rows = [[to.get(p, p) for p in row] + [-1] * (width - len(row)) for row in held]
    rest = sorted((used | spare) - low)
    listed = list(listed)
    listed[len(listed) - len(rest):] = rest
    return rows, listed, len(listed) - len(rest), moves


def adjust(row, prompt, answer, repetition=1.0, presence=0.0, frequency=0.0, biases=(),
           allowed=None):
    """(row, size): one row's logits; ``biases`` of (token, value), ``allowed`` a set."""
    x = row.double().clone()
    size = x.abs()
    counts: dict[int, int] = {}
    for t in answer:
        counts[t] = counts.get(t, 0) + 1
    for t in set(prompt) | set(counts):
        if 0 <= t < x.numel():
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
            c = counts.get(t, 0)
            size[t] = x[t].abs()
            if c:
                x[t] -= frequency * c + presence
                size[t] += abs(frequency) * c + abs(presence)
    for t, value in biases:
        if 0 <= t < x.numel():
            x[t] += value
            size[t] += abs(value)
    if allowed is not None:
        out = torch.ones(x.numel(), dtype=torch.bool)
        out[list(allowed)] = False
        x[out] = float("-inf")
    return x, size
