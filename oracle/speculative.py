"""The speculative serving step by its definitions, on the CPU in 64 bits.

Plain loops over requests, heads and tokens: paged plan, append, prompt and
tree attention, draft verification.  Test infrastructure only.
"""

from __future__ import annotations

import torch


def ancestors(parents: list[int]) -> list[list[int]]:
    """For each token the indices of itself and its ancestors."""
    out: list[list[int]] = []
    for t, p in enumerate(parents):
        out.append(([] if p < 0 else out[p]) + [t])
    return out


def tree_words(parents: list[int]) -> list[int]:
    """The same sets as signed 64-bit words."""
    words = [sum(1 << a for a in row) for row in ancestors(parents)]
    return [w - (1 << 64) if w >> 63 else w for w in words]


def plan(context, new, table, free, head, page_size, num_tokens, parents=None, reserved=None):
    """(cu, slots, positions, masks, table, head, missing) as Python lists."""
    table = [list(row) for row in table]
    width, pool = len(table[0]), list(free[head:])
    cu, slots, positions, masks = [0], [], [], []
    given = missing = 0
    for b, (c, n) in enumerate(zip(context, new)):
        reach = c if reserved is None else max(c, reserved[b])
        have, want = -(-reach // page_size), -(-(c + n) // page_size)
        for col in range(have, want):
            if col >= width:
                missing += 1
                continue
            if given < len(pool):
                table[b][col] = pool[given]
                given += 1
            else:
                table[b][col] = -1
                missing += 1
        rows = None if parents is None else parents[cu[-1]:cu[-1] + n]
        for t in range(n):
            col, row = divmod(c + t, page_size)
            page = table[b][col] if col < width else -1
            slots.append(page * page_size + row if page >= 0 else -1)
            positions.append(c + (t if rows is None else len(ancestors(rows)[t]) - 1))
            masks.append(0 if rows is None else tree_words(rows)[t])
        cu.append(cu[-1] + n)
    rest = num_tokens - len(slots)
    return (cu, slots + [-1] * rest, positions + [0] * rest, masks + [0] * rest, table,
            head + given, missing)


def attend(q, k, v, visible, scale):
    """One head: q [T, Dk], k [S, Dk], v [S, Dv], visible [T, S] -> (out, lse, size).

    ``size`` is sum_j p_j |v_j|, the scale of the error that rounding the
    weights makes.  Keys that a row does not see do not enter it, whatever
    they hold.
    """
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((q.shape[0],), float("-inf"), dtype=torch.float64)
    for t in range(q.shape[0]):
        seen = visible[t].nonzero()[:, 0]
        if seen.numel() == 0:
            continue
        s = k[seen] @ q[t] * scale
        lse[t] = torch.logsumexp(s, 0)
        if torch.isinf(lse[t]) and lse[t] < 0:
            continue
        p = torch.exp(s - lse[t])
        out[t] = p @ v[seen]
        size[t] = p @ v[seen].abs()
    return out, lse, size


def prompt_attention(q, k, v, cu_q, cu_k, scale):
    """(out [T, H, Dv], lse [T, H], size) of packed causal prompts."""
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        n, m = q1 - q0, k1 - k0
        visible = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
        for h in range(q.shape[1]):
            out[q0:q1, h], lse[q0:q1, h], size[q0:q1, h] = attend(
                q[q0:q1, h], k[k0:k1, h // group], v[k0:k1, h // group], visible, scale)
    return out, lse, size


def tree_attention(q, k_cache, v_cache, table, context, cu, masks, scale):
    """(out, lse, size) of drafted tokens over the paged cache.

    ``masks``: per token the list of tree indices it sees, or None (causal).
    Places whose page is not in the cache are absent.
    """
    pages, ps, hkv, _ = k_cache.shape
    group = q.shape[1] // hkv
    out = torch.zeros(q.shape[0], q.shape[1], v_cache.shape[3], dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    for b in range(len(cu) - 1):
        q0, q1 = cu[b], cu[b + 1]
        n, c = q1 - q0, context[b]
        places = [p for p in range(c + n)
                  if p // ps < len(table[b]) and 0 <= table[b][p // ps] < pages]
        page = torch.tensor([table[b][p // ps] for p in places], dtype=torch.long)
        row = torch.tensor([p % ps for p in places], dtype=torch.long)
        visible = torch.zeros(n, len(places), dtype=torch.bool)
        for t in range(n):
            sees = set(range(t + 1)) if masks is None else set(masks[q0 + t])
            for i, p in enumerate(places):
                visible[t, i] = p < c or (p - c) in sees
        for h in range(q.shape[1]):
            out[q0:q1, h], lse[q0:q1, h], size[q0:q1, h] = attend(
                q[q0:q1, h], k_cache[page, row, h // group], v_cache[page, row, h // group],
                visible, scale)
    return out, lse, size


def verify(logits, tokens, parents, cu, most, coin, noise, temps, probs=None):
    """(tokens, path, accepted) as lists; every request walked by the definition."""
    outs, paths, counts = [], [], []
    for b in range(len(cu) - 1):
        s, n = cu[b], cu[b + 1] - cu[b]
        if n == 0:
            outs.append([-1] * most)
            paths.append([-1] * most)
            counts.append(0)
            continue
        temp = float(temps[b])

        def target(node):
            x = logits[s + node].double()
            x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
            return x if temp == 0 else torch.softmax(x / temp, 0)

        cur, path, left = 0, [0], None
        while True:
            p = target(cur)
            left, rem, moved = p.clone(), 1.0, False
            for c in range(1, n):
                if parents[s + c] != cur:
                    continue
                x = int(tokens[s + c])
                if temp == 0:
                    if int(p.argmax()) == x:
                        moved = True
                elif probs is not None:
                    q = probs[s + c].double()
                    if float(coin[s + c]) * float(q[x]) < float(p[x]):
                        moved = True
                    else:
                        left = (p - q).clamp_min(0)
                else:
                    if float(coin[s + c]) * rem < float(left[x]):
                        moved = True
                    else:
                        rem = max(0.0, rem - float(left[x]))
                        left[x] = 0
                if moved:
                    cur = c
                    path.append(c)
                    break
            if not moved:
                break
        if temp == 0:
            last = int(p.argmax())
        else:
            if not bool((left > 0).any()):
                left = p
            last = int((left / noise[b].double()).argmax())
        got = [int(tokens[s + c]) for c in path[1:]] + [last]
        counts.append(len(path) - 1)
        outs.append(got + [-1] * (most - len(got)))
        paths.append(path + [-1] * (most - len(path)))
    return outs, paths, counts
