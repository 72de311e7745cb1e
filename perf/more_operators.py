"""Cases of serving requests that share a prompt: their linear attention, their pages, their logits.

Six operations, as a server that answers with several continuations of a prompt uses them:

  linear   linear attention with a decay for each head over packed prompts, states kept
  step     the same attention for one token of every request
  fork     rows of a paged cache that share another's full pages, and a copy of its last one
  free     pages that no request holds any more, back to the free list
  compact  pages moved to the lowest places of the pool
  logits   penalties for repeated tokens, biases and grammar masks on logits

``run`` computes them with elementary torch operations in 32 bits (running sums of decays
in 64), or, with ``own`` set, through this package's operators.  ``exact`` restates them
token by token and request by request in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    # The recurrent layers of the 27-layer model: 32 heads, 128 wide.
    kda = {"heads": 32, "q_heads": 32, "k_heads": 32, "dk": 128, "dv": 128}
    # Queries and keys shared by groups of value heads.
    shared = {"heads": 24, "q_heads": 4, "k_heads": 4, "dk": 128, "dv": 64}
    mla = {"heads": 32, "dk": 192, "dv": 128}
    gqa = {"heads": 8, "dk": 128, "dv": 128}
    return [
        # One long document read at once.
        {"name": "linear-8192", "op": "linear", "type": "bf16", **kda, "requests": 1,
         "shortest": 8192, "longest": 8192, "lens_seed": 1, "per_token": True, "state": True},
        # A server's batch of prompts of all lengths, packed, with a fixed decay a head.
        {"name": "linear-ragged", "op": "linear", "type": "bf16", **shared, "requests": 24,
         "shortest": 1, "longest": 2047, "lens_seed": 2, "per_token": False, "state": True},
        # One user's next token: latency.
        {"name": "step-b1", "op": "step", "type": "bf16", **kda, "requests": 1, "spare": 0,
         "per_token": True},
        # A decode batch whose states lie anywhere in a pool.
        {"name": "step-b256", "op": "step", "type": "bf16", **kda, "requests": 256, "spare": 5,
         "per_token": True},
        # Four continuations of one prompt.
        {"name": "fork-4", "op": "fork", "type": "bf16", **mla, "requests": 6, "forks": 4,
         "page": 64, "shortest": 777, "longest": 3001, "lens_seed": 3, "one": True},
        # Every request of a batch of 64 forked once: pages of grouped heads.
        {"name": "fork-64", "op": "fork", "type": "f16", **gqa, "requests": 128, "forks": 64,
         "page": 64, "shortest": 1, "longest": 4095, "lens_seed": 4, "one": False},
        # A few requests of a small batch are done.
        {"name": "free-32", "op": "free", "requests": 32, "page": 64, "shortest": 1,
         "longest": 8192, "lens_seed": 5, "done": 5, "cut": 0, "twins": 4},
        # A large server: a tenth done, refused drafts' pages cut off elsewhere.
        {"name": "free-2048", "op": "free", "requests": 2048, "page": 16, "shortest": 0,
         "longest": 4000, "lens_seed": 6, "done": 205, "cut": 300, "twins": 300},
        # A small pool, half full, before the rest of it is given to something else.
        {"name": "compact-16", "op": "compact", "type": "bf16", **gqa, "requests": 16,
         "page": 16, "shortest": 1, "longest": 700, "lens_seed": 7, "fill": 0.5, "twins": 2},
        # A large one.
        {"name": "compact-256", "op": "compact", "type": "bf16", **gqa, "requests": 256,
         "page": 64, "shortest": 1, "longest": 2000, "lens_seed": 8, "fill": 0.6, "twins": 40},
        # One user's drafted tree, each of its rows with the tokens above it.
        {"name": "logits-b1", "op": "logits", "type": "bf16", "requests": 1, "vocab": 163840,
         "tokens": 9, "tree": True, "shortest": 3500, "longest": 3500, "lens_seed": 9,
         "biases": 20, "masked": True},
        # A batch of 256, answers of all lengths behind their prompts.
        {"name": "logits-b256", "op": "logits", "type": "bf16", "requests": 256,
         "vocab": 163840, "tokens": 1, "tree": False, "shortest": 16, "longest": 8000,
         "lens_seed": 10, "biases": 0, "masked": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _linear_heads(rng):
    heads = rng.choice([1, 2, 3, 4, 8, 12, 16, 24, 32, 64])
    parts = [g for g in (1, 2, 3, 4, 8, 16, 32) if heads % g == 0]
    k = rng.choice([heads, heads, rng.choice(parts)])
    q = rng.choice([heads, k])
    dk, dv = rng.choice([(128, 128), (128, 128), (128, 64), (64, 64), (64, 128), (96, 80), (40, 72)])
    return {"heads": heads, "q_heads": q, "k_heads": k, "dk": dk, "dv": dv}


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "step", "step", "fork", "free", "compact",
                     "logits", "logits"])
    lens_seed = rng.randrange(10**6)
    if op == "linear":
        heads = _linear_heads(rng)
        longest, requests = _log(rng, 2, 8192), _log(rng, 1, 48)
        while heads["heads"] * longest * requests > 32 * 8192 * 2:
            longest, requests = max(2, longest * 3 // 4), max(1, requests * 3 // 4)
        if heads["heads"] * longest * requests > 32 * 8192:
            longest = max(2, longest // 2)
        return {"op": op, "type": "bf16", **heads, "requests": requests,
                "shortest": rng.choice([1, 1, max(1, longest // 2)]), "longest": longest,
                "lens_seed": lens_seed, "per_token": rng.random() < 0.7,
                "state": rng.random() < 0.7}
    if op == "step":
        heads = _linear_heads(rng)
        requests = _log(rng, 1, 512)
        while heads["heads"] * requests > 32 * 256:
            requests = max(1, requests * 2 // 3)
        return {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), **heads,
                "requests": requests, "spare": rng.choice([0, 0, 3, 17]),
                "per_token": rng.random() < 0.7}
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    dk, dv = rng.choice([(64, 64), (128, 128), (192, 128), (72, 40)])
    pool = {"type": rng.choice(["bf16", "f16"]), "heads": kv, "dk": dk, "dv": dv}
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "fork":
        one = rng.random() < 0.4
        forks = _log(rng, 1, 100)
        return {"op": op, **pool, "requests": (1 if one else forks) + forks + rng.randrange(6),
                "forks": forks, "page": page, "shortest": rng.choice([0, 1, 60]),
                "longest": _log(rng, 64, 3000), "lens_seed": lens_seed, "one": one}
    if op == "free":
        requests = _log(rng, 4, 3000)
        return {"op": op, "requests": requests, "page": page, "shortest": rng.choice([0, 1, 100]),
                "longest": _log(rng, 128, 8000), "lens_seed": lens_seed,
                "done": rng.choice([0, 1, requests // 8, requests // 2]),
                "cut": rng.choice([0, requests // 4]), "twins": rng.choice([0, requests // 4])}
    if op == "compact":
        requests = _log(rng, 2, 200)
        return {"op": op, **pool, "requests": requests, "page": page,
                "shortest": rng.choice([0, 1, 50]), "longest": _log(rng, 64, 1500),
                "lens_seed": lens_seed, "fill": rng.choice([0.3, 0.5, 0.7, 0.9]),
                "twins": rng.choice([0, requests // 5])}
    vocab = rng.choice([163840, 163840, 32000, 50257, 151936, _log(rng, 100, 100000)])
    requests, tokens = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 5, 9, 16])
    while requests * tokens > 256:
        requests = max(1, requests // 2)
    longest = _log(rng, 8, 12000)
    return {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "requests": requests,
            "vocab": vocab, "tokens": tokens, "tree": tokens > 1 and rng.random() < 0.6,
            "shortest": rng.choice([0, 1, longest // 2]), "longest": longest,
            "lens_seed": lens_seed, "biases": rng.choice([0, 0, 5, 300]),
            "masked": rng.random() < 0.6}


def _lens(case, count=None):
    """Lengths of the case's requests, spread over the logarithm."""
    r = random.Random(case["lens_seed"])
    lo, hi = case["shortest"], case["longest"]
    got = [_log(r, max(lo, 1), hi) for _ in range(count or case["requests"])]
    got[0] = hi
    if len(got) > 1:
        got[-1] = lo
    return got


def _sums(values):
    got = [0]
    for v in values:
        got.append(got[-1] + v)
    return got


def _pages(tokens, page):
    return -(-tokens // page)


def _twins(case):
    """Requests that were forked from another: (parent, child, full pages they share)."""
    lens, r = _lens(case), random.Random(case["lens_seed"] + 5)
    order = list(range(case["requests"]))
    r.shuffle(order)
    got = []
    for parent, child in zip(order[0::2], order[1::2]):
        if len(got) < case["twins"]:
            got.append((parent, child, min(lens[parent], lens[child]) // case["page"]))
    return got


# ---------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _decays(gen, *shape):
    """Logarithms of decays: rates a head, from long memories to short ones, and their inputs."""
    rate = torch.empty(shape[-1], device="cuda").uniform_(-5.0, 0.7, generator=gen).exp_()
    x = torch.randn(shape, generator=gen, device="cuda")
    return -rate * torch.log1p(x.exp())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(  # noqa: E731
        shape, generator=gen, device="cuda", dtype=_TYPES[case["type"]])
    state, op = {"case": case}, case["op"]
    if op in ("linear", "step"):
        n, h, dk, dv = case["requests"], case["heads"], case["dk"], case["dv"]
        lens = _lens(case) if op == "linear" else [1] * n
        t = sum(lens)
        slots = n + case.get("spare", 0)
        state.update(
            lens=lens, q=normal(t, case["q_heads"], dk),
            k=torch.nn.functional.normalize(normal(t, case["k_heads"], dk).float(), dim=-1).to(
                _TYPES[case["type"]]),
            v=normal(t, h, dv),
            decay=_decays(gen, t, h) if case["per_token"] else _decays(gen, h),
            cu=_ints(_sums(lens)), scale=dk ** -0.5, pool=None, index=None)
        if op == "step" or case["state"]:
            state["pool"] = torch.randn((slots, h, dk, dv), generator=gen, device="cuda")
        if op == "step" and case["spare"]:
            state["index"] = torch.randperm(slots, generator=gen, device="cuda")[:n].int()
        return state
    if op == "logits":
        b, v, t, lens = case["requests"], case["vocab"], case["tokens"], _lens(case)
        rows = b * t
        some = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
        # Tokens come often or seldom; an answer repeats its own.
        words = lambda *shape: (some(*shape).pow_(4) * v).long().clamp_max_(v - 1)  # noqa: E731
        state.update(
            logits=(2.5 * torch.randn((rows, v), generator=gen, device="cuda")).to(
                _TYPES[case["type"]]),
            history=words(b, max(max(lens), 1)), lens=_ints(lens),
            prompts=(_ints(lens) * some(b)).int(),
            repetition=1.0 + 0.3 * some(b), presence=some(b), frequency=0.5 * some(b),
            ids=None, values=None, allowed=None, cu=None, tokens=None, mask=None)
        if b > 3:       # requests that ask for nothing
            state["repetition"][1::4], state["presence"][1::4], state["frequency"][1::4] = 1, 0, 0
        if case["biases"]:
            ids = words(b, case["biases"])
            ids[:, case["biases"] // 2 + 1:][some(b, case["biases"])[:, case["biases"] // 2 + 1:] < 0.3] = -1
            state["ids"] = ids
            state["values"] = 4 * torch.randn((b, case["biases"]), generator=gen, device="cuda")
        if case["masked"]:
            # Grammars that allow one token in eight, or all but a few.
            words_of = lambda: torch.randint(  # noqa: E731
                -2**31, 2**31, (rows, -(-v // 32)), generator=gen, device="cuda").int()
            few = words_of() & words_of() & words_of()
            state["allowed"] = torch.where(some(rows, 1) < 0.5, few, ~(few & words_of()))
        if t > 1:
            state["cu"], state["tokens"] = _ints(list(range(0, rows + 1, t))), words(rows)
            if case["tree"]:
                state["mask"] = _ints([w for i in range(b) for w in _words(case, i)], torch.int64)
        return state
    ps, lens = case["page"], _lens(case)
    if op == "fork":
        # The first requests are forked; the last ones are the rows they are forked to.
        n, forks = case["requests"], case["forks"]
        sources = [0] * forks if case["one"] else list(range(forks))
        targets = list(range(n - forks, n))
        lens = [0 if i in targets else x for i, x in enumerate(lens)]
        have = [_pages(x, ps) for x in lens]
        total = sum(have) + forks + 3
        width = max(have) + 2
    else:
        have = [_pages(x, ps) for x in lens]
        fill = case.get("fill", 0.8)
        total, width = int(sum(have) / fill) + 8, max(have) + 1
    ids = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]] = ids[:sum(have)]
    head, free = 5, torch.cat((ids[:5], ids[sum(have):]))
    if op != "fork":
        for parent, child, pages in _twins(case):
            table[child, :pages] = table[parent, :pages]
        # Pages that no row names any more are free too; the list has room in front.
        held = torch.zeros(total, dtype=torch.bool, device="cuda")
        held[table[table >= 0].long()] = True
        rest = ids[~held[ids.long()]]
        head, free = total - rest.shape[0], torch.cat((ids[:total - rest.shape[0]], rest))
    state.update(table=table, reserved=_ints(lens), free=free, head=_ints([head]), pages=total)
    if op == "fork":
        state.update(sources=_ints(sources), targets=_ints(targets), context=_ints(lens))
    if op == "free":
        r, keep = random.Random(case["lens_seed"] + 9), list(lens)
        order = list(range(len(lens)))
        r.shuffle(order)
        for i in order[:case["done"]]:
            keep[i] = 0
        for i in order[case["done"]:case["done"] + case["cut"]]:
            keep[i] = max(0, lens[i] - r.randrange(3 * ps))
        state["keep"] = _ints(keep)
        return state
    h = case["heads"]
    # Pages hold one head's rows together; users see [page, row, head, width].
    state.update(k_cache=normal(total, h, ps, case["dk"]).transpose(1, 2),
                 v_cache=normal(total, h, ps, case["dv"]).transpose(1, 2))
    return state


def _words(case, i):
    """For each token of a request's tree the bits of itself and its ancestors."""
    r, words = random.Random(case["lens_seed"] + 77 + i), [1]
    for t in range(1, case["tokens"]):
        words.append((1 << t) | words[r.randint(max(0, t - 4), t - 1)])
    return words


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return _OWN[state["case"]["op"]](state) if own else _PLAIN[state["case"]["op"]](state)


_CHUNK = 64


def _plain_linear(s):
    case = s["case"]
    b, h, c, dk, dv = case["requests"], case["heads"], _CHUNK, case["dk"], case["dv"]
    t = s["q"].shape[0]
    most = -(-max(s["lens"]) // c) * c
    cu = s["cu"].long()
    at = cu[:-1, None] + torch.arange(most, device="cuda")[None, :]
    real = at < cu[1:, None]
    at = at.clamp_max(t - 1)

    def blocks(x, heads):     # [requests, heads, chunks, c, width], zero past a request's end
        x = (x.float()[at] * real[:, :, None, None]).repeat_interleave(h // heads, dim=2)
        return x.view(b, most // c, c, h, -1).permute(0, 3, 1, 2, 4)

    q, k = blocks(s["q"], case["q_heads"]) * s["scale"], blocks(s["k"], case["k_heads"])
    v = blocks(s["v"], h)
    g = s["decay"].double().expand(t, h)[at] * real[:, :, None]
    g = g.view(b, most // c, c, h).permute(0, 3, 1, 2).cumsum(-1)
    last = g[..., -1:]
    near = (g[..., :, None] - g[..., None, :]).float()
    near = near.masked_fill_(torch.ones((c, c), dtype=torch.bool, device="cuda").triu(1), -math.inf)
    out = (q @ k.transpose(-1, -2)).mul_(near.exp_()) @ v
    gain = (k * (last - g).exp().float()[..., None]).transpose(-1, -2) @ v
    keep, q = last.exp().float()[..., None], q * g.exp().float()[..., None]
    total = torch.zeros((b, h, dk, dv), device="cuda") if s["pool"] is None else s["pool"].clone()
    for i in range(most // c):
        out[:, :, i] += q[:, :, i] @ total
        total = total * keep[:, :, i] + gain[:, :, i]
    out = out.permute(0, 2, 3, 1, 4).reshape(b, most, h, dv)[real].to(s["q"].dtype)
    if s["pool"] is None:
        return out
    s["pool"].copy_(total)
    return {"out": out, "state": s["pool"]}


def _own_linear(s):
    from local_kimi_b200 import ops

    out = ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["cu"], max(s["lens"]),
                               state=s["pool"], scale=s["scale"])
    return out if s["pool"] is None else {"out": out, "state": s["pool"]}


def _plain_step(s):
    case = s["case"]
    q = s["q"].float().repeat_interleave(case["heads"] // case["q_heads"], dim=1) * s["scale"]
    k = s["k"].float().repeat_interleave(case["heads"] // case["k_heads"], dim=1)
    now = s["pool"] if s["index"] is None else s["pool"][s["index"].long()]
    g = s["decay"].float().exp().expand(case["requests"], case["heads"])
    now = now * g[:, :, None, None] + k[..., None] * s["v"].float()[..., None, :]
    out = (q[..., None, :] @ now)[..., 0, :].to(s["q"].dtype)
    if s["index"] is None:
        s["pool"].copy_(now)
    else:
        s["pool"][s["index"].long()] = now
    return {"out": out, "state": s["pool"]}


def _own_step(s):
    from local_kimi_b200 import ops

    out = ops.linear_attention_step(s["pool"], s["q"], s["k"], s["v"], s["decay"],
                                    state_index=s["index"], scale=s["scale"])
    return {"out": out, "state": s["pool"]}


def _plain_fork(s):
    ps, width = s["case"]["page"], s["table"].shape[1]
    sources, targets = s["sources"].long(), s["targets"].long()
    lens = s["context"][sources]
    full, part = lens // ps, lens % ps
    need = (part > 0).int()
    place = s["head"] + need.cumsum(0) - need
    given = (need > 0) & (place < s["free"].shape[0])
    made = given | (need == 0)
    fresh = s["free"][place.clamp_max(s["free"].shape[0] - 1).long()]
    column = torch.arange(width, device="cuda")[None, :]
    rows = torch.where(column < full[:, None], s["table"][sources], -1)
    rows = torch.where((column == full[:, None]) & given[:, None], fresh[:, None], rows)
    s["table"][targets] = torch.where(made[:, None], rows, -1)
    s["context"][targets] = torch.where(made, lens, 0)
    old = s["table"][sources, full.clamp_max(width - 1).long()]
    move_from, move_to = torch.where(given, old, -1), torch.where(given, fresh, -1)
    count = torch.where(given, part, 0)
    row = torch.arange(ps, device="cuda")
    pick, r = (row[None, :] < count[:, None]).nonzero(as_tuple=True)
    a, z = move_from.long()[pick], move_to.long()[pick]
    s["k_cache"][z, r] = s["k_cache"][a, r]
    s["v_cache"][z, r] = s["v_cache"][a, r]
    return {"table": s["table"], "context": s["context"], "from": move_from, "to": move_to,
            "rows": count, "head": (s["head"] + given.sum()).int(), "k": s["k_cache"],
            "v": s["v_cache"]}


def _own_fork(s):
    from local_kimi_b200 import ops

    got = ops.paged_fork(s["context"], s["table"], s["sources"], s["targets"], s["free"],
                         s["head"], s["case"]["page"])
    ops.paged_copy(s["k_cache"], s["v_cache"], got.copy_from, got.copy_to, got.copy_rows)
    return {"table": s["table"], "context": s["context"], "from": got.copy_from,
            "to": got.copy_to, "rows": got.copy_rows, "head": got.free_head, "k": s["k_cache"],
            "v": s["v_cache"]}


def _plain_free(s):
    ps, pages = s["case"]["page"], s["pages"]
    have = (s["reserved"] + ps - 1) // ps
    keep = (torch.minimum(s["keep"], s["reserved"]) + ps - 1) // ps
    column = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    # One place more, for what counts nowhere.
    kept = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    gone = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    table = s["table"].long()
    kept[torch.where((column < keep[:, None]) & (table >= 0), table, pages)] = True
    gone[torch.where((column >= keep[:, None]) & (column < have[:, None]) & (table >= 0), table,
                     pages)] = True
    gone = (gone & ~kept)[:pages]
    head = s["head"] - gone.sum()
    rank = gone.cumsum(0) - 1 + head
    s["free"][rank[gone]] = torch.arange(pages, dtype=torch.int32, device="cuda")[gone]
    return {"head": head.int(), "free": s["free"]}


def _own_free(s):
    from local_kimi_b200 import ops

    head = ops.paged_free(s["table"], s["reserved"], s["keep"], s["free"], s["head"],
                          s["case"]["page"], s["pages"])
    return {"head": head, "free": s["free"]}


def _plain_compact(s):
    ps, pages, table = s["case"]["page"], s["pages"], s["table"].long()
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    inside = (column < ((s["reserved"] + ps - 1) // ps)[:, None]) & (table >= 0)
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(inside, table, pages)] = True
    used = used[:pages]
    listed_ = torch.arange(s["free"].shape[0], device="cuda") >= s["head"]
    free = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    free[torch.where(listed_, s["free"].long(), pages)] = True
    free = free[:pages] & ~used
    # The lowest places of the pages that are used or free, as many as are used.
    low = (used | free).cumsum(0) <= used.sum()
    ids = torch.arange(pages, device="cuda")
    moved, holes = ids[used & ~low], ids[free & low]
    to = ids.clone()
    to[moved] = holes
    new = torch.where(inside, to[table.clamp_min(0)], -1).int()
    rest = ((used | free) & ~low).nonzero()[:, 0]
    out = s["free"].clone()
    out[s["free"].shape[0] - rest.shape[0]:] = rest.int()
    s["k_cache"][holes] = s["k_cache"][moved]
    s["v_cache"][holes] = s["v_cache"][moved]
    blank = torch.full((pages // 2,), -1, dtype=torch.int32, device="cuda")
    a, z = blank.clone(), blank.clone()
    a[:moved.shape[0]], z[:moved.shape[0]] = moved.int(), holes.int()
    return {"table": new, "free": out, "from": a, "to": z, "k": s["k_cache"], "v": s["v_cache"]}


def _own_compact(s):
    from local_kimi_b200 import ops

    got = ops.paged_compact(s["table"], s["reserved"], s["free"], s["head"], s["case"]["page"],
                            s["pages"])
    ops.paged_copy(s["k_cache"], s["v_cache"], got.copy_from, got.copy_to)
    return {"table": got.block_table, "free": got.free_pages, "from": got.copy_from,
            "to": got.copy_to, "k": s["k_cache"], "v": s["v_cache"]}


def _plain_logits(s):
    case = s["case"]
    b, v, t = case["requests"], case["vocab"], case["tokens"]
    x = s["logits"].float()
    step = torch.arange(s["history"].shape[1], device="cuda")[None, :]
    there = step < s["lens"][:, None]
    answer = there & (step >= s["prompts"][:, None])
    said = torch.zeros((b, v), device="cuda").scatter_add_(1, s["history"], answer.float())
    seen = torch.zeros((b, v), device="cuda").scatter_add_(1, s["history"], there.float())
    said, seen = said.repeat_interleave(t, 0), seen.repeat_interleave(t, 0)
    if s["tokens"] is not None:
        place = torch.arange(t, device="cuda")[None, :]
        if s["mask"] is None:
            above = (place <= place.T).repeat(b, 1)
        else:
            above = ((s["mask"][:, None] >> place) & 1) == 1
        drafted = s["tokens"].view(b, t).repeat_interleave(t, 0)
        said.scatter_add_(1, drafted, above.float())
        seen.scatter_add_(1, drafted, above.float())
    each = lambda p: p.repeat_interleave(t)[:, None]  # noqa: E731
    r = each(s["repetition"])
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - each(s["frequency"]) * said
    x = x - each(s["presence"]) * (said > 0)
    if s["ids"] is not None:
        bias = torch.zeros((b, v), device="cuda").scatter_add_(
            1, s["ids"].clamp_min(0), torch.where(s["ids"] >= 0, s["values"], 0.0))
        x = x + bias.repeat_interleave(t, 0)
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device="cuda")) & 1
        x = x.masked_fill(bits.flatten(1)[:, :v] == 0, -math.inf)
    return x.to(s["logits"].dtype)


def _own_logits(s):
    from local_kimi_b200 import ops

    return ops.adjust_logits(
        s["logits"], history=s["history"], history_lens=s["lens"], prompt_lens=s["prompts"],
        repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
        bias_ids=s["ids"], bias_values=s["values"], allowed=s["allowed"], cu_tokens=s["cu"],
        tokens=s["tokens"], tree_mask=s["mask"])


_PLAIN = {"linear": _plain_linear, "step": _plain_step, "fork": _plain_fork, "free": _plain_free,
          "compact": _plain_compact, "logits": _plain_logits}
_OWN = {"linear": _own_linear, "step": _own_step, "fork": _own_fork, "free": _own_free,
        "compact": _own_compact, "logits": _own_logits}


# ---------------------------------------------------------------------------
# the work, and the definition
# ---------------------------------------------------------------------------


def work(case):
    size = 4 if case.get("type") == "f32" else 2
    op, n = case["op"], case["requests"]
    if op in ("linear", "step"):
        t = sum(_lens(case)) if op == "linear" else n
        h, dk, dv = case["heads"], case["dk"], case["dv"]
        kept = n if op == "step" or case["state"] else 0
        rows = t * ((case["q_heads"] + case["k_heads"]) * dk + 2 * h * dv) * size
        return {"bytes": rows + (t if case["per_token"] else 1) * h * 4 + 8 * kept * h * dk * dv,
                "flops": 4 * t * h * dk * dv}
    if op == "logits":
        rows, v, lens = n * case["tokens"], case["vocab"], _lens(case)
        return {"bytes": rows * v * 2 * size + 8 * sum(lens) + 12 * n * case["biases"]
                + (rows * v // 8 if case["masked"] else 0),
                "flops": 2 * sum(lens)}
    ps, lens = case["page"], _lens(case)
    ints = 4 * sum(_pages(x, ps) for x in lens) + 8 * n
    if op == "free":
        return {"bytes": ints, "flops": 0}
    row = case["heads"] * (case["dk"] + case["dv"]) * size
    if op == "fork":
        forks = case["forks"]
        from_ = [lens[0]] * forks if case["one"] else lens[:forks]
        return {"bytes": 2 * row * sum(x % ps for x in from_) + 4 * sum(x // ps for x in from_),
                "flops": 0}
    # About as many pages move as random places leave above the lowest.
    pages = sum(_pages(x, ps) for x in lens)
    return {"bytes": int(2 * row * ps * pages * (1 - case["fill"])) + 2 * ints, "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s, case)


def _exact_linear(s, case):
    """Token after token, all requests and heads at once."""
    h, n = case["heads"], case["requests"]
    q = s["q"].double().repeat_interleave(h // case["q_heads"], dim=1) * s["scale"]
    k = s["k"].double().repeat_interleave(h // case["k_heads"], dim=1)
    v, cu = s["v"].double(), _sums(s["lens"])
    keep = s["decay"].double().exp().expand(q.shape[0], h)
    total = (torch.zeros((n, h, case["dk"], case["dv"]), dtype=torch.float64, device="cuda")
             if s["pool"] is None else s["pool"].double())
    if s["index"] is not None:
        total = total[s["index"].long()]
    out = torch.empty_like(v)
    # Longest first, so that those still running are the first ones.
    order = sorted(range(n), key=lambda i: -s["lens"][i])
    total = total[_ints(order, torch.int64)]
    firsts = _ints([cu[i] for i in order], torch.int64)
    lens = [s["lens"][i] for i in order]
    live = n
    for t in range(max(lens)):
        while live and lens[live - 1] <= t:
            live -= 1
        at = firsts[:live] + t
        now = total[:live]
        now *= keep[at][:, :, None, None]
        now += k[at][..., None] * v[at][..., None, :]
        out[at] = (q[at][..., None, :] @ now)[..., 0, :]
    if s["pool"] is None:
        return out
    end = s["pool"].double()
    rows = _ints(order, torch.int64)
    end[rows if s["index"] is None else s["index"].long()[rows]] = total
    return {"out": out, "state": end}


def _exact_fork(s, case):
    k, v = s["k_cache"].double(), s["v_cache"].double()
    ps, head, free = case["page"], int(s["head"]), s["free"].tolist()
    context, table = s["context"].tolist(), s["table"].tolist()
    for a in s["sources"].tolist():
        full, part = divmod(context[a], ps)
        if part and head < len(free):
            k[free[head], :part] = s["k_cache"][table[a][full], :part].double()
            v[free[head], :part] = s["v_cache"][table[a][full], :part].double()
            head += 1
    return {"table": None, "context": None, "from": None, "to": None, "rows": None,
            "head": None, "k": k, "v": v}


def _exact_compact(s, case):
    k, v = s["k_cache"].double(), s["v_cache"].double()
    held = {p for row, n in zip(s["table"].tolist(), s["reserved"].tolist())
            for p in row[:_pages(n, case["page"])]}
    spare = set(s["free"].tolist()[int(s["head"]):]) - held
    low = set(sorted(held | spare)[:len(held)])
    moved, holes = sorted(held - low), sorted(spare & low)
    if moved:
        a, z = _ints(moved, torch.int64), _ints(holes, torch.int64)
        k[z], v[z] = s["k_cache"][a].double(), s["v_cache"][a].double()
    return {"table": None, "free": None, "from": None, "to": None, "k": k, "v": v}


def _exact_logits(s, case):
    b, v, t = case["requests"], case["vocab"], case["tokens"]
    out = s["logits"].double()
    for i in range(b):
        n, p = int(s["lens"][i]), int(s["prompts"][i])
        words = s["history"][i, :n]
        for j in range(t):
            row, extra = i * t + j, words[:0]
            if s["tokens"] is not None:
                word = (1 << (j + 1)) - 1 if s["mask"] is None else int(s["mask"][row])
                extra = s["tokens"][[i * t + a for a in range(t) if word >> a & 1]]
            said = torch.bincount(torch.cat((words[p:], extra)), minlength=v).double()
            seen = torch.bincount(torch.cat((words, extra)), minlength=v) > 0
            x, r = out[row], s["repetition"][i].double()
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
            x = x - s["frequency"][i].double() * said - s["presence"][i].double() * (said > 0)
            if s["ids"] is not None:
                real = s["ids"][i] >= 0
                x = x.index_add(0, s["ids"][i][real], s["values"][i][real].double())
            if s["allowed"] is not None:
                at = torch.arange(v, device="cuda")
                x = torch.where((s["allowed"][row][at // 32] >> (at % 32)) & 1 == 1, x, -math.inf)
            out[row] = x
    return out


_EXACT = {"linear": _exact_linear, "step": _exact_linear, "fork": _exact_fork,
          "free": lambda s, case: None, "compact": _exact_compact, "logits": _exact_logits}
