"""Cases of the speculative serving step: prompts, paged cache, drafted tokens, verification.

Five operators, as one serving step uses them:

  plan     pages, slots and positions for the new tokens of every request
  append   the new tokens' keys and values into the paged cache
  prompt   causal attention over packed whole prompts
  tree     attention of drafted tokens (or one token a request) over the paged cache
  verify   which drafted tokens the target accepts, and the token after them

``run`` computes them with elementary torch operations in 32 bits, or, with
``own`` set, through this package's operators.  ``exact`` restates the
attention outputs in 64 bits.
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
    # The attention layers of the 27-layer model: 32 heads, keys 192 wide, values 128;
    # grouped layouts (8 key/value heads, 128 wide) stand for other target models.
    mla = {"heads": 32, "kv_heads": 32, "dk": 192, "dv": 128}
    gqa = {"heads": 32, "kv_heads": 8, "dk": 128, "dv": 128}
    small = {"heads": 8, "kv_heads": 2, "dk": 64, "dv": 64}
    return [
        # One long document read at once: throughput of the prompt phase.
        {"name": "prompt-8192", "op": "prompt", "type": "bf16", **mla, "requests": 1,
         "shortest": 8192, "longest": 8192, "lens_seed": 1, "prefix": 0, "lse": False},
        # A server's batch of prompts of all lengths, packed; log-sum-exp kept to join parts.
        {"name": "prompt-ragged", "op": "prompt", "type": "bf16", **gqa, "requests": 24,
         "shortest": 1, "longest": 2047, "lens_seed": 2, "prefix": 0, "lse": True},
        # A few short chat turns, each behind an earlier part of its prompt: latency.
        {"name": "prompt-short", "op": "prompt", "type": "f16", **small, "requests": 5,
         "shortest": 3, "longest": 90, "lens_seed": 3, "prefix": 37, "lse": False},
        # One user's next token over a 4096-token context: latency of a read of the cache.
        {"name": "token-b1", "op": "tree", "type": "bf16", **mla, "requests": 1, "page": 64,
         "shortest": 4096, "longest": 4096, "lens_seed": 4, "tokens": 1, "ragged": False,
         "tree": False, "lse": False},
        # A serving batch, contexts of all lengths up to 8192: bandwidth.
        {"name": "token-b32", "op": "tree", "type": "bf16", **mla, "requests": 32, "page": 64,
         "shortest": 512, "longest": 8192, "lens_seed": 5, "tokens": 1, "ragged": False,
         "tree": False, "lse": False},
        # Trees of up to 24 drafted tokens for a batch with grouped heads and small pages.
        {"name": "tree-b16", "op": "tree", "type": "f16", **gqa, "requests": 16, "page": 16,
         "shortest": 100, "longest": 4095, "lens_seed": 6, "tokens": 24, "ragged": True,
         "tree": True, "lse": True},
        # One user's drafted tree after a step of the full vocabulary.
        {"name": "verify-b1", "op": "verify", "type": "bf16", "requests": 1, "vocab": 163840,
         "tokens": 9, "ragged": False, "tree": True, "probs": False, "greedy": 0},
        # A batch of 256 with four drafted tokens each from a draft model's probabilities.
        {"name": "verify-b256", "op": "verify", "type": "bf16", "requests": 256,
         "vocab": 163840, "tokens": 5, "ragged": True, "tree": False, "probs": True,
         "greedy": 8},
        # The step of a small batch of drafted trees.
        {"name": "plan-b32", "op": "plan", "requests": 32, "page": 64, "shortest": 1,
         "longest": 8192, "lens_seed": 7, "tokens": 9, "ragged": True, "tree": True},
        # A large server takes in whole prompts beside its running requests.
        {"name": "plan-b2048", "op": "plan", "requests": 2048, "page": 16, "shortest": 0,
         "longest": 4000, "lens_seed": 8, "tokens": 200, "ragged": True, "tree": False},
        # The new tokens of a decode batch.
        {"name": "append-256", "op": "append", "type": "bf16", **mla, "tokens": 256, "page": 64,
         "skipped": 3},
        # A whole prompt's keys and values.
        {"name": "append-8192", "op": "append", "type": "f16", **gqa, "tokens": 8192,
         "page": 16, "skipped": 0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "tree", "verify", "verify", "plan",
                     "append"])
    kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
    group = rng.choice([g for g in (1, 1, 2, 3, 4, 5, 8, 16) if g * kv <= 64])
    dk, dv = rng.choice([(64, 64), (128, 128), (192, 128), (192, 128), (96, 96), (72, 40)])
    heads = {"heads": kv * group, "kv_heads": kv, "dk": dk, "dv": dv}
    kind = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "prompt":
        # No more than the largest listed case: 8192 tokens of 32 heads.
        longest = _log(rng, 2, 8192)
        requests = _log(rng, 1, 32)
        while kv * group * longest * (longest + 600) * requests > 32 * 8192 * 8192:
            longest, requests = max(2, longest * 3 // 4), max(1, requests * 3 // 4)
        return {"op": op, "type": kind, **heads, "requests": requests,
                "shortest": rng.choice([1, 1, max(1, longest // 2)]), "longest": longest,
                "lens_seed": rng.randrange(10**6), "prefix": rng.choice([0, 0, 0, rng.randrange(1, 300)]),
                "lse": rng.random() < 0.5}
    if op == "tree":
        longest = _log(rng, 1, 16000)
        requests = _log(rng, 1, 64)
        while kv * longest * requests > 32 * 8192 * 8:
            longest, requests = max(1, longest * 2 // 3), max(1, requests // 2)
        tree = rng.random() < 0.6
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 48)
        return {"op": op, "type": kind, **heads, "requests": requests, "page": page,
                "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest,
                "lens_seed": rng.randrange(10**6), "tokens": tokens,
                "ragged": rng.random() < 0.5, "tree": tree, "lse": rng.random() < 0.5}
    if op == "verify":
        vocab = rng.choice([163840, 163840, 32000, 50257, 151936, _log(rng, 100, 100000)])
        requests = _log(rng, 1, 200)
        tokens = rng.choice([1, 2, 5, 9, 16])
        while requests * tokens > 1200:
            requests //= 2
        tree = rng.random() < 0.5
        return {"op": op, "type": rng.choice(["bf16", "f16", "f32"]), "requests": requests,
                "vocab": vocab, "tokens": tokens, "ragged": rng.random() < 0.5, "tree": tree,
                "probs": not tree and rng.random() < 0.6,
                "greedy": rng.choice([0, 0, requests // 2, requests])}
    if op == "plan":
        tree = rng.random() < 0.5
        return {"op": op, "requests": _log(rng, 1, 3000), "page": page,
                "shortest": rng.choice([0, 1, 100]), "longest": _log(rng, 128, 30000),
                "lens_seed": rng.randrange(10**6),
                "tokens": _log(rng, 1, 64) if tree else _log(rng, 1, 300),
                "ragged": rng.random() < 0.7, "tree": tree}
    tokens = _log(rng, 1, 8192 * 24 // kv if kv > 24 else 8192)
    return {"op": op, "type": kind, **heads, "tokens": tokens, "page": page,
            "skipped": rng.choice([0, min(3, tokens - 1)])}


def _lens(case):
    """Context (or prompt) lengths of the case's requests, spread over the logarithm."""
    r = random.Random(case["lens_seed"])
    lo, hi = case["shortest"], case["longest"]
    got = [_log(r, max(lo, 1), hi) if hi > 0 else 0 for _ in range(case["requests"])]
    got[0] = hi
    if len(got) > 1:
        got[-1] = lo
    return got


def _counts(case):
    """New tokens of each request (the first is the root of a drafted tree)."""
    r = random.Random(case.get("lens_seed", 11) + 1)
    n, b = case["tokens"], case["requests"]
    return [r.randint(1, n) if case["ragged"] and i else n for i in range(b)]


def _parents(case, counts):
    """For each tree token the index of its parent in the request (-1 for the root)."""
    r = random.Random(case.get("lens_seed", 11) + 2)
    return [[-1] + [r.randint(max(0, t - 4), t - 1) for t in range(1, n)] for n in counts]


def _sums(values):
    got = [0]
    for v in values:
        got.append(got[-1] + v)
    return got


# ---------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    normal = lambda *shape: torch.randn(  # noqa: E731
        shape, generator=gen, device="cuda", dtype=_TYPES[case["type"]])
    op = case["op"]
    if op == "prompt":
        lens = _lens(case)
        keys = [n + case["prefix"] for n in lens]
        state.update(
            q_lens=lens, k_lens=keys, longest=max(lens),
            q=normal(sum(lens), case["heads"], case["dk"]),
            k=normal(sum(keys), case["kv_heads"], case["dk"]),
            v=normal(sum(keys), case["kv_heads"], case["dv"]),
            cu_q=_ints(_sums(lens)), cu_k=_ints(_sums(keys)), scale=case["dk"] ** -0.5)
        return state
    if op == "tree":
        ctx, new = _lens(case), _counts(case)
        ps, b = case["page"], case["requests"]
        pages = [-(-(c + n) // ps) for c, n in zip(ctx, new)]
        total = sum(pages)
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        cells = (torch.arange(max(pages), device="cuda")[None, :]
                 < _ints(pages)[:, None])
        table = torch.zeros((b, max(pages)), dtype=torch.int32, device="cuda")
        table[cells] = order
        h = case["kv_heads"]
        # Pages hold one head's rows together; users see [page, row, head, width].
        state.update(
            ctx=ctx, new=new, most=max(new), k_cache=normal(total, h, ps, case["dk"]).transpose(1, 2),
            v_cache=normal(total, h, ps, case["dv"]).transpose(1, 2), table=table,
            q=normal(sum(new), case["heads"], case["dk"]), cu=_ints(_sums(new)),
            ctx_dev=_ints(ctx), scale=case["dk"] ** -0.5, mask=None)
        if case["tree"]:
            state["mask"] = _ints(_masks(_parents(case, new)), torch.int64)
        return state
    if op == "verify":
        new, v = _counts(case), case["vocab"]
        rows, b = sum(new), case["requests"]
        par = _parents(case, new) if case["tree"] else [list(range(-1, n - 1)) for n in new]
        base = 2.5 * torch.randn((rows, v), generator=gen, device="cuda")
        cu = _sums(new)
        parent_row = _ints([cu[i] + max(p, 0) for i, r in enumerate(par) for p in r], torch.int64)
        # Each drafted token comes from a nearby distribution at its parent.
        draft = base[parent_row] + 0.5 * torch.randn((rows, v), generator=gen, device="cuda")
        draft = torch.softmax(draft, dim=-1)
        race = torch.empty((rows, v), device="cuda").exponential_(generator=gen)
        tokens = (draft / race).argmax(dim=-1)
        del race
        temps = [0.0 if i < case["greedy"] else 1.0 for i in range(b)]
        if not case["probs"]:
            draft = None
        state.update(
            new=new, most=max(new), parents=par, logits=base.to(_TYPES[case["type"]]),
            tokens=tokens, cu=_ints(cu), probs=draft,
            parents_dev=_ints([p for r in par for p in r]) if case["tree"] else None,
            parent_row=parent_row,
            coin=torch.rand((rows,), generator=gen, device="cuda"),
            noise=torch.empty((b, v), device="cuda").exponential_(generator=gen).clamp_min(1e-30),
            temps=torch.tensor(temps, device="cuda"))
        return state
    if op == "plan":
        ctx, new, ps = _lens(case), _counts(case), case["page"]
        have = [-(-c // ps) for c in ctx]
        want = [-(-(c + n) // ps) for c, n in zip(ctx, new)]
        b, width, total = len(ctx), max(want) + 1, sum(want) + 7
        ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
        cells = torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]
        table[cells] = ids[:sum(have)]
        state.update(
            total=sum(new), table=table, ctx=_ints(ctx), new=_ints(new),
            free=torch.cat((ids[:5], ids[sum(have):])), head=_ints([5]), parents=None)
        if case["tree"]:
            state["parents"] = _ints([p for r in _parents(case, new) for p in r])
        return state
    n, ps, h = case["tokens"], case["page"], case["kv_heads"]
    pages = n // ps + 9
    slots = torch.randperm(pages * ps, generator=gen, device="cuda")[:n]
    if case["skipped"]:
        slots[-case["skipped"]:] = -1
    state.update(
        k=normal(n, h, case["dk"]), v=normal(n, h, case["dv"]), slots=slots,
        k_cache=normal(pages, h, ps, case["dk"]).transpose(1, 2),
        v_cache=normal(pages, h, ps, case["dv"]).transpose(1, 2))
    return state


def _masks(parents):
    """For each tree token the bits of itself and its ancestors, as signed 64-bit words."""
    got = []
    for row in parents:
        words = []
        for t, p in enumerate(row):
            words.append((1 << t) | (words[p] if p >= 0 else 0))
        got += [w - (1 << 64) if w >> 63 else w for w in words]
    return got


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return _OWN[state["case"]["op"]](state) if own else _PLAIN[state["case"]["op"]](state)


def _attend(q, k, v, visible, scale, dtype):
    """q [B, T, H, Dk], k [B, S, G, Dk], v [B, S, G, Dv], visible [B, T, S]: (out, lse)."""
    b, t, h, _ = q.shape
    g = k.shape[2]
    qf = (q.float() * scale).view(b, t, g, h // g, -1).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(qf.reshape(b, g, h // g * t, -1), k.float().permute(0, 2, 3, 1))
    scores = scores.view(b, g, h // g, t, -1).masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp_min_(-1e30)
    weights = scores.sub_(top).exp_()
    total = weights.sum(dim=-1, keepdim=True)
    out = torch.matmul(weights.view(b, g, h // g * t, -1), v.float().permute(0, 2, 1, 3))
    out = out.view(b, g, h // g, t, -1) / total.clamp_min(1e-30)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    return (out.permute(0, 3, 1, 2, 4).reshape(b, t, h, -1).to(dtype),
            lse.permute(0, 3, 1, 2).reshape(b, t, h))


def _plain_prompt(s):
    outs, lses, q0, k0 = [], [], 0, 0
    for n, m in zip(s["q_lens"], s["k_lens"]):
        rows = torch.arange(n, device="cuda")[:, None] + (m - n)
        visible = torch.arange(m, device="cuda")[None, :] <= rows
        out, lse = _attend(s["q"][None, q0:q0 + n], s["k"][None, k0:k0 + m],
                           s["v"][None, k0:k0 + m], visible[None], s["scale"], s["q"].dtype)
        outs.append(out[0])
        lses.append(lse[0])
        q0, k0 = q0 + n, k0 + m
    out = torch.cat(outs)
    return {"out": out, "lse": torch.cat(lses)} if s["case"]["lse"] else out


def _own_prompt(s):
    from local_kimi_b200 import ops

    got = ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["longest"],
                               cu_seqlens_k=s["cu_k"], scale=s["scale"],
                               return_lse=s["case"]["lse"])
    return {"out": got[0], "lse": got[1]} if s["case"]["lse"] else got


def _plain_tree(s):
    b, t, ps = len(s["new"]), s["most"], s["case"]["page"]
    cu, ctx, rows = s["cu"].long(), s["ctx_dev"].long(), s["q"].shape[0]
    count = cu[1:] - cu[:-1]
    idx = (cu[:-1, None] + torch.arange(t, device="cuda")[None, :])
    real = torch.arange(t, device="cuda")[None, :] < count[:, None]
    q = s["q"][idx.clamp_max(rows - 1)]
    k = s["k_cache"][s["table"].long()].flatten(1, 2)
    v = s["v_cache"][s["table"].long()].flatten(1, 2)
    key = torch.arange(s["table"].shape[1] * ps, device="cuda")
    drafted = key[None, :] - ctx[:, None]
    if s["mask"] is None:
        visible = drafted[:, None, :] <= torch.arange(t, device="cuda")[None, :, None]
    else:
        words = s["mask"][idx.clamp_max(rows - 1)]
        bit = (words[:, :, None] >> drafted.clamp(0, 63)[:, None, :]) & 1
        visible = (drafted < 0)[:, None, :] | ((bit == 1) & (drafted < 64)[:, None, :])
    visible = visible & (drafted < count[:, None])[:, None, :] & real[:, :, None]
    out, lse = _attend(q, k, v, visible, s["scale"], s["q"].dtype)
    return {"out": out[real], "lse": lse[real]} if s["case"]["lse"] else out[real]


def _own_tree(s):
    from local_kimi_b200 import ops

    got = ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["ctx_dev"],
                             s["cu"], s["most"], tree_mask=s["mask"], scale=s["scale"],
                             return_lse=s["case"]["lse"])
    return {"out": got[0], "lse": got[1]} if s["case"]["lse"] else got


def _plain_verify(s):
    b, t = len(s["new"]), s["most"]
    cu, rows = s["cu"].long(), s["logits"].shape[0]
    request = torch.repeat_interleave(torch.arange(b, device="cuda"), cu[1:] - cu[:-1])
    x = s["logits"].float()
    greedy = s["temps"][request] == 0
    w = x / torch.where(greedy, 1.0, s["temps"][request])[:, None]
    best = x.argmax(dim=-1)
    w = (w - w.amax(dim=-1, keepdim=True)).exp_()
    p = w / w.sum(dim=-1, keepdim=True)
    at = torch.arange(rows, device="cuda")
    # p of each drafted token at its parent, and the draft's own probability of it.
    px = p[s["parent_row"], s["tokens"]]
    qx = None if s["probs"] is None else s["probs"][at, s["tokens"]]
    cur = cu[:-1].clone()
    rem = torch.ones(b, device="cuda")
    lost = torch.full((b, t), -1, dtype=torch.int64, device="cuda")
    path = torch.full((b, t), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    accepted = torch.zeros(b, dtype=torch.int32, device="cuda")
    refused = torch.full((b,), -1, dtype=torch.int64, device="cuda")
    each = torch.arange(b, device="cuda")
    for i in range(1, t):
        node = (cu[:-1] + i).clamp_max(rows - 1)
        live = (cu[:-1] + i < cu[1:]) & (s["parent_row"][node] == cur)
        token = s["tokens"][node]
        again = (lost == token[:, None]).any(dim=1)
        mass = torch.where(again, 0.0, px[node])
        bar = s["coin"][node] * (rem if qx is None else qx[node])
        take = torch.where(s["temps"] == 0, best[cur] == token, bar < mass) & live
        drop = live & ~take
        refused = torch.where(drop, node, refused)
        lost[:, i] = torch.where(drop, token, -1)
        rem = torch.where(drop, (rem - mass).clamp_min(0.0), rem)
        accepted = accepted + take.int()
        slot = torch.where(take, accepted, 0).long()
        path[each, slot] = torch.where(take, torch.full_like(accepted, i), path[each, slot])
        cur = torch.where(take, node, cur)
        rem = torch.where(take, 1.0, rem)
        refused = torch.where(take, -1, refused)
        lost = torch.where(take[:, None], -1, lost)
    left = p[cur]
    if s["probs"] is None:
        cut = torch.zeros_like(left, dtype=torch.bool)
        cut.scatter_(1, lost.clamp_min(0), lost >= 0)
        zero = (lost == 0).any(dim=1)
        cut[:, 0] = zero
        res = left.masked_fill(cut, 0.0)
    else:
        q = s["probs"][refused.clamp_min(0)]
        res = torch.where((refused >= 0)[:, None], (left - q).clamp_min(0.0), left)
    res = torch.where((res > 0).any(dim=1, keepdim=True), res, left)
    last = torch.where(s["temps"] == 0, best[cur], (res / s["noise"]).argmax(dim=-1))
    out = torch.full((b, t), -1, dtype=torch.int64, device="cuda")
    step = torch.arange(t, device="cuda")[None, :]
    inner = (step < accepted[:, None])
    ahead = torch.cat((path[:, 1:].long(), torch.zeros((b, 1), dtype=torch.int64, device="cuda")), 1)
    took = s["tokens"][(cu[:-1, None] + ahead.clamp_min(0)).clamp_max(rows - 1)]
    out = torch.where(inner, took, torch.where(step == accepted[:, None], last[:, None], out))
    return {"tokens": out, "path": path, "accepted": accepted}


def _own_verify(s):
    from local_kimi_b200 import ops

    got = ops.verify_drafts(s["logits"], s["tokens"], s["cu"], s["most"], s["coin"], s["noise"],
                            s["temps"], parents=s["parents_dev"], draft_probs=s["probs"])
    return {"tokens": got.tokens, "path": got.path, "accepted": got.accepted}


def _plain_plan(s):
    ps, total = s["case"]["page"], s["total"]
    ctx, new = s["ctx"].long(), s["new"].long()
    b, width = s["table"].shape
    have, want = (ctx + ps - 1) // ps, (ctx + new + ps - 1) // ps
    ends = (want - have).cumsum(0)
    first = s["head"].long() + ends - (want - have)
    column = torch.arange(width, device="cuda")[None, :]
    fresh = (column >= have[:, None]) & (column < want[:, None])
    source = (first[:, None] + column - have[:, None]).clamp(0, s["free"].shape[0] - 1)
    s["table"].copy_(torch.where(fresh, s["free"][source], s["table"]))
    cu = torch.cat((new.new_zeros(1), new.cumsum(0)))
    token = torch.arange(total, device="cuda")
    request = torch.searchsorted(cu[1:], token, right=True)
    step = token - cu[request]
    place = ctx[request] + step
    slots = s["table"][request, place // ps].long() * ps + place % ps
    got = {"cu": cu.int(), "slots": slots, "table": s["table"], "head": (s["head"] + ends[-1]).int()}
    if s["parents"] is None:
        return {**got, "positions": place.int()}
    # Ancestors by doubling: each round joins the words of the row reached so far.
    up = torch.where(s["parents"] >= 0, cu[request] + s["parents"], token)
    words = torch.ones_like(step) << step
    depth = (up != token).int()
    for _ in range(6):
        words = words | words[up]
        depth = depth + depth[up]
        up = up[up]
    return {**got, "positions": (ctx[request] + depth).int(), "mask": words}


def _own_plan(s):
    from local_kimi_b200 import ops

    got = ops.paged_plan(s["ctx"], s["new"], s["table"], s["free"], s["head"], s["case"]["page"],
                         s["total"], parents=s["parents"])
    out = {"cu": got.cu_tokens, "slots": got.slots, "table": s["table"], "head": got.free_head,
           "positions": got.positions}
    return out if s["parents"] is None else {**out, "mask": got.tree_mask}


def _plain_append(s):
    ps = s["case"]["page"]
    kept = s["slots"] >= 0
    slots = s["slots"][kept]
    s["k_cache"][slots // ps, slots % ps] = s["k"][kept]
    s["v_cache"][slots // ps, slots % ps] = s["v"][kept]
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _own_append(s):
    from local_kimi_b200 import ops

    ops.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    return {"k": s["k_cache"], "v": s["v_cache"]}


_PLAIN = {"prompt": _plain_prompt, "tree": _plain_tree, "verify": _plain_verify,
          "plan": _plain_plan, "append": _plain_append}
_OWN = {"prompt": _own_prompt, "tree": _own_tree, "verify": _own_verify, "plan": _own_plan,
        "append": _own_append}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    op = case["op"]
    size = torch.empty(0, dtype=_TYPES[case["type"]]).element_size() if "type" in case else 0
    if op == "prompt":
        lens, pre = _lens(case), case["prefix"]
        h, g, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
        pairs = sum(n * pre + n * (n + 1) // 2 for n in lens)
        rows, keys = sum(lens), sum(lens) + pre * len(lens)
        return {"bytes": size * (rows * h + keys * g) * (dk + dv) + 4 * rows * h * case["lse"],
                "flops": 2 * (dk + dv) * h * pairs}
    if op == "tree":
        ctx, new = _lens(case), _counts(case)
        h, g, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
        if case["tree"]:
            seen = [[bin(w & ((1 << 64) - 1)).count("1") for w in _masks([r])]
                    for r in _parents(case, new)]
        else:
            seen = [list(range(1, n + 1)) for n in new]
        pairs = sum(c * n + sum(w) for c, n, w in zip(ctx, new, seen))
        rows, keys = sum(new), sum(ctx) + sum(new)
        return {"bytes": size * (rows * h + keys * g) * (dk + dv) + 4 * rows * h * case["lse"],
                "flops": 2 * (dk + dv) * h * pairs}
    if op == "verify":
        new, v, b = _counts(case), case["vocab"], case["requests"]
        sampled = b - case["greedy"]
        # Every logit once; a row of noise (and of draft probabilities) where one is sampled.
        return {"bytes": size * v * sum(new) + 4 * v * sampled * (2 if case["probs"] else 1),
                "flops": 3 * v * sum(new)}
    if op == "plan":
        ctx, new, ps = _lens(case), _counts(case), case["page"]
        fresh = sum(-(-(c + n) // ps) - (-(-c // ps)) for c, n in zip(ctx, new))
        n = sum(new)
        return {"bytes": 12 * case["requests"] + 8 * fresh + (24 if case["tree"] else 12) * n,
                "flops": 4 * n}
    n = case["tokens"] - case["skipped"]
    return {"bytes": 2 * size * n * case["kv_heads"] * (case["dk"] + case["dv"]) + 8 * n,
            "flops": 0}


# ---------------------------------------------------------------------------
# the attention outputs in 64 bits, one head of one request at a time
# ---------------------------------------------------------------------------


def _exact_rows(q, k, v, hidden, scale):
    """q [T, Dk], k [S, Dk], v [S, Dv] in 64 bits, hidden [T, S]: softmax by its definition."""
    scores = (q @ k.T) * scale
    scores[hidden] = -math.inf
    lse = torch.logsumexp(scores, dim=1)
    share = torch.exp(scores - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    return share @ v, lse


def exact(case, seed):
    if case["op"] not in ("prompt", "tree"):
        return None
    s = prepare(case, seed)
    rows, h, g = s["q"].shape[0], case["heads"], case["kv_heads"]
    out = torch.empty((rows, h, case["dv"]), dtype=torch.float64, device="cuda")
    lse = torch.empty((rows, h), dtype=torch.float64, device="cuda")
    if case["op"] == "prompt":
        parts = []
        cq, ck = _sums(s["q_lens"]), _sums(s["k_lens"])
        for i, (n, m) in enumerate(zip(s["q_lens"], s["k_lens"])):
            hidden = torch.ones((n, m), dtype=torch.bool, device="cuda").triu(m - n + 1)
            parts.append((cq[i], n, s["k"][ck[i]:ck[i + 1]], s["v"][ck[i]:ck[i + 1]], hidden))
    else:
        parts = []
        trees = _parents(case, s["new"]) if case["tree"] else [
            list(range(-1, n - 1)) for n in s["new"]]
        cq = _sums(s["new"])
        for i, (c, n) in enumerate(zip(s["ctx"], s["new"])):
            places = torch.arange(c + n, device="cuda")
            page = s["table"][i].long()[places // case["page"]]
            line = [[True] * n for _ in range(n)]
            for t in range(n):
                a = t
                while a >= 0:
                    line[t][a] = False
                    a = trees[i][a]
            hidden = torch.cat((torch.zeros((n, c), dtype=torch.bool, device="cuda"),
                                torch.tensor(line, dtype=torch.bool, device="cuda")), dim=1)
            parts.append((cq[i], n, s["k_cache"][page, places % case["page"]],
                          s["v_cache"][page, places % case["page"]], hidden))
    for q0, n, k, v, hidden in parts:
        for head in range(h):
            kv = head // (h // g)
            got = _exact_rows(s["q"][q0:q0 + n, head].double(), k[:, kv].double(),
                              v[:, kv].double(), hidden, s["scale"])
            out[q0:q0 + n, head], lse[q0:q0 + n, head] = got
    return {"out": out, "lse": lse} if case["lse"] else out
