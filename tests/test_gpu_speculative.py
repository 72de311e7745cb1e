"""The speculative serving operators against their definitions in 64 bits (GPU).

Attention tolerance.  Products of 16-bit inputs and their sums are held in
fp32, the softmax weights are rounded once to the inputs' type before they
meet the values (relative 2^-9 bf16, 2^-12 f16, so at most that times
sum_j p_j |v_j|) and the result once more (that times |o|).  The tests allow
twice this bound, for the fp32 sums and exponentials in between.  The
log-sum-exp comes from fp32 scores alone: a score of up to 192 products is
within 192 * 2^-24 * sum |q k| * scale, below 2e-4 for the inputs here.
Whole numbers (slots, tokens, paths) have to be equal.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from local_kimi_b200 import _lib, ops
from oracle import speculative as ref

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
LSE_TOL = 2e-4


def check_attention(out, lse, want, want_lse, size, dtype):
    o, e = out.detach().double().cpu(), want
    assert torch.isfinite(o).all()
    room = 2 * STEP[dtype] * (size + e.abs()) + 1e-6
    bad = (o - e).abs() > room
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} outputs off by up to "
        f"{float(((o - e).abs() / room).max()):.3g} times the bound; first at "
        f"{bad.nonzero()[0].tolist()}")
    if lse is not None:
        got = lse.double().cpu()
        assert torch.equal(torch.isinf(got), torch.isinf(want_lse))
        fin = torch.isfinite(want_lse)
        assert float((got[fin] - want_lse[fin]).abs().max() if fin.any() else 0.0) < LSE_TOL


def sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def ints(values, cuda, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=cuda)


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,extra,heads,kv,dk,dv", [
    ([1], [0], 1, 1, 64, 64),
    ([5, 1, 0, 17], [0, 0, 0, 0], 4, 4, 192, 128),
    ([130, 3, 127, 128, 129], [0, 1, 200, 0, 64], 8, 2, 128, 128),
    ([257, 31], [0, 300], 6, 2, 72, 40),
    ([300], [0], 7, 1, 96, 96),
    ([513, 2], [0, 0], 3, 3, 192, 128),
    ([64, 200, 1], [100, 0, 511], 16, 1, 128, 64),
    ([40, 600], [0, 1], 5, 5, 8, 8),
])
def test_prompt_attention(cuda, dtype, lens, extra, heads, kv, dk, dv):
    gen = torch.Generator().manual_seed(sum(lens) + heads)
    keys = [n + x for n, x in zip(lens, extra)]
    q = torch.randn(sum(lens), heads, dk, generator=gen).to(dtype)
    k = torch.randn(sum(keys), kv, dk, generator=gen).to(dtype)
    v = torch.randn(sum(keys), kv, dv, generator=gen).to(dtype)
    cq, ck, scale = sums(lens), sums(keys), dk ** -0.5
    out, lse = ops.prompt_attention(q.to(cuda), k.to(cuda), v.to(cuda), ints(cq, cuda),
                                    max(lens), cu_seqlens_k=ints(ck, cuda), return_lse=True)
    check_attention(out, lse, *ref.prompt_attention(q, k, v, cq, ck, scale), dtype)


@pytest.mark.parametrize("lens,heads,kv,dk,dv", [
    ([40, 7], 400, 400, 64, 64), ([1500, 1, 900], 32, 32, 192, 128), ([2100, 300], 24, 3, 128, 128),
])
def test_prompt_attention_many_units(cuda, lens, heads, kv, dk, dv):
    # More units of rows than SMs, so a CTA goes through several; the softmax
    # by its definition in 64 bits, all heads at once on the device.
    gen = torch.Generator(device=cuda).manual_seed(len(lens) + heads)
    q = torch.randn(sum(lens), heads, dk, generator=gen, device=cuda).bfloat16()
    k = torch.randn(sum(lens), kv, dk, generator=gen, device=cuda).bfloat16()
    v = torch.randn(sum(lens), kv, dv, generator=gen, device=cuda).bfloat16()
    cu = sums(lens)
    out, lse = ops.prompt_attention(q, k, v, ints(cu, cuda), max(lens), return_lse=True)
    for a, b in zip(cu, cu[1:]):
        x = q[a:b].double().view(b - a, kv, heads // kv, dk)
        s = torch.einsum("tkgd,skd->kgts", x, k[a:b].double()) * dk ** -0.5
        s.masked_fill_(torch.ones(b - a, b - a, dtype=torch.bool, device=cuda).triu(1),
                       float("-inf"))
        w, p = s.logsumexp(-1), s.softmax(-1)
        want = torch.einsum("kgts,skd->tkgd", p, v[a:b].double()).reshape(b - a, heads, dv)
        size = torch.einsum("kgts,skd->tkgd", p, v[a:b].double().abs()).reshape(b - a, heads, dv)
        check_attention(out[a:b], lse[a:b], want.cpu(), w.permute(2, 0, 1).reshape(b - a, heads).cpu(),
                        size.cpu(), torch.bfloat16)


def test_prompt_attention_rows_without_keys(cuda):
    # More queries than keys: the first rows of a request see nothing.
    gen = torch.Generator().manual_seed(7)
    lens, keys = [200, 5, 3], [60, 0, 3]
    q = torch.randn(sum(lens), 4, 64, generator=gen).bfloat16()
    k = torch.randn(sum(keys), 2, 64, generator=gen).bfloat16()
    v = torch.randn(sum(keys), 2, 64, generator=gen).bfloat16()
    cq, ck = sums(lens), sums(keys)
    out, lse = ops.prompt_attention(q.to(cuda), k.to(cuda), v.to(cuda), ints(cq, cuda), 200,
                                    cu_seqlens_k=ints(ck, cuda), return_lse=True)
    check_attention(out, lse, *ref.prompt_attention(q, k, v, cq, ck, 0.125), torch.bfloat16)
    assert float(out[:140].abs().max()) == 0.0 and torch.isinf(lse[:140]).all()


def test_prompt_attention_strided_inputs_and_a_side_stream(cuda):
    # Slices of one projection output, on a stream of their own.
    gen = torch.Generator().manual_seed(8)
    fused = torch.randn(333, 10, 128, generator=gen).half()
    dev = fused.to(cuda)
    q, k, v = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    cq = sums([133, 200])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.prompt_attention(dev[:, :6], dev[:, 6:8], dev[:, 8:], ints(cq, cuda), 200,
                                   scale=0.1)
    side.synchronize()
    want, _, size = ref.prompt_attention(q, k, v, cq, cq, 0.1)
    check_attention(out, None, want, None, size, torch.float16)
    # A width that is not a multiple of the row alignment's stride: copied first.
    odd = torch.randn(50, 3, 67, generator=gen).half().to(cuda)[..., :64]
    got = ops.prompt_attention(odd, odd, odd, ints([0, 50], cuda), 50)
    x = odd.cpu()
    want, _, size = ref.prompt_attention(x, x, x, [0, 50], [0, 50], 0.125)
    check_attention(got, None, want, None, size, torch.float16)


def test_prompt_attention_large_scores_and_infinite_neighbours(cuda):
    # Scores up to several hundred (the running maximum moves), and a request
    # whose neighbours hold infinities and not-a-numbers.
    gen = torch.Generator().manual_seed(9)
    lens = [100, 190, 70]
    q = 6 * torch.randn(sum(lens), 2, 128, generator=gen)
    k = 6 * torch.randn(sum(lens), 2, 128, generator=gen)
    v = torch.randn(sum(lens), 2, 128, generator=gen)
    for t in (q, k, v):
        t[290:] = float("nan")
        t[:100] = float("inf")
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    cq = sums(lens)
    out, lse = ops.prompt_attention(q.to(cuda), k.to(cuda), v.to(cuda), ints(cq, cuda), 190,
                                    return_lse=True)
    want = ref.prompt_attention(q[100:290], k[100:290], v[100:290], [0, 190], [0, 190],
                                128 ** -0.5)
    # The scores are ~36 times larger than in the other tests, and so is their room.
    o, e = out[100:290].double().cpu(), want[0]
    assert torch.isfinite(o).all()
    assert bool(((o - e).abs() <= 4 * STEP[torch.bfloat16] * (want[2] + e.abs()) + 1e-6).all())
    assert float((lse[100:290].double().cpu() - want[1]).abs().max()) < 36 * LSE_TOL


def test_prompt_attention_hidden_later_tokens_do_not_matter(cuda):
    # What a row does not see does not change it, infinities included.
    gen = torch.Generator().manual_seed(10)
    x = torch.randn(150, 2, 64, generator=gen).bfloat16().to(cuda)
    cu = ints([0, 150], cuda)
    base = ops.prompt_attention(x, x, x, cu, 150)
    y = x.clone()
    y[100] = float("inf")
    y[120] = float("nan")
    got = ops.prompt_attention(x, x, y, cu, 150)
    assert torch.equal(got[:100], base[:100])
    assert not torch.isfinite(got[100:]).any()
    got = ops.prompt_attention(x, y, x, cu, 150)
    assert torch.equal(got[:100], base[:100])


def test_prompt_attention_empty(cuda):
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    assert ops.prompt_attention(q, q, q, ints([0], cuda), 0).shape == (0, 2, 64)
    assert ops.prompt_attention(q, q, q, ints([0, 0], cuda), 0).shape == (0, 2, 64)


# ---------------------------------------------------------------------------
# drafted tokens over the paged cache
# ---------------------------------------------------------------------------


def paged_case(cuda, dtype, ctx, new, heads, kv, dk, dv, ps, seed, head_major=True, tree=True):
    """Caches with not-a-numbers wherever nothing was written."""
    r, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    need = [-(-(c + n) // ps) for c, n in zip(ctx, new)]
    ids = list(range(sum(need) + 3))
    r.shuffle(ids)
    table = [[0] * (max(need) + 1) for _ in ctx]
    shape = (len(ids), kv, ps) if head_major else (len(ids), ps, kv)
    caches = []
    for d in (dk, dv):
        full = torch.full((*shape, d), float("nan"))
        caches.append(full.transpose(1, 2) if head_major else full)
    at = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        for i in range(need[b]):
            table[b][i] = ids[at]
            rows = min(ps, c + n - i * ps)
            for cache in caches:
                cache[ids[at], :rows] = torch.randn(rows, kv, cache.shape[3], generator=gen)
            at += 1
    kc, vc = (c.to(dtype) for c in caches)
    q = torch.randn(sum(new), heads, dk, generator=gen).to(dtype)
    parents = [([-1] + [r.randint(max(0, t - 3), t - 1) for t in range(1, n)])[:n] for n in new]
    sees = [a for p in parents for a in ref.ancestors(p)] if tree else None
    words = [w for p in parents for w in ref.tree_words(p)] if tree else None
    dev = dict(q=q.to(cuda), k_cache=kc.to(cuda), v_cache=vc.to(cuda),
               block_table=ints(table, cuda), context_lens=ints(ctx, cuda),
               cu_tokens=ints(sums(new), cuda), max_tokens=max(new),
               tree_mask=ints(words, cuda, torch.long) if tree else None)
    want = ref.tree_attention(q, kc, vc, table, ctx, sums(new), sees, dk ** -0.5)
    return dev, want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ctx,new,heads,kv,dk,dv,ps,tree", [
    ([0], [1], 1, 1, 64, 64, 8, False),
    ([5, 64, 0, 63], [1, 1, 1, 1], 4, 4, 192, 128, 64, False),
    ([300, 1, 700], [1, 1, 1], 32, 2, 128, 128, 16, False),
    ([129, 31, 0, 500], [7, 12, 3, 1], 8, 2, 128, 128, 16, True),
    ([100, 257], [24, 9], 8, 8, 192, 128, 32, True),
    ([77, 10, 400], [48, 64, 33], 4, 1, 64, 64, 8, True),
    ([200, 3], [5, 17], 6, 2, 72, 40, 128, True),
    ([64, 90], [9, 40], 3, 3, 96, 96, 64, False),
    ([1000, 0], [100, 70], 2, 1, 128, 128, 32, False),
    ([33, 0, 8], [2, 0, 5], 5, 1, 128, 64, 256, True),
    ([1500], [3], 64, 64, 192, 128, 64, True),
])
def test_tree_attention(cuda, dtype, ctx, new, heads, kv, dk, dv, ps, tree):
    dev, want = paged_case(cuda, dtype, ctx, new, heads, kv, dk, dv, ps, 31 + heads, tree=tree)
    out, lse = ops.tree_attention(**dev, return_lse=True)
    check_attention(out, lse, *want, dtype)
    # The workspace is left as it was found: the same call again.
    again = ops.tree_attention(**dev)
    assert torch.equal(out, again)


def test_tree_attention_row_major_pages(cuda):
    dev, want = paged_case(cuda, torch.bfloat16, [99, 200], [3, 6], 8, 2, 128, 128, 16, 5,
                           head_major=False)
    out, lse = ops.tree_attention(**dev, return_lse=True)
    check_attention(out, lse, *want, torch.bfloat16)


def test_tree_attention_many_requests(cuda):
    r = random.Random(3)
    ctx = [r.choice([0, 1, 15, 16, 17, r.randint(0, 300)]) for _ in range(150)]
    new = [r.choice([0, 1, 1, 4]) for _ in range(150)]
    new[0] = 4
    dev, want = paged_case(cuda, torch.float16, ctx, new, 4, 2, 64, 64, 16, 6)
    out, lse = ops.tree_attention(**dev, return_lse=True)
    check_attention(out, lse, *want, torch.float16)


def test_tree_attention_masks_that_hide_everything(cuda):
    # No context and an empty word: the row is zero.
    dev, _ = paged_case(cuda, torch.bfloat16, [0, 20], [3, 3], 4, 2, 64, 64, 16, 7)
    dev["tree_mask"] = ints([0, 2, 7, 0, 1, 4], cuda, torch.long)
    out, lse = ops.tree_attention(**dev, return_lse=True)
    assert float(out[0].abs().max()) == 0.0 and torch.isinf(lse[0]).all()
    q, kc, vc = (dev[n].cpu() for n in ("q", "k_cache", "v_cache"))
    want = ref.tree_attention(q, kc, vc, dev["block_table"].tolist(), [0, 20], [0, 3, 6],
                              [[], [1], [0, 1, 2], [], [0], [2]], 0.125)
    check_attention(out, lse, *want, torch.bfloat16)


def test_tree_attention_hidden_tokens_may_hold_anything(cuda):
    # A drafted token with infinities is seen by itself alone.
    dev, _ = paged_case(cuda, torch.bfloat16, [37], [4], 4, 2, 64, 64, 16, 8)
    dev["tree_mask"] = ints([1, 3, 5, 9], cuda, torch.long)
    base = ops.tree_attention(**dev)
    page, row = divmod(37 + 2, 16)
    page = int(dev["block_table"][0, page])
    dev["v_cache"][page, row] = float("inf")
    dev["k_cache"][page, row] = float("nan")
    got = ops.tree_attention(**dev)
    assert torch.equal(got[[0, 1, 3]], base[[0, 1, 3]])


def test_tree_attention_pages_outside_the_cache_count_as_absent(cuda):
    dev, _ = paged_case(cuda, torch.bfloat16, [50, 20], [2, 2], 4, 2, 64, 64, 16, 9, tree=False)
    _lib_errors()
    table = dev["block_table"]
    table[0, 1] = -1
    table[1, 0] = 10 ** 6
    dev["block_table"] = table[:, :3]      # request 0 needs a fourth page
    out, lse = ops.tree_attention(**dev, return_lse=True)
    assert _lib_errors() == 4
    q, kc, vc = (dev[n].cpu() for n in ("q", "k_cache", "v_cache"))
    want = ref.tree_attention(q, kc, vc, dev["block_table"].tolist(), [50, 20], [0, 2, 4], None,
                              0.125)
    check_attention(out, lse, *want, torch.bfloat16)


def _lib_errors():
    torch.cuda.synchronize()
    return _lib.device_errors()


# ---------------------------------------------------------------------------
# plan and append
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("requests,ps,longest,most,tree,pool,narrow", [
    (1, 16, 0, 1, False, 1, 0),
    (5, 8, 40, 9, True, 100, 0),
    (300, 16, 500, 20, False, 5000, 0),
    (3000, 64, 4000, 3, True, 9000, 0),
    (40, 32, 200, 64, True, 7, 0),          # the pool runs out
    (20, 8, 100, 30, False, 500, 4),        # the table is too narrow
])
def test_paged_plan(cuda, requests, ps, longest, most, tree, pool, narrow):
    r = random.Random(requests + ps)
    ctx = [r.choice([0, ps, ps - 1, r.randint(0, longest)]) for _ in range(requests)]
    ctx = [min(c, longest) for c in ctx]
    new = [r.choice([0, 1, most, r.randint(0, most)]) for _ in range(requests)]
    width = max(max(-(-(c + n) // ps) for c, n in zip(ctx, new)) - narrow, 1) + (0 if narrow else 1)
    table = [[r.randint(0, 10 ** 6) if i < -(-c // ps) else -7 for i in range(width)] for c in ctx]
    free = [r.randint(0, 10 ** 6) for _ in range(pool + 2)]
    total = sum(new) + 5
    parents = [p for n in new for p in
               ([-1] + [r.randint(max(0, t - 5), t - 1) for t in range(1, n)])[:n]]
    parents = (parents + [-1] * 5) if tree else None
    dev_table = ints(table, cuda)
    got = ops.paged_plan(ints(ctx, cuda), ints(new, cuda), dev_table, ints(free, cuda),
                         ints([2], cuda), ps, total,
                         parents=ints(parents, cuda) if tree else None)
    cu, slots, positions, masks, want_table, head, missing = ref.plan(
        ctx, new, table, free, 2, ps, total, parents)
    assert got.cu_tokens.tolist() == cu
    assert got.slots.tolist() == slots
    assert got.positions.tolist() == positions
    assert dev_table.tolist() == want_table
    assert got.free_head.tolist() == [head] and got.missing.tolist() == [missing]
    if tree:
        assert got.tree_mask.tolist() == masks
    else:
        assert got.tree_mask is None


def test_paged_plan_with_reserved_pages(cuda):
    # Pages that refused drafts left behind are used before new ones.
    r = random.Random(4)
    ps, requests = 8, 50
    ctx = [r.randint(0, 60) for _ in range(requests)]
    reserved = [c + r.choice([0, 0, 3, 9, 40]) for c in ctx]
    reserved[7] = 0                          # below the context: the context counts
    new = [r.randint(0, 30) for _ in range(requests)]
    table = [[r.randint(0, 999) if i < -(-max(c, h) // ps) else -1 for i in range(20)]
             for c, h in zip(ctx, reserved)]
    free = [r.randint(0, 999) for _ in range(300)]
    dev_table = ints(table, cuda)
    got = ops.paged_plan(ints(ctx, cuda), ints(new, cuda), dev_table, ints(free, cuda),
                         ints([0], cuda), ps, sum(new), reserved_lens=ints(reserved, cuda))
    cu, slots, positions, _, want_table, head, missing = ref.plan(
        ctx, new, table, free, 0, ps, sum(new), reserved=reserved)
    assert got.slots.tolist() == slots and got.positions.tolist() == positions
    assert dev_table.tolist() == want_table and got.cu_tokens.tolist() == cu
    assert got.free_head.tolist() == [head] and got.missing.tolist() == [missing]


def test_paged_plan_flags_bad_trees_and_short_outputs(cuda):
    _lib_errors()
    table = torch.full((1, 4), -1, dtype=torch.int32, device=cuda)
    args = (ints([0], cuda), ints([3], cuda), table, ints([5, 6], cuda), ints([0], cuda), 8)
    got = ops.paged_plan(*args, 3, parents=ints([-1, 2, 0], cuda))
    assert _lib_errors() == 8
    assert got.tree_mask.tolist() == [1, 2, 5]
    got = ops.paged_plan(*args, 2)
    assert _lib_errors() == 4
    assert got.cu_tokens.tolist() == [0, 2] and got.slots.tolist() == [40, 41]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,dk,dv,ps,head_major", [
    (1, 1, 64, 64, 8, True), (7, 3, 72, 40, 16, False), (300, 32, 192, 128, 64, True),
    (1000, 2, 8, 128, 8, True),
])
def test_paged_append(cuda, dtype, tokens, heads, dk, dv, ps, head_major):
    gen = torch.Generator().manual_seed(tokens)
    pages = tokens // ps + 2
    slots = torch.randperm(pages * ps, generator=gen)[:tokens]
    if tokens > 3:
        slots[2] = -1
    kv = [torch.randn(tokens, heads + 1, d, generator=gen).to(dtype)[:, 1:] for d in (dk, dv)]
    shape = (pages, heads, ps) if head_major else (pages, ps, heads)
    caches = [torch.randn(*shape, d, generator=gen).to(dtype) for d in (dk, dv)]
    views = [c.transpose(1, 2) if head_major else c for c in caches]
    dev = [v.to(cuda) for v in views]
    ops.paged_append(kv[0].to(cuda), kv[1].to(cuda), *dev, slots.to(cuda))
    for x, view, got in zip(kv, views, dev):
        want = view.clone()
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                want[s // ps, s % ps] = x[t]
        assert torch.equal(got.cpu(), want)


def test_paged_append_flags_slots_outside_the_cache(cuda):
    _lib_errors()
    x = torch.ones(2, 1, 64, dtype=torch.half, device=cuda)
    c = torch.zeros(2, 8, 1, 64, dtype=torch.half, device=cuda)
    ops.paged_append(x, x, c, c.clone(), ints([16, 3], cuda, torch.long))
    assert _lib_errors() == 4
    assert float(c.sum()) == 64 and float(c[0, 3].sum()) == 64


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------


def verify_case(requests, vocab, most, tree, probs, greedy, dtype, seed, sharp=2.0, empty=False):
    r, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    new = [r.randint(0 if empty else 1, most) for _ in range(requests)]
    new[0] = most
    cu = sums(new)
    parents = [p for n in new for p in
               ([-1] + [r.randint(max(0, t - 3), t - 1) if tree else t - 1
                        for t in range(1, n)])[:n]]
    logits = (sharp * torch.randn(cu[-1], vocab, generator=gen)).to(dtype)
    q = torch.empty(cu[-1], vocab)
    tokens = torch.zeros(cu[-1], dtype=torch.long)
    for b in range(requests):
        for t in range(new[b]):
            row = cu[b] + t
            base = logits[cu[b] + max(0, parents[row])].float()
            q[row] = torch.softmax(base + 0.7 * torch.randn(vocab, generator=gen), 0)
            tokens[row] = torch.multinomial(q[row], 1, generator=gen)
    coin = torch.rand(cu[-1], generator=gen)
    noise = torch.empty(requests, vocab).exponential_(generator=gen).clamp_min(1e-30)
    temps = torch.tensor([0.0 if i < greedy else 0.8 for i in range(requests)])
    return dict(logits=logits, tokens=tokens, parents=parents, cu=cu, most=most, coin=coin,
                noise=noise, temps=temps, probs=q if probs else None)


def run_verify(c, cuda, tree):
    return ops.verify_drafts(
        c["logits"].to(cuda), c["tokens"].to(cuda), ints(c["cu"], cuda), c["most"],
        c["coin"].to(cuda), c["noise"].to(cuda), c["temps"].to(cuda),
        parents=ints(c["parents"], cuda) if tree else None,
        draft_probs=None if c["probs"] is None else c["probs"].to(cuda))


@pytest.mark.parametrize("requests,vocab,most,tree,probs,greedy,dtype", [
    (1, 7, 1, False, False, 0, torch.float32),
    (6, 100, 5, False, True, 1, torch.float32),
    (9, 1003, 9, True, False, 2, torch.bfloat16),
    (40, 5000, 64, True, False, 0, torch.float16),
    (3, 163840, 9, True, False, 1, torch.bfloat16),
    (5, 50257, 6, False, True, 0, torch.bfloat16),
    (33, 777, 4, False, False, 33, torch.float16),
    (200, 257, 3, False, True, 7, torch.float32),
])
def test_verify_drafts(cuda, requests, vocab, most, tree, probs, greedy, dtype):
    c = verify_case(requests, vocab, most, tree, probs, greedy, dtype, 50 + requests,
                    empty=requests > 30)
    want = ref.verify(c["logits"], c["tokens"], c["parents"], c["cu"], most, c["coin"],
                      c["noise"], c["temps"], c["probs"])
    for _ in range(2):          # the counters are left at zero
        got = run_verify(c, cuda, tree)
        assert got.accepted.tolist() == want[2]
        assert got.path.tolist() == want[1]
        assert got.tokens.tolist() == want[0]


def test_verify_drafts_keeps_the_targets_distribution(cuda):
    # 4000 requests, one drafted token each from q: the first emitted token is
    # distributed as p, with and without q (5 sigma of a binomial count).
    vocab, n = 12, 4000
    gen = torch.Generator().manual_seed(77)
    row = torch.randn(vocab, generator=gen)
    p = torch.softmax(row.double(), 0)
    q = torch.softmax(row + torch.randn(vocab, generator=gen), 0)
    for probs in (True, False):
        drafts = torch.multinomial(q, n, replacement=True, generator=gen)
        tokens = torch.stack((torch.zeros_like(drafts), drafts), 1).flatten()
        got = ops.verify_drafts(
            row.expand(2 * n, vocab).contiguous().to(cuda), tokens.to(cuda),
            torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=cuda), 2,
            torch.rand(2 * n, generator=gen).to(cuda),
            torch.empty(n, vocab).exponential_(generator=gen).to(cuda),
            torch.ones(n, device=cuda),
            draft_probs=q.expand(2 * n, vocab).contiguous().to(cuda) if probs else None)
        count = torch.bincount(got.tokens[:, 0].cpu(), minlength=vocab).double()
        off = (count - n * p).abs() / (n * p * (1 - p)).sqrt()
        assert float(off.max()) < 5.0


def test_verify_drafts_not_a_number_and_infinite_logits(cuda):
    c = verify_case(4, 300, 3, True, False, 1, torch.float32, 9)
    c["logits"][:, 5] = float("nan")
    c["logits"][:, 9] = float("-inf")
    want = ref.verify(c["logits"], c["tokens"], c["parents"], c["cu"], 3, c["coin"], c["noise"],
                      c["temps"])
    got = run_verify(c, cuda, True)
    assert got.tokens.tolist() == want[0] and got.path.tolist() == want[1]
    # One infinite logit takes everything.
    c["logits"][:, 17] = float("inf")
    got = run_verify(c, cuda, True)
    last = got.tokens.gather(1, got.accepted.long()[:, None])
    taken = (got.tokens == 17).any(dim=1)
    assert bool(((last[:, 0] == 17) | taken).all())


def test_verify_drafts_flags_bad_trees_and_tokens(cuda):
    _lib_errors()
    c = verify_case(2, 50, 3, False, False, 0, torch.float32, 10)
    c["tokens"][1] = 50
    got = run_verify(c, cuda, False)
    assert _lib_errors() == 8
    assert got.accepted.tolist()[0] == 0


def test_operators_in_a_cuda_graph(cuda):
    # Plan, append, attention and verification replayed from one graph.
    dev, want = paged_case(cuda, torch.bfloat16, [50, 20], [4, 2], 4, 2, 64, 64, 16, 11)
    c = verify_case(2, 500, 3, True, False, 0, torch.bfloat16, 12)
    cd = {n: (t.to(cuda) if torch.is_tensor(t) else t) for n, t in c.items()}
    cu, par = ints(c["cu"], cuda), ints(c["parents"], cuda)

    def step():
        out = ops.tree_attention(**dev)
        got = ops.verify_drafts(cd["logits"], cd["tokens"], cu, 3, cd["coin"], cd["noise"],
                                cd["temps"], parents=par)
        return out, got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], eager[0])
    assert torch.equal(held[1].tokens, eager[1].tokens)
    check_attention(held[0], None, want[0], None, want[2], torch.bfloat16)
    assert math.isfinite(float(held[0].float().sum()))


# ---------------------------------------------------------------------------
# what is visible and no finite number
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("new,heads,kv", [([1, 1], 4, 2), ([5, 2], 6, 2), ([24, 5], 8, 2),
                                          ([60, 3], 8, 2)])
def test_tree_attention_a_query_that_is_no_number_is_seen(cuda, new, heads, kv):
    # Over a context that several CTAs share, as over one that a single CTA has.
    dev, _ = paged_case(cuda, torch.bfloat16, [6000, 20], new, heads, kv, 128, 128, 16, 41)
    base, base_lse = ops.tree_attention(**dev, return_lse=True)
    last = sum(new) - 1
    for value in (float("nan"), float("inf")):
        q = dev["q"].clone()
        q[0, 1] = value
        q[last, 0] = value
        out, lse = ops.tree_attention(**{**dev, "q": q}, return_lse=True)
        for t, h in ((0, 1), (last, 0)):
            assert torch.isnan(out[t, h]).all() and torch.isnan(lse[t, h])
            out[t, h], lse[t, h] = base[t, h], base_lse[t, h]
        assert torch.equal(out, base) and torch.equal(lse, base_lse)


@pytest.mark.parametrize("ctx", [40, 6000])
@pytest.mark.parametrize("new", [1, 24])
def test_tree_attention_infinite_values_meet_weights_of_zero(cuda, ctx, new):
    # The last cached key takes all the weight; the first one's value is infinite, and
    # zero times infinity is no number, whichever CTA had the key.
    dev, _ = paged_case(cuda, torch.bfloat16, [ctx], [new], 4, 2, 128, 128, 16, 42)
    table, kc, vc = dev["block_table"][0], dev["k_cache"], dev["v_cache"]
    dev["q"].copy_(torch.ones_like(dev["q"]))
    page, row = divmod(ctx - 1, 16)
    kc[int(table[page]), row] = 64.0          # score 724, the others' are of order ten
    vc[int(table[0]), 0, :, :8] = float("inf")
    out, lse = ops.tree_attention(**dev, return_lse=True)
    assert torch.isfinite(lse).all() and torch.isfinite(out[..., 8:]).all()
    assert not torch.isfinite(out[..., :8]).any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("key", list(range(64, 80)) + [127])
def test_prompt_attention_a_visible_key_that_is_no_number_is_seen(cuda, value, key):
    # At any place of a step that all rows of a tile see whole.
    gen = torch.Generator().manual_seed(11)
    q = torch.rand(400, 4, 64, generator=gen).add_(0.1).bfloat16().to(cuda)
    k, v = (torch.randn(400, 2, 64, generator=gen).bfloat16().to(cuda) for _ in range(2))
    cu = ints([0, 400], cuda)
    base, base_lse = ops.prompt_attention(q, k, v, cu, 400, return_lse=True)
    k[key, 1] = value                        # its score is infinite or not a number
    out, lse = ops.prompt_attention(q, k, v, cu, 400, return_lse=True)
    assert torch.equal(out[:, :2], base[:, :2]) and torch.equal(lse[:, :2], base_lse[:, :2])
    assert torch.equal(out[:key], base[:key]) and torch.equal(lse[:key], base_lse[:key])
    assert torch.isnan(out[key:, 2:]).all() and not torch.isfinite(lse[key:, 2:]).any()


@pytest.mark.parametrize("new", [1, 24, 60])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_tree_attention_a_visible_key_that_is_no_number_is_seen(cuda, new, value):
    dev, _ = paged_case(cuda, torch.float16, [3000], [new], 8, 2, 64, 64, 16, 43)
    dev["q"].abs_().add_(0.1)
    base, base_lse = ops.tree_attention(**dev, return_lse=True)
    for key in (0, 6, 15, 70, 1031, 2990):
        page, row = int(dev["block_table"][0, key // 16]), key % 16
        held = dev["k_cache"][page, row, 1].clone()
        dev["k_cache"][page, row, 1] = value
        out, lse = ops.tree_attention(**dev, return_lse=True)
        assert torch.equal(out[:, :4], base[:, :4]) and torch.equal(lse[:, :4], base_lse[:, :4])
        assert torch.isnan(out[:, 4:]).all() and not torch.isfinite(lse[:, 4:]).any()
        dev["k_cache"][page, row, 1] = held


def test_attention_scores_of_minus_infinity_count_nothing(cuda):
    # Rows with no other score are zero; the others see the finite keys alone.
    gen = torch.Generator().manual_seed(12)
    q = torch.rand(100, 2, 64, generator=gen).add_(0.1).bfloat16().to(cuda)
    k, v = (torch.randn(400, 2, 64, generator=gen).bfloat16().to(cuda) for _ in range(2))
    k[:350] = float("-inf")
    out, lse = ops.prompt_attention(q, k, v, ints([0, 100], cuda), 100,
                                    cu_seqlens_k=ints([0, 400], cuda), return_lse=True)
    assert not out[:50].any() and (lse[:50] == float("-inf")).all()
    # Queries 50 to 99 see the finite keys 350 to 350 + t - 50.
    want = ref.prompt_attention(q[50:].cpu(), k[350:].cpu(), v[350:].cpu(), [0, 50], [0, 50],
                                0.125)
    check_attention(out[50:], lse[50:], *want, torch.bfloat16)
    # The same over pages: one token a request, and more than 16 rows.
    for n in (1, 40):
        cache = [t[:384].view(24, 16, 2, 64) for t in (k, v)]
        table = torch.arange(24, dtype=torch.int32, device=cuda)[None]
        out, lse = ops.tree_attention(q[:n], *cache, table, ints([340 - n], cuda), ints([0, n], cuda),
                                      n, return_lse=True)
        assert not out.any() and (lse == float("-inf")).all()


def test_attention_scores_that_leave_fp32_are_no_numbers(cuda):
    # Finite products of 1.6e38 times a scale of 4.
    for n in (1, 300):
        q = torch.zeros(n, 1, 64, dtype=torch.bfloat16, device=cuda)
        k, v = q.clone(), torch.ones_like(q)
        q[:, :, 0] = 1.25e19
        k[:, :, 0] = 1.25e19
        out, lse = ops.prompt_attention(q, k, v, ints([0, n], cuda), n, scale=4.0,
                                        return_lse=True)
        assert torch.isnan(out).all() and not torch.isfinite(lse).any()


@pytest.mark.parametrize("greedy", [0, 9])
def test_verify_drafts_scratch_may_hold_anything(cuda, greedy, monkeypatch):
    c = verify_case(9, 5000, 5, True, False, greedy, torch.bfloat16, 44)
    want = ref.verify(c["logits"], c["tokens"], c["parents"], c["cu"], 5, c["coin"], c["noise"],
                      c["temps"])
    real, kept = _lib.call, []

    def call(name, *args):
        for fill in (255, 1):
            kept.append(torch.full((args[-2],), fill, dtype=torch.uint8, device=cuda))
            real(name, *args[:-3], kept[-1].data_ptr(), *args[-2:])

    monkeypatch.setattr(_lib, "call", call)
    got = run_verify(c, cuda, True)
    assert got.accepted.tolist() == want[2] and got.tokens.tolist() == want[0]


def test_graphs_of_one_capture_stream_replay_in_any_order(cuda):
    # Captured one after the other without a stream, so that both record on torch's own;
    # the second one is replayed first, then both beside each other.
    trees = [paged_case(cuda, torch.bfloat16, [2000, 90], [n, 2], 4, 2, 64, 64, 16, 45 + n)[0]
             for n in (1, 24)]
    c = verify_case(6, 3000, 4, False, True, 1, torch.bfloat16, 46)
    gen = torch.Generator().manual_seed(47)
    hidden = torch.randn(24, 512, generator=gen).bfloat16().to(cuda)
    weight = torch.randn(64, 512, generator=gen).bfloat16().to(cuda)
    cd = {n: (t.to(cuda) if torch.is_tensor(t) else t) for n, t in c.items()}
    cu = ints(c["cu"], cuda)

    def step():
        got = ops.verify_drafts(cd["logits"], cd["tokens"], cu, 4, cd["coin"], cd["noise"],
                                cd["temps"], draft_probs=cd["probs"])
        return [ops.tree_attention(**dev) for dev in trees] + [
            got.tokens, got.path, *ops.moe_router(hidden, weight, None, 4)]

    want = step()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    sides = [torch.cuda.Stream() for _ in graphs]
    for order in ([1], [0], [1, 0, 1, 0, 0, 1]):
        for held in outs:
            for t in held:
                t.zero_()
        torch.cuda.synchronize()
        for i in order:
            with torch.cuda.stream(sides[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in order:
            for got, expected in zip(outs[i], want):
                assert torch.equal(got, expected)
    for got, expected in zip(step(), want):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("requests,ps,longest,most,pool,narrow", [
    (1, 8, 30, 40, 3, 0), (60, 16, 500, 900, 700, 0), (300, 64, 4000, 5, 40, 0),
    (40, 8, 100, 60, 10 ** 4, 3),
])
def test_paged_reserve(cuda, requests, ps, longest, most, pool, narrow):
    # What is reached after a plan: the places up to the last one with a page.
    r = random.Random(requests + most)
    ctx = [r.randint(0, longest) for _ in range(requests)]
    reserved = [c + r.choice([0, 0, 3, most]) for c in ctx]
    new = [r.choice([0, 1, most, r.randint(0, most)]) for _ in range(requests)]
    width = -(-max(longest + 2 * most, 1) // ps) - narrow
    table = [[r.randint(0, 999) if i < -(-max(c, h) // ps) else -1 for i in range(width)]
             for c, h in zip(ctx, reserved)]
    dev_table, held = ints(table, cuda), ints(reserved, cuda)
    got = ops.paged_plan(ints(ctx, cuda), ints(new, cuda), dev_table,
                         ints([r.randint(0, 999) for _ in range(pool)], cuda), ints([0], cuda), ps,
                         sum(new), reserved_lens=held)
    ops.paged_reserve(ints(ctx, cuda), ints(new, cuda), dev_table, held, ps)
    cu, slots = got.cu_tokens.tolist(), got.slots.tolist()
    want = [max(c, h, *[c + t + 1 for t in range(n) if slots[cu[b] + t] >= 0], 0)
            for b, (c, h, n) in enumerate(zip(ctx, reserved, new))]
    assert held.tolist() == want


@pytest.mark.parametrize("tokens", [3, 200])
def test_attention_takes_expanded_heads_and_tokens(cuda, tokens):
    # One key/value head, or one query, expanded to all of them (strides of zero).
    gen = torch.Generator().manual_seed(15)
    one = torch.randn(tokens, 1, 64, generator=gen).bfloat16().to(cuda)
    q = torch.randn(tokens, 4, 64, generator=gen).bfloat16().to(cuda)
    cu, k = ints([0, tokens], cuda), one.expand(tokens, 4, 64)
    want = ops.prompt_attention(q, k.contiguous(), k.contiguous(), cu, tokens)
    assert torch.equal(ops.prompt_attention(q, k, k, cu, tokens), want)
    same = q[:1].expand(tokens, 4, 64)
    want = ops.prompt_attention(same.contiguous(), k.contiguous(), k.contiguous(), cu, tokens)
    assert torch.equal(ops.prompt_attention(same, k, k, cu, tokens), want)
    pages = -(-tokens // 16)
    kc, vc = (torch.zeros(pages, 16, 4, 64, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    ops.paged_append(k, k, kc, vc, torch.arange(tokens, device=cuda))
    assert torch.equal(kc.flatten(0, 1)[:tokens], k) and torch.equal(vc, kc)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    for wide in (q, same):
        got, want = (ops.tree_attention(x, kc, vc, table, ints([0], cuda), cu, tokens)
                     for x in (wide, wide.contiguous()))
        assert torch.equal(got, want)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_drafts_infinite_logits_share_the_draw(cuda, probs):
    # Several infinite logits count as equally likely, in the acceptance and in the draw.
    c = verify_case(60, 700, 3, False, probs, 0, torch.float32, 13)
    c["logits"][:, [5, 17, 300, 698]] = float("inf")
    x = c["logits"].clone()
    x[torch.isinf(x)] = 1e30               # what is largest by far, for the oracle
    want = ref.verify(x, c["tokens"], c["parents"], c["cu"], 3, c["coin"], c["noise"],
                      c["temps"], c["probs"])
    got = run_verify(c, cuda, False)
    assert got.tokens.tolist() == want[0] and got.path.tolist() == want[1]
    last = got.tokens.gather(1, got.accepted.long()[:, None])
    assert len(set(last.flatten().tolist())) > 1


def test_verify_drafts_emits_tokens_of_the_vocabulary_whatever_the_inputs(cuda):
    # Temperatures without a usable inverse, and noise that compares with nothing.
    c = verify_case(6, 300, 3, False, False, 0, torch.float32, 14)
    c["logits"][:, 40:60] = float("-inf")
    c["temps"] = torch.tensor([1e-40, 1e-44, float("inf"), 3e38, 0.8, 0.8])
    c["noise"][4:] = float("nan")
    got = run_verify(c, cuda, False)
    last = got.tokens.gather(1, got.accepted.long()[:, None])[:, 0]
    assert bool(((last >= 0) & (last < 300)).all())
    # Next to temperature 0 the draw is the argmax, and so is what is accepted.
    cold = run_verify({**c, "temps": torch.zeros(6)}, cuda, False)
    assert torch.equal(got.tokens[:2], cold.tokens[:2])
    # Without bound the finite logits are all as likely.
    x = torch.where(torch.isinf(c["logits"]), c["logits"], torch.zeros(()))
    want = ref.verify(x, c["tokens"], c["parents"], c["cu"], 3, c["coin"], c["noise"],
                      torch.ones(6))
    assert got.tokens[2].tolist() == want[0][2]


@pytest.mark.parametrize("new,heads", [([3, 2], 4), ([9, 30], 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tree_attention_contexts_past_the_table(cuda, dtype, new, heads):
    # Lengths that nobody meant: what the table has is seen, the rest is absent, and the
    # call takes no longer than for a full table.
    dev, _ = paged_case(cuda, dtype, [58, 20], new, heads, 2, 64, 64, 16, 17, tree=False)
    dev["block_table"] = dev["block_table"][:, :3].contiguous()
    q, kc, vc = (dev[n].cpu() for n in ("q", "k_cache", "v_cache"))
    want = ref.tree_attention(q, kc, vc, dev["block_table"].tolist(), [10 ** 4, 20], sums(new),
                              None, 0.125)
    for length in (10 ** 4, 2 ** 30, 2 ** 31 - 1):
        dev["context_lens"] = ints([length, 20], cuda)
        _lib_errors()
        out, lse = ops.tree_attention(**dev, return_lse=True)
        assert _lib_errors() == 4
        check_attention(out, lse, *want, dtype)
    dev["block_table"] = dev["block_table"][:, :0]
    out, lse = ops.tree_attention(**dev, return_lse=True)
    assert _lib_errors() == 4 and not out.any() and torch.isinf(lse).all()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("ps,rows,slots,missing", [
    (1, [[9, 8], [-1, -1], [-1, -1], [7, 6], [-1, -1]], [9, 8, *[-1] * 62], 2 ** 30 + 1),
    (8, [[9, -1], [-1, 8], [-1, -1], [7, 6], [-1, -1]],
     [72, 73, 74, *[-1] * 4, *range(64, 72), *[-1] * 49], 3 * 2 ** 27 - 2),
])
def test_paged_plan_of_lengths_that_nobody_meant(cuda, ps, rows, slots, missing, tree):
    # Lengths and sums past 2^30: what comes before is planned, the rest has no place.
    _lib_errors()
    table = torch.full((5, 2), -1, dtype=torch.int32, device=cuda)
    parents = ints([-1, 0, 1, -1, *range(60)], cuda) if tree else None
    ctx = ints([0, 4, 2 ** 31 - 1, 0, -7], cuda)
    new = ints([3, 2 ** 30, 2 ** 31 - 1, 2 ** 30, 5], cuda)
    got = ops.paged_plan(ctx, new, table, ints([9, 8, 7, 6], cuda), ints([0], cuda), ps, 64,
                         parents=parents)
    assert _lib_errors() == 4
    assert got.cu_tokens.tolist() == [0, 3, 64, 64, 64, 64]
    assert table.tolist() == rows and got.slots.tolist() == slots
    assert got.missing.tolist() == [missing] and got.free_head.tolist() == [4]
    if tree:
        assert got.positions.tolist() == [0, 1, 2, *range(4, 65)]
        assert got.tree_mask[:4].tolist() == [1, 3, 7, 1]
    held = ints([0, 0, 0, 0, 0], cuda)
    ops.paged_reserve(ctx, new, table, held, ps)
    assert held.tolist() == ([2, 4, 2 ** 30 - 1, 2, 0] if ps == 1 else [3, 16, 2 ** 30 - 1, 16, 0])


@pytest.mark.parametrize("requests,longest,heads,kv,dk,dv", [
    (33, 90, 4, 2, 64, 64), (100, 150, 6, 2, 128, 128), (257, 40, 8, 8, 192, 128),
])
def test_prompt_attention_many_requests(cuda, requests, longest, heads, kv, dk, dv):
    # More requests than a warp counts at once, empty and long ones among them.
    r, gen = random.Random(requests), torch.Generator(device=cuda).manual_seed(requests)
    lens = [r.choice([0, 1, r.randint(0, longest)]) for _ in range(requests)]
    lens[requests // 2] = 700
    keys = [n + r.choice([0, 0, 65]) if n else r.choice([0, 3]) for n in lens]
    q = torch.randn(sum(lens), heads, dk, generator=gen, device=cuda).bfloat16()
    k = torch.randn(sum(keys), kv, dk, generator=gen, device=cuda).bfloat16()
    v = torch.randn(sum(keys), kv, dv, generator=gen, device=cuda).bfloat16()
    cq, ck = sums(lens), sums(keys)
    out, lse = ops.prompt_attention(q, k, v, ints(cq, cuda), 700, cu_seqlens_k=ints(ck, cuda),
                                    return_lse=True)
    for b in range(requests):
        n, m = lens[b], keys[b]
        if n == 0:
            continue
        x = q[cq[b]:cq[b + 1]].double().view(n, kv, heads // kv, dk)
        s = torch.einsum("tkgd,skd->kgts", x, k[ck[b]:ck[b + 1]].double()) * dk ** -0.5
        s.masked_fill_(torch.ones(n, m, dtype=torch.bool, device=cuda).triu(1 + m - n),
                       float("-inf"))
        w, p, vb = s.logsumexp(-1), s.softmax(-1), v[ck[b]:ck[b + 1]].double()
        want, size = (torch.einsum("kgts,skd->tkgd", p, y).reshape(n, heads, dv).cpu()
                      for y in (vb, vb.abs()))
        check_attention(out[cq[b]:cq[b + 1]], lse[cq[b]:cq[b + 1]], want,
                        w.permute(2, 0, 1).reshape(n, heads).cpu(), size, torch.bfloat16)


@pytest.mark.parametrize("most", [17, 64, 5000])
def test_tree_attention_longest_length_far_above_the_lengths(cuda, most):
    # The kernel is chosen by max_tokens; what it computes is not.
    dev, want = paged_case(cuda, torch.bfloat16, [300, 0, 70, 1000], [1, 2, 0, 5], 8, 2, 128, 128,
                           16, 48, tree=False)
    dev["max_tokens"] = most
    out, lse = ops.tree_attention(**dev, return_lse=True)
    check_attention(out, lse, *want, torch.bfloat16)
    assert torch.equal(out, ops.tree_attention(**dev))


@pytest.mark.parametrize("new", [[1, 1], [5, 3], [30, 64]])
def test_caches_past_32_bit_offsets(cuda, new):
    # The same pages at the end of a cache of over 2^32 bytes (and 2^31 elements), written
    # by paged_append; an infinite value of the step is taken from the cache itself.
    dev, _ = paged_case(cuda, torch.bfloat16, [70, 500], new, 8, 4, 128, 128, 16, 49)
    pages = dev["k_cache"].shape[0]
    most = (2 ** 31 + 2 ** 25) // (4 * 16 * 128)
    table = dev["block_table"].clone()
    slots = torch.tensor([int(table[b, p // 16]) * 16 + p % 16 for b, n in enumerate(new)
                          for p in range([70, 500][b] + n)], device=cuda)
    last = int(table[1, (500 + new[1] - 1) // 16])
    dev["v_cache"][last, (500 + new[1] - 1) % 16, 0, 3] = float("inf")
    want, want_lse = ops.tree_attention(**dev, return_lse=True)
    big = [torch.empty(most, 4, 16, 128, dtype=torch.bfloat16, device=cuda).transpose(1, 2)
           for _ in range(2)]
    k, v = (dev[n].flatten(0, 1)[slots] for n in ("k_cache", "v_cache"))
    ops.paged_append(k, v, *big, slots + (most - pages) * 16)
    out, lse = ops.tree_attention(**{**dev, "k_cache": big[0], "v_cache": big[1],
                                     "block_table": table + (most - pages)}, return_lse=True)
    assert torch.equal(lse, want_lse)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[~out.isnan()], want[~want.isnan()])
    assert not torch.isfinite(out[-1, 0, 3]) and torch.isfinite(out[..., 4:]).all()


@pytest.mark.parametrize("probs", [False, True])
def test_verify_drafts_past_32_bit_offsets(cuda, probs):
    # The last rows of over 2^31 logits, as a batch of their own and as they lie.
    c = verify_case(3, 163840, 4, False, probs, 0, torch.bfloat16, 50)
    want = run_verify(c, cuda, False)
    n, rows = c["cu"][-1], 2 ** 31 // 163840 + 20
    logits = torch.empty(rows, 163840, dtype=torch.bfloat16, device=cuda)
    logits[-n:] = c["logits"].to(cuda)
    tokens = torch.zeros(rows, dtype=torch.long, device=cuda)
    tokens[-n:] = c["tokens"].to(cuda)
    coin = torch.zeros(rows, device=cuda)
    coin[-n:] = c["coin"].to(cuda)
    q = None
    if probs:
        q = torch.empty(rows, 163840, device=cuda)
        q[-n:] = c["probs"].to(cuda)
    got = ops.verify_drafts(logits, tokens, ints([rows - n + x for x in c["cu"]], cuda), 4, coin,
                            c["noise"].to(cuda), c["temps"].to(cuda), draft_probs=q)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
