"""The serving step end to end: drafted trees emit what the target itself would (GPU)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from local_kimi_b200 import _lib, ops
from local_kimi_b200.speculative import PagedCache, children_first_tree

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "speculative_serving.py"


def load_example():
    spec = importlib.util.spec_from_file_location("speculative_serving", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_logits(model, sequence):
    """Logits after every token of a sequence, plain torch in fp32 from the decoded weights."""
    from oracle.codec import dequantise

    def dense(x, w):
        return x @ dequantise(w[0].cpu(), w[1].cpu()).float().T.cuda()

    n = len(sequence)
    x = model.embedding[torch.tensor(sequence, device="cuda")].float()
    q = dense(x, model.q).view(n, model.heads, model.dk)
    k = dense(x, model.k).view(n, model.heads, model.dk)
    v = dense(x, model.v).view(n, model.heads, model.dv)
    s = torch.einsum("thd,shd->hts", q, k) * model.dk ** -0.5
    s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    x = x + dense(torch.einsum("hts,shd->thd", s.softmax(-1), v).flatten(1), model.o)
    return dense(x, model.head)


def test_speculative_serving_emits_the_targets_tokens(cuda):
    example = load_example()
    model = example.TinyTarget(vocab=2_048, hidden=256, heads=4, dk=192, dv=128, seed=3)
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(model.vocab, (n,), generator=gen) for n in (9, 1, 70, 33)]
    _lib.device_errors()
    emitted, accepted = example.serve(model, prompts, steps=6, page_size=8)
    assert _lib.device_errors() == 0
    assert accepted > 0
    for prompt, row in zip(prompts, emitted):
        sequence = prompt.tolist() + row
        logits = plain_logits(model, sequence[:-1])[len(prompt) - 1:]
        chosen = logits.gather(1, torch.tensor(row, device="cuda")[:, None])[:, 0]
        # Every emitted token is the target's argmax, up to the bf16 rounding of
        # activations and logits on the way (a few steps of 2^-8 of values of
        # order one; the logits spread over several units).
        assert float((logits.amax(dim=1) - chosen).max()) < 0.15


def test_cache_keeps_the_accepted_rows_in_a_row(cuda):
    cache = PagedCache(2, 12, 8, 1, 64, 64, dtype=torch.half)
    parents = children_first_tree(2, 2)                    # root, 1-2, 3-4
    counts = torch.tensor([5, 5], dtype=torch.int32, device=cuda)
    tree = torch.tensor(parents * 2, dtype=torch.int32, device=cuda)
    rows = [[], []]
    for step in range(4):
        plan = cache.plan(counts, 10, tree)
        value = torch.arange(10, device=cuda, dtype=torch.half) + 10 * step
        x = value[:, None, None].expand(10, 1, 64).contiguous()
        cache.append(x, x, plan)
        path = torch.tensor([[0, 3, 4, -1, -1], [0, 1, -1, -1, -1]], dtype=torch.int32,
                            device=cuda)
        got = ops.Verification(path.long(), path, torch.tensor([2, 1], device=cuda))
        cache.keep(plan, got)
        rows[0] += [10 * step, 10 * step + 3, 10 * step + 4]
        rows[1] += [10 * step + 5, 10 * step + 6]
    assert cache.context.tolist() == [12, 8]
    for b, want in enumerate(rows):
        got = [float(cache.v[int(cache.table[b, p // 8]), p % 8, 0, 0]) for p in range(len(want))]
        assert got == want
    # Pages left by refused tokens were used again: 14 and 11 places were reached.
    assert int(cache.head) == 2 + 2


def fill(cache, plan, base):
    """Appends rows that hold base, base + 1, ... and returns how many there are."""
    n = plan.slots.shape[0]
    value = torch.arange(n, device=cache.k.device, dtype=torch.half) + base
    x = value[:, None, None].expand(n, 1, 64).contiguous()
    cache.append(x, x, plan)


def held(cache, b):
    return [float(cache.v[int(cache.table[b, p // 8]), p % 8, 0, 0])
            for p in range(int(cache.context[b]))]


def test_cache_that_runs_out_of_pages_recovers(cuda):
    # Three pages for two requests that ask for four, then more pages.
    cache = PagedCache(2, 3, 8, 1, 64, 64, dtype=torch.half, max_pages=6)
    lens = torch.tensor([10, 12], dtype=torch.int32, device=cuda)
    plan = cache.plan(lens, 22)
    assert plan.missing.tolist() == [1]
    fill(cache, plan, 0)
    cache.advance(lens)
    # What has no page is not in the context.
    assert cache.context.tolist() == [10, 8]
    assert held(cache, 0) == list(range(10)) and held(cache, 1) == list(range(10, 18))
    # Another plan still misses the page, and the tree's tokens have no slots.
    counts = torch.tensor([5, 5], dtype=torch.int32, device=cuda)
    parents = children_first_tree(2, 2)
    tree = torch.tensor(parents * 2, dtype=torch.int32, device=cuda)
    plan = cache.plan(counts, 10, tree)
    assert plan.missing.tolist() == [1]
    assert plan.slots[5:].tolist() == [-1] * 5 and min(plan.slots[:5].tolist()) >= 0
    fill(cache, plan, 100)
    path = torch.tensor([[0, 3, 4, -1, -1], [0, 1, -1, -1, -1]], dtype=torch.int32, device=cuda)
    got = ops.Verification(path.long(), path, torch.tensor([2, 1], device=cuda))
    cache.keep(plan, got)
    assert cache.context.tolist() == [13, 8]
    assert held(cache, 0) == [*range(10), 100, 103, 104]
    assert held(cache, 1) == list(range(10, 18))
    # With pages in the pool again, the same tokens find their places.
    k, v = cache.k, cache.v
    more = PagedCache(2, 6, 8, 1, 64, 64, dtype=torch.half, max_pages=6)
    more.k[:3], more.v[:3] = k, v
    cache.k, cache.v = more.k, more.v
    cache.free = torch.arange(6, dtype=torch.int32, device=cuda)
    plan = cache.plan(counts, 10, tree)
    assert plan.missing.tolist() == [0] and min(plan.slots.tolist()) >= 0
    fill(cache, plan, 200)
    cache.keep(plan, got)
    assert cache.context.tolist() == [16, 10]
    assert held(cache, 0) == [*range(10), 100, 103, 104, 200, 203, 204]
    assert held(cache, 1) == [*range(10, 18), 205, 206]
    pages = [p for row in cache.table.tolist() for p in row if p >= 0]
    assert len(pages) == len(set(pages)) == int(cache.head)


def test_cache_keeps_drafts_up_to_the_last_slot(cuda):
    # A pool that ends inside a tree: an accepted token without a slot stays out, and
    # nothing is copied from another request's rows in its place.
    cache = PagedCache(2, 2, 8, 1, 64, 64, dtype=torch.half, max_pages=3)
    lens = torch.tensor([1, 6], dtype=torch.int32, device=cuda)
    fill(cache, cache.plan(lens, 7), 0)
    cache.advance(lens)
    counts = torch.tensor([5, 5], dtype=torch.int32, device=cuda)
    tree = torch.tensor(children_first_tree(2, 2) * 2, dtype=torch.int32, device=cuda)
    plan = cache.plan(counts, 10, tree)
    assert plan.missing.tolist() == [1] and plan.slots[5:].tolist()[2:] == [-1] * 3
    fill(cache, plan, 50)
    path = torch.tensor([[0, 1, 2, -1, -1], [0, 3, 4, -1, -1]], dtype=torch.int32, device=cuda)
    cache.keep(plan, ops.Verification(path.long(), path, torch.tensor([2, 2], device=cuda)))
    assert cache.context.tolist() == [4, 7]
    assert held(cache, 0) == [0, 50, 51, 52] and held(cache, 1) == [*range(1, 7), 55]


def test_cache_steps_replay_from_a_graph(cuda):
    # Lengths, the free list's head and the reserved pages move on with every replay.
    parents = children_first_tree(2, 2)
    counts = torch.tensor([5, 5], dtype=torch.int32, device=cuda)
    tree = torch.tensor(parents * 2, dtype=torch.int32, device=cuda)
    path = torch.tensor([[0, 3, 4, -1, -1], [0, 1, -1, -1, -1]], dtype=torch.int32, device=cuda)
    got = ops.Verification(path.long(), path, torch.tensor([2, 1], device=cuda))
    gen = torch.Generator().manual_seed(16)
    rows = torch.randn(10, 1, 64, generator=gen).half().to(cuda)

    def step(cache):
        plan = cache.plan(counts, 10, tree)
        cache.append(rows, rows, plan)
        out = cache.attend(rows, plan, 5)
        cache.keep(plan, got)
        return out

    eager, captured = (PagedCache(2, 12, 8, 1, 64, 64, dtype=torch.half) for _ in range(2))
    for cache in (eager, captured):
        cache.k.zero_()
        cache.v.zero_()
        step(cache)                           # the warm-up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    for _ in range(3):
        want = step(eager)
        graph.replay()
        assert torch.equal(out, want)
    for name in ("context", "reserved", "head", "table", "k", "v"):
        assert torch.equal(getattr(captured, name), getattr(eager, name)), name
    assert captured.context.tolist() == [12, 8]
