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
