"""Speculative serving on synthetic weights: prompts, drafted trees, verification.

One attention layer of the 27-layer model's shape (32 heads, keys 192 wide,
values 128) between an embedding and the INT4 lm_head, all projections on the
W4A16 operators.  The draft model is the same network without the attention: it
proposes, for each request, a tree whose first branch is its own most likely
continuation and whose second starts with its second choice.  Decoding is greedy
(temperature 0), so the output is what one token at a time would give.

  python examples/speculative_serving.py [--requests 4] [--steps 16]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from local_kimi_b200 import ops  # noqa: E402
from local_kimi_b200.speculative import PagedCache, children_first_tree  # noqa: E402


class TinyTarget:
    """Embedding, one attention layer, lm_head; random weights."""

    def __init__(self, vocab: int = 163_840, hidden: int = 2_304, heads: int = 32, dk: int = 192,
                 dv: int = 128, seed: int = 0) -> None:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda n, k: ops.quantise(  # noqa: E731
            (torch.randn((n, k), generator=gen, device="cuda") * k ** -0.5).bfloat16(), 128)
        self.vocab, self.heads, self.dk, self.dv = vocab, heads, dk, dv
        self.embedding = torch.randn((vocab, hidden), generator=gen, device="cuda").bfloat16()
        self.q, self.k = w(heads * dk, hidden), w(heads * dk, hidden)
        self.v, self.o = w(heads * dv, hidden), w(hidden, heads * dv)
        self.head = w(vocab, hidden)

    def qkv(self, tokens: torch.Tensor):
        x = self.embedding[tokens]
        n = tokens.shape[0]
        q, k, v = ops.w4a16_dense_multi([(x, *self.q), (x, *self.k), (x, *self.v)])
        return (x, q.view(n, self.heads, self.dk), k.view(n, self.heads, self.dk),
                v.view(n, self.heads, self.dv))

    def logits(self, x: torch.Tensor, attended: torch.Tensor | None) -> torch.Tensor:
        if attended is not None:
            x = x + ops.w4a16_dense(attended.flatten(1), *self.o)
        return ops.w4a16_dense(x, *self.head)

    def draft(self, tokens: torch.Tensor, width: int, depth: int) -> torch.Tensor:
        """[requests, 1 + width * depth] tokens of the tree under each root."""
        columns = [tokens]
        first = self.logits(self.embedding[tokens], None).topk(width, dim=1).indices
        for i in range(width):
            token = first[:, i]
            columns.append(token)
            for _ in range(depth - 1):
                token = self.logits(self.embedding[token], None).argmax(dim=1)
                columns.append(token)
        return torch.stack(columns, dim=1)


def serve(model: TinyTarget, prompts: list[torch.Tensor], steps: int, width: int = 2,
          depth: int = 3, page_size: int = 16) -> tuple[list[list[int]], int]:
    """Greedy tokens of each request after ``steps`` steps, and the drafted tokens accepted."""
    n = len(prompts)
    lens = [int(p.shape[0]) for p in prompts]
    parents = children_first_tree(width, depth)
    most = len(parents)
    pages = sum(-(-(length + steps * most) // page_size) + 1 for length in lens)
    cache = PagedCache(n, pages, page_size, model.heads, model.dk, model.dv)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    # Prompts: into the cache, and their attention.
    tokens = torch.cat(prompts).cuda()
    plan = cache.plan(i32(lens), tokens.shape[0])
    x, q, k, v = model.qkv(tokens)
    cache.append(k, v, plan)
    out = ops.prompt_attention(q, k, v, plan.cu_tokens, max(lens))
    cache.advance(i32(lens))
    last = plan.cu_tokens[1:].long() - 1
    root = model.logits(x[last], out[last]).argmax(dim=1)

    # Steps: a tree of drafted tokens for every request.
    counts, tree = i32([most] * n), i32(parents * n)
    greedy = torch.zeros(n, device="cuda")
    coin = torch.zeros(n * most, device="cuda")
    noise = torch.ones((n, model.vocab), device="cuda")
    emitted = [[int(t)] for t in root]
    accepted = 0
    for _ in range(steps):
        tokens = model.draft(root, width, depth).flatten()
        plan = cache.plan(counts, n * most, tree)
        x, q, k, v = model.qkv(tokens)
        cache.append(k, v, plan)
        logits = model.logits(x, cache.attend(q, plan, most))
        got = ops.verify_drafts(logits, tokens, plan.cu_tokens, most, coin, noise, greedy,
                                parents=tree)
        cache.keep(plan, got)
        root = got.tokens.gather(1, got.accepted.long()[:, None])[:, 0]
        for row, out_tokens, count in zip(emitted, got.tokens.tolist(), got.accepted.tolist()):
            row += out_tokens[:count + 1]
            accepted += count
    return emitted, accepted


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--requests", type=int, default=4)
    parser.add_argument("--steps", type=int, default=16)
    args = parser.parse_args()
    model = TinyTarget()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(model.vocab, (int(n),), generator=gen)
               for n in torch.randint(5, 400, (args.requests,), generator=gen)]
    emitted, accepted = serve(model, prompts, args.steps)
    total = sum(len(row) for row in emitted)
    print(f"{args.requests} requests, {args.steps} steps: {total} tokens, {accepted} of them "
          f"drafted ({total / args.requests / args.steps:.2f} tokens a request and step)")


if __name__ == "__main__":
    main()
