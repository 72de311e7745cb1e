"""A paged cache and the serving step around drafted tokens.

The attention layers' part of serving that the quantised hot path leaves out:
prompts go into a paged cache with their attention, then each step takes in a
tree of drafted tokens per request (one token: plain decoding), attends over
the cache, and keeps what the target model accepts.

  cache = PagedCache(requests, pages, page_size, heads, dk, dv)
  plan = cache.plan(prompt_lens, total)                    # pages and slots
  cache.append(k, v, plan)
  out = ops.prompt_attention(q, k, v, plan.cu_tokens, longest)
  cache.advance(prompt_lens)
  ...
  plan = cache.plan(tree_lens, total, parents)             # every step
  cache.append(k, v, plan)
  out = cache.attend(q, plan, most)
  ... logits of the tree's tokens ...
  got = ops.verify_drafts(logits, tokens, plan.cu_tokens, most, u, noise, temps, parents=parents)
  cache.keep(plan, got)

Requests may share a prompt: ``cache.fork(sources, targets)`` lets requests go on from
another's context with its full pages, ``cache.release(keep_lens)`` gives pages back that no
request holds any more, and ``cache.compact()`` moves those in use to the lowest places.

Nothing here synchronizes the host; lengths, tables and the free list stay on
the device and are updated in place, so a step captured in a CUDA graph moves on
with every replay.
"""

from __future__ import annotations

import torch

from . import ops


class PagedCache:
    """Keys and values of one attention layer for a batch of requests, in pages.

    A page holds one head's rows together ([pages, heads, page_size, width] in
    memory, [pages, page_size, heads, width] to the operators).
    """

    def __init__(self, requests: int, pages: int, page_size: int, heads: int, dk: int, dv: int,
                 *, dtype: torch.dtype = torch.bfloat16, max_pages: int | None = None,
                 device: str | torch.device = "cuda") -> None:
        self.page_size = page_size
        self.k = torch.empty((pages, heads, page_size, dk), dtype=dtype,
                             device=device).transpose(1, 2)
        self.v = torch.empty((pages, heads, page_size, dv), dtype=dtype,
                             device=device).transpose(1, 2)
        ints = dict(dtype=torch.int32, device=device)
        self.table = torch.full((requests, max_pages or pages), -1, **ints)
        self.context = torch.zeros(requests, **ints)
        self.reserved = torch.zeros(requests, **ints)     # tokens the pages reach
        self.free = torch.arange(pages, **ints)
        self.head = torch.zeros(1, **ints)

    def plan(self, new_lens: torch.Tensor, num_tokens: int,
             parents: torch.Tensor | None = None) -> ops.PagedPlan:
        """Pages and slots for ``new_lens`` more tokens of each request.

        Where the pool or the table runs out, ``plan.missing`` counts the pages and the
        tokens without one have slot -1: they are not stored and do not become context.
        A later plan asks for the pages again (more may be put at the end of ``free``).
        """
        plan = ops.paged_plan(self.context, new_lens, self.table, self.free, self.head,
                              self.page_size, num_tokens, parents=parents,
                              reserved_lens=self.reserved)
        self.head.copy_(plan.free_head)
        ops.paged_reserve(self.context, new_lens, self.table, self.reserved, self.page_size)
        return plan

    def append(self, k: torch.Tensor, v: torch.Tensor, plan: ops.PagedPlan) -> None:
        ops.paged_append(k, v, self.k, self.v, plan.slots)

    def attend(self, q: torch.Tensor, plan: ops.PagedPlan, max_tokens: int,
               scale: float | None = None) -> torch.Tensor:
        """Attention of the plan's tokens over the cache they were appended to."""
        return ops.tree_attention(q, self.k, self.v, self.table, self.context, plan.cu_tokens,
                                  max_tokens, tree_mask=plan.tree_mask, scale=scale)

    def advance(self, lens: torch.Tensor) -> None:
        """The last ``lens`` appended tokens of each request become context.

        Tokens that the plan found no page for do not.
        """
        torch.minimum(self.context + lens, self.reserved, out=self.context)

    def keep(self, plan: ops.PagedPlan, got: ops.Verification) -> None:
        """The root and the accepted tokens become context, in a row behind it.

        From the first of them on that the plan found no page for, they do not.
        """
        first = plan.cu_tokens[:-1, None].long()
        places = torch.arange(got.path.shape[1], device=self.k.device)[None, :]
        last = plan.slots.shape[0] - 1
        source = plan.slots[(first + got.path.clamp_min(0)).clamp_max(last)]
        # Paths ascend and the tokens with slots come first.
        kept = torch.minimum(got.path, source) >= 0
        target = plan.slots[(first + places).clamp_max(last)].masked_fill(~kept, -1)
        # The rows are read before any is written: targets of one token are
        # sources of another.
        source = source.clamp_min(0).flatten()
        page, row = source // self.page_size, source % self.page_size
        ops.paged_append(self.k[page, row], self.v[page, row], self.k, self.v, target.flatten())
        self.context += kept.sum(dim=1, dtype=torch.int32)

    def fork(self, sources: torch.Tensor, targets: torch.Tensor) -> ops.Fork:
        """Requests ``targets`` go on from the contexts of ``sources`` (int32 [pairs]).

        They share the full pages; a page that the context ends inside is copied.  Targets hold
        no pages (``release`` them first); a target for which the pool has no page stays empty
        (``missing``).  A request that shares pages is not to be cut back into them.
        """
        got = ops.paged_fork(self.context, self.table, sources, targets, self.free, self.head,
                             self.page_size, reserved_lens=self.reserved)
        self.head.copy_(got.free_head)
        ops.paged_copy(self.k, self.v, got.copy_from, got.copy_to, got.copy_rows)
        return got

    def release(self, keep_lens: torch.Tensor) -> None:
        """Each request keeps its first ``keep_lens`` tokens (int32 [requests]; 0: it is done,
        its context: pages that refused drafts left it go back).  Pages that no request holds
        any more are free again."""
        head = ops.paged_free(self.table, self.reserved, keep_lens, self.free, self.head,
                              self.page_size, self.k.shape[0])
        self.head.copy_(head)
        keep = keep_lens.clamp_min(0)
        torch.minimum(self.reserved, keep, out=self.reserved)
        torch.minimum(self.context, keep, out=self.context)

    def compact(self) -> ops.Compaction:
        """Moves the pages in use to the lowest places of the pool."""
        got = ops.paged_compact(self.table, self.reserved, self.free, self.head, self.page_size,
                                self.k.shape[0])
        ops.paged_copy(self.k, self.v, got.copy_from, got.copy_to)
        self.table.copy_(got.block_table)
        self.free.copy_(got.free_pages)
        self.head.copy_(got.free_head)
        return got


def children_first_tree(width: int, depth: int) -> list[int]:
    """Parents of a drafted tree: a root, ``width`` children, each the head of a
    chain of ``depth`` tokens."""
    parents = [-1]
    for _ in range(width):
        at = 0
        for _ in range(depth):
            parents.append(at)
            at = len(parents) - 1
    return parents
