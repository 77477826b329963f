"""A serving step over the paged operators, as a host runs them together.

PagedCache keeps the key / value pools of a stack's layers, the block table and
the free list on the device.  A step that brings new tokens to any of its rows
(a whole prompt, a chunk of one, a single decoded token, nothing) is

    step = cache.begin([n new tokens of each row])       # qtb_paged_plan
    for layer in range(layers):
        out = cache.attend(step, layer, q, k, v)         # qtb_paged_append, qtb_paged_attention
    cache.retire([rows that are done])                   # their pages return to the free list

without a host synchronisation: the host knows the lengths, the device the pages.

Run as a program it serves a few requests in chunks beside decoding ones and
checks every token's attention against the whole prompt's:

    python qwen3-tts_b200/qtb_paged_step.py
"""
from __future__ import annotations

import os
import sys
from typing import List, NamedTuple, Sequence

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import qtb_paged as P


class Step(NamedTuple):
    plan: P.Plan
    tokens: int      # new tokens in all
    max_new: int     # most of a row
    max_kv: int      # most keys of a row


class PagedCache:
    """Rows are request slots; `pages` pages of `page` positions serve all of them, in every layer."""

    def __init__(self, layers: int, rows: int, pages: int, page: int, max_len: int, kv_heads: int, dim: int,
                 dtype=torch.bfloat16, device="cuda"):
        shape = (layers, pages, kv_heads, page, dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.page, self.device = page, self.k.device
        self.table = torch.full((rows, -(-max_len // page)), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.head = torch.zeros(1, dtype=torch.int32, device=device)
        self.taken = 0                               # what *head holds, as the host knows it
        self.length = [0] * rows
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def _pages(self, n: int) -> int:
        return -(-n // self.page)

    def pages_left(self) -> int:
        return self.free.shape[0] - self.taken

    def begin(self, new: Sequence[int]) -> Step:
        """New tokens of each row.  What does not fit is refused here, with nothing changed: the device would cut it."""
        if len(new) != len(self.length) or min(new, default=0) < 0:
            raise ValueError(f"new tokens of each of {len(self.length)} rows wanted, got {list(new)}")
        room = self.table.shape[1] * self.page
        for r, (a, n) in enumerate(zip(self.length, new)):
            if a + n > room:
                raise RuntimeError(f"row {r}: {a} and {n} tokens, room for {room}")
        need = sum(self._pages(a + n) - self._pages(a) for a, n in zip(self.length, new))
        if need > self.pages_left():
            raise RuntimeError(f"{need} pages needed, {self.pages_left()} left")
        past, fresh = torch.tensor([self.length, list(new)], dtype=torch.int32).to(self.device, non_blocking=True)
        plan = P.plan(past, fresh, self.table, self.free, self.page, sum(new), free_head=self.head, status=self.status)
        self.head, self.taken = plan.free_head, self.taken + need
        self.length = [a + n for a, n in zip(self.length, new)]
        return Step(plan, sum(new), max(new), max((a for a, n in zip(self.length, new) if n), default=0))

    def attend(self, step: Step, layer: int, q, k, v, scale=None, window: int = 0):
        """q [tokens][heads][dim], k and v [tokens][key heads][dim] of the step's new tokens, row by row."""
        k_pool, v_pool = self.k[layer], self.v[layer]
        P.append(k, v, k_pool, v_pool, step.plan.slot, status=self.status)
        out, _ = P.paged_attention(q, k_pool, v_pool, self.table, step.plan.cu_new, step.plan.kv_len, step.max_new, step.max_kv,
                                   scale=scale, window=window, status=self.status)
        return out

    def retire(self, rows: Sequence[int]) -> None:
        if len(set(rows)) < len(rows) or not all(0 <= r < len(self.length) for r in rows):
            raise ValueError(f"different rows below {len(self.length)} wanted, got {list(rows)}")
        pages = [self.table[r, :self._pages(self.length[r])] for r in rows]
        self.free = torch.cat([self.free[self.taken:], *pages])
        self.head, self.taken = torch.zeros_like(self.head), 0
        for r in rows:
            self.length[r] = 0

    def check(self) -> None:
        P.check_status(self.status)


def serve(lengths: Sequence[int], prompts: Sequence[int], rows: int, chunk: int, layers: int = 2, heads: int = 16, kv_heads: int = 8,
          dim: int = 128, page: int = 16, seed: int = 0, dtype=torch.bfloat16) -> List[List[torch.Tensor]]:
    """Requests of lengths[i] tokens, the first prompts[i] of which come in chunks and the others one by one, through `rows`
    slots with room for about two thirds of them at once.  Every token's q, k and v are given beforehand (random, from
    the seed).  Returns for each request and layer the largest difference of its attention from the whole sequence's
    (qtb_prompt_attention), relative to the largest output."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    data = [[tuple(torch.randn(n, h, dim, generator=gen, device="cuda").to(dtype) for h in (heads, kv_heads, kv_heads))
             for _ in range(layers)] for n in lengths]
    longest = max(lengths)
    pages = max(-(-longest // page), 2 * sum(-(-n // page) for n in lengths) // 3) + rows
    cache = PagedCache(layers, rows, pages, page, longest, kv_heads, dim, dtype)
    waiting, slot, got = list(range(len(lengths))), [None] * rows, [[[] for _ in range(layers)] for _ in lengths]
    promised = 0
    while waiting or any(s is not None for s in slot):
        for r in range(rows):
            if slot[r] is None and waiting and promised + -(-lengths[waiting[0]] // page) <= pages:
                slot[r] = waiting.pop(0)
                promised += -(-lengths[slot[r]] // page)
        new = []
        for r, i in enumerate(slot):
            at = cache.length[r]
            new.append(0 if i is None else min(chunk, prompts[i] - at) if at < prompts[i] else 1)
        step = cache.begin(new)
        spans = [(i, cache.length[r] - n, cache.length[r]) for r, (i, n) in enumerate(zip(slot, new)) if n]
        for layer in range(layers):
            q, k, v = (torch.cat([data[i][layer][x][a:b] for i, a, b in spans]) for x in range(3))
            for part, (i, _, _) in zip(cache.attend(step, layer, q, k, v).split([b - a for _, a, b in spans]), spans):
                got[i][layer].append(part)
        done = [r for r, i in enumerate(slot) if i is not None and cache.length[r] == lengths[i]]
        if done:
            cache.retire(done)
        for r in done:
            promised -= -(-lengths[slot[r]] // page)
            slot[r] = None
    cache.check()
    worst = []
    for i, n in enumerate(lengths):
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        worst.append([])
        for layer in range(layers):
            whole, _ = P.prompt_attention(*data[i][layer], cu, n)
            mine = torch.cat(got[i][layer])
            worst[i].append((mine.float() - whole.float()).abs().max() / whole.float().abs().max())
    return worst


if __name__ == "__main__":
    sizes = [700, 64, 1, 333, 2048, 90, 17]
    for n, w in zip(sizes, serve(sizes, [600, 64, 1, 300, 2000, 30, 1], rows=4, chunk=256)):
        print("request of %4d tokens: largest difference from the whole prompt's attention %.2g" % (n, max(float(x) for x in w)))
