"""The pool of pages that the paged caches (KV4Cache, KV8Cache) have in common: page table, lengths and the stack
of free pages, all on the device."""
from __future__ import annotations

import torch

from openattention_amd import ops

REFUSED = {1: "a negative count, or a request longer than max_len", 2: "too few free pages", 4: "more tokens than `total`"}


class PagedCache:
    def __init__(self, B: int, max_len: int, dev, layers: int, kv_heads: int, head_dim: int, page: int, pages: int | None):
        """Up to B requests of up to max_len tokens (rounded up to whole pages) out of a pool of `pages`
        pages (B * max_len tokens' worth unless given: fewer where requests are mostly shorter)."""
        if head_dim not in (64, 128) or B < 1 or max_len < 1 or layers < 1 or kv_heads < 1:
            raise ValueError("head_dim: 64 or 128; B, max_len, layers, kv_heads: at least 1")
        self.B, self.layers, self.page = B, layers, page
        self.width = -(-max_len // page)
        self.pages = B * self.width if pages is None else pages
        i32 = dict(device=dev, dtype=torch.int32)
        self.lens = torch.zeros(B, **i32)
        self.table = torch.full((B, self.width), -1, **i32)
        self.free = torch.arange(self.pages, **i32)
        self.nfree = torch.full((1,), self.pages, **i32)
        self.status = torch.zeros(1, **i32)
        self.one = torch.ones(B, **i32)

    def extend(self, add: torch.Tensor | None = None, total: int | None = None):
        """(slots, pos, cu) of the tokens that requests add (ops.kv_pages_extend); add None: one each."""
        if add is None:
            add, total = self.one, self.B
        elif total is None:
            raise ValueError("total: the sum of add")
        return ops.kv_pages_extend(add, self.lens, self.table, self.free, self.nfree, self.status, self.page, total)

    def truncate(self, keep: torch.Tensor) -> None:
        """Requests keep their first `keep` tokens (ops.kv_pages_truncate)."""
        ops.kv_pages_truncate(keep, self.lens, self.table, self.free, self.nfree, self.status, self.page)

    def check(self) -> None:
        """Raises for an extension or truncation that was refused since the last check (waits for the
        device)."""
        bad = int(self.status)
        if bad:
            self.status.zero_()
            raise RuntimeError(f"{type(self).__name__}: refused: " + "; ".join(t for b, t in REFUSED.items() if bad & b))
