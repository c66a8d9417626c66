"""A paged KV cache held in 4 bits, and a decoder's calls on it.

The pool of pages, the page table and the lengths of the requests live on the device, so that a decode
step (extend, then write and attend in every layer) is captured once in a hipGraph and crosses into new
pages as it is replayed:

    cache = KV4Cache(B, max_len=40000, dev="cuda", layers=32)
    slots, pos, cu = cache.extend(new, total)          # the step's tokens: (B,) counts, their sum
    for l in range(32):
        q, k = ops.qk_norm_rope(q, k, pos, cos, sin)
        cache.write(l, k, v, slots)
        o = cache.attend(l, q, cu, max_q)               # (T, HQ, D); cu None where each request adds one token
    cache.truncate(keep)                                # drafts not taken, requests that ended (0)

What a request's rows hold is in include/openattention_amd.h: 17 bytes for 32 values, an eighth more than
a quarter of bf16.
"""
from __future__ import annotations

import torch

from openattention_amd import ops

REFUSED = {1: "a negative count, or a request longer than max_len", 2: "too few free pages", 4: "more tokens than `total`"}


class KV4Cache:
    def __init__(self, B: int, max_len: int, dev, layers: int = 1, kv_heads: int = 8, head_dim: int = 128,
                 page: int = 64, pages: int | None = None):
        """Up to B requests of up to max_len tokens (rounded up to whole pages) out of a pool of `pages`
        pages (B * max_len tokens' worth unless given: fewer where requests are mostly shorter)."""
        ops._page(page)
        if head_dim not in (64, 128) or B < 1 or max_len < 1 or layers < 1 or kv_heads < 1:
            raise ValueError("head_dim: 64 or 128; B, max_len, layers, kv_heads: at least 1")
        self.B, self.layers, self.page = B, layers, page
        self.width = -(-max_len // page)
        self.pages = B * self.width if pages is None else pages
        u8 = dict(device=dev, dtype=torch.uint8)
        shape = (layers, self.pages, kv_heads, page)
        codes = [torch.zeros(*shape, head_dim // 2, **u8) for _ in range(2)]
        scales = [torch.zeros(*shape, head_dim // ops.KV4_BLOCK, **u8) for _ in range(2)]
        # a layer's cache as the operators take it: kc, ks, vc, vs
        self.rows = [(codes[0][l], scales[0][l], codes[1][l], scales[1][l]) for l in range(layers)]
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

    def write(self, l: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        ops.kv4_write(k, v, slots, *self.rows[l])

    def read(self, l: int, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        return ops.kv4_read(slots, *self.rows[l], dtype=dtype)

    def attend(self, l: int, q: torch.Tensor, cu_q: torch.Tensor | None = None, max_q: int = 1,
               sm_scale: float | None = None, out: torch.Tensor | None = None, max_len: int | None = None) -> torch.Tensor:
        """Causal attention of the newest tokens of every request over layer l (ops.kv4_attn)."""
        return ops.kv4_attn(q, *self.rows[l], self.table, self.lens, sm_scale, cu_q=cu_q, max_q=max_q, out=out,
                            max_len=max_len)

    def check(self) -> None:
        """Raises for an extension or truncation that was refused since the last check (waits for the
        device)."""
        bad = int(self.status)
        if bad:
            self.status.zero_()
            raise RuntimeError("KV4Cache: refused: " + "; ".join(t for b, t in REFUSED.items() if bad & b))
