"""A paged KV cache held in 8 bits, and a decoder's calls on it: attention over all that a request holds, or over
the blocks of it whose keys can score highest for each query token.

The pool of pages, the page table and the lengths of the requests live on the device, as KV4Cache's do, so that a
decode step is captured once in a hipGraph and crosses into new pages as it is replayed:

    cache = KV8Cache(B, max_len=40000, dev="cuda", layers=32)
    slots, pos, cu = cache.extend(new, total)          # the step's tokens: (B,) counts, their sum
    for l in range(32):
        q, k = ops.qk_norm_rope(q, k, pos, cos, sin)
        cache.write(l, k, v, cu)
        blocks = cache.select(l, q, 64, cu)             # 64 blocks of a page each for every token and KV head
        o = cache.attend(l, q, cu, max_q, blocks=blocks)   # (T, HQ, D); without blocks: over all keys
    cache.truncate(keep)                                # drafts not taken, requests that ended (0)

A page is a block: its keys and its values of a head share a scale each, which tokens that are added may raise.
What a request's rows hold is in include/openattention_kv8.h: a byte a value, and for a block of a head two scales
and two bounds of every channel of its keys (of pages of 64 tokens 1.6 in 100 more).
"""
from __future__ import annotations

import torch

from openattention_amd import ops
from openattention_amd.paged import PagedCache


class KV8Cache(PagedCache):
    def __init__(self, B: int, max_len: int, dev, layers: int = 1, kv_heads: int = 8, head_dim: int = 128,
                 page: int = 64, pages: int | None = None):
        """Up to B requests of up to max_len tokens (rounded up to whole pages of 32, 64 or 128) out of a pool of
        `pages` pages (B * max_len tokens' worth unless given: fewer where requests are mostly shorter)."""
        if page not in (32, 64, 128):
            raise ValueError(f"page: 32, 64 or 128 (got {page})")
        super().__init__(B, max_len, dev, layers, kv_heads, head_dim, page, pages)
        u8 = dict(device=dev, dtype=torch.uint8)
        shape = (layers, self.pages, kv_heads)
        codes = [torch.zeros(*shape, page, head_dim, **u8) for _ in range(2)]
        scales = [torch.zeros(*shape, **u8) for _ in range(2)]
        bounds = torch.zeros(*shape, 2, head_dim, device=dev, dtype=torch.int8)
        # a layer's cache as the operators take it: kc, ks, vc, vs; and its bounds
        self.rows = [(codes[0][l], scales[0][l], codes[1][l], scales[1][l]) for l in range(layers)]
        self.bounds = [bounds[l] for l in range(layers)]

    def write(self, l: int, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, request: int | None = None) -> None:
        """The rows of the tokens that requests have just added (ops.kv8_write): cu as extend gave it, so that an
        extension which was refused writes nothing.  request: the rows are that one's alone, cu (2,) 0 and their
        number."""
        table, lens = self.table, self.lens
        if request is not None:
            table, lens = table[request:request + 1], lens[request:request + 1]
        ops.kv8_write(k, v, *self.rows[l], self.bounds[l], table, lens, cu)

    def read(self, l: int, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        return ops.kv8_read(slots, *self.rows[l], dtype=dtype)

    def select(self, l: int, q: torch.Tensor, n: int, cu_q: torch.Tensor | None = None, first: int = 1, last: int = 2,
               max_len: int | None = None) -> torch.Tensor:
        """The n blocks of layer l to read for every query token and KV head (ops.kv8_select)."""
        return ops.kv8_select(q, self.rows[l][1], self.bounds[l], self.table, self.lens, self.page, n, cu_q, first, last,
                              max_len)

    def attend(self, l: int, q: torch.Tensor, cu_q: torch.Tensor | None = None, max_q: int = 1,
               sm_scale: float | None = None, out: torch.Tensor | None = None, max_len: int | None = None,
               blocks: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the newest tokens of every request over layer l, over all keys or over the blocks
        listed for each token and KV head (ops.kv8_attn)."""
        return ops.kv8_attn(q, *self.rows[l], self.table, self.lens, sm_scale, cu_q, max_q, blocks, out, max_len)
