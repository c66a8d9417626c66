"""A Llama-3.1-8B-shaped decoder with random-init bf16 weights, for timing a whole decode step
with the sparse attention stage against dense decode attention.

Shapes follow Llama-3.1-8B (32 layers, hidden 4096, 32 query / 8 KV heads of 128, SwiGLU FFN
14336, vocabulary 128256, RMSNorm eps 1e-5, RoPE theta 500000 with the Llama-3 frequency
scaling).  The attention of each layer is the reference's decode hook contract
(methods_eager.py:198-224, graph_runner.py:469-482): the new K/V row is written at position
n - 1 of the cache C.K[l], C.V[l] before the attention runs, and n lives on the device
(C.n_dev), so a whole step -- embedding, 32 layers, final norm, LM head and the greedy next
token -- is captured once in a hipGraph and replayed with n advancing on the device.

With `method` an OursHIP the attention is its decode (the gfx950 sparse stage); with
method = None it is the dense split-K decode kernel over [0, n) on the same cache.  With `cache` a
KV4Cache or a KV8Cache keys and values are held in 4 or 8 bits in its pages instead: the step extends every
sequence by its token, and positions and lengths are the cache's, one for each sequence.  With `blocks` a step
reads of a KV8Cache only so many blocks for every sequence and KV head, those whose keys can score highest.
`qk_norm` gives every layer norms of the query and key heads.

`prefill` runs a prompt through the model one batch row at a time, as the reference's runner
does (graph_runner.py:615-622): every layer's attention goes through the hook's prefill branch
(method.attn_hook: K, V into the cache, dense causal attention, the method's index build with the
prompt's last `qlen` query rows as the question chunk).  `probe(layers)` makes each decode step
copy the attention's inputs and decisions of those layers into per-layer buffers (inside a
captured graph too): the query rows, sel, quota, exp_idx and the attention output.
"""
from __future__ import annotations

import torch

import types

from openattention_amd import ops
from openattention_amd.kv8 import KV8Cache
from openattention_amd.method import C as CTX, Method, attn_hook, prefill_attention
from openattention_amd.synth import llama31_inv_freq

HID, NLAYER, HQ, HKV, D, FFN, VOCAB = 4096, 32, 32, 8, 128, 14336, 128256
EPS = 1e-5


def rmsnorm(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + EPS)).to(x.dtype) * w


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x (N, H, D) at one position per row n; cos, sin (N, 1, D) (or (1, 1, D) for one shared
    position)."""
    h = D // 2
    xf = x.float()
    rot = torch.cat([-xf[..., h:], xf[..., :h]], -1)
    return (xf * cos + rot * sin).to(x.dtype)


class LlamaShaped:
    def __init__(self, B: int, Lmax: int, dev, layers: int = NLAYER, seed: int = 0, method=None, cache=None,
                 qk_norm: bool = False, blocks: int | None = None):
        """method: an OursHIP over these layers (sparse attention) or None (dense attention).
        The KV cache is C.K / C.V (set by the caller), (B, 8, Lmax, 128) bf16 per layer, or `cache`, a
        KV4Cache or KV8Cache of B requests and these layers (method None): steps go on to the end of its pages, also
        past Lmax.  blocks: a step's attention reads that many blocks (at least 3) of a KV8Cache (KV8Cache.select);
        prompts are attended to densely."""
        if blocks is not None and (not isinstance(cache, KV8Cache) or blocks < 3):
            raise ValueError("blocks: at least 3, of a KV8Cache")
        if cache is not None and (method is not None or cache.B != B or cache.layers != layers):
            raise ValueError("cache: for B requests and these layers, without a method")
        self.B, self.Lmax, self.dev, self.L = B, Lmax, dev, layers
        self.method, self.cache, self.qk_norm, self.blocks = method, cache, qk_norm, blocks
        g = torch.Generator(device=dev).manual_seed(seed)

        def w(*shape):
            return torch.randn(*shape, generator=g, device=dev, dtype=torch.bfloat16) * 0.02

        bf = dict(device=dev, dtype=torch.bfloat16)
        self.embed = w(VOCAB, HID)
        self.wqkv = [w(HID, (HQ + 2 * HKV) * D) for _ in range(layers)]
        self.wo = [w(HQ * D, HID) for _ in range(layers)]
        self.w13 = [w(HID, 2 * FFN) for _ in range(layers)]
        self.w2 = [w(FFN, HID) for _ in range(layers)]
        self.ln1 = [torch.ones(HID, **bf) for _ in range(layers)]
        self.ln2 = [torch.ones(HID, **bf) for _ in range(layers)]
        self.lnf = torch.ones(HID, **bf)
        self.lm_head = w(HID, VOCAB)
        inv = llama31_inv_freq().to(dev)
        P = Lmax if cache is None else max(Lmax, cache.width * cache.page)      # (a paged cache's length is in whole pages)
        t = torch.arange(P, device=dev, dtype=torch.float32)
        fr = torch.outer(t, inv)
        emb = torch.cat([fr, fr], -1)
        self.cos, self.sin = emb.cos(), emb.sin()                       # (P, D) fp32
        self.half = self.cos[:, :D // 2], self.sin[:, :D // 2]           # (a head's halves turn by the same angles)
        self.qn, self.kn = ([1 + w(D) * 5 for _ in range(layers)] if qk_norm else [None] * layers for _ in range(2))
        self.tok = torch.zeros(B, device=dev, dtype=torch.long)         # token at position n - 1
        self.ws = None
        self.mods = [types.SimpleNamespace(layer_idx=l) for l in range(layers)]
        self.probes = {}

    def params(self) -> int:
        per = HID * (HQ + 2 * HKV) * D + HQ * D * HID + HID * 2 * FFN + FFN * HID + 2 * HID
        return self.L * per + 2 * VOCAB * HID + HID

    def probe(self, layers) -> dict:
        """Per-layer probe buffers that every later decode step fills (inside a captured graph
        too): q (B*HQ, D) bf16, and with a sparse method sel, quota, exp_idx and the attention
        output out (B*HQ, D) in the method's output dtype.  Returns {layer: {name: tensor}}."""
        R = self.B * HQ
        self.probes = {}
        for l in layers:
            p = {"q": torch.empty(R, D, device=self.dev, dtype=torch.bfloat16)}
            if self.method is not None:
                m = self.method
                p["quota"] = torch.empty_like(m.quota)
                p["exp_idx"] = torch.empty_like(m.exp_idx)
                p["out"] = torch.empty_like(m.out)
                p["sel"] = None          # sized at the first step (the sel width follows n)
            self.probes[l] = p
        return self.probes

    def _qkv(self, l: int, qkv: torch.Tensor, pos: torch.Tensor):
        """Layer l's query and key rows of a product, normalised where the model has head norms and turned
        to their positions, and its value rows, each (N, heads, D)."""
        N = qkv.shape[0]
        q, k = ops.qk_norm_rope(qkv[:, :HQ * D].view(N, HQ, D), qkv[:, HQ * D:(HQ + HKV) * D].view(N, HKV, D), pos,
                                *self.half, self.qn[l], self.kn[l], EPS)
        return q, k, qkv[:, (HQ + HKV) * D:].view(N, HKV, D)

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, qlen: int = 64) -> torch.Tensor:
        """Prompt prefill of every batch row (tokens (B, T) int64), one row at a time through all
        layers (graph_runner.py:615-622).  Each layer's attention is attn_hook's prefill branch:
        the row's K, V are written to C.K[l][b, :, :T], its causal attention is dense and the
        method builds the row's index (C.qlen[b] = qlen question rows).  Leaves C.phase at
        "decode" and the greedy next token of every row in self.tok; returns it.  With a paged cache the
        rows extend its requests (empty ones; all of them, or none where the cache refuses: RuntimeError), a
        row's keys and values are written to the new slots and its own attention is dense over the unrounded
        rows."""
        B, T = tokens.shape
        if B != self.B or T > self.Lmax:
            raise ValueError(f"tokens must be ({self.B}, <= {self.Lmax})")
        if self.cache is not None:
            return self._prefill_cache(tokens)
        CTX.phase = "prefill"
        CTX.qlen = [qlen] * B
        CTX.method = self.method if self.method is not None else Method(None, B, self.Lmax, self.dev)
        cos, sin = self.cos[:T].unsqueeze(1), self.sin[:T].unsqueeze(1)           # (T, 1, D)
        where = torch.arange(T, device=self.dev)
        for b in range(B):
            CTX.brow = b
            x = self.embed.index_select(0, tokens[b])                              # (T, HID)
            for l in range(self.L):
                h = rmsnorm(x, self.ln1[l])
                qkv = h @ self.wqkv[l]
                if self.qk_norm:
                    q, k, v = (t.transpose(0, 1).unsqueeze(0) for t in self._qkv(l, qkv, where))
                else:
                    q = rope(qkv[:, :HQ * D].view(T, HQ, D), cos, sin).transpose(0, 1).unsqueeze(0)
                    k = rope(qkv[:, HQ * D:(HQ + HKV) * D].view(T, HKV, D), cos, sin).transpose(0, 1).unsqueeze(0)
                    v = qkv[:, (HQ + HKV) * D:].view(T, HKV, D).transpose(0, 1).unsqueeze(0)
                del qkv
                o, _ = attn_hook(self.mods[l], q, k, v, None)                       # (1, T, HQ, D)
                x = x + o.reshape(T, HQ * D) @ self.wo[l]
                del q, k, v, o
                h = rmsnorm(x, self.ln2[l])
                gu = h @ self.w13[l]
                x = x + (torch.nn.functional.silu(gu[:, :FFN]) * gu[:, FFN:]) @ self.w2[l]
                del gu
            logits = rmsnorm(x[-1:], self.lnf) @ self.lm_head
            self.tok[b] = logits.argmax(-1)[0]
        CTX.phase = "decode"
        return self.tok

    def _prefill_cache(self, tokens: torch.Tensor) -> torch.Tensor:
        B, T = tokens.shape
        cache = self.cache
        if bool((cache.lens != 0).any()):
            raise ValueError("prefill: the cache's requests must be empty (truncate)")
        cache.check()                                                              # (an earlier call's refusal)
        slots, pos, cu = cache.extend(torch.full_like(cache.lens, T), B * T)       # all requests or none
        cache.check()
        where = pos[:T]
        eight = isinstance(cache, KV8Cache)
        for b in range(B):
            at = slots[b * T:(b + 1) * T]
            x = self.embed.index_select(0, tokens[b])                              # (T, HID)
            for l in range(self.L):
                h = rmsnorm(x, self.ln1[l])
                q, k, v = self._qkv(l, h @ self.wqkv[l], where)
                if eight:
                    cache.write(l, k, v, cu[:2], b)                                # (0 and T)
                else:
                    cache.write(l, k, v, at)
                o = prefill_attention(*(t.transpose(0, 1).unsqueeze(0) for t in (q, k, v)), D ** -0.5)
                x = x + o[0].transpose(0, 1).reshape(T, HQ * D) @ self.wo[l]
                del q, k, v, o
                h = rmsnorm(x, self.ln2[l])
                gu = h @ self.w13[l]
                x = x + (torch.nn.functional.silu(gu[:, :FFN]) * gu[:, FFN:]) @ self.w2[l]
                del gu
            logits = rmsnorm(x[-1:], self.lnf) @ self.lm_head
            self.tok[b] = logits.argmax(-1)[0]
        return self.tok

    def _step_cache(self) -> torch.Tensor:
        B, cache = self.B, self.cache
        slots, pos, cu = cache.extend()
        eight = isinstance(cache, KV8Cache)
        x = self.embed.index_select(0, self.tok)                        # (B, HID)
        for l in range(self.L):
            h = rmsnorm(x, self.ln1[l])
            q, k, v = self._qkv(l, h @ self.wqkv[l], pos)
            cache.write(l, k, v, cu if eight else slots)
            if self.blocks is None:
                o = cache.attend(l, q)
            else:
                o = cache.attend(l, q, blocks=cache.select(l, q, self.blocks))
            x = x + o.view(B, HQ * D) @ self.wo[l]
            h = rmsnorm(x, self.ln2[l])
            gu = h @ self.w13[l]
            x = x + (torch.nn.functional.silu(gu[:, :FFN]) * gu[:, FFN:]) @ self.w2[l]
        logits = rmsnorm(x, self.lnf) @ self.lm_head
        # (a refused step's positions are -1: its tokens wait for the next one)
        self.tok.copy_(torch.where(pos >= 0, logits.argmax(-1), self.tok))
        return self.tok

    @torch.no_grad()
    def step(self, n: int | None = None) -> torch.Tensor:
        """One decode step: the token in self.tok sits at position n - 1 (n = C.n_dev on the
        device; the host n only fixes the sparse stage's sink/local/top-k counts).  Writes the
        greedy next token into self.tok and returns it.  With a paged cache n is not used: each token
        sits at its request's length, which the step extends (a step that the cache refuses, out of
        pages or past max_len, leaves lengths, rows and self.tok as they were: its check())."""
        if self.cache is not None:
            return self._step_cache()
        B = self.B
        pos = (CTX.n_dev - 1).long()                                    # (1,) on the device
        cos = self.cos.index_select(0, pos).unsqueeze(0)                # (1, 1, D)
        sin = self.sin.index_select(0, pos).unsqueeze(0)
        x = self.embed.index_select(0, self.tok)                        # (B, HID)
        for l in range(self.L):
            h = rmsnorm(x, self.ln1[l])
            qkv = h @ self.wqkv[l]
            if self.qk_norm:
                q, k, v = self._qkv(l, qkv, pos.expand(B).contiguous())
            else:
                q = rope(qkv[:, :HQ * D].view(B, HQ, D), cos, sin)
                k = rope(qkv[:, HQ * D:(HQ + HKV) * D].view(B, HKV, D), cos, sin)
                v = qkv[:, (HQ + HKV) * D:].view(B, HKV, D)
            CTX.K[l].index_copy_(2, pos, k.unsqueeze(2))
            CTX.V[l].index_copy_(2, pos, v.unsqueeze(2))
            p = self.probes.get(l)
            if p is not None:
                p["q"].copy_(q.reshape(B * HQ, D))
            if self.method is not None:
                o = self.method.decode(l, q.reshape(B, HQ, 1, D), n)
                if p is not None:
                    m = self.method
                    if p["sel"] is None or p["sel"].shape != m.last_sel.shape:
                        p["sel"] = torch.empty_like(m.last_sel)
                    p["sel"].copy_(m.last_sel)
                    p["quota"].copy_(m.quota)
                    p["exp_idx"].copy_(m.exp_idx)
                    p["out"].copy_(o.reshape(B * HQ, D))
                o = o.reshape(B, HQ * D).to(x.dtype)
            else:
                R = B * HQ
                need = R * ops.DENSE_SPLITS * (D + 2)
                if self.ws is None or self.ws.numel() < need:
                    self.ws = torch.empty(need, device=self.dev, dtype=torch.float32)
                o = ops.dense_decode(q.reshape(R, D).contiguous(), CTX.K[l].view(-1, self.Lmax, D),
                                     CTX.V[l].view(-1, self.Lmax, D), CTX.n_dev, ws=self.ws).reshape(B, HQ * D)
            x = x + o @ self.wo[l]
            h = rmsnorm(x, self.ln2[l])
            gu = h @ self.w13[l]
            x = x + (torch.nn.functional.silu(gu[:, :FFN]) * gu[:, FFN:]) @ self.w2[l]
        logits = rmsnorm(x, self.lnf) @ self.lm_head
        self.tok.copy_(logits.argmax(-1))
        return self.tok
