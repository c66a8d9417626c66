"""Performance cases of the 8-bit paged KV cache and of what chooses and reads its blocks, from the public
entry points of openattention_amd.ops.

  write   ops.kv8_write: key and value rows of the newest tokens of every sequence rounded to 8 bits in
          the sequence's pages; and ops.kv8_read: the values that slots hold.
  select  ops.kv8_select: for each query token and KV head the blocks whose keys can score highest.
  attn    ops.kv8_attn: causal attention of the newest tokens of every sequence over its pages.
  blocks  ops.kv8_attn(blocks=...): the same over chosen blocks alone.

A page of the cache holds one block of 32, 64 or 128 tokens of each KV head: codes in e4m3 and one byte s, which
scales the block's codes by 2^e, e = s - 127.  e is the smallest with max |x| <= 448 * 2^e, -117 <= e <= 120; it
starts afresh with the block's first token and otherwise only grows, the codes of earlier tokens then being rounded
again.  A row with a value that is not finite is held as NaN and counts for nothing else.  Beside the keys' codes lie
bounds of every channel of a block in steps of 4 * 2^e: hi, the least integer with code <= 4 hi, and nlo, that with
-code <= 4 nlo, for all of its codes (-112 where there are none); rounded up again where e grows.

A block's score for a query token and KV head is max over its query heads of sum_d max(q8_d, 0) hi_d + max(-q8_d, 0)
nlo_d, times 2^min(e, 100), where q8 = rint(q / 2^u), u the smallest with |q8| <= 127 for the heads together.  Whole
numbers times powers of two: scores are exact, ties go to the lower block.

Shapes are the ones this framework decodes (32 query heads, 8 KV heads, head dimension 128; 32K and
128K contexts, batches of 32) and generic others.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FIRST, LAST = 1, 2           # blocks that are always chosen: sinks, and the newest tokens'


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 32 sequences: a launch's latency
        dict(name="write step b32", kind="write", B=32, longest=8192, add=1, HKV=8, D=128, page=64, type="bf16", mix=1),
        # a long prompt of one sequence, an odd number of tokens
        dict(name="write prompt 32k", kind="write", B=1, longest=0, add=32767, HKV=8, D=128, page=64, type="bf16", mix=0),
        # pieces of prompts go on in the middle of blocks, small heads in fp16
        dict(name="write pieces d64 fp16", kind="write", B=61, longest=3001, add=500, HKV=2, D=64, page=32, type="fp16", mix=3),
        # the blocks of a decode step
        dict(name="select step b32 32k", kind="select", B=32, longest=32768, q=1, HQ=32, HKV=8, D=128, page=64, n=64, type="bf16", mix=0),
        # the blocks of every token of two questions asked of long documents
        dict(name="select question 32k", kind="select", B=2, longest=32768, q=64, HQ=32, HKV=8, D=128, page=64, n=64, type="bf16", mix=0),
        # one long conversation: few rows, work split along the keys
        dict(name="attn b1 128k", kind="attn", B=1, longest=131072, q=1, HQ=32, HKV=8, D=128, page=64, type="bf16", mix=0),
        # the serving batch of this framework's decode step
        dict(name="attn b32 32k", kind="attn", B=32, longest=32768, q=1, HQ=32, HKV=8, D=128, page=64, type="bf16", mix=0),
        # requests of all ages, some just begun
        dict(name="attn b61 ragged", kind="attn", B=61, longest=16001, q=1, HQ=32, HKV=8, D=128, page=32, type="bf16", mix=3),
        # drafts of up to 5 tokens checked at once, 7 query heads to a KV head, small heads, fp16 queries
        dict(name="attn drafts d64 fp16", kind="attn", B=7, longest=9001, q=5, HQ=14, HKV=2, D=64, page=128, type="fp16", mix=4),
        # questions of up to 64 tokens asked of long documents
        dict(name="attn question 32k", kind="attn", B=2, longest=32768, q=64, HQ=32, HKV=8, D=128, page=64, type="bf16", mix=0),
        # a decode step that reads an eighth of its keys
        dict(name="blocks step b32 32k", kind="blocks", B=32, longest=32768, q=1, HQ=32, HKV=8, D=128, page=64, n=64, type="bf16", mix=0),
        # a question's tokens, each with blocks of its own
        dict(name="blocks question 32k", kind="blocks", B=2, longest=32768, q=64, HQ=32, HKV=8, D=128, page=64, n=64, type="bf16", mix=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("write", "select", "attn", "attn", "blocks"))
    HQ, HKV, D = rng.choice(((32, 8, 128), (32, 8, 128), (14, 2, 64), (8, 8, 128), (40, 8, 128), (16, 2, 64), (16, 1, 128)))
    page = rng.choice((32, 64, 128))
    mix = rng.randrange(1, 1 << 20)
    if kind == "write":
        B = _log(rng, 1, 64)
        return dict(kind=kind, B=B, longest=_log(rng, 1, 8192), add=rng.choice((1, _log(rng, 2, 32767 // B))), HKV=HKV, D=D,
                    page=page, type=rng.choice(("bf16", "bf16", "fp16")) if HKV == 8 else rng.choice(("bf16", "fp16", "fp32")), mix=mix)
    q = rng.choice((1, 1, 1, _log(rng, 2, 64)))
    B = _log(rng, 1, 64 if q == 1 else 4)
    longest = _log(rng, 32 * page if kind == "select" else 16, min(131072 // (1 if q == 1 else 4), (1 << 20) // B))
    mix = mix if rng.random() < 0.7 else 0
    case = dict(kind=kind, B=B, longest=longest, q=q, HQ=HQ, HKV=HKV, D=D, page=page, type=rng.choice(("bf16", "bf16", "fp16")), mix=mix)
    if kind != "attn":                                  # (select: where there is something to choose)
        case["n"] = _log(rng, 8, longest // page // 2) if kind == "select" else _log(rng, 4, max(4, min(4096 // page, longest // page)))
    return case


def _lens(case):
    """Tokens that each sequence holds before the call (write) or with its newest ones, by the case alone: all the
    longest (mix 0), or spread over their logarithm, the longest first and, in larger batches, an empty one and one of
    one token."""
    B, n = case["B"], case["longest"]
    if not case["mix"]:
        return [n] * B
    r = random.Random(case["mix"])
    ls = [n] + [_log(r, 1, n) for _ in range(B - 1)]
    if B >= 8:
        ls[3], ls[5] = 0, 1
    return ls


def _rows(case):
    """New tokens of each sequence: of a write case up to `add`, otherwise up to `q` and as many as it holds at most."""
    r = random.Random(case["mix"] + 5)
    ls = _lens(case)
    if case["kind"] == "write":
        return [case["add"] if not case["mix"] or case["add"] == 1 else r.randint(1, case["add"]) for _ in ls]
    if case["q"] == 1:
        return [1] * len(ls)
    return [min(n, case["q"] if not case["mix"] else r.randint(1, case["q"])) for n in ls]


def _up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def _pages_of(lens, page, g, spare=2):
    """A page table over a shuffled pool, and the pool's size."""
    held = torch.tensor([_up(n, page) for n in lens], device=DEV)
    NP = int(held.sum()) + spare
    MP = max(int(held.max()), 1)
    perm = torch.randperm(NP, generator=g, device=DEV).int()
    col = torch.arange(MP, device=DEV)
    k = (held.cumsum(0) - held)[:, None] + col
    table = torch.where(col[None] < held[:, None], perm[k.clamp(max=NP - 1)], torch.full_like(k, -1, dtype=torch.int32))
    return table.contiguous(), NP


def _fill(st, g, NP, HKV, page, D, codes=True):
    """Pages of keys with strong channels, whose blocks differ from one another, and of values."""
    u8 = dict(device=DEV, dtype=torch.uint8)
    spread = 0.5 + 3 * torch.rand(HKV, 1, D, generator=g, device=DEV) ** 4
    st.update(ks=torch.empty(NP, HKV, **u8), vs=torch.empty(NP, HKV, **u8), kb=torch.empty(NP, HKV, 2, D, device=DEV, dtype=torch.int8))
    if codes:
        st.update(kc=torch.empty(NP, HKV, page, D, **u8), vc=torch.empty(NP, HKV, page, D, **u8))
    step = max(1, (1 << 26) // (HKV * page * D))
    for p in range(0, NP, step):
        n = min(step, NP - p)
        k = (_normal(g, n, HKV, page, D) * 0.8 + _normal(g, n, HKV, 1, D) * 0.6) * spread
        e = _exponent(k.abs().amax((-1, -2)))
        c = _to8(k, e)
        st["ks"][p:p + n] = (e + 127).byte()
        st["kb"][p:p + n] = _bounds(c, torch.ones_like(c[..., 0], dtype=torch.bool))
        if codes:
            st["kc"][p:p + n] = c
            v = _normal(g, n, HKV, page, D)
            e = _exponent(v.abs().amax((-1, -2)))
            st["vc"][p:p + n], st["vs"][p:p + n] = _to8(v, e), (e + 127).byte()


def prepare(case, seed):
    g = _gen(seed)
    kind, HKV, D, page = case["kind"], case["HKV"], case["D"], case["page"]
    before, rows = _lens(case), _rows(case)
    lens = [a + b for a, b in zip(before, rows)] if kind == "write" else before
    table, NP = _pages_of(lens, page, g)
    one = case["add" if kind == "write" else "q"] == 1
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    st = dict(kind=kind, table=table, lens=_i32(lens), cu=None if one else _i32(starts))
    _fill(st, g, NP, HKV, page, D, kind != "select")
    T, dt = starts[-1], TYPES[case["type"]]
    if kind == "write":
        spread = 0.5 + 3 * torch.rand(HKV, D, generator=g, device=DEV) ** 4
        # rows of the layer's product, keys and values side by side
        kv = torch.cat([_normal(g, T, HKV, D) * spread, _normal(g, T, HKV, D)], 1).to(dt)
        st.update(k=kv[:, :HKV], v=kv[:, HKV:])
        # slots of the blocks that the new tokens lie in, from their first token on
        at = [(b, p) for b, (n, r) in enumerate(zip(lens, rows)) for p in range((n - r) // page * page, n)]
        b, p = (torch.tensor(x, device=DEV) for x in zip(*at))
        st["slots"] = (table[b, p // page].long() * page + p % page).int()
        return st
    st.update(q=_normal(g, T, case["HQ"], D).to(dt), max_q=max(rows))
    if kind == "select":
        st.update(n=case["n"], page=page)
    else:
        st["scale"] = D ** -0.5
    if kind == "blocks":
        n, W = case["n"], table.shape[1]
        b, j = _places(st["cu"], T, len(lens))
        seen = ((st["lens"][b] - _i32(rows)[b] + j) // page + 1).clamp(min=0)[:, None, None]
        col = torch.arange(W, device=DEV)
        r = torch.rand(T, HKV, W, generator=g, device=DEV)
        r = torch.where((col < FIRST) | (col >= seen - LAST), 2.0, r)
        r = torch.where(col < seen, r, -1.0)
        top = r.topk(min(n, W), -1)
        idx = torch.where(top.values < 0, W, top.indices).sort(-1).values
        idx = torch.where(idx == W, -1, idx).int()
        st["blocks"] = torch.nn.functional.pad(idx, (0, n - idx.shape[-1]), value=-1).contiguous()
    return st


def _places(cu, T, B):
    """Sequence and number in it of every token."""
    t = torch.arange(T, device=DEV)
    if cu is None:
        return t, torch.zeros_like(t)
    b = torch.searchsorted(cu[1:].contiguous(), t.int(), right=True).clamp(max=B - 1)
    return b, t - cu[b].long()


# ------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _run_own(st)
    return {"write": _plain_write, "select": _plain_select, "attn": _plain_attn, "blocks": _plain_blocks}[st["kind"]](st)


def _run_own(st):
    from openattention_amd import ops
    kind = st["kind"]
    if kind == "select":
        return ops.kv8_select(st["q"], st["ks"], st["kb"], st["table"], st["lens"], st["page"], st["n"], cu_q=st["cu"],
                              first=FIRST, last=LAST)
    cache = (st["kc"], st["ks"], st["vc"], st["vs"])
    if kind == "write":
        ops.kv8_write(st["k"], st["v"], *cache, st["kb"], st["table"], st["lens"], cu=st["cu"])
        return ops.kv8_read(st["slots"], *cache) + (st["ks"], st["vs"], st["kb"])
    return ops.kv8_attn(st["q"], *cache, st["table"], st["lens"], st["scale"], cu_q=st["cu"], max_q=st["max_q"],
                        blocks=st.get("blocks"))


# ------------------------------------------------------------------ plain forms
def _exponent(top):
    """The smallest e with top <= 448 * 2^e, -117 <= e <= 120."""
    m, x = torch.frexp(top)                             # top = m * 2^x, 0.5 <= m < 1
    e = (x - 9 + (m > 0.875).int()).clamp(-117, 120)
    return torch.where(top == 0, -117, e)


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127."""
    return ((e + 127) << 23).int().view(torch.float32)


def _to8(x, e):
    """Codes of float values (..., page, D) by the exponents (...) of their blocks; NaN of values that are not finite."""
    y = x.float() * _power(-e)[..., None, None]
    return torch.where(torch.isfinite(x), y, math.nan).to(torch.float8_e4m3fn).view(torch.uint8)


def _code(c):
    return c.view(torch.float8_e4m3fn).float()


def _bounds(c, counts):
    """hi and nlo (..., 2, D) of the codes (..., page, D) of the rows that count."""
    x = _code(c)
    x = torch.where(counts[..., None] & ~torch.isnan(x).any(-1, keepdim=True), torch.stack([x, -x]), -448.0).amax(-2)
    return torch.ceil(x / 4).to(torch.int8).movedim(0, -2)


def _plain_write(st):
    table, lens, cu = st["table"], st["lens"].long(), st["cu"]
    NP, HKV, page, D = st["kc"].shape
    T, B = st["k"].shape[0], lens.numel()
    cu = torch.arange(B + 1, device=DEV) if cu is None else cu.long()
    first = lens - (cu[1:] - cu[:-1])                   # position of the first new token
    # the blocks with new tokens, sequence by sequence
    n = torch.where(lens > first, (lens + page - 1) // page - first // page, 0)
    end = n.cumsum(0)
    i = torch.arange(T // page + 2 * B, device=DEV)
    i = i[i < end[-1]]
    b = torch.searchsorted(end, i, right=True)
    blk = first[b] // page + i - (end - n)[b]
    pid = table[b, blk].long()
    pos = blk[:, None] * page + torch.arange(page, device=DEV)
    new = (pos >= first[b][:, None]) & (pos < lens[b][:, None])
    old = pos < first[b][:, None]
    tok = (cu[b][:, None] + pos - first[b][:, None]).clamp(0, T - 1)
    fresh = (blk * page >= first[b])[:, None]

    def side(x, c, s):
        x = x[tok].transpose(1, 2).float()              # (blocks, HKV, page, D)
        fine = torch.isfinite(x).all(-1) & new[:, None]
        e = _exponent(torch.where(fine[..., None], x.abs(), 0).amax((-1, -2)))
        was = st[s][pid].int() - 127
        e = torch.where(fresh, e, torch.maximum(e, was))
        drop = torch.where(fresh, 0, e - was)           # (a block's earlier codes shrink by 2^-drop)
        y = torch.where(fine[..., None], x, math.nan)
        held = st[c][pid]
        again = (_code(held) * _power(-drop.clamp(max=126))[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        codes = torch.where(new[:, None, :, None], _to8(y, e), torch.where(old[:, None, :, None], again, held))
        st[c][pid], st[s][pid] = codes, (e + 127).byte()
        return codes, drop

    codes, drop = side(st["k"], "kc", "ks")
    kb = st["kb"][pid].int()
    kb = torch.where(fresh[..., None, None], -112, -((-kb) >> drop.clamp(max=31)[..., None, None]))
    st["kb"][pid] = torch.maximum(kb, _bounds(codes, new[:, None].expand(-1, HKV, -1)).int()).to(torch.int8)
    side(st["v"], "vc", "vs")
    slots = st["slots"].long()
    p, o = slots // page, slots % page
    out = [(_code(st[c][p, :, o]) * _power(st[s][p].int() - 127)[..., None]).to(torch.bfloat16) for c, s in (("kc", "ks"), ("vc", "vs"))]
    return (*out, st["ks"], st["vs"], st["kb"])


def _by_sequence(st):
    """Queries (B, HKV, tokens * G, D) in 32 bits, by sequence; positions (B, tokens) of their tokens."""
    q, lens, cu = st["q"], st["lens"].long(), st["cu"]
    T, HQ, D = q.shape
    B, HKV, M = lens.numel(), st["ks"].shape[1], st["max_q"]
    cu = torch.arange(B + 1, device=DEV) if cu is None else cu.long()
    j = torch.arange(M, device=DEV)
    at = (cu[:-1, None] + j).clamp(max=T - 1)
    x = q[at].float().view(B, M, HKV, -1, D).permute(0, 2, 1, 3, 4).reshape(B, HKV, -1, D)
    return x, (lens - cu[1:] + cu[:-1])[:, None] + j


def _by_token(x, cu, T):
    """Rows (B, tokens, ...) of sequences as rows (T, ...) of tokens."""
    b, j = _places(cu, T, x.shape[0])
    return x[b, j]


def _plain_select(st):
    q, table, n = st["q"], st["table"].clamp(min=0).long(), st["n"]
    T, HQ, D = q.shape
    HKV, W = st["ks"].shape[1], table.shape[1]
    page = st["page"]
    x, pos = _by_sequence(st)
    B, M = pos.shape
    x = x.view(B, HKV, M, -1, D)
    m, u = torch.frexp(x.abs().amax((-1, -2), keepdim=True))
    u = (u - 7 + (m > 127 / 128).int()).clamp(min=-120)         # |q| <= 127 * 2^u
    q8 = torch.round(x * _power(-u))
    q8 = torch.cat([q8.clamp(min=0), (-q8).clamp(min=0)], -1).view(B, HKV, -1, 2 * D)
    kb = st["kb"][table].transpose(1, 2).reshape(B, HKV, W, 2 * D).float()
    s = torch.matmul(q8, kb.transpose(2, 3)).view(B, HKV, M, -1, W).amax(3)
    s = s * _power((st["ks"][table].int() - 127).clamp(max=100)).transpose(1, 2)[:, :, None]
    seen = (torch.div(pos, page, rounding_mode="floor") + 1)[:, None, :, None]
    col = torch.arange(W, device=DEV)
    s = torch.where((col < FIRST) | (col >= seen - LAST), math.inf, s)
    s = torch.where(col < seen, s, -math.inf)
    val, idx = s.sort(dim=-1, descending=True, stable=True)
    idx = torch.where(val[..., :n] == -math.inf, W, idx[..., :n]).sort(-1).values
    idx = torch.nn.functional.pad(torch.where(idx == W, -1, idx), (0, max(0, n - W)), value=-1)
    return _by_token(idx.transpose(1, 2), st["cu"], T).int().contiguous()


def _plain_attn(st):
    q, lens, table = st["q"], st["lens"].long(), st["table"]
    T, HQ, D = q.shape
    HKV, page = st["kc"].shape[1:3]
    x, pos = _by_sequence(st)
    B, M = pos.shape
    pages = table.clamp(min=0).long()

    def rows_of(c, s):
        y = _code(c[pages].transpose(1, 2)) * _power(s[pages].int() - 127).transpose(1, 2)[..., None, None]
        return y.flatten(2, 3)                          # (B, HKV, keys, D)

    s = torch.matmul(x, rows_of(st["kc"], st["ks"]).transpose(2, 3)) * st["scale"]
    t = torch.arange(s.shape[-1], device=DEV)
    seen = (t <= pos[..., None]).repeat_interleave(HQ // HKV, 1)[:, None]
    s = torch.where(seen, s, -math.inf)
    some = seen.any(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(some, s.amax(-1, keepdim=True), 0)), 0)
    v = torch.where((t < lens[:, None])[:, None, :, None], rows_of(st["vc"], st["vs"]), 0)
    o = torch.matmul(p, v) / torch.where(some, p.sum(-1, keepdim=True), 1)
    o = o.view(B, HKV, M, -1, D).permute(0, 2, 1, 3, 4).reshape(B, M, HQ, D).to(q.dtype)
    return _by_token(o, st["cu"], T)


def _plain_blocks(st):
    q, lens, table, blocks = st["q"], st["lens"].long(), st["table"], st["blocks"].long()
    T, HQ, D = q.shape
    HKV, page = st["kc"].shape[1:3]
    B, n = lens.numel(), blocks.shape[-1]
    cu = torch.arange(B + 1, device=DEV) if st["cu"] is None else st["cu"].long()
    b, j = _places(st["cu"], T, B)
    pos = (lens - cu[1:] + cu[:-1])[b] + j
    pages = torch.where(blocks >= 0, table[b[:, None, None], blocks.clamp(min=0)], 0).long()         # (T, HKV, n)
    h = torch.arange(HKV, device=DEV)[None, :, None]

    def rows_of(c, s):
        return (_code(c[pages, h]) * _power(s[pages, h].int() - 127)[..., None, None]).flatten(2, 3)   # (T, HKV, n * page, D)

    at = blocks[..., None] * page + torch.arange(page, device=DEV)
    seen = ((blocks[..., None] >= 0) & (at <= pos[:, None, None, None])).flatten(2, 3)[:, :, None]
    s = torch.matmul(q.float().view(T, HKV, -1, D), rows_of(st["kc"], st["ks"]).transpose(2, 3)) * st["scale"]
    s = torch.where(seen, s, -math.inf)
    some = seen.any(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(some, s.amax(-1, keepdim=True), 0)), 0)
    v = torch.where(seen.transpose(2, 3), rows_of(st["vc"], st["vs"]), 0)
    o = torch.matmul(p, v) / torch.where(some, p.sum(-1, keepdim=True), 1)
    return o.view(T, HQ, D).to(q.dtype)


# ------------------------------------------------------------------ work
def work(case):
    kind, HKV, D, page = case["kind"], case["HKV"], case["D"], case["page"]
    lens, rows, size = _lens(case), _rows(case), TYPES[case["type"]].itemsize
    T = sum(rows)
    if kind == "write":
        blocks = sum(_up(n + r, page) - n // page for n, r in zip(lens, rows))
        back = sum(r + n % page for n, r in zip(lens, rows))
        # rows read, codes, scales and bounds written; codes read back, values written
        return dict(bytes=2 * T * HKV * D * (size + 1) + blocks * HKV * (2 * D + 2) + 2 * back * HKV * D * 3 + 4 * back,
                    flops=6 * T * HKV * D)
    HQ = case["HQ"]
    at = [(n, range(max(0, n - r), n)) for n, r in zip(lens, rows)]
    if kind == "select":
        seen = sum(p // page + 1 for _, ps in at for p in ps)
        return dict(bytes=sum(_up(n, page) for n in lens) * HKV * (2 * D + 1) + T * HQ * D * size + 4 * T * HKV * case["n"],
                    flops=4 * D * HQ * seen)
    if kind == "attn":
        keys = sum(lens)
        seen = sum(p + 1 for _, ps in at for p in ps)
    else:
        n = case["n"]
        keys = sum(min(m, len(ps) * n * page) for m, ps in at)
        seen = sum(min(p + 1, n * page) for _, ps in at for p in ps)
    return dict(bytes=keys * HKV * 2 * D + 2 * T * HQ * D * size + (4 * T * HKV * case["n"] if kind == "blocks" else 0),
                flops=4 * D * HQ * seen)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "select": _exact_select, "attn": _exact_attn, "blocks": _exact_blocks}[case["kind"]](st)


def _values(c, s):
    """Values in 64 bits of codes (..., page, D) and scale bytes (...), by sign, exponent and mantissa."""
    c = c.int()
    e, m = c // 8 % 16, c % 8
    x = torch.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m.double() / 8) * torch.exp2(e.double() - 7))
    x = torch.where(c % 128 == 127, math.nan, x) * (1 - 2 * (c // 128))
    return x * torch.exp2(s.double() - 127)[..., None, None]


def _nearest(y):
    """The e4m3 value nearest to y (64 bits, at most 448), ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_write(st):
    """Sequence by sequence and block by block: the values of every block's tokens; the scales and bounds are whole numbers, which
    the plain form gives."""
    page, HKV = st["kc"].shape[2], st["kc"].shape[1]
    lens, table = st["lens"].tolist(), st["table"].tolist()
    cu = list(range(len(lens) + 1)) if st["cu"] is None else st["cu"].tolist()
    out = []
    for x, c, s in ((st["k"], "kc", "ks"), (st["v"], "vc", "vs")):
        got = []
        for b, n in enumerate(lens):
            first = n - (cu[b + 1] - cu[b])
            for blk in range(first // page, _up(n, page)):
                p0, p1 = max(first, blk * page), min(n, (blk + 1) * page)
                y = x[cu[b] + p0 - first:cu[b] + p1 - first].double().transpose(0, 1)          # (HKV, tokens, D)
                e = torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448)).clamp(-117, 120)
                pid, had = table[b][blk], p0 - blk * page
                if had:
                    e = torch.maximum(e, st[s][pid].double() - 127)
                    y = torch.cat([_values(st[c][pid, :, :had], st[s][pid]), y], 1)
                f = torch.exp2(e)[:, None, None]
                got.append((_nearest(y / f) * f).transpose(0, 1))
        out.append(torch.cat(got))
    return (*out, None, None, None)


def _exact_select(st):
    """Every token on its own, in whole numbers of 64 bits."""
    q, n, table, page = st["q"], st["n"], st["table"], st["page"]
    T, HQ, D = q.shape
    HKV = st["ks"].shape[1]
    lens = st["lens"].tolist()
    cu = list(range(len(lens) + 1)) if st["cu"] is None else st["cu"].tolist()
    out = torch.full((T, HKV, n), -1, dtype=torch.int32, device=DEV)
    for b, m in enumerate(lens):
        ids = table[b, :_up(m, page)].long()
        hi, nlo = st["kb"][ids].long().unbind(2)                                               # (blocks, HKV, D)
        e = (st["ks"][ids].double() - 127).clamp(max=100)
        for t in range(cu[b], cu[b + 1]):
            seen = (m - (cu[b + 1] - t)) // page + 1
            if seen <= 0:
                continue
            x = q[t].double().view(HKV, 1, -1, D)
            top = x.abs().amax((1, 2, 3), keepdim=True)
            u = torch.ceil(torch.log2(top / 127)).clamp(min=-120)
            x = torch.round(x / torch.exp2(u))
            s = torch.where(x > 0, x * hi[:seen].transpose(0, 1)[:, :, None], -x * nlo[:seen].transpose(0, 1)[:, :, None]).sum(-1)
            s = s.amax(-1) * torch.exp2(e[:seen]).t()                                          # (HKV, blocks)
            s[:, :FIRST] = math.inf
            s[:, max(0, seen - LAST):] = math.inf
            best = s.sort(dim=-1, descending=True, stable=True).indices[:, :n].sort(-1).values
            out[t, :, :best.shape[1]] = best.int()
    return out


def _exact_attn(st):
    q, page = st["q"].double(), st["kc"].shape[2]
    HKV = st["kc"].shape[1]
    T, HQ, D = q.shape
    lens = st["lens"].tolist()
    cu = list(range(T + 1)) if st["cu"] is None else st["cu"].tolist()
    out = torch.zeros(T, HQ, D, device=q.device, dtype=torch.float64)
    for b, n in enumerate(lens):
        if not n or cu[b + 1] == cu[b]:
            continue
        ids = st["table"][b, :_up(n, page)].long()
        R = cu[b + 1] - cu[b]
        k, v = (_values(st[c][ids], st[s][ids]).transpose(0, 1).flatten(1, 2)[:, :n] for c, s in (("kc", "ks"), ("vc", "vs")))
        x = q[cu[b]:cu[b + 1]].view(R, HKV, -1, D).permute(1, 0, 2, 3).reshape(HKV, -1, D)      # rows by token, then head
        w = torch.bmm(x, k.transpose(1, 2).contiguous()) * st["scale"]
        last = (n - R + torch.arange(R, device=q.device)).repeat_interleave(HQ // HKV)
        w = w.masked_fill(torch.arange(n, device=q.device)[None, None] > last[None, :, None], -math.inf)
        w = torch.softmax(w, -1)
        out[cu[b]:cu[b + 1]] = torch.bmm(w, v).view(HKV, R, -1, D).permute(1, 0, 2, 3).reshape(R, HQ, D)
    return out


def _exact_blocks(st):
    q, page = st["q"].double(), st["kc"].shape[2]
    HKV = st["kc"].shape[1]
    T, HQ, D = q.shape
    lens = st["lens"].tolist()
    cu = list(range(T + 1)) if st["cu"] is None else st["cu"].tolist()
    out = torch.zeros(T, HKV, HQ // HKV, D, device=q.device, dtype=torch.float64)
    head = torch.arange(HKV, device=q.device)[:, None]
    for b, n in enumerate(lens):
        for t in range(cu[b], cu[b + 1]):
            blk = st["blocks"][t].long()                                                       # (HKV, n)
            at = (blk[..., None] * page + torch.arange(page, device=q.device)).flatten(1)
            seen = (blk[..., None] >= 0).expand(-1, -1, page).flatten(1) & (at <= n - (cu[b + 1] - t))
            if not bool(seen.any()):
                continue
            ids = torch.where(blk >= 0, st["table"][b].long()[blk.clamp(min=0)], 0)
            k, v = (_values(st[c][ids, head], st[s][ids, head]).flatten(1, 2) for c, s in (("kc", "ks"), ("vc", "vs")))
            w = torch.bmm(q[t].view(HKV, -1, D), k.transpose(1, 2).contiguous()) * st["scale"]
            w = torch.softmax(w.masked_fill(~seen[:, None], -math.inf), -1)
            out[t] = torch.bmm(w, torch.where(seen[..., None], v, 0))
    return out.view(T, HQ, D)
