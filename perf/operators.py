"""Performance cases of the 4-bit paged KV cache and of what feeds and reads it, from the public
entry points of openattention_amd.ops.

  rope   ops.qk_norm_rope: a layer's query and key rows, each head normalised and turned to its
         position in one pass.
  pages  ops.kv_pages_extend: the pages, slots and positions of the tokens that requests add,
         formed on the device; and ops.kv_pages_truncate, which gives pages back (drafts that were
         not taken, requests that end).
  cache  ops.kv4_write: key and value rows rounded to 4 bits and put at their slots; ops.kv4_read:
         the values that slots hold.
  attn   ops.kv4_attn: causal attention of the newest tokens of every sequence over its pages.

The cache holds blocks of 32 values of a row: a 4-bit code for each (sign, two bits of exponent, one
of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6; the even value of a row in the low half of the byte) and one
byte s for the block, which scales them by 2^(s - 127).  The scale is the smallest power of two 2^e
with max |x| < 7 * 2^e, -125 <= e <= 125; values are rounded to the nearest code, ties to the even
one, at most 6; a block with a value that is not finite is held as s = 255, which stands for NaN.

Shapes are the ones this framework decodes (32 query heads, 8 KV heads, head dimension 128; 32K and
128K contexts, batches of 32) and generic others.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-5
THETA = 500000.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 32 sequences: a launch's latency
        dict(name="rope step b32", kind="rope", T=32, HQ=32, HKV=8, D=128, P=32896, type="bf16", norm=True),
        # a long prompt of one sequence, an odd number of tokens
        dict(name="rope prompt 32k", kind="rope", T=32767, HQ=32, HKV=8, D=128, P=32896, type="bf16", norm=True),
        # chunks of a model with small heads in fp16, without norms
        dict(name="rope chunk d64 fp16", kind="rope", T=4099, HQ=14, HKV=2, D=64, P=131072, type="fp16", norm=False),
        # every sequence of a decode batch grows by one token
        dict(name="pages step b32", kind="pages", B=32, page=64, longest=32768, add=1, mix=1),
        # a full server takes up prompts and steps together, and gives them back
        dict(name="pages admit b1000", kind="pages", B=1000, page=64, longest=16384, add=1500, mix=2),
        # the new token of 32 sequences
        dict(name="cache step b32", kind="cache", T=32, HKV=8, D=128, page=64, type="bf16"),
        # a prompt's rows
        dict(name="cache prompt 32k", kind="cache", T=32767, HKV=8, D=128, page=64, type="bf16"),
        # one long conversation: few rows, work split along the keys
        dict(name="attn b1 128k", kind="attn", B=1, longest=131072, q=1, HQ=32, HKV=8, D=128, page=64, mix=0),
        # the serving batch of this framework's decode step
        dict(name="attn b32 32k", kind="attn", B=32, longest=32768, q=1, HQ=32, HKV=8, D=128, page=64, mix=0),
        # requests of all ages, some just begun
        dict(name="attn b61 ragged", kind="attn", B=61, longest=16001, q=1, HQ=32, HKV=8, D=128, page=32, mix=3),
        # drafts of up to 5 tokens checked at once, 7 query heads to a KV head, small heads
        dict(name="attn drafts d64", kind="attn", B=7, longest=9001, q=5, HQ=14, HKV=2, D=64, page=128, mix=4),
        # questions of up to 64 tokens asked of long documents
        dict(name="attn question 32k", kind="attn", B=2, longest=32768, q=64, HQ=32, HKV=8, D=128, page=64, mix=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope", "pages", "cache", "attn", "attn"))
    HQ, HKV, D = rng.choice(((32, 8, 128), (32, 8, 128), (14, 2, 64), (8, 8, 128), (40, 8, 128), (16, 2, 64)))
    page = rng.choice((32, 64, 128))
    if kind == "rope":
        return dict(kind=kind, T=_log(rng, 1, 32767), HQ=HQ, HKV=HKV, D=D, P=_log(rng, 32768, 131072),
                    type=rng.choice(("bf16", "bf16", "fp16", "fp32")) if D == 64 else "bf16", norm=rng.random() < 0.7)
    if kind == "pages":
        return dict(kind=kind, B=_log(rng, 1, 1000), page=page, longest=_log(rng, 64, 16384),
                    add=_log(rng, 1, 1500), mix=rng.randrange(1, 1 << 20))
    if kind == "cache":
        return dict(kind=kind, T=_log(rng, 1, 32767), HKV=HKV, D=D, page=page,
                    type=rng.choice(("bf16", "bf16", "fp16", "fp32")) if HKV < 8 else "bf16")
    q = rng.choice((1, 1, 1, _log(rng, 2, 64)))
    B = _log(rng, 1, 64 if q == 1 else 4)
    return dict(kind=kind, B=B, longest=_log(rng, 16, min(131072 // (1 if q == 1 else 4), (1 << 20) // B)), q=q, HQ=HQ,
                HKV=HKV, D=D, page=page, mix=rng.randrange(0, 1 << 20) if rng.random() < 0.7 else 0)


def _lens(case):
    """Tokens that each sequence holds, by the case alone: all the longest (mix 0), or spread over
    their logarithm, the longest first and, in larger batches, an empty one and one of one token."""
    B, n = case["B"], case["longest"]
    if not case["mix"]:
        return [n] * B
    r = random.Random(case["mix"])
    ls = [n] + [_log(r, 1, n) for _ in range(B - 1)]
    if B >= 8:
        ls[3], ls[5] = 0, 1
    return ls


def _adds(case):
    """Tokens that each request of a pages case adds: one for each where add is 1, otherwise one for
    half of them and up to `add` for the others."""
    r = random.Random(case["mix"] + 7)
    return [1 if case["add"] == 1 or r.random() < 0.5 else r.randint(1, case["add"]) for _ in range(case["B"])]


def _rows(case):
    """Query tokens of each sequence of an attn case: as many as it holds at most."""
    r = random.Random(case["mix"] + 5)
    ls = _lens(case)
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


def prepare(case, seed):
    g = _gen(seed)
    return dict({"rope": _prepare_rope, "pages": _prepare_pages, "cache": _prepare_cache,
                 "attn": _prepare_attn}[case["kind"]](case, g), kind=case["kind"])


def _prepare_rope(case, g):
    T, HQ, HKV, D, P, dt = case["T"], case["HQ"], case["HKV"], case["D"], case["P"], TYPES[case["type"]]
    # rows of the layer's product, queries, keys and values side by side
    qkv = _normal(g, T, (HQ + 2 * HKV) * D).to(dt)
    inv = THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(P, device=DEV, dtype=torch.float64)[:, None] * inv
    if T > 64:      # a prompt's or chunk's successive positions
        pos = int(torch.randint(0, P - T + 1, (), generator=g, device=DEV)) + torch.arange(T, device=DEV)
    else:
        pos = torch.randint(0, P, (T,), generator=g, device=DEV)
    st = dict(q=qkv[:, :HQ * D].view(T, HQ, D), k=qkv[:, HQ * D:(HQ + HKV) * D].view(T, HKV, D),
              pos=pos.int(), cos=ang.cos().float(), sin=ang.sin().float(), wq=None, wk=None)
    if case["norm"]:
        st["wq"], st["wk"] = ((1 + 0.2 * _normal(g, D)).to(dt) for _ in range(2))
    return st


def _pages_of(lens, page, g, extra=0, width=0):
    """A page table over a shuffled pool, and the free pages."""
    held = torch.tensor([_up(n, page) for n in lens], device=DEV)
    NP = int(held.sum()) + extra
    MP = max(int(held.max()), width, 1)
    perm = torch.randperm(NP, generator=g, device=DEV).int()
    col = torch.arange(MP, device=DEV)
    has = col[None] < held[:, None]
    k = (held.cumsum(0) - held)[:, None] + col
    table = torch.where(has, perm[k.clamp(max=NP - 1)], torch.full_like(k, -1, dtype=torch.int32))
    free = torch.cat([perm[int(held.sum()):], perm[:int(held.sum())]])
    return table.contiguous(), free.contiguous(), NP


def _prepare_pages(case, g):
    lens, adds, page = _lens(case), _adds(case), case["page"]
    width = _up(case["longest"] + case["add"], page)
    extra = sum(_up(n + a, page) - _up(n, page) for n, a in zip(lens, adds)) + 5
    table, free, NP = _pages_of(lens, page, g, extra, width)
    i32 = dict(device=DEV, dtype=torch.int32)
    return dict(new=torch.tensor(adds, **i32), lens=torch.tensor(lens, **i32), keep=torch.tensor(lens, **i32), table=table,
                free=free, nfree=torch.tensor([extra], **i32), status=torch.zeros(1, **i32), page=page, total=sum(adds))


def _prepare_cache(case, g):
    T, HKV, D, page = case["T"], case["HKV"], case["D"], case["page"]
    dt = TYPES[case["type"]]
    spread = 0.5 + 3 * torch.rand(HKV, D, generator=g, device=DEV) ** 4          # keys have strong channels
    NP = _up(T, page) + 3
    u8 = dict(device=DEV, dtype=torch.uint8)
    st = dict(k=(_normal(g, T, HKV, D) * spread).to(dt), v=_normal(g, T, HKV, D).to(dt))
    for n in ("k", "v"):
        st[n + "c"], st[n + "s"] = torch.zeros(NP, HKV, page, D // 2, **u8), torch.zeros(NP, HKV, page, D // 32, **u8)
    if T > 64:      # a prompt's tokens fill pages
        pages = torch.randperm(NP, generator=g, device=DEV)[:_up(T, page)]
        slots = (pages[:, None] * page + torch.arange(page, device=DEV)).flatten()[:T]
    else:           # a step's tokens lie anywhere
        slots = torch.randperm(NP * page, generator=g, device=DEV)[:T]
    return dict(st, slots=slots.int())


def _prepare_attn(case, g):
    HQ, HKV, D, page = case["HQ"], case["HKV"], case["D"], case["page"]
    lens, rows = _lens(case), _rows(case)
    table, _, NP = _pages_of(lens, page, g)
    u8 = dict(device=DEV, dtype=torch.uint8)
    st = {}
    spread = 0.5 + 3 * torch.rand(HKV, 1, D, generator=g, device=DEV) ** 4
    step = max(1, (1 << 26) // (HKV * page * D))
    for n in ("k", "v"):
        st[n + "c"], st[n + "s"] = torch.empty(NP, HKV, page, D // 2, **u8), torch.empty(NP, HKV, page, D // 32, **u8)
        for p in range(0, NP, step):
            x = _normal(g, min(step, NP - p), HKV, page, D)
            st[n + "c"][p:p + step], st[n + "s"][p:p + step] = _to4(x * spread if n == "k" else x)
    T = sum(rows)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], device=DEV, dtype=torch.int32)
    return dict(st, q=_normal(g, T, HQ, D).to(torch.bfloat16), table=table, scale=D ** -0.5,
                lens=torch.tensor(lens, device=DEV, dtype=torch.int32), cu=None if case["q"] == 1 else cu, max_q=max(rows))


# ------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _run_own(st)
    return {"rope": _plain_rope, "pages": _plain_pages, "cache": _plain_cache, "attn": _plain_attn}[st["kind"]](st)


def _run_own(st):
    from openattention_amd import ops
    kind = st["kind"]
    if kind == "rope":
        return ops.qk_norm_rope(st["q"], st["k"], st["pos"], st["cos"], st["sin"], st["wq"], st["wk"], EPS)
    if kind == "pages":
        slots, pos, cu = ops.kv_pages_extend(st["new"], st["lens"], st["table"], st["free"], st["nfree"], st["status"],
                                             st["page"], st["total"])
        ops.kv_pages_truncate(st["keep"], st["lens"], st["table"], st["free"], st["nfree"], st["status"], st["page"])
        return slots, pos, cu, st["lens"], st["table"], st["free"], st["nfree"], st["status"]
    cache = (st["kc"], st["ks"], st["vc"], st["vs"])
    if kind == "cache":
        ops.kv4_write(st["k"], st["v"], st["slots"], *cache)
        return ops.kv4_read(st["slots"], *cache)
    return ops.kv4_attn(st["q"], *cache, st["table"], st["lens"], st["scale"], cu_q=st["cu"], max_q=st["max_q"])


# ------------------------------------------------------------------ plain forms
def _plain_rope(st):
    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)

    pos = st["pos"].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    return one(st["q"], st["wq"]), one(st["k"], st["wk"])


def _plain_pages(st):
    new, lens, table, free, nfree = (st[n] for n in ("new", "lens", "table", "free", "nfree"))
    page, total = st["page"], st["total"]
    B, MP = table.shape
    NP = free.numel()
    col = torch.arange(MP, device=DEV)[None]
    # the tokens that requests add
    held, after = (lens + page - 1) // page, (lens + new + page - 1) // page
    need = after - held
    bad = ((new < 0).any() | (lens + new > MP * page).any()).int() + 2 * (need.sum() > nfree[0]).int() + 4 * (new.sum() > total).int()
    st["status"] |= bad
    take = bad == 0
    need, new = need * take, new * take
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0, dtype=torch.int32)])
    base = need.cumsum(0) - need
    t = torch.arange(total, device=DEV, dtype=torch.int32)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    pos = lens[r] + t - cu[r]
    at = pos // page
    fresh = free[(nfree - 1 - (base[r] + at - held[r])).clamp(0, NP - 1)]
    ids = torch.where(at >= held[r], fresh, table[r, at.clamp(max=MP - 1)])
    inside = t < cu[-1]
    slots = torch.where(inside, ids * page + pos % page, -1).int()
    pos = torch.where(inside, pos, -1).int()
    k = nfree - 1 - (base[:, None] + col - held[:, None])
    table.copy_(torch.where((col >= held[:, None]) & (col < (held + need)[:, None]), free[k.clamp(0, NP - 1)], table))
    lens += new
    nfree -= need.sum()
    # what they give back
    keep = torch.where(st["keep"] < 0, lens, torch.minimum(st["keep"], lens))
    held, left = (lens + page - 1) // page, (keep + page - 1) // page
    back = held - left
    gone = (col >= left[:, None]) & (col < held[:, None])
    k = nfree + back.sum() - 1 - ((back.cumsum(0) - back)[:, None] + col - left[:, None])
    more = torch.cat([free, free[:1]])
    more.scatter_(0, torch.where(gone, k, NP).flatten(), table.flatten())
    free.copy_(more[:NP])
    table.copy_(torch.where(gone, -1, table))
    lens.copy_(keep)
    nfree += back.sum()
    return slots, pos, cu, lens, table, free, nfree, st["status"]


def _to4(x):
    """(codes, scales) of rows of float values."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    m, e = torch.frexp(top)                             # top = m * 2^e, 0.5 <= m < 1
    e = (e - 3 + (m >= 0.875).int()).clamp(-125, 125)
    e = torch.where(top == 0, -125, e)
    y = b.abs() * ((127 - e) << 23).view(torch.float32)[..., None]
    c = ((y > 0.25).byte() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5))
    c = c + 8 * torch.signbit(b).byte()
    fine = torch.isfinite(b).all(-1)
    c = torch.where(fine[..., None], c, 0).flatten(-2)
    return c[..., 0::2] + 16 * c[..., 1::2], torch.where(fine, e + 127, 255).byte()


def _from4(c, s):
    """Values, in 32 bits, of rows of codes and scales."""
    lut = torch.tensor(CODES + tuple(-x for x in CODES), device=c.device)
    x = lut[torch.stack([c & 15, c >> 4], -1).flatten(-2).int()].unflatten(-1, (-1, 32))
    f = torch.where(s == 255, math.nan, (s.int() << 23).view(torch.float32))
    return (x * f[..., None]).flatten(-2)


def _plain_cache(st):
    page = st["kc"].shape[2]
    slots = st["slots"].long()
    p, o = slots // page, slots % page
    out = []
    for n in ("k", "v"):
        c, s = _to4(st[n])
        st[n + "c"][p, :, o], st[n + "s"][p, :, o] = c, s
        out.append(_from4(st[n + "c"][p, :, o], st[n + "s"][p, :, o]).to(torch.bfloat16))
    return tuple(out)


def _plain_attn(st):
    q, lens, table, cu = st["q"], st["lens"].long(), st["table"], st["cu"]
    T, HQ, D = q.shape
    B = lens.numel()
    HKV, page = st["kc"].shape[1:3]
    M, G = st["max_q"], HQ // HKV
    if cu is None:
        cu = torch.arange(B + 1, device=DEV)
    cu = cu.long()
    j = torch.arange(M, device=DEV)
    rows = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + j).clamp(max=T - 1)                                           # (B, M)
    qf = q[at].float().view(B, M, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(B, HKV, M * G, D)
    pages = table.clamp(min=0).long()

    def rows_of(c, s):
        return _from4(c[pages].transpose(1, 2).flatten(2, 3), s[pages].transpose(1, 2).flatten(2, 3))   # (B, HKV, MP * page, D)

    s = torch.matmul(qf, rows_of(st["kc"], st["ks"]).transpose(2, 3)) * st["scale"]
    last = (lens - rows)[:, None] + j                                                   # a row's own position
    t = torch.arange(s.shape[-1], device=DEV)
    seen = (t[None, None] <= last[..., None]).repeat_interleave(G, 1)[:, None]          # (B, 1, M * G, keys)
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(seen.any(-1, keepdim=True), m, 0)), 0)
    v = torch.where((t[None] < lens[:, None])[:, None, :, None], rows_of(st["vc"], st["vs"]), 0)
    o = torch.matmul(p, v) / torch.where(seen.any(-1, keepdim=True), p.sum(-1, keepdim=True), 1)
    o = o.view(B, HKV, M, G, D).permute(0, 2, 1, 3, 4).reshape(B, M, HQ, D).to(q.dtype)
    r = torch.searchsorted(cu[1:], torch.arange(T, device=DEV), right=True)
    return o[r, torch.arange(T, device=DEV) - cu[r]]


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "rope":
        T, H, D = case["T"], case["HQ"] + case["HKV"], case["D"]
        size = TYPES[case["type"]].itemsize
        return dict(bytes=2 * T * H * D * size + 4 * T + 4 * min(T, case["P"]) * D, flops=T * H * D * (8 if case["norm"] else 4))
    if kind == "pages":
        lens, adds, page = _lens(case), _adds(case), case["page"]
        pages = sum(_up(n + a, page) - _up(n, page) for n, a in zip(lens, adds))
        # slots and positions written; lengths, counts and starts; each page off the stack, into the table and back
        return dict(bytes=8 * sum(adds) + 24 * case["B"] + 24 * pages, flops=sum(adds) + case["B"])
    if kind == "cache":
        n = case["T"] * case["HKV"] * case["D"]
        size = TYPES[case["type"]].itemsize
        # both rows read, their codes and scales written, and those read and their values written
        return dict(bytes=2 * n * size + 4 * n * 17 // 32 + 4 * n + 8 * case["T"], flops=8 * n)
    lens, rows, D, HQ = _lens(case), _rows(case), case["D"], case["HQ"]
    held = sum(lens) * case["HKV"] * (D + D // 16)
    seen = sum(max(0, n - r + i + 1) for n, r in zip(lens, rows) for i in range(r))
    return dict(bytes=held + 4 * sum(rows) * HQ * D + 4 * sum(_up(n, case["page"]) for n in lens) + 8 * case["B"],
                flops=4 * D * HQ * seen)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "pages": _exact_pages, "cache": _exact_cache, "attn": _exact_attn}[case["kind"]](st)


def _exact_rope(st):
    """Pairs (x_i, x_(i + D/2)) of a normalised head as complex numbers, times cos + i sin."""
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, None]
    out = []
    for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
        x = x.double()
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        h = x.shape[-1] // 2
        z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * turn
        out.append(torch.cat([z.real, z.imag], -1))
    return tuple(out)


def _exact_pages(st):
    """Requests one by one on the host; afterwards everything is as it was."""
    page, table, free = st["page"], st["table"].cpu().numpy(), st["free"].cpu().numpy()
    top = int(st["nfree"])
    slots, pos, cu = [], [], [0]
    for i, (n, a) in enumerate(zip(st["lens"].tolist(), st["new"].tolist())):
        ids = list(table[i, :_up(n, page)])
        while len(ids) * page < n + a:
            top -= 1
            ids.append(free[top])
        p = np.arange(n, n + a)
        slots.append(np.asarray(ids, dtype=np.int64)[p // page] * page + p % page)
        pos.append(p)
        cu.append(cu[-1] + a)
    ints = [torch.from_numpy(np.concatenate(x)).int() for x in (slots, pos)] + [torch.tensor(cu, dtype=torch.int32)]
    return tuple(ints) + (st["lens"], st["table"], st["free"], st["nfree"], st["status"])


def _exact_cache(st):
    """Each block's value nearest to what was put in, from distances to all codes."""
    out = []
    for x in (st["k"], st["v"]):
        b = x.double().unflatten(-1, (-1, 32))
        e = (torch.floor(torch.log2(b.abs().amax(-1, keepdim=True) / 7)) + 1).clamp(-125, 125)
        y = b / torch.exp2(e)
        best = torch.zeros_like(y)
        far = torch.full_like(y, math.inf)
        for c in (0, 2, 4, 6, 1, 3, 5, 7):              # a tie stays with the even code
            d = (y.abs() - CODES[c]).abs()
            best = torch.where(d < far, CODES[c], best)
            far = torch.minimum(far, d)
        out.append((best * y.sign() * torch.exp2(e)).flatten(-2))
    return tuple(out)


def _exact_attn(st):
    q, page = st["q"].double(), st["kc"].shape[2]
    HKV = st["kc"].shape[1]
    T, HQ, D = q.shape
    lens = st["lens"].tolist()
    cu = list(range(T + 1)) if st["cu"] is None else st["cu"].tolist()
    out = torch.zeros(T, HQ, D, device=q.device, dtype=torch.float64)

    def values(c, s, ids, n):
        """Rows 0 .. n - 1 of the pages `ids`, by sign, exponent and mantissa of every code."""
        c = c[ids].transpose(0, 1).flatten(1, 2)[:, :n].int()
        s = s[ids].transpose(0, 1).flatten(1, 2)[:, :n].double() - 127
        c = torch.stack([c % 16, c // 16], -1).flatten(-2)
        e, m = c // 2 % 4, c % 2
        x = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1)) * (1 - 2 * (c // 8))
        return x * torch.exp2(s).repeat_interleave(32, -1)

    for b, n in enumerate(lens):
        if not n or cu[b + 1] == cu[b]:
            continue
        ids = st["table"][b, :_up(n, page)].long()
        R = cu[b + 1] - cu[b]
        k, v = values(st["kc"], st["ks"], ids, n), values(st["vc"], st["vs"], ids, n)
        x = q[cu[b]:cu[b + 1]].view(R, HKV, -1, D).permute(1, 0, 2, 3).reshape(HKV, -1, D)      # rows by token, then head
        w = torch.bmm(x, k.transpose(1, 2).contiguous()) * st["scale"]
        last = (n - R + torch.arange(R, device=q.device)).repeat_interleave(HQ // HKV)
        w = w.masked_fill(torch.arange(n, device=q.device)[None, None] > last[None, :, None], -math.inf)
        w = torch.softmax(w, -1)
        out[cu[b]:cu[b + 1]] = torch.bmm(w, v).view(HKV, R, -1, D).permute(1, 0, 2, 3).reshape(R, HQ, D)
    return out
