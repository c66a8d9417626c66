"""The 4-bit paged cache on the GPU: head norms with rotation, page tables, cache rows and attention
against 64-bit references (tests/kv4_ref.py), alone and as a decode loop runs them."""
import math
import random

import pytest
import torch

from openattention_amd import ops
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def tables(P, D, half=None):
    inv = 500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(P, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


# ================================================================== head norms with rotation
def check_rope(out, x, pos, cos, sin, w, eps):
    want, size = ref.rope(x, pos, cos, sin, w, eps)
    # fp32: 16 squares a lane and four joins, halved by the root (10), mean, root, quotient, two products
    # (5), a product and a sum of the rotation (2): under 20 steps of 2^-24; then the type's own rounding
    half = torch.finfo(x.dtype).eps / 2
    tol = 20 * 2.0 ** -24 * size
    tol = tol + half * (want.abs() + tol) + (2.0 ** -24 if x.dtype == torch.float16 else 0)
    bad = ~((out.double() - want).abs() <= tol)
    assert torch.equal(torch.isnan(want), torch.isnan(out))
    assert not (bad & ~torch.isnan(want)).any()


@pytest.mark.parametrize("T,HQ,HKV,D,dtype,norm,pos64", [
    (1, 32, 8, 128, torch.bfloat16, True, False), (33, 32, 8, 128, torch.bfloat16, True, True),
    (257, 14, 2, 64, torch.float16, False, False), (5, 3, 1, 256, torch.float32, True, True),
    (70, 7, 7, 128, torch.float16, True, False), (1001, 5, 1, 64, torch.bfloat16, False, True),
    (9, 1, 0, 128, torch.bfloat16, True, False), (3, 40, 8, 128, torch.float32, False, False)])
def test_rope(T, HQ, HKV, D, dtype, norm, pos64):
    print(f"[case] rope {T} {HQ} {HKV} {D} {dtype} norm={norm}", flush=True)
    g = gen(T)
    qkv = randn(g, T, (HQ + 2 * HKV) * D, dtype=dtype)
    q = qkv[:, :HQ * D].view(T, HQ, D)
    k = qkv[:, HQ * D:(HQ + HKV) * D].view(T, HKV, D)
    cos, sin = tables(5000, D)
    pos = torch.randint(0, 5000, (T,), generator=g, device=DEV)
    pos = pos if pos64 else pos.int()
    wq, wk = (randn(g, D, dtype=dtype), randn(g, D, dtype=dtype)) if norm else (None, None)
    keep = qkv.clone()
    qo, ko = ops.qk_norm_rope(q, k, pos, cos, sin, wq, wk, 1e-5)
    assert torch.equal(qkv, keep)
    check_rope(qo, q, pos, cos, sin, wq, 1e-5)
    check_rope(ko, k, pos, cos, sin, wk, 1e-5)


def test_rope_layouts_padding_and_in_place():
    """Head-major rows, wider tables, one norm only, zero rows, padding, positions past the tables, outputs
    that are the inputs; what the call does not own stays as it was."""
    g = gen(7)
    T, HQ, HKV, D = 13, 4, 2, 128
    q = randn(g, HQ, T, D, dtype=torch.bfloat16).transpose(0, 1)
    k = randn(g, HKV, T, D + 8, dtype=torch.bfloat16).transpose(0, 1)[..., :D]
    q[4] = 0
    cos, sin = tables(100, 2 * D)
    cos, sin = cos[:, :D // 2], sin[:, :D // 2]
    pos = torch.randint(0, 100, (T,), generator=g, device=DEV)
    pos[2], pos[5], pos[7], pos[9] = -1, 100, -(1 << 40), 1 << 40
    wk = randn(g, D, dtype=torch.bfloat16)
    for wq in (None, randn(g, D, dtype=torch.bfloat16)):
        qo = torch.full((T + 1, HQ, D), 7.0, device=DEV, dtype=torch.bfloat16)
        a, b = ops.qk_norm_rope(q, k, pos, cos, sin, wq, wk, 1e-5, q_out=qo[:T])
        assert a.data_ptr() == qo.data_ptr() and (qo[T] == 7).all()
        check_rope(a, q, pos, cos, sin, wq, 1e-5)
        check_rope(b, k, pos, cos, sin, wk, 1e-5)
    q2, k2 = q.clone(memory_format=torch.preserve_format), k.clone()
    ops.qk_norm_rope(q2, k2, pos, cos, sin, wq, wk, 1e-5, q_out=q2, k_out=k2)
    assert torch.equal(q2.isnan(), a.isnan()) and torch.equal(q2.nan_to_num(), a.nan_to_num())
    assert torch.equal(k2.nan_to_num(), b.nan_to_num())
    e = ops.qk_norm_rope(q[:0], k[:0], pos[:0], cos, sin, wq, wk)
    assert e[0].shape == (0, HQ, D)


# ================================================================== pages
def pool_state(seed, B, width, page, spare):
    r = random.Random(seed)
    lens = [r.choice((0, 1, page - 1, page, page + 1, r.randrange(width * page // 2))) for _ in range(B)]
    lens = [min(n, width * page) for n in lens]
    held = [-(-n // page) for n in lens]
    NP = sum(held) + spare
    ids = list(range(NP))
    r.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[at:] + [0] * at
    return lens, table, free, spare


def same(pool, lens, table, free, nfree, status):
    assert lens.tolist() == pool.lens and table.tolist() == pool.table and int(nfree) == pool.nfree
    assert free.tolist() == pool.free and int(status) == pool.status


@pytest.mark.parametrize("B,width,page,most", [(1, 4, 32, 40), (5, 9, 64, 100), (64, 12, 32, 60), (300, 5, 128, 30), (40, 6, 32, 4), (200, 6, 64, 3),
                                               (1500, 6, 32, 9), (1500, 6, 32, 1), (4500, 4, 32, 3)])
def test_pages_follow_the_pool(B, width, page, most):
    print(f"[case] pages {B} {width} {page} {most}", flush=True)
    lens, table, free, spare = pool_state(B, B, width, page, 4 * B)
    pool = ref.Pool(lens, table, free, spare, page)
    st = [i32(lens), i32(table), i32(free), i32([spare]), i32([0])]
    r = random.Random(B + 1)
    for it in range(8):
        add = [r.choice((0, 1, 1, r.randint(0, most))) for _ in range(B)]
        if it == 3:
            add[r.randrange(B)] = -1
        total = sum(max(a, 0) for a in add) + r.choice((0, 0, 3))
        if it == 5:
            total = max(0, sum(add) - 1)
        want = pool.extend(add, total)
        got = ops.kv_pages_extend(i32(add), *st, page, total)
        for w, x in zip(want, got):
            assert x.dtype == torch.int32 and x.tolist() == w
        same(pool, *st)
        keep = [r.choice((-1, n, max(0, n - 1), r.randint(0, n + 2), 0)) for n in pool.lens]
        pool.truncate(keep)
        ops.kv_pages_truncate(i32(keep), *st, page)
        same(pool, *st)


def test_pages_refusals_change_nothing():
    page = 32
    # (30 and 32 tokens in a page each, one page free, rows of 128 tokens: 30 + 3 and 32 + 3 take a page each,
    # 30 + 97 three more)
    for add, total, why in (([1, -1], 9, 1), ([1, 97], 99, 1), ([40, 40], 80, 2), ([3, 3], 5, 2 | 4), ([97, 60], 9, 2 | 4),
                            ([1, 0], 0, 4), ([2, 3], 4, 4), ([99, 1], 0, 1 | 4)):
        lens, table, free = i32([30, 32]), i32([[3, -1, -1, -1], [0, -1, -1, -1]]), i32([1, 2, 9, 9])
        st = [lens, table, free, i32([1]), i32([0])]
        keep = [t.clone() for t in st]
        slots, pos, cu = ops.kv_pages_extend(i32(add), *st, page, total)
        assert int(st[4]) == why
        assert (slots == -1).all() and (pos == -1).all() and (cu == 0).all() and cu.numel() == 3
        assert all(torch.equal(a, b) for a, b in zip(st[:4], keep[:4]))
        st[4] |= 8                                        # the word is added to, never cleared
        ops.kv_pages_extend(i32([1, 0]), *st, page, 4)
        assert int(st[4]) == why | 8 and st[0].tolist() == [31, 32]
    # more pages than the stack can hold go back to nothing
    st = [i32([64, 64]), i32([[0, 1], [2, 3]]), i32([5, 6, 7, 8]), i32([2]), i32([0])]
    ops.kv_pages_truncate(i32([0, 0]), *st, 32)
    assert int(st[4]) == 2 and st[0].tolist() == [64, 64] and st[1].tolist() == [[0, 1], [2, 3]] and int(st[3]) == 2
    # lengths outside of a row, ids outside of the pool: no slot is given
    st = [i32([-5, 0]), i32([[0, 1], [2, 3]]), i32([5, 6, 7, 8]), i32([2]), i32([0])]
    assert (ops.kv_pages_extend(i32([1, 1]), *st, 32, 2)[0] == -1).all() and int(st[4]) == 1
    st = [i32([0, 3]), i32([[0, 1], [1 << 27, 3]]), i32([5, -7, 7, 8]), i32([2]), i32([0])]
    assert ops.kv_pages_extend(i32([1, 1]), *st, 32, 2)[0].tolist() == [-1, -1]


def test_pages_rows_of_a_wider_table():
    wide = torch.full((3, 10), 77, device=DEV, dtype=torch.int32)
    table = wide[:, 2:6]
    table.fill_(-1)
    st = [i32([0, 0, 0]), table, i32(range(9)), i32([9]), i32([0])]
    slots, pos, cu = ops.kv_pages_extend(i32([33, 0, 5]), *st, 32, 38)
    assert table.tolist() == [[8, 7, -1, -1], [-1] * 4, [6, -1, -1, -1]] and cu.tolist() == [0, 33, 33, 38]
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()


# ================================================================== cache rows
def new_cache(NP, HKV, page, D, fill=None, g=None):
    out = []
    for w in (D // 2, D // 32, D // 2, D // 32):
        if fill is None:
            out.append(torch.randint(0, 256, (NP, HKV, page, w), generator=g, device=DEV, dtype=torch.uint8))
        else:
            out.append(torch.full((NP, HKV, page, w), fill, device=DEV, dtype=torch.uint8))
    return out


def hard_rows(T, HKV, D, dtype, g):
    """Rows whose blocks meet every rule: borders between codes and their neighbours, all magnitudes,
    zeros of both signs, values that are not finite."""
    x = randn(g, T, HKV, D)
    e = torch.randint(-40 if dtype != torch.float16 else -12, 40 if dtype != torch.float16 else 12, (T, HKV, D // 32, 1),
                      generator=g, device=DEV).float()
    x = (x.unflatten(-1, (-1, 32)) * torch.exp2(e)).flatten(-2)
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.99, 7.0, 0.0, -0.0, -0.25, -5.0, 3.0, 0.5], device=DEV)
    b = x.view(T, HKV, -1, 32)
    b[0::3, :, 0, :16] = edge * torch.exp2(e[0::3, :, 0])
    b[0::3, :, 0, 16:] = b[0::3, :, 0, :16] * (1 + 2.0 ** -8)
    b[1::3, :, 0] = 7.0 * torch.exp2(e[1::3, :, 0]) * torch.where(torch.arange(32, device=DEV) == 9, 1.0, 2.0 ** -6)
    b[2::7, :, 1] = 0
    x = x.to(dtype)
    flat = x.view(T, HKV, -1, 32)
    if T > 8:
        flat[3, 0, 0, 5], flat[4, 0, 0, 31], flat[5, 0, 1, 0] = math.nan, math.inf, -math.inf
        if dtype != torch.float16:
            flat[6, 0, 0] = torch.tensor([2.0 ** -126, -2.0 ** -127, 2.0 ** -128, 3 * 2.0 ** -128] * 8).to(dtype)
            flat[7, 0, 0, 3] = torch.finfo(dtype).max
            flat[8, 0, 1, :2] = torch.tensor([1.75 * 2.0 ** 127, 1.7 * 2.0 ** 127]).to(dtype)
    return x


@pytest.mark.parametrize("T,HKV,D,page,dtype", [(1, 8, 128, 64, torch.bfloat16), (50, 3, 128, 32, torch.bfloat16),
                                                (301, 2, 64, 128, torch.float16), (77, 5, 64, 32, torch.float32),
                                                (40, 1, 128, 64, torch.float32), (33, 8, 128, 64, torch.float16)])
def test_cache_rows_are_the_nearest_codes(T, HKV, D, page, dtype):
    print(f"[case] cache rows {T} {HKV} {D} {page} {dtype}", flush=True)
    g = gen(T + D)
    NP = -(-T // page) + 2
    cache = new_cache(NP, HKV, page, D, g=g)
    before = [t.clone() for t in cache]
    kv = torch.cat([hard_rows(T, HKV, D, dtype, g), hard_rows(T, HKV, D, dtype, g)], 1)       # side by side, as in a product
    k, v = kv[:, :HKV], kv[:, HKV:]
    slots = torch.randperm(NP * page, generator=g, device=DEV)[:T].int()
    ops.kv4_write(k, v, slots, *cache)
    p, o = slots.long() // page, slots.long() % page
    for x, c, s in ((k, 0, 1), (v, 2, 3)):
        qc, qs = ref.quantise(x)
        before[c][p, :, o], before[s][p, :, o] = qc, qs
        assert torch.equal(cache[s], before[s])
        assert torch.equal(cache[c], before[c])
    for dt in (torch.bfloat16, torch.float32):
        for x, c, s in zip(ops.kv4_read(slots, *cache, dtype=dt), (0, 2), (1, 3)):
            want = ref.rows_at(cache[c], cache[s], slots)
            assert x.dtype == dt and torch.equal(x.isnan(), want.isnan())
            assert torch.equal(x.double().nan_to_num(7.0), want.nan_to_num(7.0))


def test_cache_every_bf16_value():
    """Each of the 65536 bf16 patterns, in blocks with a larger neighbour and alone."""
    bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    alone = torch.zeros(65536, 32, device=DEV, dtype=torch.bfloat16)
    alone[:, 11] = bits
    beside = alone.clone()
    beside[:, 3] = (bits.float().abs() * 5.3).clamp(max=3e38).to(torch.bfloat16)
    x = torch.cat([alone, beside]).view(1024, 32, 2, 64)
    k, v = x[:, :, 0], x[:, :, 1]
    cache = new_cache(32, 32, 32, 64, fill=0)
    slots = torch.arange(1024, device=DEV, dtype=torch.int32)
    ops.kv4_write(k, v, slots, *cache)
    for y, c, s in ((k, 0, 1), (v, 2, 3)):
        qc, qs = ref.quantise(y)
        assert torch.equal(cache[s].transpose(1, 2).reshape(1024, 32, 2), qs)
        assert torch.equal(cache[c].transpose(1, 2).reshape(1024, 32, 32), qc)


def test_cache_padding_and_layers_of_one_tensor():
    """Slots outside of the cache are passed over and read as zeros; the caches of several layers lie in one
    tensor, page by page; the neighbours keep what they hold."""
    g = gen(3)
    NP, HKV, page, D, T = 5, 2, 32, 128, 20
    big = [torch.randint(0, 256, (NP, 3, HKV, page, w), generator=g, device=DEV, dtype=torch.uint8) for w in (64, 4, 64, 4)]
    keep = [t.clone() for t in big]
    cache = [t[:, 1] for t in big]
    k, v = randn(g, T, HKV, D, dtype=torch.bfloat16), randn(g, T, HKV, D, dtype=torch.bfloat16)
    slots = torch.randperm(NP * page, generator=g, device=DEV)[:T].int()
    slots[3], slots[8], slots[19] = -1, NP * page, -(1 << 31)
    ops.kv4_write(k, v, slots, *cache)
    ok = (slots >= 0) & (slots < NP * page)
    p, o = slots[ok].long() // page, slots[ok].long() % page
    for x, c in ((k, 0), (v, 2)):
        qc, qs = ref.quantise(x[ok])
        keep[c][p, 1, :, o], keep[c + 1][p, 1, :, o] = qc, qs
    assert all(torch.equal(a, b) for a, b in zip(big, keep))
    kr, vr = ops.kv4_read(slots, *cache)
    assert (kr[~ok] == 0).all() and (vr[~ok] == 0).all()
    assert torch.equal(kr[ok].double(), ref.rows_at(cache[0], cache[1], slots[ok]))
    ops.kv4_write(k[:0], v[:0], slots[:0], *cache)
    assert ops.kv4_read(slots[:0], *cache)[0].shape == (0, HKV, D)


# ================================================================== attention
def paged(lens, HKV, D, page, g, spare=2, extra_width=0):
    """A cache of garbage with the sequences' rows put into shuffled pages of it."""
    held = [-(-n // page) for n in lens]
    NP = sum(held) + spare
    cache = new_cache(NP, HKV, page, D, g=g)
    for s in (1, 3):                                      # garbage scales, NaN among them
        cache[s].copy_(torch.where(cache[s] % 3 == 0, 255, cache[s] % 252 + 2))
    perm = torch.randperm(NP, generator=g, device=DEV).tolist()
    width = max(max(held), 1) + extra_width
    table, at = [], 0
    for h in held:
        table.append(perm[at:at + h] + [-1] * (width - h))
        at += h
    table = i32(table)
    for slots in ref.held(table, lens, page):
        if slots.numel():
            k, v = randn(g, slots.numel(), HKV, D) * 1.5, randn(g, slots.numel(), HKV, D)
            ops.kv4_write(k, v, slots.int().to(DEV), *cache)
    return cache, table


def want_attn(q, cache, table, lens, cu, scale, page):
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(out)
    most = max(b - a for a, b in zip(cu, cu[1:])) * q.shape[1] // cache[0].shape[1]
    for b, slots in enumerate(ref.held(table, lens, page)):
        r = slice(cu[b], cu[b + 1])
        slots = slots.to(DEV)
        k, v = ref.rows_at(cache[0], cache[1], slots), ref.rows_at(cache[2], cache[3], slots)
        out[r], err[r] = ref.attn(q[r], k, v, lens[b], scale, 2.0 ** -11 if most > 64 else 2.0 ** -16)
    return out, err


def check_attn(out, want, err):
    half = torch.finfo(torch.bfloat16).eps / 2
    assert torch.equal(out.isnan(), want.isnan())
    bad = ~((out.double() - want).abs() <= err + half * (want.abs() + err)) & ~want.isnan()
    assert not bad.any(), ((out.double() - want).abs() - err - half * want.abs()).nan_to_num(0).max()


def starts(rows):
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    return cu


CASES = [  # lens, rows (None: one each), HQ, HKV, D, page
    ([1], None, 4, 1, 128, 32), ([31], None, 32, 8, 128, 64), ([33, 0, 1, 64, 65, 32, 700], None, 32, 8, 128, 32),
    ([129, 127, 128], None, 8, 8, 128, 64), ([300, 5], None, 14, 2, 64, 128), ([1025], None, 40, 8, 128, 1024),
    ([97], None, 48, 2, 64, 32), ([515, 1, 40], [2, 1, 2], 32, 8, 128, 64), ([100, 33, 7, 0], [4, 0, 4, 0], 16, 4, 128, 32),
    ([260, 90], [33, 65], 8, 2, 128, 64), ([130], [130], 6, 2, 64, 32), ([400, 3, 77], [5, 3, 1], 14, 2, 64, 64),
    ([4000], None, 4, 1, 128, 64), ([2, 5], [4, 9], 4, 2, 128, 32), ([2500, 800], [20, 3], 7, 1, 128, 32)]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("chunk,copies", [(None, 1), (128, 1), (1 << 20, 1), (256, 5)])
def test_attention(case, chunk, copies, monkeypatch):
    print(f"[case] attn {CASES[case]} chunk={chunk} copies={copies}", flush=True)
    lens, rows, HQ, HKV, D, page = CASES[case]
    if chunk:
        monkeypatch.setattr(ops, "kv4_chunk", lambda cap, units, rows: min(chunk, -(-cap // 128) * 128))
    lens, rows = lens * copies, rows and rows * copies
    g = gen(case)
    cache, table = paged(lens, HKV, D, page, g, extra_width=case % 3)
    cu = starts(rows or [1] * len(lens))
    # the rows of a product, every second token's
    q = randn(g, 2 * cu[-1], HQ + 2, D, dtype=torch.bfloat16)[::2, 1:-1] * 1.3
    scale = D ** -0.5 if case % 2 else 0.11
    out = ops.kv4_attn(q, *cache, table, i32(lens), scale, cu_q=i32(cu) if rows else None, max_q=max(rows) if rows else 1)
    check_attn(out, *want_attn(q, cache, table, lens, cu, scale, page))


@pytest.mark.parametrize("rows", [17, 40])
def test_attention_values_of_all_sizes(rows):
    """Values whose scales lie up to 2^24 apart from key to key and block to block, a first tile of zeros, of
    NaN in masked places: what fp16 does not hold is done in bf16."""
    g = gen(rows + 1)
    page, lens = 32, [300, 200, 150, 70]
    cache, table = paged(lens, 2, 128, page, g)
    for b, slots in enumerate(ref.held(table, lens, page)):
        n = lens[b]
        k, v = randn(g, n, 2, 128), randn(g, n, 2, 128).view(n, 2, 4, 32)
        if b == 0:
            v *= torch.exp2(torch.randint(-12, 13, (n, 2, 4, 1), generator=g, device=DEV).float())
        elif b == 1:
            v[:64] = 0                                    # nothing to go by in the first tile
            v[100:] *= 2.0 ** 60
        elif b == 2:
            v *= 2.0 ** -100
            v[:, :, 2] *= torch.exp2(torch.arange(n, device=DEV).float() / 12)[:, None, None]
        ops.kv4_write(k, v.view(n, 2, 128), slots.int().to(DEV), *cache)
    cu = starts([rows] * 4)
    q = randn(g, cu[-1], 8, 128, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=rows)
    check_attn(out, *want_attn(q, cache, table, lens, cu, 128 ** -0.5, page))


@pytest.mark.parametrize("n,size", [(20001, 11.0 / 8), (60001, 1.953125)])
def test_attention_of_small_weights(n, size):
    """One key takes a weight of 1 and the others e^(-8 size) each: about 2^-16, a quarter of the sum together, or
    2^-22.5, a hundredth of it, which fp16 holds as numbers under its least normal one."""
    g = gen(8)
    rows, page = 40, 64
    cache, table = paged([n], 1, 64, page, g)
    k = torch.zeros(n, 1, 64, device=DEV)
    k[0, 0, :8] = 1.0
    v = torch.ones(n, 1, 64, device=DEV)
    v[0] = -1.0
    ops.kv4_write(k, v, ref.held(table, [n], page)[0].int().to(DEV), *cache)
    q = torch.zeros(rows, 4, 64, device=DEV, dtype=torch.bfloat16)
    q[..., :8] = size
    for R in (1, rows):
        out = ops.kv4_attn(q[:R], *cache, table, i32([n]), 1.0, cu_q=i32([0, R]), max_q=R)
        check_attn(out, *want_attn(q[:R], cache, table, [n], [0, R], 1.0, page))


def test_attention_of_many_sequences():
    """More sequences than a workgroup has threads, most of them short or empty."""
    g = gen(77)
    r = random.Random(4)
    lens = [r.choice((0, 0, 1, 2, 33, 100, 200)) for _ in range(700)]
    lens[650] = 1500
    rows = [min(n, r.choice((0, 1, 2, 3))) if n else r.choice((0, 1)) for n in lens]
    cache, table = paged(lens, 1, 64, 32, g)
    cu = starts(rows)
    q = randn(g, cu[-1], 4, 64, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=3)
    check_attn(out, *want_attn(q, cache, table, lens, cu, 0.125, 32))
    q = randn(g, 700, 2, 64, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens))
    check_attn(out, *want_attn(q, cache, table, lens, list(range(701)), 0.125, 32))


@pytest.mark.parametrize("rows", [1, 3, 33])
def test_attention_scales(rows):
    """A negative scale, one of zero, large scores (one key takes all), scores past what fp32 tells apart, equal
    keys, and queries that are not finite."""
    g = gen(5)
    lens = [150, 70]
    cache, table = paged(lens, 2, 128, 32, g)
    cu = [0, rows, 2 * rows]
    q = randn(g, 2 * rows, 8, 128, dtype=torch.bfloat16)

    def run(q, scale):
        return ops.kv4_attn(q, *cache, table, i32(lens), scale, cu_q=i32(cu), max_q=rows)

    for scale in (-0.09, 0.0, 30.0):
        check_attn(run(q, scale), *want_attn(q, cache, table, lens, cu, scale, 32))
    for size in (2.0 ** 22, 2.0 ** 24, 2.0 ** 27, 2.0 ** 60):
        out = run(q, size)
        assert not out.isnan().any()
        # the one key that takes all, wherever fp32 tells the best two apart
        out, err = run(q, size), None
        for b, slots in enumerate(ref.held(table, lens, 32)):
            k, v = (ref.rows_at(cache[i], cache[i + 1], slots.to(DEV)) for i in (0, 2))
            for j in range(rows):
                n = lens[b] - rows + j + 1
                x = q[cu[b] + j].double().view(2, 4, 1, 128)
                s = (x * k[:n].transpose(0, 1)[:, None]).sum(-1)                     # (2, 4, n)
                size_of = (x.abs() * k[:n].transpose(0, 1)[:, None].abs()).sum(-1).amax(-1)
                top = s.topk(2, -1)
                clear = (top.values[..., 0] - top.values[..., 1]) > 2 * size_of * 132 * 2.0 ** -24 + 40 / size
                want = v.transpose(0, 1)[torch.arange(2, device=DEV)[:, None], top.indices[..., 0]]
                got = out[cu[b] + j].double().view(2, 4, 128)
                assert clear.any() and torch.equal(got[clear], want[clear])
    k = torch.ones(150, 2, 128, device=DEV)
    slots = ref.held(table, lens, 32)[0].int().to(DEV)
    v = randn(g, 150, 2, 128)
    ops.kv4_write(k * 2.0 ** 90, v, slots, *cache)
    check_attn(run(torch.full_like(q, 2.0 ** 30), 1e-6)[:rows],
               *want_attn(torch.full_like(q[:rows], 2.0 ** 30), cache, table[:1], lens[:1], cu[:2], 1e-6, 32))
    q[0, 1, 5], q[rows, 3, 9] = math.nan, math.inf
    out = run(q, 0.1)
    assert out[0, 1].isnan().all() and out[rows, 3].isnan().all()
    assert not out[0, 0].isnan().any() and not out[0, 2:].isnan().any() and not out[rows, :3].isnan().any()


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_nan_stays_with_who_sees_it(rows):
    """A key or a value that is not finite makes NaN of the rows that see it (a value: of its block of
    dims), and of no others: not of earlier tokens, other heads or other sequences."""
    g = gen(rows)
    lens, page = [70, 70, 70], 32
    cache, table = paged(lens, 2, 128, page, g)
    held = ref.held(table, lens, page)
    for b, key in ((0, 69 - rows // 2), (1, 50), (2, 69)):
        k, v = randn(g, 1, 2, 128), randn(g, 1, 2, 128)
        v[0, 1, 40] = math.nan
        if b == 1:
            k[0, 0, 3] = math.inf
        ops.kv4_write(k, v, held[b][key:key + 1].int().to(DEV), *cache)
    cu = starts([rows] * 3)
    q = randn(g, cu[-1], 8, 128, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=rows)
    want, err = want_attn(q, cache, table, lens, cu, 128 ** -0.5, page)
    # a row that does not see the key is formed without it; matmul's 0 * NaN of the reference is not
    assert want.isnan().any() and not want.isnan().all()
    check_attn(out, want, err)


def test_attention_bad_pages_lengths_and_starts():
    """Page ids outside of the cache, lengths past the table, starts that do not fit: NaN, or rows left as
    they were, and no access outside of the cache."""
    g = gen(11)
    lens, page = [100, 100, 100, 40], 32
    cache, table = paged(lens, 2, 128, page, g)
    q = randn(g, 4, 8, 128, dtype=torch.bfloat16)
    table[0, 1], table[1, 3], table[3, 3] = -1, 1 << 30, 12345
    out = ops.kv4_attn(q, *cache, table, i32([100, 100, 100, 40]))
    assert out[:2].isnan().all() and not out[2:].isnan().any()
    out = ops.kv4_attn(q, *cache, table, i32([100, 1 << 30, 100, -3]), max_len=128)
    assert out[1].isnan().all() and (out[3] == 0).all() and not out[2].isnan().any()
    own = torch.full_like(q, 5.0)
    ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32([0, 0, 0, 1, 2]), max_q=1, out=own)
    assert not own[0].isnan().any() and (own[2:] == 5).all()
    own.fill_(5.0)
    ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32([9, 3, -4, 1 << 30, -(1 << 31)]), max_q=2, out=own)
    assert (own == 5).all()
    new = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32([0, 0, 0, 1, 1]), max_q=1)
    assert (new[1:] == 0).all()
    assert ops.kv4_attn(q[:0], *cache, table[:0], i32([])).shape == (0, 8, 128)


@pytest.mark.parametrize("D,HQ,HKV,rows,n", [(128, 8, 2, 3, 100), (128, 8, 2, 3, 5000), (64, 14, 2, 3, 900), (128, 32, 2, 3, 900),
                                             (128, 64, 2, 3, 5000), (64, 80, 1, 3, 100)])
def test_rows_of_no_sequence_are_zeros(D, HQ, HKV, rows, n):
    """An output that the call makes: 0 before the first sequence, behind the last and past max_q, over memory that held
    NaN, by every kernel and with one piece of keys or several; elsewhere what a given output gets."""
    g = gen(31)
    lens = [n, n // 2, n - 7]
    cache, table = paged(lens, HKV, D, 32, g)
    q = randn(g, 300, HQ, D, dtype=torch.bfloat16)
    for cu in ([2, 4, 4, 9], [0, 1, 3, 8], [0, 0, 0, 0], [299, 300, 300, 300], [4, 9, 11, 301], [-1, 2, 3, 3]):
        own = torch.full_like(q, float("nan"))
        ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=rows, out=own)
        used = torch.full_like(q, float("nan"))
        del used
        made = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=rows)
        taken = torch.zeros(300, dtype=torch.bool)
        for r0, r1 in zip(cu, cu[1:]):
            if 0 <= r0 <= r1 <= 300:
                taken[r0:min(r1, r0 + rows)] = True
        assert (own.isnan().all((1, 2)).cpu() != taken).all()
        assert torch.equal(made, torch.where(taken.to(DEV)[:, None, None], own, 0.0))


@pytest.mark.parametrize("HQ,HKV,rows", [(8, 2, 4), (64, 2, 4)])
def test_replays_follow_starts_and_lengths(HQ, HKV, rows):
    """A captured call whose starts and lengths change between replays gives the eager call's rows, zeros among them."""
    g = gen(33)
    lens = [4000, 2500, 700]
    cache, table = paged(lens, HKV, 128, 64, g)
    q = randn(g, 16, HQ, 128, dtype=torch.bfloat16)
    cu, n = i32([0, 4, 8, 12]), i32(lens)

    def call():
        return ops.kv4_attn(q, *cache, table, n, cu_q=cu, max_q=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for starts, held in (([0, 4, 8, 12], lens), ([0, 1, 1, 2], [3999, 1, 0]), ([3, 3, 7, 10], [64, 2000, 3]), ([0, 0, 0, 0], lens),
                         ([0, 4, 8, 12], lens)):
        cu.copy_(i32(starts))
        n.copy_(i32(held))
        want = call().clone()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and not want.isnan().any()
        assert (out[:starts[0]] == 0).all() and (out[starts[-1]:] == 0).all()


def test_pages_far_apart():
    """Offsets past 32 bits: pages of codes 2^31 + 4096 bytes apart."""
    step = (1 << 31) + 4096
    base = [torch.empty(2 * step + 8192, device=DEV, dtype=torch.uint8) for _ in range(2)]
    sc = [torch.empty(3, 1, 32, 4, device=DEV, dtype=torch.uint8) for _ in range(2)]
    cache = [base[0].as_strided((3, 1, 32, 64), (step, 2048, 64, 1)), sc[0],
             base[1].as_strided((3, 1, 32, 64), (step, 2048, 64, 1)), sc[1]]
    g = gen(2)
    table, lens = i32([[2, 0, 1]]), [90]
    slots = ref.held(table, lens, 32)[0].int().to(DEV)
    k, v = randn(g, 90, 1, 128), randn(g, 90, 1, 128)
    ops.kv4_write(k, v, slots, *cache)
    kr, _ = ops.kv4_read(slots, *cache, dtype=torch.float32)
    qc, qs = ref.quantise(k)
    assert torch.equal(kr.double(), ref.values(qc, qs))
    q = randn(g, 1, 4, 128, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens))
    check_attn(out, *want_attn(q, cache, table, lens, [0, 1], 128 ** -0.5, 32))


# ================================================================== together
def decode_loop(steps, graph, B=3, HQ=8, HKV=2, D=128, page=32, seed=0):
    """Tokens of B sequences through extension, norm and rotation, cache and attention, one step after the
    other, eagerly or as one captured step that is replayed; returns outputs of every step and the state."""
    g = gen(seed)
    width, NP = 4, 14
    cache = new_cache(NP, HKV, page, D, fill=255)
    lens, table = i32([29, 0, 63][:B]), torch.full((B, width), -1, device=DEV, dtype=torch.int32)
    free, nfree, status = torch.arange(NP, device=DEV, dtype=torch.int32), i32([NP]), i32([0])
    cos, sin = tables(width * page, D)
    wq, wk = randn(g, D, dtype=torch.bfloat16), randn(g, D, dtype=torch.bfloat16)
    # the prompts
    start = lens.clone()
    lens.zero_()
    total = int(start.sum())
    slots, pos, cu = ops.kv_pages_extend(start, lens, table, free, nfree, status, page, total)
    prompt = randn(g, total, (HQ + 2 * HKV) * D, dtype=torch.bfloat16)
    xs = randn(g, steps, B, (HQ + 2 * HKV) * D, dtype=torch.bfloat16)
    one = torch.ones(B, device=DEV, dtype=torch.int32)
    x = torch.empty_like(xs[0])

    def layer(x, slots, pos, **kw):
        n = x.shape[0]
        q, k = ops.qk_norm_rope(x[:, :HQ * D].view(n, HQ, D), x[:, HQ * D:(HQ + HKV) * D].view(n, HKV, D), pos, cos, sin,
                                wq, wk)
        ops.kv4_write(k, x[:, (HQ + HKV) * D:].view(n, HKV, D), slots, *cache)
        return ops.kv4_attn(q, *cache, table, lens, **kw), q, k

    def step():
        slots, pos, _ = ops.kv_pages_extend(one, lens, table, free, nfree, status, page, B)
        return layer(x, slots, pos)

    outs = [layer(prompt, slots, pos, cu_q=cu, max_q=63)[0].clone()]
    if graph:
        x.copy_(xs[0])
        state = [t.clone() for t in (lens, table, free, nfree, status, *cache)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step()
        for t, u in zip((lens, table, free, nfree, status, *cache), state):
            t.copy_(u)
    for i in range(steps):
        x.copy_(xs[i])
        if graph:
            gr.replay()
        else:
            res = step()
        outs.append(res[0].clone())
        if i % 3 == 0:
            torch.cuda.synchronize()
    return outs, [lens, table, free, nfree, status, *cache], (prompt, xs, start, cos, sin, wq, wk)


def test_decode_loop_eager_and_captured():
    """40 steps that cross pages: a captured step replayed gives what the eager loop gives, bit for bit, and
    both what the sequences' own rows give in 64 bits."""
    steps, HQ, HKV, D, page = 40, 8, 2, 128, 32
    eager, st, (prompt, xs, start, cos, sin, wq, wk) = decode_loop(steps, False)
    captured, st2, _ = decode_loop(steps, True)
    assert all(torch.equal(a, b) for a, b in zip(eager, captured))
    assert all(torch.equal(a, b) for a, b in zip(st, st2))
    assert int(st[4]) == 0
    lens, first = start.tolist(), starts(start.tolist())
    for b in range(3):
        rows = torch.cat([prompt[first[b]:first[b + 1]], xs[:, b]])
        n = rows.shape[0]
        q, k = ops.qk_norm_rope(rows[:, :HQ * D].view(n, HQ, D), rows[:, HQ * D:(HQ + HKV) * D].view(n, HKV, D),
                                torch.arange(n, device=DEV), cos, sin, wq, wk)
        kk = ref.values(*ref.quantise(k))
        vv = ref.values(*ref.quantise(rows[:, (HQ + HKV) * D:].view(n, HKV, D)))
        want, err = ref.attn(q, kk, vv, n, D ** -0.5)
        err[:lens[b]] = ref.attn(q[:lens[b]], kk[:lens[b]], vv[:lens[b]], lens[b], D ** -0.5, 2.0 ** -11)[1]
        check_attn(eager[0][first[b]:first[b + 1]], want[:lens[b]], err[:lens[b]])
        check_attn(torch.stack([eager[1 + i][b] for i in range(steps)]), want[lens[b]:], err[lens[b]:])


def test_two_streams_at_once():
    """Two attentions and two extensions over different states on two streams give what each gives alone."""
    g = gen(9)
    sets = []
    for n in (3000, 2000):
        cache, table = paged([n], 8, 128, 64, g)
        sets.append((randn(g, 1, 32, 128, dtype=torch.bfloat16), cache, table, i32([n])))
    alone = [ops.kv4_attn(q, *c, t, n) for q, c, t, n in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, ((q, c, t, n), s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.kv4_attn(q, *c, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, a) for xs, a in zip(got, alone) for x in xs)
