"""The 8-bit paged cache on the GPU: rows rounded into it, blocks chosen by their bounds, attention over all keys or
over listed blocks, against 64-bit references (tests/kv8_ref.py), alone and as a decode loop runs them."""
import math
import random

import pytest
import torch

from openattention_amd import ops
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=FS):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def starts(rows):
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    return cu


def new_cache(NP, HKV, page, D, g):
    """Tensors full of anything."""
    any8 = lambda *s: torch.randint(0, 256, s, generator=g, device=DEV, dtype=torch.uint8)  # noqa: E731
    return [any8(NP, HKV, page, D), any8(NP, HKV), any8(NP, HKV, page, D), any8(NP, HKV), any8(NP, HKV, 2, D).view(torch.int8)]


def new_table(lens, page, g, spare=2, extra_width=0):
    held = [-(-n // page) for n in lens]
    NP = sum(held) + spare
    perm = torch.randperm(NP, generator=g, device=DEV).tolist()
    width, table, at = max(max(held), 1) + extra_width, [], 0
    for h in held:
        table.append(perm[at:at + h] + [-1] * (width - h))
        at += h
    return i32(table), NP


def host_write(cache, k, v, table, lens, cu, page):
    """What kv8_write leaves, worked out on the host from the cache as it was."""
    c = [t.cpu() for t in cache]
    k, v, table = k.cpu(), v.cpu(), table.cpu()
    for b, n in enumerate(lens):
        if cu[b + 1] > cu[b]:
            ref.write(c[0], c[1], c[4], k[cu[b]:cu[b + 1]], table[b], n, page)
            ref.write(c[2], c[3], None, v[cu[b]:cu[b + 1]], table[b], n, page)
    return c


def same_cache(cache, want):
    for t, w, name in zip(cache, want, ("kc", "ks", "vc", "vs", "kb")):
        assert torch.equal(t.cpu(), w), f"{name}: {int((t.cpu() != w).sum())} differ"


def hard_rows(T, HKV, D, dtype, g):
    """Rows of all sizes, borders between codes and their neighbours, zeros of both signs, values that are not finite."""
    x = randn(g, T, HKV, D)
    e = torch.randint(-9 if dtype == FH else -30, 10 if dtype == FH else 30, (T, HKV, 1), generator=g, device=DEV).float()
    x *= torch.exp2(e)
    mid = torch.cat([ref.MIDDLES, ref.CODES[:127]]).float().to(DEV)
    pick = mid[torch.randint(0, mid.numel(), (T, HKV, D), generator=g, device=DEV)] * torch.where(x < 0, -1.0, 1.0)
    x[0::4] = pick[0::4]
    x[1::4] = pick[1::4] * (1 + 2.0 ** -8)
    x[2::9] = 0
    x[2::9, :, 1::2] = -0.0
    x = x.to(dtype)
    if T > 8:
        x[3, 0, 5], x[5, -1, D - 1], x[7, 0, 0] = math.nan, math.inf, -math.inf
    return x


# ================================================================== cache rows
WRITES = [  # tokens before, new ones, HKV, D, page, type
    ([0], [1], 8, 128, 64, BF), ([63, 64, 0, 5], None, 3, 128, 64, BF), ([40], [200], 2, 64, 32, FH), ([5, 31, 32, 0, 90], [3, 1, 70, 0, 33], 5, 64, 32, FS),
    ([127, 130], [2, 300], 2, 128, 128, FH), ([17, 0, 64], [120, 1, 64], 1, 128, 32, FS), ([0], [257], 8, 128, 64, BF), ([11], [90], 3, 64, 128, BF),
    ([2] * 70, [1, 2, 0, 5, 40, 1, 33] * 10, 1, 64, 32, BF)]


@pytest.mark.parametrize("case", range(len(WRITES)))
def test_rows_written_and_read(case):
    print(f"[case] kv8 write {WRITES[case]}", flush=True)
    before, new, HKV, D, page, dtype = WRITES[case]
    g = gen(case)
    rows = new or [1] * len(before)
    lens = [a + b for a, b in zip(before, rows)]
    table, NP = new_table(lens, page, g, extra_width=case % 3)
    cache = new_cache(NP, HKV, page, D, g)
    cu = starts(rows)
    T = cu[-1]
    # what the blocks held before, then the new rows, side by side as in a product
    for had, rws in ((before, before), (lens, rows)):
        c2 = starts(rws)
        kv = torch.cat([hard_rows(c2[-1], HKV, D, dtype, g), hard_rows(c2[-1], HKV, D, dtype, g)], 1)
        k, v = kv[:, :HKV], kv[:, HKV:]
        want = host_write(cache, k, v, table, had, c2, page)
        one = rws is rows and new is None
        ops.kv8_write(k, v, *cache, table, i32(had), cu=None if one else i32(c2))
        same_cache(cache, want)
    slots = torch.randperm(NP * page, generator=g, device=DEV)[:300].int()
    slots[1], slots[2] = -1, NP * page
    inside = (slots >= 0) & (slots < NP * page)
    for dt in (BF, FS):
        for x, c, s in zip(ops.kv8_read(slots, *cache[:4], dtype=dt), (0, 2), (1, 3)):
            w = ref.rows_at(cache[c], cache[s], slots.clamp(0, NP * page - 1))
            w = torch.where(inside[:, None, None], w, 0.0)
            fine = (cache[s][slots.clamp(0, NP * page - 1).long() // page] % 128 > 9)[..., None] & (cache[s][slots.clamp(0, NP * page - 1).long() // page] < 248)[..., None]
            x, w = torch.where(fine, x.double(), 0.0), torch.where(fine, w, 0.0)       # (scales that a write leaves)
            assert torch.equal(x.isnan(), w.isnan()) and torch.equal(x.nan_to_num(7.0), w.nan_to_num(7.0))
    assert T == sum(rows)


@pytest.mark.parametrize("D,page,dtype", [(64, 32, BF), (128, 64, FS), (128, 128, FH)])
def test_scales_that_grow_token_by_token(D, page, dtype):
    """Tokens one at a time, some many times as large as those before: the block's codes are rounded again each time, the
    bounds enclose what it holds, and a block that is begun again forgets its scale."""
    g = gen(D + page)
    B, HKV, steps = 3, 2, page + 9
    table, NP = new_table([steps] * B, page, g)
    cache = new_cache(NP, HKV, page, D, g)
    lens = [0] * B
    r = random.Random(page)
    for it in range(steps):
        lens = [n + 1 for n in lens]
        if it == 20:
            lens = [5, 1, lens[2]]                         # (drafts taken back, a request that ended)
        x = hard_rows(B, HKV, D, dtype, g).float() if it % 5 else randn(g, B, HKV, D)
        k, v = ((x * 2.0 ** r.randint(-6, 3 + it // 8)).to(dtype) for _ in range(2))
        want = host_write(cache, k, v, table, lens, list(range(B + 1)), page)
        ops.kv8_write(k, v, *cache, table, i32(lens))
        same_cache(cache, want)
        for b, n in enumerate(lens):
            pid, o = int(table[b, (n - 1) // page]), (n - 1) % page + 1
            held = ref.CODES.to(DEV)[cache[0][pid, :, :o].long()]
            held = torch.where(held.isnan(), 0.0 * held, held)
            hi, lo = (torch.where(held.isnan(), -448.0, s * held).amax(1) for s in (1, -1))
            bound = 4 * cache[4][pid].int()
            assert (hi <= bound[:, 0]).all() and (lo <= bound[:, 1]).all()


def test_every_bf16_value():
    """Each of the 65536 bf16 patterns, alone in a block's row of zeros and beside a larger neighbour."""
    bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(BF)
    alone = torch.zeros(65536, 32, device=DEV, dtype=BF)
    alone[:, 11] = bits
    beside = alone.clone()
    beside[:, 3] = (bits.float().abs() * 300).clamp(max=3e38).to(BF)
    # a block of 32 tokens holds one pattern in its first row and zeros in the others
    x = torch.zeros(2 * 65536 // 4, 4, 64, device=DEV, dtype=BF)
    x[:, :, :32] = torch.cat([alone, beside]).view(-1, 4, 32)
    NB = x.shape[0]
    table = torch.randperm(NB, generator=gen(1), device=DEV).int()[:, None].contiguous()
    cache = new_cache(NB, 4, 32, 64, gen(2))
    ops.kv8_write(x, x, *cache, table, torch.ones(NB, device=DEV, dtype=torch.int32))
    y = x.double().cpu()
    fine = torch.isfinite(y).all(-1, keepdim=True)
    top = torch.where(fine, y.abs(), 0.0).amax(-1)
    e = torch.full_like(top, -117)
    for i in range(-117, 120):
        e = torch.where(top > 448 * 2.0 ** i, float(i + 1), e)
    want = ref.codes_of(torch.where(fine, y, math.nan) / torch.exp2(e)[..., None])
    at = table[:, 0].long()
    for c, s in ((0, 1), (2, 3)):
        assert torch.equal(cache[s][at].cpu(), (e + 127).byte())
        assert torch.equal(cache[c][at][:, :, 0].cpu(), want)


def test_writes_that_have_no_place():
    """Pages outside of the cache, sequences longer than their table row, tokens of negative position, starts that leave
    the rows, rows behind the last sequence: passed over, and nothing else changes.  Pages of a layer lie apart."""
    g = gen(9)
    HKV, D, page = 2, 128, 32
    big = [torch.randint(0, 256, (9, 3, *s), generator=g, device=DEV, dtype=torch.uint8)
           for s in ((HKV, page, D), (HKV,), (HKV, page, D), (HKV,), (HKV, 2, D))]
    big[4] = big[4].view(torch.int8)
    cache = [t[:, 1] for t in big]
    table = i32([[0, 1], [9, 2], [3, -1], [4, 5], [6, 7], [1 << 30, 8]])
    lens, rows = [40, 40, 40, 65, 3, 33], [10, 40, 40, 5, 7, 2]
    cu = starts(rows)
    k, v = randn(g, cu[-1] + 3, HKV, D, dtype=BF), randn(g, cu[-1] + 3, HKV, D, dtype=BF)
    keep = [t.clone() for t in big]
    want = [t.cpu() for t in cache]
    for b in (0, 1, 2, 4, 5):                               # (3: 65 tokens in two pages)
        x = slice(cu[b], cu[b + 1])
        ref.write(want[0], want[1], want[4], k[x].cpu(), table[b].cpu(), lens[b], page)
        ref.write(want[2], want[3], None, v[x].cpu(), table[b].cpu(), lens[b], page)
    ops.kv8_write(k, v, *cache, table, i32(lens), cu=i32(cu))
    same_cache(cache, want)
    for t, s in zip(big, keep):
        assert torch.equal(t[:, 0], s[:, 0]) and torch.equal(t[:, 2], s[:, 2])
    state = [t.clone() for t in big]
    for bad in ([0, 10, 9, 200, 210, 220, 230], [-5, -1, -1, -1, -1, -1, -1], [0, 200, 200, 200, 200, 200, 200]):
        ops.kv8_write(k, v, *cache, i32([[0, 1]] * 6), i32([40] * 6) * 0 + i32([0] * 6), cu=i32(bad))
        ops.kv8_write(k, v, *cache, i32([[0, 1]] * 6), i32([-7] * 6), cu=i32(bad))
    assert all(torch.equal(a, b) for a, b in zip(big, state))
    ops.kv8_write(k[:0], v[:0], *cache, table, i32(lens), cu=i32([0] * 7))
    assert all(torch.equal(a, b) for a, b in zip(big, state))
    ops.kv8_write(k[:cu[-1]], v[:cu[-1]], *cache[:4], None, table, i32(lens), cu=i32(cu))       # without bounds
    assert torch.equal(big[4], state[4])
    assert ops.kv8_read(i32([])[:0], *cache[:4])[0].shape == (0, HKV, D)


# ================================================================== blocks chosen
def filled(lens, HKV, D, page, g, spare=2, extra_width=0, size=1.5):
    """A cache of anything with the sequences' rows put into shuffled pages of it, some at a time."""
    table, NP = new_table(lens, page, g, spare, extra_width)
    cache = new_cache(NP, HKV, page, D, g)
    cache[1] %= 100
    cache[3] %= 100
    spread = 0.3 + 2 * torch.rand(HKV, D, generator=g, device=DEV) ** 4
    part = [n // 2 for n in lens]
    for n, r in ((part, part), (lens, [a - b for a, b in zip(lens, part)])):
        T = sum(r)
        if T:
            ops.kv8_write(randn(g, T, HKV, D) * spread * size, randn(g, T, HKV, D), *cache, table, i32(n), cu=i32(starts(r)))
    return cache, table


SELECTS = [  # lens, rows, HQ, HKV, D, page, n, first, last, type
    ([1], None, 4, 1, 128, 32, 3, 1, 2, BF), ([400, 0, 1, 31, 700, 64], None, 32, 8, 128, 32, 5, 1, 2, BF),
    ([900, 300], [40, 5], 14, 2, 64, 32, 6, 0, 1, FH), ([3000], [9], 8, 8, 128, 64, 4, 2, 2, BF), ([1500, 2, 800], [3, 2, 1], 40, 2, 128, 32, 9, 1, 1, FH),
    ([700], [1], 48, 1, 64, 32, 7, 1, 2, BF), ([640, 100, 500], [30, 0, 2], 6, 2, 64, 32, 8, 1, 2, BF), ([2000], [7], 3, 1, 128, 128, 3, 1, 2, BF),
    ([5, 1000], [9, 4], 16, 1, 128, 32, 10, 3, 4, BF), ([16000, 300], [17, 3], 2, 2, 64, 32, 20, 1, 2, BF), ([32700, 40, 9000], None, 4, 2, 64, 32, 300, 1, 2, FH),
    ([17000], [3], 1, 1, 64, 32, 5, 1, 2, BF)]


def want_select(q, cache, table, lens, cu, page, n, first, last):
    out = torch.full((q.shape[0], cache[1].shape[1], n), -1, dtype=torch.int32)
    for b, m in enumerate(lens):
        if cu[b + 1] > cu[b]:
            out[cu[b]:cu[b + 1]] = ref.select(q[cu[b]:cu[b + 1]].cpu(), cache[1].cpu(), cache[4].cpu(), table[b].cpu(), m, page, n, first, last)
    return out


@pytest.mark.parametrize("case", range(len(SELECTS)))
def test_selection(case):
    print(f"[case] kv8 select {SELECTS[case]}", flush=True)
    lens, rows, HQ, HKV, D, page, n, first, last, dtype = SELECTS[case]
    g = gen(case + 50)
    cache, table = filled(lens, HKV, D, page, g, extra_width=case % 3)
    cu = starts(rows or [1] * len(lens))
    q = randn(g, 2 * cu[-1], HQ + 2, D, dtype=dtype)[::2, 1:-1]
    if cu[-1] > 3:
        q[1, 0, 5], q[2, :, 3], q[3] = math.nan, math.inf, 0
    got = ops.kv8_select(q, cache[1], cache[4], table, i32(lens), page, n, cu_q=i32(cu) if rows else None, first=first, last=last)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), want_select(q, cache, table, lens, cu, page, n, first, last))


def test_selection_of_ties_and_sizes():
    """Equal scores go to the lower block, scales of all sizes keep their order, pages outside of the cache come last."""
    g = gen(3)
    page, NB, D = 32, 300, 64
    table = torch.randperm(NB, generator=g, device=DEV).int()[None].contiguous()
    kb = torch.randint(-3, 4, (NB, 1, 2, D), generator=g, device=DEV, dtype=torch.int8)
    ks = torch.randint(120, 128, (NB, 1), generator=g, device=DEV, dtype=torch.uint8)
    kb[100:200], ks[100:200] = kb[100], ks[100]
    q = randn(g, 1, 2, D, dtype=BF)
    lens = [NB * page]
    cache = [None, ks, None, None, kb]
    for n, first, last in ((1, 0, 1), (4, 0, 1), (4, 1, 2), (120, 5, 1), (150, 0, 150), (299, 0, 1), (300, 1, 1), (310, 1, 1)):
        for scales in (ks, torch.full_like(ks, 127), torch.randint(10, 248, ks.shape, generator=g, device=DEV, dtype=torch.uint8)):
            cache[1] = scales
            for x in (q, q * 0, (q.float() * 2.0 ** 100).to(BF), (q.float() * 2.0 ** -120).to(BF)):
                got = ops.kv8_select(x, scales, kb, table, i32(lens), page, n, first=first, last=last)
                assert torch.equal(got.cpu(), want_select(x, cache, table, lens, [0, 1], page, n, first, last))
    cache[1] = ks
    holes = table.clone()
    holes[0, 7:250:3] = -1
    holes[0, 8:250:9] = NB
    for n in (150, 260):
        got = ops.kv8_select(q, ks, kb, holes, i32(lens), page, n)
        assert torch.equal(got.cpu(), want_select(q, cache, holes, lens, [0, 1], page, n, 1, 2))


def test_selection_of_many_blocks():
    """More scores than a workgroup keeps in registers."""
    g = gen(4)
    page, HKV, D, lens = 32, 2, 64, [32 * 5003 - 7, 32 * 2048, 32 * 2049, 900]
    table, NP = new_table(lens, page, g)
    kb = torch.randint(0, 113, (NP, HKV, 2, D), generator=g, device=DEV, dtype=torch.int8)
    ks = torch.randint(118, 124, (NP, HKV), generator=g, device=DEV, dtype=torch.uint8)
    q = randn(g, 4, 4, D, dtype=BF)
    for n in (3, 64, 1000, 4000):
        got = ops.kv8_select(q, ks, kb, table, i32(lens), page, n)
        assert torch.equal(got.cpu(), want_select(q, [None, ks, None, None, kb], table, lens, [0, 1, 2, 3, 4], page, n, 1, 2))


def test_selection_that_has_no_place():
    """Sequences past their table row or max_len, starts that leave the rows, rows of no sequence: -1 alone."""
    g = gen(6)
    cache, table = filled([300, 200], 2, 64, 32, g)
    q = randn(g, 6, 4, 64, dtype=BF)
    one = ops.kv8_select(q[:2], cache[1], cache[4], table, i32([300, 200]), 32, 4)
    assert (one >= 0).all()
    got = ops.kv8_select(q[:2], cache[1], cache[4], table, i32([321, 200]), 32, 4)
    assert (got[0] == -1).all() and torch.equal(got[1], one[1])
    got = ops.kv8_select(q[:2], cache[1], cache[4], table, i32([300, 200]), 32, 4, max_len=200)
    assert (got[0] == -1).all() and torch.equal(got[1], one[1])
    got = ops.kv8_select(q, cache[1], cache[4], table, i32([300, 200]), 32, 4, cu_q=i32([1, 3, 5]))
    assert (got[[0, 5]] == -1).all() and (got[1:5] >= 0).all()
    for cu in ([-1, 2, 4], [0, 7, 7], [4, 2, 1]):
        got = ops.kv8_select(q, cache[1], cache[4], table, i32([300, 200]), 32, 4, cu_q=i32(cu))
        assert ((got >= -1) & (got < 10)).all()
    assert ops.kv8_select(q[:0], cache[1], cache[4], table, i32([300, 200]), 32, 4, cu_q=i32([0, 0, 0])).shape == (0, 2, 4)


def test_selection_of_no_sequences():
    """Rows that no sequence takes, as there is none: -1 alone, at once and again."""
    cache, table = filled([100], 2, 64, 32, gen(61))
    q = randn(gen(62), 3, 4, 64, dtype=BF)
    for _ in range(3):
        junk = torch.full((3 * 2 * 4,), 7, device=DEV, dtype=torch.int32)
        del junk                                             # (what the next tensor of this size is likely to hold)
        got = ops.kv8_select(q, cache[1], cache[4], table[:0], i32([]), 32, 4, cu_q=i32([0]))
        assert got.shape == (3, 2, 4) and (got == -1).all()


@pytest.mark.parametrize("HQ,blocks,rows", [(1, 512, 16), (1, 512, 1), (2, 1024, 9), (16, 1024, 2), (16, 8, 1)])
def test_selection_of_the_largest_tiles(HQ, blocks, rows):
    """As many scores as one launch holds, with rows of the larger head dimension."""
    g = gen(63)
    page, D = 32, 128
    table = torch.randperm(blocks, generator=g, device=DEV).int()[None].contiguous()
    kb = torch.randint(-5, 113, (blocks, 1, 2, D), generator=g, device=DEV, dtype=torch.int8)
    ks = torch.randint(118, 124, (blocks, 1), generator=g, device=DEV, dtype=torch.uint8)
    q = randn(g, rows, HQ, D, dtype=BF)
    for n in (4, blocks // 2, blocks - 1):
        if n < 3:
            continue
        got = ops.kv8_select(q, ks, kb, table, i32([blocks * page]), page, n, cu_q=i32([0, rows]))
        assert torch.equal(got.cpu(), want_select(q, [None, ks, None, None, kb], table, [blocks * page], [0, rows], page, n, 1, 2))


# ================================================================== attention
def values_of(cache, table, lens, page):
    """fp64 keys and values of every sequence"""
    out = []
    for row, n in zip(table.tolist(), lens):
        t = torch.arange(n, device=DEV)
        ids = torch.tensor(row, device=DEV)
        slots = ids[t // page] * page + t % page
        out.append((ref.rows_at(cache[0], cache[1], slots), ref.rows_at(cache[2], cache[3], slots)))
    return out


def want_attn(q, cache, table, lens, cu, scale, page, blocks=None):
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(out)
    most = max(b - a for a, b in zip(cu, cu[1:])) * q.shape[1] // cache[0].shape[1]
    for b, (k, v) in enumerate(values_of(cache, table, lens, page)):
        r = slice(cu[b], cu[b + 1])
        out[r], err[r] = ref.attn(q[r], k, v, lens[b], scale, 2.0 ** -11 if most > 64 and blocks is None else 2.0 ** -16,
                                  None if blocks is None else blocks[r], page)
    return out, err


def check_attn(out, want, err):
    half = torch.finfo(out.dtype).eps / 2
    least = 2.0 ** -25 if out.dtype == FH else 0.0          # (fp16 below 2^-14)
    assert torch.equal(out.isnan(), want.isnan())
    bad = ~((out.double() - want).abs() <= err + half * (want.abs() + err) + least) & ~want.isnan()
    assert not bad.any(), ((out.double() - want).abs() - err - half * want.abs()).nan_to_num(0).max()


CASES = [  # lens, rows (None: one each), HQ, HKV, D, page, type
    ([1], None, 4, 1, 128, 32, BF), ([31], None, 32, 8, 128, 64, FH), ([33, 0, 1, 64, 65, 32, 700], None, 32, 8, 128, 32, BF),
    ([129, 127, 128], None, 8, 8, 128, 64, FH), ([300, 5], None, 14, 2, 64, 128, BF), ([1025], None, 40, 8, 128, 128, BF),
    ([97], None, 48, 2, 64, 32, FH), ([515, 1, 40], [2, 1, 2], 32, 8, 128, 64, BF), ([100, 33, 7, 0], [4, 0, 4, 0], 16, 4, 128, 32, FH),
    ([260, 90], [33, 65], 8, 2, 128, 64, BF), ([130], [130], 6, 2, 64, 32, FH), ([400, 3, 77], [5, 3, 1], 14, 2, 64, 64, BF),
    ([4000], None, 4, 1, 128, 64, BF), ([2, 5], [4, 9], 4, 2, 128, 32, BF), ([2500, 800], [20, 3], 7, 1, 128, 32, FH),
    ([700, 300], [40, 64], 16, 4, 128, 128, FH)]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("chunk,copies", [(None, 1), (128, 1), (1 << 20, 1), (256, 5)])
def test_attention(case, chunk, copies, monkeypatch):
    print(f"[case] kv8 attn {CASES[case]} chunk={chunk} copies={copies}", flush=True)
    lens, rows, HQ, HKV, D, page, dtype = CASES[case]
    if chunk:
        monkeypatch.setattr(ops, "kv8_chunk", lambda cap, units, rows, listed: min(chunk, -(-cap // 128) * 128))
    lens, rows = lens * copies, rows and rows * copies
    g = gen(case)
    cache, table = filled(lens, HKV, D, page, g, extra_width=case % 3)
    cu = starts(rows or [1] * len(lens))
    # the rows of a product, every second token's
    q = randn(g, 2 * cu[-1], HQ + 2, D, dtype=dtype)[::2, 1:-1] * 1.3
    scale = D ** -0.5 if case % 2 else 0.11
    out = ops.kv8_attn(q, *cache[:4], table, i32(lens), scale, cu_q=i32(cu) if rows else None, max_q=max(rows) if rows else 1)
    assert out.dtype == dtype
    check_attn(out, *want_attn(q, cache, table, lens, cu, scale, page))


def lists(T, HKV, n, W, g):
    """Blocks in any order, numbers that name nothing among them."""
    r = torch.rand(T, HKV, W + 6, generator=g, device=DEV).argsort(-1)[..., :n] - 3
    return torch.where(r < 0, r * 1000003, r).int().contiguous()


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("n,chunk", [(1, None), (3, 128), (9, None), (40, 256)])
def test_attention_over_blocks(case, n, chunk, monkeypatch):
    print(f"[case] kv8 blocks {CASES[case]} n={n} chunk={chunk}", flush=True)
    lens, rows, HQ, HKV, D, page, dtype = CASES[case]
    if chunk:
        monkeypatch.setattr(ops, "kv8_chunk", lambda cap, units, rows, listed: min(chunk, -(-cap // 128) * 128))
    g = gen(case + 30)
    cache, table = filled(lens, HKV, D, page, g, extra_width=case % 3)
    cu = starts(rows or [1] * len(lens))
    q = randn(g, 2 * cu[-1], HQ + 2, D, dtype=dtype)[::2, 1:-1] * 1.3
    W = table.shape[1]
    blocks = lists(cu[-1], HKV, min(n, W + 6), W, g)
    out = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu) if rows else None, max_q=max(rows) if rows else 1, blocks=blocks)
    check_attn(out, *want_attn(q, cache, table, lens, cu, D ** -0.5, page, blocks))


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("listed", [False, True])
def test_attention_scales(rows, listed):
    """A negative scale, one of zero, large scores (one key takes all), scores past what fp32 tells apart."""
    g = gen(5)
    lens, page = [150, 70], 32
    cache, table = filled(lens, 2, 128, page, g)
    cu = [0, rows, 2 * rows]
    q = randn(g, 2 * rows, 8, 128, dtype=BF)
    blocks = i32([[[0, 1, 2, 3, 4]] * 2] * (2 * rows)) if listed else None

    def run(q, scale):
        return ops.kv8_attn(q, *cache[:4], table, i32(lens), scale, cu_q=i32(cu), max_q=rows, blocks=blocks)

    for scale in (-0.09, 0.0, 30.0):
        check_attn(run(q, scale), *want_attn(q, cache, table, lens, cu, scale, page, blocks))
    for size in (2.0 ** 22, 2.0 ** 24, 2.0 ** 27, 2.0 ** 60):
        out = run(q, size)
        assert not out.isnan().any()
        # the one key that takes all, wherever fp32 tells the best two apart
        for b, (k, v) in enumerate(values_of(cache, table, lens, page)):
            for j in range(rows):
                n = lens[b] - rows + j + 1
                x = q[cu[b] + j].double().view(2, 4, 1, 128)
                s = (x * k[:n].transpose(0, 1)[:, None]).sum(-1)                     # (2, 4, n)
                size_of = (x.abs() * k[:n].transpose(0, 1)[:, None].abs()).sum(-1).amax(-1)
                top = s.topk(2, -1)
                clear = (top.values[..., 0] - top.values[..., 1]) > 2 * size_of * 132 * 2.0 ** -24 + 40 / size
                want = v.transpose(0, 1)[torch.arange(2, device=DEV)[:, None], top.indices[..., 0]]
                got = out[cu[b] + j].double().view(2, 4, 128)
                assert clear.any() and ((got - want).abs() <= 2.0 ** -8 * want.abs())[clear].all()


@pytest.mark.parametrize("rows", [1, 5, 17, 40])
@pytest.mark.parametrize("listed", [False, True])
def test_attention_values_of_all_sizes(rows, listed):
    """Values whose blocks' scales lie far apart, zeros among them."""
    g = gen(rows + 1)
    page, lens = 32, [300, 200, 150, 70]
    table, NP = new_table(lens, page, g)
    cache = new_cache(NP, 2, page, 128, g)
    for b, n in enumerate(lens):
        k, v = randn(g, n, 2, 128), randn(g, n, 2, 128)
        blk = torch.arange(n, device=DEV) // page
        if b == 0:
            v *= torch.exp2(torch.randint(-20, 21, (10, 2), generator=g, device=DEV).float())[blk][..., None]
        elif b == 1:
            v[:64] = 0
            v[100:] *= 2.0 ** 60
        elif b == 2:
            v *= 2.0 ** -100
            v *= torch.exp2(blk.float() * 40)[:, None, None]
        ops.kv8_write(k, v, *cache, table[b:b + 1], i32([n]), cu=i32([0, n]))
    cu = starts([rows] * 4)
    q = randn(g, cu[-1], 8, 128, dtype=BF)
    blocks = lists(cu[-1], 2, 7, 10, g) if listed else None
    out = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=rows, blocks=blocks)
    check_attn(out, *want_attn(q, cache, table, lens, cu, 128 ** -0.5, page, blocks))


@pytest.mark.parametrize("n,size", [(20001, 11.0 / 8), (60001, 1.953125)])
def test_attention_of_small_weights(n, size):
    """One key takes a weight of 1 and the others e^(-8 size) each: about 2^-16, a quarter of the sum together, or
    2^-22.5, a hundredth of it."""
    rows, page = 40, 64
    table, NP = new_table([n], page, gen(8))
    cache = new_cache(NP, 1, page, 64, gen(9))
    k = torch.zeros(n, 1, 64, device=DEV)
    k[0, 0, :8] = 1.0
    v = torch.ones(n, 1, 64, device=DEV)
    v[0] = -1.0
    ops.kv8_write(k, v, *cache, table, i32([n]), cu=i32([0, n]))
    q = torch.zeros(rows, 4, 64, device=DEV, dtype=BF)
    q[..., :8] = size
    for R in (1, rows):
        out = ops.kv8_attn(q[:R], *cache[:4], table, i32([n]), 1.0, cu_q=i32([0, R]), max_q=R)
        check_attn(out, *want_attn(q[:R], cache, table, [n], [0, R], 1.0, page))


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("HQ", [8, 32])
def test_attention_of_nan(rows, listed, HQ):
    """Keys, values and queries that are not finite reach the rows that see them and no others; what lies past a sequence's
    end is never seen."""
    g = gen(12)
    page, n = 32, 140
    cache, table = filled([n], 2, 128, page, g)
    for what, at in (("k", n - 2), ("v", n - 2), ("v", 33), ("k", 40)):
        c2 = [t.clone() for t in cache]
        pid, o = int(table[0, at // page]), at % page
        c2[0 if what == "k" else 2][pid, 1, o] = 0x7f if at == 33 else 0xff
        q = randn(g, rows, HQ, 128, dtype=BF)
        blocks = i32([[[0, 1, 4]] * 2] * rows) if listed else None
        out = ops.kv8_attn(q, *c2[:4], table, i32([n]), cu_q=i32([0, rows]), max_q=rows, blocks=blocks)
        want, err = want_attn(q, c2, table, [n], [0, rows], 128 ** -0.5, page, blocks)
        check_attn(out, want, err)
        assert want.isnan().any()
    q = randn(g, rows, HQ, 128, dtype=BF)
    q[0, 1, 3], q[0, HQ - 1, 7] = math.nan, math.inf
    out = ops.kv8_attn(q, *cache[:4], table, i32([n]), cu_q=i32([0, rows]), max_q=rows, blocks=i32([[[0, 1, 4]] * 2] * rows) if listed else None)
    nan = out.isnan().all(-1)
    assert nan[0, 1] and nan[0, HQ - 1] and int(nan.sum()) == 2 and int(out.isnan().sum()) == 256


def test_attention_that_has_no_place():
    """Pages outside of the cache and sequences past their row give NaN rows, lists that name nothing and rows that see no
    key 0; rows that no sequence takes are left alone in a given output and 0 in a new one."""
    g = gen(13)
    page = 32
    for D, HQ, HKV in ((128, 8, 2), (64, 34, 2)):
        cache, table = filled([100, 64, 40], HKV, D, page, g)
        lens = i32([100, 64, 40])
        q = randn(g, 3, HQ, D, dtype=BF)
        good = ops.kv8_attn(q, *cache[:4], table, lens)
        bad = table.clone()
        bad[0, 3], bad[1, 0] = -1, 1 << 29
        out = ops.kv8_attn(q, *cache[:4], bad, lens)
        assert out[:2].isnan().all() and torch.equal(out[2], good[2])
        long = ops.kv8_attn(q, *cache[:4], table, i32([129, 64, 40]))
        assert long[0].isnan().all() and torch.equal(long[1:], good[1:])
        every = i32([[[0, 1, 2, 3]] * HKV] * 3)
        assert ops.kv8_attn(q, *cache[:4], table, i32([129, 64, 40]), blocks=every)[0].isnan().all()
        out = ops.kv8_attn(q, *cache[:4], bad, lens, blocks=i32([[[0, 1]] * HKV, [[1, -1]] * HKV, [[5, -1]] * HKV]))
        assert not out.isnan().any() and (out[2] == 0).all() and (out[:2] != 0).any()
        assert ops.kv8_attn(q, *cache[:4], bad, lens, blocks=every)[:2].isnan().all()
        zero = ops.kv8_attn(q, *cache[:4], table, i32([0, -3, 40]))
        assert (zero[:2] == 0).all() and torch.equal(zero[2], good[2])
        x = randn(g, 9, HQ, D, dtype=BF)
        for n in (None, 4):
            blocks = None if n is None else i32([[[0, 1, 2, 3]] * HKV] * 9)
            cu = i32([1, 3, 3, 7])
            new = ops.kv8_attn(x, *cache[:4], table, lens, cu_q=cu, max_q=2, blocks=blocks)
            kept = torch.full((10, HQ, D), 7.0, device=DEV, dtype=BF)
            ops.kv8_attn(x, *cache[:4], table, lens, cu_q=cu, max_q=2, blocks=blocks, out=kept[:9])
            took = [1, 2, 3, 4]
            rest = [0, 5, 6, 7, 8]
            assert (new[rest] == 0).all() and (kept[rest] == 7).all() and (kept[9] == 7).all()
            assert torch.equal(new[took], kept[took])
            for c in ([-1, 2, 4, 5], [0, 30, 30, 30], [5, 3, 2, 1]):
                ops.kv8_attn(x, *cache[:4], table, lens, cu_q=i32(c), max_q=2, blocks=blocks)


def test_attention_of_many_sequences():
    """More sequences than a wave has lanes squared, most of them short or empty."""
    g = gen(77)
    r = random.Random(4)
    B = 4200
    lens = [r.choice((0, 0, 1, 2, 33)) for _ in range(B)]
    lens[3650] = 500
    rows = [min(n, r.choice((0, 1, 2, 3))) if n else r.choice((0, 1)) for n in lens]
    cache, table = filled(lens, 1, 64, 32, g)
    cu = starts(rows)
    q = randn(g, cu[-1], 4, 64, dtype=BF)
    want, err = want_attn(q, cache, table, lens, cu, 0.125, 32)
    check_attn(ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=3), want, err)
    blocks = ops.kv8_select(q, cache[1], cache[4], table, i32(lens), 32, table.shape[1], cu_q=i32(cu))
    check_attn(ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=3, blocks=blocks), want, err)


def test_all_blocks_are_all_keys():
    """Where a list names every block the sums are those of the call without one, up to their order."""
    g = gen(21)
    lens, rows = [500, 77], [4, 3]
    cache, table = filled(lens, 2, 128, 64, g)
    cu = starts(rows)
    q = randn(g, cu[-1], 8, 128, dtype=BF)
    blocks = ops.kv8_select(q, cache[1], cache[4], table, i32(lens), 64, 12, cu_q=i32(cu))
    assert (blocks[0, 0] == i32([0, 1, 2, 3, 4, 5, 6, 7, -1, -1, -1, -1])).all()
    a = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=4, blocks=blocks)
    b = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=4)
    assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs().clamp(min=2.0 ** -8)).all()


@pytest.mark.parametrize("rows", [2, 20, 70])
def test_bad_pages_reach_the_rows_that_see_them(rows):
    """A page outside of the cache makes NaN of the tokens behind its beginning and of no others, however many rows share
    their keys."""
    g = gen(14)
    page, n = 32, 97
    cache, table = filled([n], 2, 128, page, g)
    bad = table.clone()
    bad[0, 3] = -1
    for HQ in (4, 8):
        q = randn(g, rows, HQ, 128, dtype=BF)
        good = ops.kv8_attn(q, *cache[:4], table, i32([n]), cu_q=i32([0, rows]), max_q=rows)
        out = ops.kv8_attn(q, *cache[:4], bad, i32([n]), cu_q=i32([0, rows]), max_q=rows)
        assert out[-1].isnan().all() and torch.equal(out[:-1], good[:-1])
        last = ops.kv8_attn(q, *cache[:4], table, i32([n - 1]), cu_q=i32([0, rows]), max_q=rows)
        none = ops.kv8_attn(q, *cache[:4], bad, i32([n - 1]), cu_q=i32([0, rows]), max_q=rows)
        assert torch.equal(last, none) and not none.isnan().any()


def test_pages_past_32_bits():
    """Codes more than 2^32 bytes from the first page's: every operator gives what it gives over near pages, bit by bit."""
    g = gen(31)
    HKV, page, D, lens, rows = 8, 64, 128, [700, 150], [70, 40]
    table, NP = new_table(lens, page, g)
    far = (1 << 32) // (HKV * page * D) + NP + 3
    near, cu = new_cache(NP, HKV, page, D, g), i32(starts(lens))
    wide = [torch.empty(far, *t.shape[1:], device=DEV, dtype=t.dtype) for t in near]
    away = torch.where(table >= 0, far - 1 - table, table)
    assert (away[table >= 0].long() * HKV * page * D >= 1 << 32).all()
    k, v = randn(g, sum(lens), HKV, D, dtype=BF), randn(g, sum(lens), HKV, D, dtype=BF)
    n = i32(lens)
    ops.kv8_write(k, v, *near, table, n, cu)
    ops.kv8_write(k, v, *wide, away, n, cu)
    slots, back = [i32([int(t[b, i // page]) * page + i % page for b, m in enumerate(lens) for i in range(m)]) for t in (table, away)]
    for a, b in zip(ops.kv8_read(slots, *near[:4]), ops.kv8_read(back, *wide[:4])):
        assert torch.equal(a, b)
    for r, HQ in ((None, 32), ([1, 1], 64), ([5, 3], 32), (rows, 16)):
        c = None if r is None else i32(starts(r))
        q = randn(g, 2 if r is None else sum(r), HQ, D, dtype=BF)
        m = 1 if r is None else max(r)
        assert torch.equal(ops.kv8_attn(q, *near[:4], table, n, cu_q=c, max_q=m), ops.kv8_attn(q, *wide[:4], away, n, cu_q=c, max_q=m))
        x, y = ops.kv8_select(q, near[1], near[4], table, n, page, 5, c), ops.kv8_select(q, wide[1], wide[4], away, n, page, 5, c)
        assert torch.equal(x, y)
        assert torch.equal(ops.kv8_attn(q, *near[:4], table, n, cu_q=c, max_q=m, blocks=x),
                           ops.kv8_attn(q, *wide[:4], away, n, cu_q=c, max_q=m, blocks=x))


@pytest.mark.parametrize("HQ,HKV,D,page,dtype", [(32, 8, 128, 64, BF), (14, 2, 64, 32, FH), (5, 1, 128, 128, FH)])
def test_short_sequences_beside_long_ones(HQ, HKV, D, page, dtype, monkeypatch):
    """Sequences of few rows in a call that holds one of many: what they give on their own, bit by bit."""
    g = gen(33)
    rows, lens = [70, 1, 2, 0, 3, 9, 1, 16], [700, 1300, 2, 40, 333, 95, 0, 1100]
    cache, table = filled(lens, HKV, D, page, g)
    cu = starts(rows)
    q = randn(g, cu[-1] + 1, HQ, D, dtype=dtype)
    for chunk in (1 << 20, 256):
        monkeypatch.setattr(ops, "kv8_chunk", lambda cap, units, rows, listed: min(chunk, -(-cap // 128) * 128))
        out = torch.full_like(q, 3.0)
        got = ops.kv8_attn(q[:-1], *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=70)
        assert ops.kv8_attn(q[:-1], *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=70, out=out[:-1]).data_ptr() == out.data_ptr()
        assert torch.equal(out[:-1], got) and (out[-1] == 3).all()
        check_attn(got, *want_attn(q[:-1], cache, table, lens, cu, D ** -0.5, page))
        for b, r in enumerate(rows):
            if 0 < r and r * HQ // HKV <= 64:
                own = ops.kv8_attn(q[cu[b]:cu[b + 1]], *cache[:4], table[b:b + 1], i32(lens[b:b + 1]), cu_q=i32([0, r]), max_q=r)
                if r * HQ // HKV <= 8 or r * HQ // HKV > 16:          # (between them the sums of 16 rows, not of 32)
                    assert torch.equal(got[cu[b]:cu[b + 1]], own)
    # a page outside of the cache, and a sequence past its table row, beside the others
    monkeypatch.undo()
    bad, long = table.clone(), list(lens)
    bad[1, 0], long[4] = -1, table.shape[1] * page + 1
    out = ops.kv8_attn(q[:-1], *cache[:4], bad, i32(long), cu_q=i32(cu), max_q=70)
    good = ops.kv8_attn(q[:-1], *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=70)
    assert out[cu[1]:cu[2]].isnan().all() and out[cu[4]:cu[5]].isnan().all()
    rest = [t for t in range(cu[-1]) if not (cu[1] <= t < cu[2] or cu[4] <= t < cu[5])]
    assert torch.equal(out[rest], good[rest])


@pytest.mark.parametrize("listed", [False, True])
def test_sparse_calls(listed, monkeypatch):
    """Few tokens of the many that the sequences may have, in pieces: rows that no sequence takes before, behind and past
    max_q, left as they were or 0, and starts that do not fit the rows."""
    monkeypatch.setattr(ops, "kv8_chunk", lambda cap, units, rows, listed: 128)
    g = gen(34)
    HQ, HKV, D, page, rows, lens = 8, 2, 64, 32, [40, 1, 2, 0, 1, 1, 3, 1], [300, 170, 90, 0, 1, 0, 260, 64]
    cache, table = filled(lens, HKV, D, page, g)
    cu = [2 + c for c in starts(rows)]
    T = cu[-1] + 3
    q = randn(g, T, HQ, D, dtype=BF)
    W = table.shape[1]
    blocks = lists(T, HKV, 6, W, g) if listed else None
    want, err = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    own = None if blocks is None else blocks[2:cu[-1]]
    want[2:cu[-1]], err[2:cu[-1]] = want_attn(q[2:cu[-1]], cache, table, lens, starts(rows), D ** -0.5, page, own)
    out = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=40, blocks=blocks)
    check_attn(out, want, err)
    kept = torch.full_like(q, 7.0)
    ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=40, blocks=blocks, out=kept)
    assert (kept[:2] == 7).all() and (kept[cu[-1]:] == 7).all() and torch.equal(kept[2:cu[-1]], out[2:cu[-1]])
    # 25 of the first sequence's 40 tokens
    fewer = ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(cu), max_q=25, blocks=blocks)
    assert (fewer[27:42] == 0).all()
    check_attn(torch.cat([fewer[2:27], fewer[42:cu[-1]]]), torch.cat([want[2:27], want[42:cu[-1]]]), torch.cat([err[2:27], err[42:cu[-1]]]))
    for bad in ([-1] + cu[1:], cu[:-1] + [T + 1], [5, 3] + cu[2:], [T + 9] * 9):
        ops.kv8_attn(q, *cache[:4], table, i32(lens), cu_q=i32(bad), max_q=40, blocks=blocks)
