"""What the operators of the 4-bit paged cache hand to the library, and refuse, where their first tests do not look (CPU
tensors stand in for device ones; the launch is recorded instead)."""
import random

import pytest
import torch

from openattention_amd import lib, ops
from tests.test_gpu_kv4 import CASES
from tests.test_kv4_cpu import cache, calls, rope_args  # noqa: F401


def attn_sizes(call):
    """(chunk, nchunk) of a recorded oa_kv4_attn"""
    name, a = call
    assert name == "oa_kv4_attn" and len(a) + 1 == len(lib.SIGNATURES[name])
    return a[23:25]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_the_rule_for_pieces_is_looked_up_in_every_call(calls, case, monkeypatch):  # noqa: F811
    """Sizes are looked up by value, and the rule that cuts the keys is one of the values: another rule in its place is
    followed from the next call on, and the first one again once it is back."""
    lens, rows, HQ, HKV, D, page = CASES[case]
    width = max(1, -(-max(lens) // page)) + case % 3
    T, cap = sum(rows or [1] * len(lens)), width * page
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731

    def call():
        ops.kv4_attn(torch.zeros(T, HQ, D, dtype=torch.bfloat16), **cache(NP=2, H=HKV, page=page, D=D), table=z(len(lens), width),
                     lens=z(len(lens)), cu_q=z(len(lens) + 1) if rows else None, max_q=max(rows) if rows else 1)
        return attn_sizes(calls[-1])
    own = call()
    for chunk in (128, 1 << 20, 256):
        with monkeypatch.context() as m:
            m.setattr(ops, "kv4_chunk", lambda cap, units, rows: min(chunk, -(-cap // 128) * 128))
            want = min(chunk, -(-cap // 128) * 128)
            assert call() == call() == (want, -(-cap // want))
    assert call() == own


@pytest.mark.parametrize("B", [65535, 65536, 1 << 20])
def test_more_sequences_than_a_grids_axis_holds_take_one_piece_each(calls, B):  # noqa: F811
    """The join counts sequences along an axis of 65535; so many fill the card with a piece each."""
    c = cache(NP=2, H=1, page=32, D=64)
    q, lens = torch.zeros(B, 1, 64, dtype=torch.bfloat16), torch.zeros(B, dtype=torch.int32)
    ops.kv4_attn(q, **c, table=torch.zeros(B, 40, dtype=torch.int32), lens=lens)
    chunk, n = attn_sizes(calls[-1])
    assert chunk * n >= 1280 and (n > 1) == (B == 65535) and (n > 1 or chunk == 1280)
    ops.kv4_attn(q, **c, table=torch.zeros(B, 40, dtype=torch.int32), lens=lens, max_len=100)
    assert attn_sizes(calls[-1]) == (128, 1)


def test_what_a_grid_does_not_hold_is_refused_by_name(calls):  # noqa: F811
    """More than 2^24 - 1 workgroups: the library's own answer would be its invalid argument."""
    for H, HQ, B, width, rows in ((1, 1, 1 << 24, 2, None), (2, 8, 1 << 23, 2, None), (64, 64, 1 << 18, 1, None), (1, 65, 1 << 23, 2, 4),
                                  (1, 1, 130, 400, 1 << 24), (1 << 16, 1 << 16, 1, 1, None)):
        c = cache(NP=1, H=H, page=32, D=64)
        T = B if rows is None else 9
        q = torch.zeros(1, 1, 64, dtype=torch.bfloat16).expand(T, HQ, 64)
        kw = {} if rows is None else dict(cu_q=torch.zeros(B + 1, dtype=torch.int32), max_q=rows)
        table = torch.zeros(B, width, dtype=torch.int32)
        with pytest.raises(ValueError, match="workgroups"):
            ops.kv4_attn(q, **c, table=table, lens=torch.zeros(B, dtype=torch.int32), out=torch.empty(T, HQ, 64, dtype=torch.bfloat16), **kw)
    assert not calls


def touched(t):
    """The addresses of a tensor's elements"""
    n = torch.zeros(t.shape, dtype=torch.int64)
    for d, (size, step) in enumerate(zip(t.shape, t.stride())):
        n += (torch.arange(size) * step).view(-1, *[1] * (t.dim() - 1 - d))
    return set((n * t.element_size() + t.data_ptr()).flatten().tolist())


def layouts(buf, r, T, H):
    """Rows (T, H, 64) somewhere in a buffer, each way that a caller lays them out"""
    D = 64
    gap = r.choice((0, 0, 8, 64))
    if r.random() < 0.7:
        s1 = r.choice((D, D, D + 8, 2 * D))
        s0 = s1 * (H - 1) + D + gap if r.random() < 0.5 else r.choice((384, 512))       # (a common distance: views of one product)
        s0 = max(s0, s1 * (H - 1) + D)
    else:
        s0 = r.choice((D, D + 8, 2 * D))
        s1 = max(s0 * (T - 1) + D + gap, r.choice((0, 512)))
    span = s0 * (T - 1) + s1 * (H - 1) + D
    at = 8 * r.randrange((buf.numel() - span) // 8 + 1) if r.random() < 0.5 else 64 * r.randrange((buf.numel() - span) // 64 + 1)
    return buf.as_strided((T, H, D), (s0, s1, 1), at)


@pytest.mark.parametrize("seed", range(4))
def test_outputs_over_rows_that_are_read(calls, seed):  # noqa: F811
    """An output that shares an element with rows that the call reads, or writes besides, is refused, one that lies between
    them is taken: by the elements' addresses."""
    r = random.Random(seed)
    buf = torch.zeros(4096, dtype=torch.bfloat16)
    buf = buf[(-buf.data_ptr() // 2) % 8:][:4000]                 # (16-byte aligned)
    c = cache(NP=2, H=1, page=32, D=64)
    seen = [0, 0]
    for _ in range(300):
        T, H, D = r.choice((1, 1, 2, 3, 5)), r.choice((1, 2, 3)), 64
        q, o = layouts(buf, r, T, H), layouts(buf, r, T, H)
        meet = bool(touched(q) & touched(o))
        if o.data_ptr() == q.data_ptr() and all(n == 1 or x == y for n, x, y in zip(q.shape, q.stride(), o.stride())):
            continue                                              # (in place)
        seen[meet] += 1
        tab, one, pos, cos = torch.zeros(T, 2, dtype=torch.int32), torch.zeros(T, dtype=torch.int32), torch.zeros(T, dtype=torch.int32), torch.zeros(9, 32)
        far = torch.zeros(T, H, D, dtype=torch.bfloat16)
        tries = [lambda: ops.kv4_attn(q, **c, table=tab, lens=one, out=o), lambda: ops.qk_norm_rope(q, far, pos, cos, cos, q_out=o),
                 lambda: ops.qk_norm_rope(far, q, pos, cos, cos, q_out=o), lambda: ops.qk_norm_rope(q, far, pos, cos, cos, k_out=o),
                 lambda: ops.qk_norm_rope(far, q, pos, cos, cos, k_out=o), lambda: ops.qk_norm_rope(far, far, pos, cos, cos, q_out=q, k_out=o)]
        for call in tries:
            n = len(calls)
            if meet:
                with pytest.raises(ValueError, match="share"):
                    call()
            else:
                call()
            assert len(calls) == n + (not meet)
    assert min(seen) > 50


def test_outputs_in_place_and_over_small_operands(calls):  # noqa: F811
    """Rows of one product turned in place, both or one of them, also in many tokens; not k's rows in q's place, nor rows over
    the tables, weights or positions."""
    for T in (1, 7, 3000):
        x = torch.zeros(T, 12 * 128, dtype=torch.bfloat16)
        q, k, v = x[:, :1024].view(T, 8, 128), x[:, 1024:1280].view(T, 2, 128), x[:, 1280:].view(T, 2, 128)
        a = rope_args(q=q, k=k, pos=torch.zeros(T, dtype=torch.int32))
        ops.qk_norm_rope(**a, q_out=q, k_out=k)
        ops.qk_norm_rope(**a, q_out=q)
        ops.qk_norm_rope(**a, k_out=v)
        n = len(calls)
        for bad in (dict(k_out=q[:, 6:]), dict(q_out=x[:, 256:1280].view(T, 8, 128)), dict(q_out=q, k_out=q[:, 2:4])):
            with pytest.raises(ValueError, match="share"):
                ops.qk_norm_rope(**a, **bad)
        with pytest.raises(ValueError, match="share"):            # k's rows are q's: both would be read after one is written
            ops.qk_norm_rope(**dict(a, k=q[:, :2]), q_out=q)
        assert len(calls) == n
    x = torch.zeros(5, 1024, dtype=torch.bfloat16).view(5, 8, 128)
    ops.qk_norm_rope(**rope_args(q=x, k=x[:, 3:3]), q_out=x)      # (rows of no head share nothing)
    ops.qk_norm_rope(**rope_args(q=x[2:2], k=x[3:3], pos=torch.zeros(0, dtype=torch.int32)), q_out=x[2:2], k_out=x[1:1])
    mem = torch.zeros(4096, dtype=torch.float32)
    out = mem.view(torch.bfloat16)[64:64 + 5 * 1024].view(5, 8, 128)
    for bad in (dict(wq=out[0, 0]), dict(wk=out[4, 7]), dict(cos=mem[:576].view(9, 64)), dict(sin=mem[:576].view(9, 64)),
                dict(pos=mem.view(torch.int32)[40:45])):
        with pytest.raises(ValueError, match="share"):
            ops.qk_norm_rope(**rope_args(**bad), q_out=out)
    ops.qk_norm_rope(**rope_args(pos=mem.view(torch.int32)[:5]), q_out=out)
    c = cache()
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(2048, dtype=torch.int32)
    o = i.view(torch.bfloat16)[64:64 + 3072].view(3, 8, 128)
    kw = dict(table=torch.zeros(3, 2, dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32), cu_q=torch.zeros(4, dtype=torch.int32))
    for bad in (dict(lens=i[40:43]), dict(cu_q=i[1560:1564]), dict(table=i[30:36].view(3, 2))):
        with pytest.raises(ValueError, match="share"):
            ops.kv4_attn(q, **c, **dict(kw, **bad), out=o)
    ops.kv4_attn(q, **c, **dict(kw, lens=i[:3], cu_q=i[1568:1572]), out=o)
