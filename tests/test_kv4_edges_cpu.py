"""What the operators of the 4-bit paged cache hand to the library, and refuse, where their first tests do not look (CPU
tensors stand in for device ones; the launch is recorded instead)."""
import pytest
import torch

from openattention_amd import lib, ops
from tests.test_gpu_kv4 import CASES
from tests.test_kv4_cpu import cache, calls  # noqa: F401


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
