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
