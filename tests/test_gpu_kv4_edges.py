"""The 4-bit paged cache on the GPU where its first tests do not reach: values that are not finite among keys that every
row sees, truncations that are refused, very many sequences, outputs among their inputs."""
import math

import pytest
import torch

from openattention_amd import ops
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import DEV, check_attn, gen, i32, new_cache, paged, randn, starts, want_attn

pytestmark = pytest.mark.gpu


# 380 keys are one piece of the many-row kernel's, 900 three; 40 tokens of 4 query heads are 160 rows (two workgroups),
# 17 are 68 (one, most of whose waves have no row), 16 are 64: the other kernel
@pytest.mark.parametrize("rows", [16, 17, 40])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [380, 900])
def test_a_value_that_every_row_sees_and_is_not_finite(rows, D, n):
    """It makes NaN of its block of 32 dims in every row, in the first tile and in a later one, of one block or of a whole
    tile's, whatever codes lie under the scale of NaN; the other blocks, heads and sequences keep their numbers."""
    print(f"[case] NaN values: {rows} tokens, D {D}, {n} keys", flush=True)
    g = gen(n + rows)
    lens, page, HKV = [n] * 4, 32, 2
    cache, table = paged(lens, HKV, D, page, g)
    held = ref.held(table, lens, page)

    def put(b, keys, head, dim, value):
        k, v = randn(g, len(keys), HKV, D), randn(g, len(keys), HKV, D)
        v[:, head, dim] = value
        ops.kv4_write(k, v, held[b][keys].int().to(DEV), *cache)
    put(0, [3], 1, 40, math.nan)                              # the first tile
    put(1, [n // 2], 0, D - 1, math.inf)                      # a tile in the middle
    put(2, list(range(32)), 1, 1, -math.inf)                  # a whole tile, the first one
    put(3, [n // 2 + 1], 0, 5, math.nan)                      # beside a value that fp16 does not hold by the others' scale
    put(3, [9, 11], 0, D - 2, 2.0 ** 40)
    at = int(held[2][n // 2])                                 # codes that are not 0 under NaN's scale
    cache[3][at // page, 0, at % page, 1] = 255
    assert (cache[2][at // page, 0, at % page, 16:32] & 0x77 != 0).any()
    cu = starts([rows] * 4)
    q = randn(g, cu[-1], 8, D, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32(cu), max_q=rows)
    want, err = want_attn(q, cache, table, lens, cu, D ** -0.5, page)
    blocks = want.isnan().view(4, rows, HKV, 4, D // 32, 32)
    there = torch.zeros(4, 1, HKV, 1, D // 32, 1, dtype=torch.bool, device=DEV)
    there[0, :, 1, :, 1], there[1, :, 0, :, -1], there[2, :, 1, :, 0], there[2, :, 0, :, 1] = True, True, True, True
    there[3, :, 0, :, 0] = True
    assert torch.equal(blocks, there.expand_as(blocks))
    check_attn(out, want, err)


@pytest.mark.parametrize("B", [3, 40, 300, 1100])
@pytest.mark.parametrize("wrong", [-5, 129, 1 << 30])
def test_truncation_of_a_length_outside_of_the_row(B, wrong):
    """It is refused as an extension is: the status says so, and nothing changes for any request, also not a length
    that is to be kept as it is."""
    g = gen(B)
    table = torch.randperm(4 * B, generator=g, device=DEV).int().view(B, 4)
    lens = torch.randint(0, 129, (B,), generator=g, device=DEV, dtype=torch.int32)
    lens[B // 2] = wrong
    for keep in (torch.full_like(lens, -1), torch.zeros_like(lens), lens // 2):
        st = [lens.clone(), table.clone(), torch.full((8 * B,), 9, device=DEV, dtype=torch.int32), i32([B]), i32([8])]
        before = [t.clone() for t in st]
        ops.kv_pages_truncate(keep, *st, 32)
        assert int(st[4]) == 8 | 1
        assert all(torch.equal(a, b) for a, b in zip(st[:4], before[:4]))
    # too many pages for the stack as well
    st = [torch.where(lens == wrong, wrong, 128).int(), table.clone(), torch.full((B,), 9, device=DEV, dtype=torch.int32), i32([B]), i32([0])]
    ops.kv_pages_truncate(torch.zeros_like(lens), *st, 32)
    assert int(st[4]) == 3 and torch.equal(st[1], table) and int(st[3]) == B


def test_attention_of_more_sequences_than_a_grids_axis_holds():
    """65537 sequences in a table whose width alone would cut each into pieces."""
    g = gen(65)
    B, HQ, D, page, NP = 65537, 2, 64, 32, 300
    cache = new_cache(NP, 1, page, D, g=g)
    for slots in torch.arange(NP * page, device=DEV, dtype=torch.int32).split(4096):
        ops.kv4_write(randn(g, slots.numel(), 1, D), randn(g, slots.numel(), 1, D), slots, *cache)
    table = torch.randint(0, NP, (B, 40), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.randint(0, 90, (B,), generator=g, device=DEV, dtype=torch.int32)
    some = [0, 1, 77, 32768, 65534, 65535, 65536]
    lens[some] = i32([1280, 0, 1100, 33, 700, 1, 1280])
    q = randn(g, B, HQ, D, dtype=torch.bfloat16)
    out = ops.kv4_attn(q, *cache, table, lens)
    at = torch.tensor(some, device=DEV)
    check_attn(out[at], *want_attn(q[at], cache, table[at], lens[at].tolist(), list(range(len(some) + 1)), D ** -0.5, page))
    # and the others as they are in a batch of their own
    assert torch.equal(out[1000:9000], ops.kv4_attn(q[1000:9000], *cache, table[1000:9000], lens[1000:9000], max_len=96))


@pytest.mark.parametrize("T", [1, 33, 3001])
def test_outputs_beside_their_inputs_in_one_product(T):
    """Rows of a product turned in place, and attention written between the rows of its queries, give what outputs of
    their own get; the product's other columns stay as they were."""
    g = gen(T)
    HQ, HKV, D, page = 8, 2, 128, 32
    x = randn(g, T, (2 * HQ + 2 * HKV) * D, dtype=torch.bfloat16)
    q, free, k, v = (t.unflatten(1, (-1, D)) for t in x.split([HQ * D, HQ * D, HKV * D, HKV * D], 1))
    a = torch.arange(T, dtype=torch.float64)[:, None] * 0.7 ** torch.arange(D // 2, dtype=torch.float64)
    cos, sin, pos = a.cos().float().to(DEV), a.sin().float().to(DEV), torch.arange(T, device=DEV)
    w = randn(g, D, dtype=torch.bfloat16)
    keep = x.clone()
    want = ops.qk_norm_rope(q, k, pos, cos, sin, w, w)
    ops.qk_norm_rope(q, k, pos, cos, sin, w, w, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    q.copy_(want[0])
    lens = [T + 70]
    cache, table = paged(lens, HKV, D, page, g)
    want = ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32([0, T]), max_q=T)
    was = q.clone()
    ops.kv4_attn(q, *cache, table, i32(lens), cu_q=i32([0, T]), max_q=T, out=free)
    assert torch.equal(free, want) and not want.isnan().any() and torch.equal(q, was)
    assert torch.equal(v, keep.view(T, -1, D)[:, 2 * HQ + HKV:])
