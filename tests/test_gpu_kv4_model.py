"""The Llama-shaped model over a 4-bit paged cache: prompts, captured decode steps, drafts taken back."""
import pytest
import torch

from openattention_amd import KV4Cache
from openattention_amd.method import C as CTX
from openattention_amd.model import D, HKV, HQ, VOCAB, LlamaShaped
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import check_attn, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model_of(B, T, layers, qk_norm, page=32, extra=64, pages=None):
    cache = KV4Cache(B, T + extra, DEV, layers=layers, page=page, pages=pages)
    return LlamaShaped(B, T + extra, DEV, layers=layers, seed=3, cache=cache, qk_norm=qk_norm), cache


@pytest.mark.parametrize("qk_norm", [False, True])
def test_decode_over_the_cache(qk_norm):
    """After a prompt the next tokens are those of the dense model (whose prompt attention is the same); then
    30 decode steps, eagerly and as one captured step replayed over page borders, give the same tokens and the
    same cache, and an eager step's attention is that of the values which the cache holds."""
    print(f"[case] model over a 4-bit cache, qk_norm={qk_norm}", flush=True)
    B, T, layers, steps = 3, 61, 2, 30
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    model, cache = model_of(B, T, layers, qk_norm)
    first = model.prefill(tokens).clone()
    dense = LlamaShaped(B, T + 64, DEV, layers=layers, seed=3, qk_norm=qk_norm)
    CTX.K = [torch.zeros(B, HKV, T + 64, D, device=DEV, dtype=torch.bfloat16) for _ in range(layers)]
    CTX.V = [torch.zeros_like(k) for k in CTX.K]
    if qk_norm:                                             # (otherwise the dense model turns its rows step by step)
        assert torch.equal(first, dense.prefill(tokens))
        n = CTX.n_dev = i32([T + 1])
        dense.step(T + 1)
        assert int(n) == T + 1 and dense.tok.shape == (B,)
    assert cache.lens.tolist() == [T] * B
    state = [t.clone() for t in (cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], *cache.rows[1], model.tok)]
    now = (cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], *cache.rows[1], model.tok)

    def restore():
        for t, s in zip(now, state):
            t.copy_(s)

    eager = []
    for i in range(steps):
        eager.append(model.step().clone())
    cache.check()
    after = [t.clone() for t in now]
    assert cache.lens.tolist() == [T + steps] * B
    # an eager step's attention, layer by layer
    seen = []
    attend = cache.attend
    cache.attend = lambda l, q, *a, **kw: seen.append((l, q.clone(), attend(l, q, *a, **kw))) or seen[-1][2]
    model.step()
    cache.attend = attend
    for l, q, out in seen:
        for b, slots in enumerate(ref.held(cache.table, cache.lens.tolist(), cache.page)):
            k, v = cache.read(l, slots.int().to(DEV), dtype=torch.float32)
            check_attn(out[b:b + 1], *ref.attn(q[b:b + 1], k.double(), v.double(), T + steps + 1, D ** -0.5))
    restore()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        model.step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step()
    restore()
    for i in range(steps):
        graph.replay()
        assert torch.equal(model.tok, eager[i]), i
    assert all(torch.equal(a, b) for a, b in zip(now, after))
    CTX.K, CTX.V = [], []


def test_requests_end_and_pages_return():
    """A pool with less than all requests could take: a step past it is refused and changes nothing, and goes
    through after one request has ended; a prompt over requests that are not empty is refused."""
    B, T = 2, 40
    model, cache = model_of(B, T, 1, False, pages=4, extra=64)
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(2)).to(DEV)
    model.prefill(tokens)
    for _ in range(24):
        model.step()
    cache.check()
    assert cache.lens.tolist() == [64, 64] and int(cache.nfree) == 0
    table = cache.table.clone()
    model.step()
    assert cache.lens.tolist() == [64, 64] and torch.equal(cache.table, table)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    cache.check()
    cache.truncate(i32([0, -1]))
    assert cache.lens.tolist() == [0, 64] and int(cache.nfree) == 2
    model.step()
    cache.check()
    assert cache.lens.tolist() == [1, 65] and int(cache.nfree) == 0
    with pytest.raises(ValueError, match="empty"):
        model.prefill(tokens)
    with pytest.raises(ValueError):
        LlamaShaped(3, 64, DEV, layers=1, cache=cache)


def test_draft_tokens_checked_at_once():
    """Five tokens of every request at once give, row by row, what five single steps give up to rounding, and
    taken back leave the cache as it was."""
    B, T, R = 2, 50, 5
    g = torch.Generator(device=DEV).manual_seed(4)
    cache = KV4Cache(B, 96, DEV, page=32)
    x = lambda n, h: torch.randn(n, h, D, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    slots, pos, cu = cache.extend(i32([T, T - 7]), 2 * T - 7)
    cache.write(0, x(2 * T - 7, HKV), x(2 * T - 7, HKV), slots)
    before = [t.clone() for t in (cache.lens, cache.table, cache.free, cache.nfree)]
    q, k, v = x(B * R, HQ), x(B * R, HKV), x(B * R, HKV)
    one = []
    for j in range(R):
        at = torch.tensor([j, R + j], device=DEV)
        s1, _, _ = cache.extend()
        cache.write(0, k[at], v[at], s1)
        one.append(cache.attend(0, q[at]))
    cache.truncate(i32([T, T - 7]))
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.lens, cache.table, cache.free, cache.nfree)))
    s2, p2, cu = cache.extend(i32([R, R]), B * R)
    assert p2.tolist() == list(range(T, T + R)) + list(range(T - 7, T - 7 + R))
    cache.write(0, k, v, s2)
    out = cache.attend(0, q, cu, R)
    cache.check()
    for j in range(R):
        got, want = out[[j, R + j]].float(), one[j].float()
        # (both are within rounding of the same sums: at most one step of bf16 apart)
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs().clamp(min=2.0 ** -8)).all()
