"""The Llama-shaped model over an 8-bit paged cache, read whole or by blocks: prompts, captured decode steps, refused
ones, drafts taken back; and the operators as a run of calls on streams, in graphs and by plans kept from call to call."""
import pytest
import torch

from openattention_amd import KV8Cache, ops
from openattention_amd.method import C as CTX
from openattention_amd.model import D, HKV, HQ, VOCAB, LlamaShaped
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import check_attn, filled, gen, i32, randn, starts, values_of, want_attn, want_select

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def state_of(cache, model=None):
    return [cache.lens, cache.table, cache.free, cache.nfree, *(t for r in cache.rows for t in r), *cache.bounds] + ([model.tok] if model else [])


@pytest.mark.parametrize("qk_norm,blocks", [(False, None), (True, None), (True, 4)])
def test_decode_over_the_cache(qk_norm, blocks):
    """After a prompt the next tokens are those of the dense model (whose prompt attention is the same); then decode
    steps, eagerly and as one captured step replayed over page borders, give the same tokens and the same cache, and an eager
    step's attention is that of the values which the cache holds, in the blocks that its bounds name."""
    print(f"[case] model over an 8-bit cache, qk_norm={qk_norm} blocks={blocks}", flush=True)
    B, T, layers, steps, page = 3, 190, 2, 40, 32
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    cache = KV8Cache(B, T + 64, DEV, layers=layers, page=page)
    model = LlamaShaped(B, T + 64, DEV, layers=layers, seed=3, cache=cache, qk_norm=qk_norm, blocks=blocks)
    first = model.prefill(tokens).clone()
    if qk_norm:
        dense = LlamaShaped(B, T + 64, DEV, layers=layers, seed=3, qk_norm=qk_norm)
        CTX.K = [torch.zeros(B, HKV, T + 64, D, device=DEV, dtype=BF) for _ in range(layers)]
        CTX.V = [torch.zeros_like(k) for k in CTX.K]
        assert torch.equal(first, dense.prefill(tokens))
        CTX.K, CTX.V = [], []
    assert cache.lens.tolist() == [T] * B
    now = state_of(cache, model)
    state = [t.clone() for t in now]

    def restore():
        for t, s in zip(now, state):
            t.copy_(s)

    eager = [model.step().clone() for _ in range(steps)]
    cache.check()
    after = [t.clone() for t in now]
    assert cache.lens.tolist() == [T + steps] * B
    # an eager step's attention, layer by layer
    seen = []
    attend = cache.attend
    cache.attend = lambda l, q, *a, **kw: seen.append((l, q.clone(), attend(l, q, *a, **kw), kw.get("blocks"))) or seen[-1][2]
    model.step()
    cache.attend = attend
    lens, cu = cache.lens.tolist(), list(range(B + 1))
    assert len(seen) == layers
    for l, q, out, chosen in seen:
        held = [*cache.rows[l], cache.bounds[l]]
        if blocks:
            assert torch.equal(chosen.cpu(), want_select(q, held, cache.table, lens, cu, page, blocks, 1, 2))
        check_attn(out, *want_attn(q, held, cache.table, lens, cu, D ** -0.5, page, chosen))
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


def test_refused_steps_write_nothing():
    """A pool with less than all requests could take: a step past it is refused and changes nothing, the newest rows among
    it, and goes through after one request has ended."""
    B, T = 2, 40
    cache = KV8Cache(B, T + 64, DEV, page=32, pages=4)
    model = LlamaShaped(B, T + 64, DEV, layers=1, seed=3, cache=cache, blocks=3)
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(2)).to(DEV)
    model.prefill(tokens)
    for _ in range(24):
        model.step()
    cache.check()
    assert cache.lens.tolist() == [64, 64] and int(cache.nfree) == 0
    keep = [t.clone() for t in state_of(cache, model)]
    model.step()
    assert all(torch.equal(a, b) for a, b in zip(keep, state_of(cache, model)))
    with pytest.raises(RuntimeError, match="KV8Cache: refused: too few free pages"):
        cache.check()
    cache.truncate(i32([0, -1]))
    model.step()
    cache.check()
    assert cache.lens.tolist() == [1, 65] and int(cache.nfree) == 0
    with pytest.raises(ValueError, match="empty"):
        model.prefill(tokens)
    for bad in (dict(blocks=2, cache=cache), dict(blocks=4)):
        with pytest.raises(ValueError):
            LlamaShaped(B, 64, DEV, layers=1, **bad)
    for bad in (dict(page=256), dict(page=16), dict(head_dim=96), dict(max_len=0)):
        with pytest.raises(ValueError):
            KV8Cache(**dict(dict(B=2, max_len=64, dev=DEV), **bad))


def test_drafts_taken_back():
    """Drafts written, attended to at once and taken back, others in their place: what the cache holds, and the attention
    of it, follow the definition all along."""
    B, page, R = 3, 32, 5
    g = gen(4)
    cache = KV8Cache(B, 200, DEV, page=page, kv_heads=2, head_dim=64)
    x = lambda n, h: torch.randn(n, h, 64, generator=g, device=DEV).to(BF)  # noqa: E731
    held = [t.cpu() for t in (*cache.rows[0], cache.bounds[0])]
    for it, (add, keep) in enumerate((([50, 61, 30], None), ([R] * 3, [51, 61, 35]), ([R, 1, R], [52, 62, 0]), ([3, 3, 33], [-1, 60, 33]), ([R, 2, 4], None))):
        T = sum(add)
        slots, pos, cu = cache.extend(i32(add), T)
        k, v, q = x(T, 2) * (1 + it), x(T, 2), x(T, 8)
        cache.write(0, k, v, cu)
        lens = cache.lens.tolist()
        for b in range(B):
            at = slice(int(cu[b]), int(cu[b + 1]))
            ref.write(held[0], held[1], held[4], k[at].cpu(), cache.table[b].cpu(), lens[b], page)
            ref.write(held[2], held[3], None, v[at].cpu(), cache.table[b].cpu(), lens[b], page)
        now = [*cache.rows[0], cache.bounds[0]]
        assert all(torch.equal(a.cpu(), b) for a, b in zip(now, held))
        blocks = cache.select(0, q, 3, cu)
        for bl in (None, blocks):
            out = cache.attend(0, q, cu, max(add), blocks=bl)
            check_attn(out, *want_attn(q, now, cache.table, lens, cu.tolist(), 0.125, page, bl))
        kk, vv = cache.read(0, slots, torch.float32)
        assert torch.equal(kk.double(), ref.rows_at(now[0], now[1], slots)) and torch.equal(vv.double(), ref.rows_at(now[2], now[3], slots))
        if keep:
            cache.truncate(i32(keep))
    cache.check()


def test_calls_on_streams_and_in_graphs():
    """The same calls on two streams at once and as two captured graphs that share their inputs, replayed in turn with
    eager work between them, give what they give alone."""
    g = gen(31)
    page, lens, rows = 32, [900, 333, 64], [3, 1, 2]
    cache, table = filled(lens, 2, 128, page, g)
    n, cu = i32(lens), i32(starts(rows))
    q = randn(g, 6, 8, 128, dtype=BF)
    x = randn(g, 6, 2, 128, dtype=BF)
    side = [t.clone() for t in cache]

    def calls(q):
        ops.kv8_write(x, x, *side, table, n, cu)
        blocks = ops.kv8_select(q, cache[1], cache[4], table, n, page, 5, cu)
        return (blocks, ops.kv8_attn(q, *cache[:4], table, n, cu_q=cu, max_q=3, blocks=blocks), ops.kv8_attn(q, *cache[:4], table, n, cu_q=cu, max_q=3),
                *ops.kv8_read(i32([5, 700, -1]), *side[:4]))

    want = [t.clone() for t in calls(q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(calls(q))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for o in got:
            assert all(torch.equal(a, b) for a, b in zip(o, want))
    graphs, outs, inputs = [], [], [q.clone(), q.clone()]
    slots = i32([5, 700, -1])
    for y in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            blocks = ops.kv8_select(y, cache[1], cache[4], table, n, page, 5, cu)
            outs.append((blocks, ops.kv8_attn(y, *cache[:4], table, n, cu_q=cu, max_q=3, blocks=blocks),
                         ops.kv8_attn(y, *cache[:4], table, n, cu_q=cu, max_q=3), *ops.kv8_read(slots, *side[:4])))
        graphs.append(graph)
    for it in range(4):
        inputs[1].copy_(q * (1 + it))
        fresh = [t.clone() for t in calls(inputs[1])]
        for i in (1, 0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[0], want))
        assert all(torch.equal(a, b) for a, b in zip(outs[1], fresh))
    # lengths and lists that change between replays
    lens2 = [1, 333, 40]
    n.copy_(i32(lens2))
    for gph in graphs:
        gph.replay()
    inputs[1].copy_(q)
    graphs[1].replay()
    check_attn(outs[1][2], *want_attn(q, cache, table, lens2, starts(rows), 128 ** -0.5, page))
    assert torch.equal(outs[1][0].cpu(), want_select(q, cache, table, lens2, starts(rows), page, 5, 1, 2))


def test_kept_plans_look_at_every_call(monkeypatch):
    """A call of sizes seen before is made from what is kept, and still refuses what it refused, takes numbers by value,
    follows new pointers and another rule for pieces, and leaves the unusual to Python."""
    g = gen(8)
    page, lens = 32, [700, 90]
    cache, table = filled(lens, 2, 128, page, g)
    n = i32(lens)
    q = randn(g, 2, 8, 128, dtype=BF)
    want = ops.kv8_attn(q, *cache[:4], table, n)
    ran = []
    run = ops._run
    monkeypatch.setattr(ops, "_run", lambda *a: ran.append(a[1]) or run(*a))
    for _ in range(3):
        assert torch.equal(ops.kv8_attn(q, *cache[:4], table, n), want)
    q2 = randn(g, 2, 8, 128, dtype=BF)
    check_attn(ops.kv8_attn(q2, *cache[:4], table, n), *want_attn(q2, cache, table, lens, [0, 1, 2], 128 ** -0.5, page))
    assert not ran                                          # (all of these by the plan of the first)
    wide = torch.zeros(2, 8, 136, device=DEV, dtype=BF)
    wide[..., :128], wide[..., 4:132] = q, q
    off = torch.cat([torch.zeros(1, device=DEV, dtype=BF), q.flatten()])[1:].view(2, 8, 128)
    for bad in (off, q.clone().requires_grad_()):
        with pytest.raises(ValueError):
            ops.kv8_attn(bad, *cache[:4], table, n)
    with torch.no_grad():
        assert torch.equal(ops.kv8_attn(q.clone().requires_grad_(), *cache[:4], table, n), want)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.kv8_attn(q, *cache[:4], table.cpu(), n)
    with pytest.raises(TypeError):
        ops.kv8_attn(q, *cache[:4], table, n, max_q=1.0)
    assert torch.equal(ops.kv8_attn(torch.nn.Parameter(q, requires_grad=False), *cache[:4], table, n), want)
    out = torch.full_like(q, 3.0)
    assert ops.kv8_attn(q, *cache[:4], table, n, out=out) is out and torch.equal(out, want)
    scale = torch.tensor(0.5)
    for s in (0.5, 0.25, 0.25):
        scale.fill_(s)
        a, b = ops.kv8_attn(q, *cache[:4], table, n, scale), ops.kv8_attn(q, *cache[:4], table, n, s)
        assert torch.equal(a, b)
        check_attn(a, *want_attn(q, cache, table, lens, [0, 1, 2], s, page))
    # another rule for pieces, and one that takes its place in memory
    for size in (128, 256, 128):
        seen = []
        monkeypatch.setattr(ops, "kv8_chunk", lambda cap, units, rows, listed, size=size: seen.append(size) or size)
        check_attn(ops.kv8_attn(q, *cache[:4], table, n), *want_attn(q, cache, table, lens, [0, 1, 2], 128 ** -0.5, page))
        assert seen == [size]
    # rows, lists and caches of other types, sizes and strides
    monkeypatch.undo()
    for y in (q.half(), wide[..., :128], q):
        check_attn(ops.kv8_attn(y, *cache[:4], table, n), *want_attn(y, cache, table, lens, [0, 1, 2], 128 ** -0.5, page))
    sel = ops.kv8_select(q, cache[1], cache[4], table, n, page, 4)
    assert torch.equal(ops.kv8_select(q, cache[1], cache[4], table, n, page, 4), sel)
    assert ops.kv8_select(q, cache[1], cache[4], table, n, page, 5).shape == (2, 2, 5)
    assert (ops.kv8_select(q, cache[1], cache[4], table, n, page, 4, max_len=90)[0] == -1).all()
    assert torch.equal(ops.kv8_select(q, cache[1], cache[4], table, n, page, 4, max_len=704), sel)
    slots = table[0, :2] * page + 3
    for dt in (BF, torch.float32, BF):
        k, v = ops.kv8_read(slots, *cache[:4], dtype=dt)
        assert k.dtype == v.dtype == dt
        assert torch.equal(k.double(), ref.rows_at(cache[0], cache[1], slots)) and torch.equal(v.double(), ref.rows_at(cache[2], cache[3], slots))
    with pytest.raises(ValueError):
        ops.kv8_read(slots, *cache[:4], dtype=torch.float16)
    x = randn(g, 2, 2, 128, dtype=BF)
    keep = [t.clone() for t in cache]
    for _ in range(2):
        for t, s in zip(cache, keep):
            t.copy_(s)
        ops.kv8_write(x, x, *cache, table, n)
        newest = i32([int(table[b, (m - 1) // page]) * page + (m - 1) % page for b, m in enumerate(lens)])
        v = ops.kv8_read(newest, *cache[:4])[1]
        assert ((v.float() - x.float()).abs() <= 2.0 ** -4 * x.float().abs() + 2.0 ** -9).all()
    bad = x.clone().requires_grad_()
    with pytest.raises(ValueError):
        ops.kv8_write(bad, x, *cache, table, n)
    assert values_of(cache, table, lens, page)[0][0].shape == (700, 2, 128)


def test_calls_of_two_threads():
    """Calls of two host threads at once, each on a stream and a cache of its own, by plans that both keep."""
    import threading
    g = gen(9)
    page, lens = 32, [300, 64]
    work, errors = [], []
    for _ in range(2):
        cache, table = filled(lens, 2, 128, page, g)
        work.append((cache, table, i32(lens), randn(g, 2, 8, 128, dtype=BF), torch.cuda.Stream()))

    def run(cache, table, n, q, stream, times):
        outs = []
        with torch.cuda.stream(stream):
            for i in range(times):
                blocks = ops.kv8_select(q, cache[1], cache[4], table, n, page, 4 + i % 3)
                outs.append(ops.kv8_attn(q, *cache[:4], table, n, blocks=blocks, sm_scale=0.05 + 0.01 * (i % 5)))
        stream.synchronize()
        return outs

    torch.cuda.synchronize()
    want = [run(*w, 15) for w in work]
    got = [None, None]

    def thread(i):
        try:
            got[i] = run(*work[i], 60)
        except Exception as e:                              # (said by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, o in zip(want, got):
        assert len(o) == 60 and all(torch.equal(x, w[i % 15]) for i, x in enumerate(o))
