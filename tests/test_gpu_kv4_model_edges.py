"""The Llama-shaped model over a 4-bit paged cache at the cache's limits: its last positions, steps and prompts that are
refused."""
import pytest
import torch

from openattention_amd import KV4Cache
from openattention_amd.model import VOCAB, LlamaShaped
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import DEV, i32
from tests.test_gpu_kv4_model import model_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_a_refused_steps_token_is_taken_up_again(captured):
    """A step that lacks pages leaves the tokens where they were: the step after a request has ended gives the others
    what they would have got with pages enough."""
    B, T = 2, 31
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(6)).to(DEV)
    model, cache = model_of(B, T, 1, False)
    model.prefill(tokens)
    want = [model.step().clone() for _ in range(2)]
    model, cache = model_of(B, T, 1, False, pages=3)
    model.prefill(tokens)
    step = model.step
    if captured:
        state = [t.clone() for t in (cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], model.tok)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            model.step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            model.step()
        for t, u in zip((cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], model.tok), state):
            t.copy_(u)
        step = graph.replay
    step()
    assert torch.equal(model.tok, want[0])
    for _ in range(2):
        step()
        assert cache.lens.tolist() == [32, 32] and torch.equal(model.tok, want[0])
        with pytest.raises(RuntimeError, match="free pages"):
            cache.check()
    cache.truncate(i32([-1, 0]))
    step()
    cache.check()
    assert cache.lens.tolist() == [33, 1] and int(model.tok[0]) == int(want[1][0])


def test_steps_up_to_the_caches_last_token():
    """A cache's length is rounded up to whole pages: steps behind the length that was asked for are as good as those of a
    model made for all of them, and the first one past the pages is refused and changes nothing, the token included."""
    B, T, Lmax = 2, 120, 125
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(5)).to(DEV)
    took, rows = [], []
    for length in (Lmax, 128):
        cache = KV4Cache(B, length, DEV, page=32)
        model = LlamaShaped(B, length, DEV, layers=1, seed=3, cache=cache)
        took.append([model.prefill(tokens).clone()] + [model.step().clone() for _ in range(8)])
        cache.check()
        assert cache.lens.tolist() == [128, 128]
        rows.append(cache.read(0, ref.held(cache.table, [128, 128], 32)[1].int().to(DEV)))
        now = [t.clone() for t in (cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], model.tok)]
        model.step()
        assert all(torch.equal(a, b) for a, b in zip(now, (cache.lens, cache.table, cache.free, cache.nfree, *cache.rows[0], model.tok)))
        with pytest.raises(RuntimeError, match="max_len"):
            cache.check()
    assert all(torch.equal(a, b) for a, b in zip(*took))
    assert all(torch.equal(a, b) and not a.isnan().any() for a, b in zip(*rows))
    # a cache for more tokens than the model was made for
    cache = KV4Cache(B, 160, DEV, page=32)
    model = LlamaShaped(B, Lmax, DEV, layers=1, seed=3, cache=cache)
    assert torch.equal(model.prefill(tokens), took[0][0])
    for want in took[0][1:]:
        assert torch.equal(model.step(), want)
    model.step()
    cache.check()
    assert cache.lens.tolist() == [129, 129] and not cache.read(0, ref.held(cache.table, [129, 129], 32)[0].int().to(DEV))[0].isnan().any()


def test_prompts_that_do_not_fit_change_nothing():
    """Prompts for which the pool has too few pages, or that meet a refusal nobody has looked at, are refused as a whole:
    no request is extended, and the same prompts go through where they fit."""
    B, T = 3, 40
    tokens = torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(7)).to(DEV)
    model, cache = model_of(B, T, 1, False, pages=5)
    for _ in range(2):
        model.tok.fill_(11)
        with pytest.raises(RuntimeError, match="free pages"):
            model.prefill(tokens)
        assert cache.lens.tolist() == [0] * B and int(cache.nfree) == 5 and (cache.table == -1).all() and (model.tok == 11).all()
    first = model.prefill(tokens[:, :32]).clone()
    assert cache.lens.tolist() == [32] * B and int(cache.nfree) == 2
    cache.truncate(i32([0] * B))
    cache.extend(i32([999, 0, 0]), 999)                       # refused
    with pytest.raises(RuntimeError, match="max_len"):
        model.prefill(tokens[:, :32])
    assert cache.lens.tolist() == [0] * B and int(cache.nfree) == 5
    assert torch.equal(model.prefill(tokens[:, :32]), first)
