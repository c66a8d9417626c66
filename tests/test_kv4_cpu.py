"""What the operators of the 4-bit paged cache refuse on the host, before anything is launched, and what they
hand to the library (CPU tensors stand in for device ones; the launch is recorded instead)."""
import pytest
import torch

from openattention_amd import lib, ops


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(ops, "_where", lambda *ts: 0)
    monkeypatch.setattr(ops, "_run", lambda i, name, *a: got.append((name, a)))
    return got


def rope_args(**kw):
    a = dict(q=torch.zeros(5, 8, 128, dtype=torch.bfloat16), k=torch.zeros(5, 2, 128, dtype=torch.bfloat16),
             pos=torch.zeros(5, dtype=torch.int32), cos=torch.zeros(9, 64), sin=torch.zeros(9, 64), wq=None, wk=None, eps=1e-6)
    a.update(kw)
    return a


ROPE_BAD = [
    dict(q=torch.zeros(5, 8, 128)), dict(q=torch.zeros(5, 8, 96, dtype=torch.bfloat16), k=torch.zeros(5, 2, 96, dtype=torch.bfloat16)),
    dict(q=torch.zeros(4, 8, 128, dtype=torch.bfloat16)), dict(q=torch.zeros(5, 1024, dtype=torch.bfloat16)),
    dict(q=torch.zeros(5, 8, 128, dtype=torch.int16), k=torch.zeros(5, 2, 128, dtype=torch.int16)),
    dict(q=torch.zeros(5, 8, 129, dtype=torch.bfloat16)[..., :128]), dict(q=torch.zeros(5 * 8 * 128 + 8, dtype=torch.bfloat16)[1:5121].view(5, 8, 128)),
    dict(q=torch.zeros(5, 128, 8, dtype=torch.bfloat16).transpose(1, 2)), dict(pos=torch.zeros(5)), dict(pos=torch.zeros(4, dtype=torch.int32)),
    dict(pos=torch.zeros(10, dtype=torch.int32)[::2]), dict(cos=torch.zeros(9, 128)), dict(cos=torch.zeros(8, 64)),
    dict(cos=torch.zeros(9, 64, dtype=torch.float64)), dict(sin=torch.zeros(9, 128)[:, :64]), dict(cos=torch.zeros(0, 64), sin=torch.zeros(0, 64)),
    dict(cos=torch.zeros(9, 66)[:, :64], sin=torch.zeros(9, 66)[:, :64]), dict(wq=torch.zeros(128)), dict(wk=torch.zeros(64, dtype=torch.bfloat16)),
    dict(wk=torch.zeros(256, dtype=torch.bfloat16)[::2]), dict(wq=torch.zeros(129, dtype=torch.bfloat16)[1:]), dict(eps=-1.0), dict(eps=float("nan")),
    dict(q_out=torch.zeros(5, 8, 128)), dict(k_out=torch.zeros(5, 3, 128, dtype=torch.bfloat16)),
    dict(q_out=torch.zeros(5, 1, 128, dtype=torch.bfloat16).expand(5, 8, 128)), dict(q_out=torch.zeros(1, 8, 128, dtype=torch.bfloat16).expand(5, 8, 128)),
    dict(q_out=torch.zeros(4000, dtype=torch.bfloat16).as_strided((5, 8, 128), (512, 128, 1))),
    dict(q=torch.zeros(5, 8, 128, dtype=torch.bfloat16, requires_grad=True)), dict(wk=torch.zeros(128, dtype=torch.bfloat16, requires_grad=True)),
    dict(cos=torch.zeros(9, 64, dtype=torch.complex64).conj().imag, sin=torch.zeros(9, 64, dtype=torch.complex64).conj().imag)]


@pytest.mark.parametrize("bad", range(len(ROPE_BAD)))
def test_rope_refuses(calls, bad):
    with pytest.raises(ValueError):
        ops.qk_norm_rope(**rope_args(**ROPE_BAD[bad]))
    assert not calls


def test_rope_hands_on_strides(calls):
    x = torch.zeros(5, 12 * 128, dtype=torch.bfloat16)
    q, k = x[:, :1024].view(5, 8, 128), x[:, 1024:1280].view(5, 2, 128)
    w = torch.zeros(128, dtype=torch.bfloat16, requires_grad=True)
    with torch.no_grad():
        a, b = ops.qk_norm_rope(**rope_args(q=q, k=k, wq=w, pos=torch.zeros(5, dtype=torch.int64)))
    (name, c), = calls
    assert name == "oa_qk_norm_rope" and len(c) + 1 == len(lib.SIGNATURES[name])
    assert c[:6] == (q.data_ptr(), 1536, 128, k.data_ptr(), 1536, 128) and c[6:11] == (5, 8, 2, 128, 0) and c[12] == 1
    assert c[15:20] == (64, 9, w.data_ptr(), None, 1e-6) and c[20:] == (a.data_ptr(), 1024, 128, b.data_ptr(), 256, 128)
    # one token: its stride may be anything
    one = torch.zeros(3, 4, 128, dtype=torch.bfloat16).as_strided((1, 4, 128), (3, 128, 1))
    ops.qk_norm_rope(one, one[:, :0], torch.zeros(1, dtype=torch.int32), torch.zeros(9, 64), torch.zeros(9, 64))
    assert calls[1][1][1] == 0


def pool(B=3, width=4, NP=9):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return dict(lens=z(B), table=z(B, width), free=z(NP), nfree=z(1), status=z(1), page=64)


PAGES_BAD = [dict(lens=torch.zeros(4, dtype=torch.int32)), dict(lens=torch.zeros(3)), dict(lens=torch.zeros(6, dtype=torch.int32)[::2]),
             dict(table=torch.zeros(12, dtype=torch.int32)), dict(table=torch.zeros(3, 4, dtype=torch.int64)),
             dict(table=torch.zeros(4, 3, dtype=torch.int32).t()), dict(table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)),
             dict(table=torch.zeros(3, 0, dtype=torch.int32)), dict(table=torch.zeros(0, 4, dtype=torch.int32), lens=torch.zeros(0, dtype=torch.int32)),
             dict(free=torch.zeros(9)), dict(free=torch.zeros(0, dtype=torch.int32)), dict(free=torch.zeros(3, 3, dtype=torch.int32)),
             dict(nfree=torch.zeros(2, dtype=torch.int32)), dict(status=torch.zeros((), dtype=torch.int32)), dict(page=48), dict(page=16), dict(page=2048),
             dict(page=0), dict(add=torch.zeros(2, dtype=torch.int32)), dict(add=torch.zeros(3, dtype=torch.int64)),
             dict(free=torch.zeros(1, dtype=torch.int32).expand(1 << 26))]


@pytest.mark.parametrize("bad", range(len(PAGES_BAD)))
def test_pages_refuse(calls, bad):
    a = dict(pool(), add=torch.zeros(3, dtype=torch.int32), **{})
    a.update(PAGES_BAD[bad])
    with pytest.raises(ValueError):
        ops.kv_pages_extend(**a, total=3)
    a["keep"] = a.pop("add")
    with pytest.raises(ValueError):
        ops.kv_pages_truncate(**a)
    assert not calls


def test_pages_hand_on_their_buffers(calls):
    a = pool()
    with pytest.raises(ValueError):
        ops.kv_pages_extend(torch.zeros(3, dtype=torch.int32), **a, total=-1)
    slots, pos, cu = ops.kv_pages_extend(torch.zeros(3, dtype=torch.int32), **a, total=7)
    (name, c), = calls
    assert len(c) + 1 == len(lib.SIGNATURES[name]) and c[12:] == (slots.data_ptr(), pos.data_ptr(), cu.data_ptr(), None)
    assert slots.shape == pos.shape == (7,) and cu.shape == (4,)
    ops.kv_pages_truncate(torch.zeros(3, dtype=torch.int32), **a)
    assert len(calls[1][1]) + 1 == len(lib.SIGNATURES["oa_kv_pages_truncate"]) and calls[1][1][-1] is None
    # scratch where a second launch needs it
    ops.kv_pages_extend(torch.zeros(3, dtype=torch.int32), **a, total=2049)
    many = pool(B=1025)
    ops.kv_pages_extend(torch.zeros(1025, dtype=torch.int32), **many, total=7)
    ops.kv_pages_truncate(torch.zeros(1025, dtype=torch.int32), **many)
    assert all(c[1][-1] is not None for c in calls[2:])


def cache(NP=4, H=2, page=32, D=128, **kw):
    z = lambda w: torch.zeros(NP, H, page, w, dtype=torch.uint8)  # noqa: E731
    a = dict(kc=z(D // 2), ks=z(D // 32), vc=z(D // 2), vs=z(D // 32))
    a.update(kw)
    return a


CACHE_BAD = [cache(D=96), cache(D=256), cache(page=16), cache(page=48), cache(NP=0), cache(H=0),
             cache(kc=torch.zeros(4, 2, 32, 64)), cache(vc=torch.zeros(4, 2, 32, 64, dtype=torch.int8)),
             cache(ks=torch.zeros(4, 2, 32, 2, dtype=torch.uint8)), cache(vs=torch.zeros(4, 2, 64, 4, dtype=torch.uint8)),
             cache(kc=torch.zeros(4, 64, dtype=torch.uint8)), cache(kc=torch.zeros(4, 32, 2, 64, dtype=torch.uint8).transpose(1, 2)),
             cache(vc=torch.zeros(4, 3, 2, 32, 64, dtype=torch.uint8)[:, 1]), cache(kc=torch.zeros(1, 2, 32, 64, dtype=torch.uint8).expand(4, 2, 32, 64),
                                                                                    vc=torch.zeros(1, 2, 32, 64, dtype=torch.uint8).expand(4, 2, 32, 64)),
             cache(kc=torch.zeros(4 * 4096 + 16, dtype=torch.uint8)[1:16385].view(4, 2, 32, 64))]


@pytest.mark.parametrize("bad", range(len(CACHE_BAD)))
def test_cache_tensors_refused(calls, bad):
    c = CACHE_BAD[bad]
    D = 128
    k = torch.zeros(3, 2, D, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv4_write(k, k, slots, **c)
    with pytest.raises(ValueError):
        ops.kv4_read(slots, **c)
    with pytest.raises(ValueError):
        ops.kv4_attn(torch.zeros(3, 8, D, dtype=torch.bfloat16), **c, table=torch.zeros(3, 2, dtype=torch.int32), lens=slots)
    assert not calls


def test_cache_rows_refused(calls):
    c = cache()
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    s = torch.zeros(3, dtype=torch.int32)
    for a, b, t in ((k[:, :1], k, s), (k, k.float(), s), (k, k[:2], s), (k[0], k[0], s), (k, k, s.long()), (k, k, s[:2]), (k, k, s[None]),
                    (k.to(torch.int16), k.to(torch.int16), s), (k, k.clone().requires_grad_(), s),
                    (torch.zeros(3, 2, 129, dtype=torch.bfloat16)[..., 1:], k, s), (k, torch.zeros(3, 2, 132, dtype=torch.bfloat16)[..., :128], s)):
        with pytest.raises(ValueError):
            ops.kv4_write(a, b, t, **c)
    for t, dt in ((s.long(), torch.bfloat16), (s[None], torch.bfloat16), (s, torch.float16), (torch.zeros(6, dtype=torch.int32)[::2], torch.float32)):
        with pytest.raises(ValueError):
            ops.kv4_read(t, **c, dtype=dt)
    assert not calls
    ops.kv4_write(k, k, s, **c)
    ops.kv4_read(s, **c)
    # layers of one tensor: pages 3 layers apart
    big = [torch.zeros(4, 3, 2, 32, w, dtype=torch.uint8)[:, 1] for w in (64, 4, 64, 4)]
    ops.kv4_write(k, k, s, *big)
    for name, a in calls:
        assert len(a) + 1 == len(lib.SIGNATURES[name])
    assert calls[2][1][-4:] == (3 * 4096, 3 * 256, 4, 32)


def test_attention_refused(calls):
    c = cache()
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    t, n = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    cu = torch.zeros(4, dtype=torch.int32)
    ok = dict(q=q, table=t, lens=n)
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(q=q[0]), dict(q=q[:2]), dict(q=q[:, :0]),
                dict(q=torch.zeros(3, 8, 136, dtype=torch.bfloat16)[..., 4:132]), dict(q=q.clone().requires_grad_()),
                dict(table=t.long()), dict(table=t[0]), dict(table=torch.zeros(2, 3, dtype=torch.int32).t()), dict(table=t[:, :0]),
                dict(lens=n.long()), dict(lens=n[:2]), dict(cu_q=cu.long()), dict(cu_q=cu[:3]), dict(max_q=2), dict(cu_q=cu, max_q=0),
                dict(cu_q=cu, max_q=-1), dict(sm_scale=float("nan")), dict(max_len=-1), dict(out=q.float()), dict(out=q[:2]), dict(out=q),
                dict(out=torch.zeros(3, 1, 128, dtype=torch.bfloat16).expand(3, 8, 128)), dict(cu_q=cu, max_q=1 << 30)):
        with pytest.raises(ValueError):
            ops.kv4_attn(**dict(ok, **bad), **c)
    assert not calls
    ops.kv4_attn(**ok, **c)
    ops.kv4_attn(**ok, **c, cu_q=cu, max_q=5, max_len=4000)
    for name, a in calls:
        assert len(a) + 1 == len(lib.SIGNATURES[name])


def test_tensors_on_the_host_or_two_devices():
    z = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.kv_pages_truncate(z, **pool())
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.qk_norm_rope(**rope_args())
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        a = rope_args()
        for f in ("k", "pos", "cos", "sin"):
            b = {n: torch.empty_like(t, device="cpu" if n == f else "cuda") if isinstance(t, torch.Tensor) else t
                 for n, t in a.items()}
            with pytest.raises(RuntimeError, match="HIP device|different devices"):
                ops.qk_norm_rope(**b)


def test_library_refuses_before_a_launch():
    """The C entry points' own checks (no device is touched)."""
    L = lib.load()
    rope = [16, 1024, 128, 16, 256, 128, 5, 8, 2, 128, 0, 16, 0, 16, 16, 64, 9, None, None, 1e-6, 16, 1024, 128, 16, 256, 128, None]
    for i, v in ((0, None), (0, 24), (1, 1028), (9, 96), (10, 3), (11, None), (13, 20), (15, 66), (16, 0), (17, 20), (19, -1.0), (6, -1), (20, None),
                 (6, 1 << 27)):
        assert L.oa_qk_norm_rope(*rope[:i], v, *rope[i + 1:]) == -22, (i, v)
    assert L.oa_qk_norm_rope(*rope[:6], 0, *rope[7:]) == 0
    ext = [16, 16, 16, 4, 16, 16, 16, 3, 4, 9, 64, 7, 16, 16, 16, 16, None]
    for i, v in ((0, None), (2, None), (3, 3), (7, 0), (8, 0), (9, 0), (10, 48), (10, 16), (10, 2048), (11, -1), (12, None), (14, None),
                 (9, 1 << 26), (8, 1 << 25)):
        assert L.oa_kv_pages_extend(*ext[:i], v, *ext[i + 1:]) == -22, (i, v)
    assert L.oa_kv_pages_extend(*ext[:7], 1025, *ext[8:15], None, None) == -22 and L.oa_kv_pages_extend(*ext[:11], 2049, *ext[12:15], None, None) == -22
    assert L.oa_kv_pages_truncate(16, 16, 16, 4, 16, 16, 16, 257, 4, 9, 64, None, None) == -22
    wr = [16, 256, 128, 16, 256, 128, 3, 2, 128, 0, 16, 16, 16, 16, 16, 4096, 256, 4, 32, None]
    for i, v in ((0, 8), (1, 4), (6, -1), (7, 0), (8, 96), (9, 3), (10, None), (11, 8), (12, None), (15, 4080), (15, 4104), (16, 240), (17, 0), (18, 33),
                 (6, 1 << 26)):
        assert L.oa_kv4_write(*wr[:i], v, *wr[i + 1:]) == -22, (i, v)
    assert L.oa_kv4_write(*wr[:6], 0, *wr[7:]) == 0
    rd = [16, 16, 16, 16, 16, 4096, 256, 4, 32, 16, 256, 128, 16, 256, 128, 3, 2, 128, 0, None]
    assert L.oa_kv4_read(*rd[:18], 1, None) == -22 and L.oa_kv4_read(None, *rd[1:]) == -22
    at = [16, 1024, 128, 16, 16, 16, 16, 4096, 256, 4, 32, 16, 2, 2, 16, None, 3, 3, 1, 8, 2, 128, 0.1, 128, 2, 16, 16, 16, 32, 1024, 128, 0, None]
    for i, v in ((0, 8), (1, 4), (3, 8), (7, 4000), (9, 0), (10, 31), (11, None), (12, 1), (13, 0), (13, 1 << 26), (14, None), (16, 2), (18, 0), (18, 2), (19, 7), (20, 0),
                 (21, 96), (22, float("nan")), (23, 64), (23, 200), (24, 0), (25, None), (26, None), (28, None), (29, 2), (23, 1 << 30), (24, 1 << 24), (28, 16)):
        assert L.oa_kv4_attn(*at[:i], v, *at[i + 1:]) == -22, (i, v)
    assert L.oa_kv4_attn(*at[:16], 0, 0, *at[18:]) == 0
    many = [*at[:15], 16, 3, 64, 17, *at[19:]]           # 68 rows of a KV head
    # more workgroups, or rows to join, than a grid holds
    assert L.oa_kv4_attn(*at[:15], 16, 1 << 20, 1 << 20, 1 << 10, *at[19:]) == -22
    assert L.oa_kv4_attn(*at[:15], 16, 3, 1 << 22, 1 << 22, *at[19:]) == -22 and L.oa_kv4_attn(*at[:15], 16, 65536, 8, 1, *at[19:]) == -22
    assert L.oa_kv4_attn(*many[:27], None, *many[28:]) == -22 and L.oa_kv4_attn(*many[:27], 2, *many[28:]) == -22


def test_a_numbers_value_counts_in_every_call(calls):
    """Sizes are looked up by value: a scalar tensor, or numpy's integer, that has changed since gives its new value,
    and good sizes that were seen before do not let in a misaligned or a gradient-bearing tensor."""
    c = cache()
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    t, n, cu = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    s, m = torch.tensor(0.5), torch.tensor(2)
    for scale, rows in ((0.5, 2), (0.25, 3)):
        s.fill_(scale)
        m.fill_(rows)
        ops.kv4_attn(q, table=t, lens=n, cu_q=cu, sm_scale=s, max_q=m, **c)
        name, a = calls[-1]
        types = [x.__name__ for x in lib.SIGNATURES[name]]
        assert [x for x, k in zip(a, types) if k == "c_float"] == [scale] and rows in a
    with pytest.raises(TypeError):
        ops.kv4_attn(q, table=t, lens=n, cu_q=cu, max_q=2.0, **c)
    wide = torch.zeros(3, 8, 136, dtype=torch.bfloat16)
    ops.kv4_attn(wide[..., :128], table=t, lens=n, cu_q=cu, max_q=2, **c)
    ops.kv4_attn(q, table=t, lens=n, cu_q=cu, max_q=2, out=wide[..., :128], **c)
    count, off = len(calls), wide[..., 1:129]
    for bad in (off, q.clone().requires_grad_()):
        with pytest.raises(ValueError):
            ops.kv4_attn(bad, table=t, lens=n, cu_q=cu, max_q=2, **c)
        with pytest.raises(ValueError):
            ops.kv4_attn(q, table=t, lens=n, cu_q=cu, max_q=2, out=bad, **c)
    assert len(calls) == count


def test_forward_tangents_refused(calls):
    """An operator would drop the tangent of a dual tensor in silence."""
    from torch.autograd import forward_ad as fw
    c = cache()
    q, k, s = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    t = torch.zeros(3, 2, dtype=torch.int32)
    with fw.dual_level():
        dq, dk = fw.make_dual(q, torch.ones_like(q)), fw.make_dual(k, torch.ones_like(k))
        for call in (lambda: ops.kv4_attn(dq, table=t, lens=s, **c), lambda: ops.kv4_write(k, dk, s, **c),
                     lambda: ops.qk_norm_rope(**rope_args(q=fw.make_dual(torch.zeros(5, 8, 128), torch.ones(5, 8, 128)), k=torch.zeros(5, 2, 128)))):
            with pytest.raises(ValueError):
                call()
        assert not calls
        ops.kv4_attn(q, table=t, lens=s, **c)
        ops.kv4_write(k, k, s, **c)
    assert len(calls) == 2
