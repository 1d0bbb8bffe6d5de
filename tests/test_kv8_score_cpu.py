"""Refusals of the 8-bit cache and of token_logprobs: bad shapes, types, devices and sizes end in an error before any launch."""
import ctypes as C

import pytest
import torch

from kv8_reference import VALUES, Cache, encode, need_exp


def _lib():
    from transvae_amd import _lib
    return _lib


def test_definition_of_the_codes():
    "the reference of the GPU tests against torch's own e4m3 type"
    assert torch.equal(torch.nan_to_num(VALUES), torch.nan_to_num(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()))
    x = torch.cat([torch.randn(20000, dtype=torch.float64) * 50, torch.linspace(-448, 448, 40001, dtype=torch.float64), torch.randn(20000, dtype=torch.float64) * 0.01])
    x = x.clamp(-448, 448).float().double()
    assert torch.equal(encode(x), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    for v, e in ((448.0, 127), (448.1, 128), (1.75, 119), (1.0, 119), (0.0, 27), (3.4e38, 246), (1e-40, 27)):
        assert need_exp(torch.tensor([v, float("nan"), float("inf")], dtype=torch.float64)) == e
    c = Cache(4, 1, 32, 16)
    c.store(torch.ones(2, 3, 1, 32), torch.ones(2, 3, 1, 32), [15, -1], [3, 3], None, 2)
    assert int((c.k != 0).sum()) == 3 * 32 and float(c.load(3, [15, 0], [3, 3], None, 2, 2)[0][0].min()) == 1.0


P = C.c_void_p(4096)            # an aligned address that is never read: every call below is refused first


def _store(**kw):
    a = dict(k=P, ldkb=64, ldkt=64, ldkh=64, v=P, ldvb=64, ldvt=64, ldvh=64, dtype=0, kc=P, vc=P, ke=P, ve=P, n_pages=8, table=None, per=4,
             start=None, start0=0, count=None, n=2, T=3, h=1, dk=64, page=32, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib().lib().tvae_kv8_store(*a.values())


def _load(**kw):
    a = dict(kc=P, vc=P, ke=P, ve=P, n_pages=8, table=None, per=4, start=None, start0=0, count=None, k=P, v=P, dtype=0, n=2, T=3, h=1, dk=64,
             page=32, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib().lib().tvae_kv8_load(*a.values())


def _attn(**kw):
    a = dict(q=P, b=64, i=64, h_=64, o=P, ob=64, oi=64, oh=64, dtype=0, kc=P, vc=P, ke=P, ve=P, n_pages=8, table=None, per=4, lens=None, len0=5,
             mask=None, ldm=0, mw=0, causal=1, n=2, h=1, G=1, Lq=1, dk=64, page=32, scale=1.0, splits=1, ws=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib().lib().tvae_kv8_attn(*a.values())


ODD = C.c_void_p(4100)
CACHE = [dict(kc=None), dict(vc=None), dict(ke=None), dict(ve=None), dict(dtype=2), dict(dtype=-1), dict(dk=48), dict(dk=0), dict(page=8), dict(page=24),
         dict(page=512), dict(h=0), dict(n=-1), dict(n_pages=7), dict(n_pages=-1), dict(per=0), dict(per=1 << 30, page=256), dict(kc=ODD), dict(vc=ODD)]


@pytest.mark.parametrize("bad", CACHE + [dict(k=None), dict(v=None), dict(k=ODD), dict(ldkt=66), dict(ldvb=1), dict(start0=-1), dict(start0=126), dict(T=-1),
                                         dict(T=129), dict(n=2000000, T=1000000, start0=0, table=P, per=40000)])
def test_store_refuses(bad):
    assert _store(**bad) < 0 and _lib().lib().tvae_last_error()


@pytest.mark.parametrize("bad", CACHE + [dict(k=None), dict(v=None), dict(v=ODD), dict(T=-2), dict(n=1 << 20, table=P, T=1 << 20)])
def test_load_refuses(bad):
    assert _load(**bad) < 0 and _lib().lib().tvae_last_error()


@pytest.mark.parametrize("bad", CACHE + [dict(q=None), dict(o=None), dict(q=ODD), dict(oh=2), dict(G=0), dict(Lq=-1), dict(len0=-1), dict(len0=129),
                                         dict(mask=P, mw=10, ldm=5), dict(mask=P, mw=-1), dict(splits=0), dict(splits=2), dict(splits=2000, ws=P),
                                         dict(n=1 << 20, table=P, Lq=1 << 12), dict(splits=4, ws=ODD), dict(n=1 << 19, table=P, Lq=4, splits=1000, ws=P)])
def test_attend_refuses(bad):
    assert _attn(**bad) < 0 and _lib().lib().tvae_last_error()


def test_nothing_to_do_is_no_error():
    assert _store(n=0) == 0 and _store(T=0) == 0 and _load(n=0) == 0 and _load(T=0) == 0 and _attn(n=0) == 0 and _attn(Lq=0) == 0


def _fwd(**kw):
    a = dict(x=P, ld=30, dtype=0, tok=None, ldt=1, sub=0, rows=4, V=30, top=3, logp=P, ldl=1, ent=P, lde=1, stat=P, tl=P, ti=P, segs=1, ws=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib().lib().tvae_token_logp(*a.values())


def _bwd(**kw):
    a = dict(x=P, ld=30, dtype=0, tok=None, ldt=1, sub=0, rows=4, V=30, top=3, stat=P, ent=P, lde=1, ti=P, gl=P, ge=P, gt=P, dx=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib().lib().tvae_token_logp_bwd(*a.values())


SHAPE = [dict(x=None), dict(x=C.c_void_p(4097)), dict(dtype=2), dict(rows=-1), dict(rows=1 << 40), dict(V=0), dict(V=31), dict(V=1 << 32, ld=1 << 32),
         dict(top=-1), dict(top=31), dict(top=65, V=100, ld=100), dict(stat=None), dict(ent=None)]


@pytest.mark.parametrize("bad", SHAPE + [dict(logp=None), dict(tl=None), dict(ti=None), dict(segs=0), dict(segs=2), dict(segs=2000, ws=P)])
def test_token_logp_refuses(bad):
    assert _fwd(**bad) < 0 and _lib().lib().tvae_last_error()


def test_token_logp_refuses_a_workspace_off_its_border():
    assert _fwd(segs=2, ws=C.c_void_p(4100)) < 0 and b"aligned to 8" in _lib().lib().tvae_last_error()


@pytest.mark.parametrize("bad", SHAPE + [dict(dx=None), dict(ti=None), dict(dx=C.c_void_p(4098))])
def test_token_logp_bwd_refuses(bad):
    assert _bwd(**bad) < 0 and _lib().lib().tvae_last_error()


def test_python_side_refuses():
    from transvae_amd.kv8 import KV8Cache
    from transvae_amd.loss import token_logprobs
    E = _lib().TvaeError
    mk = lambda *s, d=torch.uint8: torch.zeros(s, dtype=d)
    ok = KV8Cache(mk(6, 2, 32, 64), mk(6, 2, 32, 64), mk(6, 2), mk(6, 2), n_seq=2)
    for args in ((mk(6, 2, 32, 64), mk(6, 2, 32, 32), mk(6, 2), mk(6, 2)), (mk(6, 2, 32, 64), mk(6, 2, 32, 64), mk(6, 3), mk(6, 3)),
                 (mk(6, 2, 32, 64, d=torch.int8), mk(6, 2, 32, 64), mk(6, 2), mk(6, 2)), (mk(6, 2, 32, 48), mk(6, 2, 32, 48), mk(6, 2), mk(6, 2)),
                 (mk(6, 2, 24, 64), mk(6, 2, 24, 64), mk(6, 2), mk(6, 2)), (mk(6, 32, 2, 64).transpose(1, 2), mk(6, 2, 32, 64), mk(6, 2), mk(6, 2))):
        with pytest.raises(E):
            KV8Cache(*args)
    for bad in (dict(n=0, max_len=5), dict(n=1, max_len=0)):
        with pytest.raises(E):
            KV8Cache.for_batch(heads=2, dk=64, device="cpu", **bad)
    with pytest.raises(E):
        KV8Cache(mk(6, 2, 32, 64), mk(6, 2, 32, 64), mk(6, 2), mk(6, 2), n_seq=4)
    r = torch.zeros(2, 1, 2, 64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    calls = [lambda: ok.store(r, r), lambda: ok.attend(r, 1), lambda: ok.load(3),                                   # host memory
             lambda: ok.store(r.double(), r.double()), lambda: ok.store(r, r.half()), lambda: ok.store(r[..., :32], r[..., :32]), lambda: ok.store(r[0], r[0]),
             lambda: ok.store(r[:1], r[:1]), lambda: ok.attend(r[:1], 1), lambda: ok.attend(torch.zeros(2, 1, 3, 64), 1), lambda: ok.attend(r, i32(3)),
             lambda: ok.attend(r, torch.zeros(2)), lambda: ok.attend(r, 1, key_mask=torch.zeros(2, 5)), lambda: ok.attend(r, 1, key_mask=torch.zeros(3, 5, dtype=torch.bool)),
             lambda: ok.attend(r, 1, table=i32(3, 2)), lambda: ok.attend(r, 1, table=i32(2, 0)), lambda: ok.attend(r, 1, table=torch.zeros(2, 2)),
             lambda: ok.attend(r, 1, out=r.half()), lambda: ok.attend(r, 1 << 32), lambda: ok.store(r, r, start=1 << 33), lambda: ok.load(1, start=-(1 << 40)),
             lambda: ok.attend(r, 1, out=torch.zeros(1, 1, 2, 64).expand(2, 1, 2, 64)), lambda: ok.load(3, dtype=torch.float64), lambda: ok.store(r, r, count=torch.zeros(2)),
             lambda: KV8Cache(mk(6, 2, 32, 64), mk(6, 2, 32, 64), mk(6, 2), mk(6, 2)).load(3)]
    for c in calls:
        with pytest.raises(E):
            c()
    x = torch.zeros(4, 9)
    for c in (lambda: token_logprobs(x.double()), lambda: token_logprobs(x, top=10), lambda: token_logprobs(x, top=-1), lambda: token_logprobs(torch.zeros(4, 0)),
              lambda: token_logprobs(x, torch.zeros(3, dtype=torch.int64)), lambda: token_logprobs(x, torch.zeros(4)), lambda: token_logprobs(x, torch.zeros(4, dtype=torch.bool)),
              lambda: token_logprobs(torch.zeros(2, 100), top=65), lambda: token_logprobs(torch.tensor(1.0)), lambda: token_logprobs(x)):
        with pytest.raises(E):
            c()


def test_sequence_logp_stops_behind_the_first_end():
    from transvae_amd.tvae_util import sequence_logp
    ids = torch.tensor([[3, 25, 7, 25], [1, 2, 3, 4], [25, 25, 25, 25]], dtype=torch.uint8)
    logp = torch.tensor([[-1.0, -2.0, -4.0, -8.0]] * 3)
    assert sequence_logp(ids, logp, 25).tolist() == [-3.0, -15.0, -1.0]


def test_decoder_refuses_an_unknown_cache():
    from transvae_amd.decode import GreedyDecoder
    with pytest.raises(_lib().TvaeError):
        GreedyDecoder(None, 4, kv_cache="int8")
