"""The 8-bit key/value cache (transvae_amd/kv8.py) against loops in 64 bits (tests/kv8_reference.py)."""
import math

import pytest
import torch

from kv8_reference import VALUES, Cache, attend_bound

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def pair(n, per, h, dk, page, paged, seed=0, extra=2):
    "(cache on the GPU, the same on the CPU, block table on the GPU or None, the same on the CPU)"
    from transvae_amd.kv8 import KV8Cache
    g = torch.Generator().manual_seed(seed)
    pages = n * per + (extra if paged else 0)
    ref = Cache(pages, h, dk, page)
    table = torch.randperm(pages, generator=g)[:n * per].view(n, per).to(torch.int32) if paged else None
    gpu = KV8Cache.empty(pages, h, dk, page, "cuda:0", n_seq=None if paged else n)
    return gpu, ref, None if table is None else table.cuda(), table


def fill(gpu, ref, seed=1):
    "random codes without NaN and exponents around 1 in both"
    g = torch.Generator().manual_seed(seed)
    for name in ("k", "v"):
        c = torch.randint(0, 256, ref.k.shape, generator=g, dtype=torch.uint8)
        c[(c & 127) == 127] = 126
        e = torch.randint(117, 122, ref.ke.shape, generator=g, dtype=torch.uint8)
        getattr(ref, name).copy_(c)
        getattr(ref, name + "e").copy_(e)
        getattr(gpu, name).copy_(c.cuda())
        getattr(gpu, name + "_exp").copy_(e.cuda())


def same_cache(gpu, ref):
    for name in ("k", "v"):
        a, b = getattr(gpu, name).cpu(), getattr(ref, name)
        nan = ((a & 127) == 127) & ((b & 127) == 127)              # either sign of NaN
        assert torch.equal(getattr(gpu, name + "_exp").cpu(), getattr(ref, name + "e")), name
        bad = ((a != b) & ~nan).nonzero()
        assert not len(bad), (name, bad[:4].tolist(), [(int(a[tuple(i)]), int(b[tuple(i)])) for i in bad[:4]])


def ints(x):
    return x if isinstance(x, int) else torch.tensor(x, dtype=torch.int32).cuda()


# ---------------------------------------------------------------------------------------------- load
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,page", [(32, 16), (64, 32), (128, 64), (256, 256)])
def test_every_code_reads_back_exactly(dtype, dk, page):
    gpu, ref, _, _ = pair(2, 2, 3, dk, page, False)
    codes = (torch.arange(ref.k.numel()) % 256).to(torch.uint8).view(ref.k.shape)
    gpu.k.copy_(codes.cuda())
    gpu.v.copy_(codes.flip(0).cuda())
    exps = torch.tensor([27, 100, 118, 127, 130, 246]).repeat(ref.ke.numel())[:ref.ke.numel()].view(ref.ke.shape).to(torch.uint8)
    gpu.k_exp.copy_(exps.cuda())
    gpu.v_exp.copy_(exps.cuda())
    k, v = gpu.load(2 * page, dtype=dtype)
    for got, c in ((k, codes), (v, codes.flip(0))):
        want = (VALUES[c.long()] * torch.exp2(exps.double() - 127)[:, :, None, None]).view(2, 2, 3, page, dk).transpose(2, 3).reshape(2, 2 * page, 3, dk)
        want = want.to(torch.float32).to(dtype)                    # one rounding: a code has 4 significant bits
        assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got).cpu(), torch.nan_to_num(want))


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("T,start,count", [(1, 0, None), (5, 31, None), (70, 3, [70, 0, 1, 33]), (40, [0, 95, 64, 90], [40, 40, 3, 40]),
                                           (4, [-2, 96, 1000, 0], None), (3, 0, 2)])
def test_load_of_any_part(T, start, count, paged):
    n, per, h, dk, page = 4, 3, 2, 64, 32
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, paged, seed=3)
    fill(gpu, ref)
    if paged:
        rtab[1, 0], rtab[2, 2] = -1, ref.n_pages                   # no such pages
        tab.copy_(rtab.cuda())
    k, v = gpu.load(T, start=ints(start), count=None if count is None else ints(count), table=tab)
    lst = lambda x, d: [d] * n if x is None else [x] * n if isinstance(x, int) else x
    wk, wv = ref.load(T, lst(start, 0), lst(count, T), rtab, per, n)
    assert torch.equal(k.cpu().double(), wk) and torch.equal(v.cpu().double(), wv)


# ---------------------------------------------------------------------------------------------- store
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,T,h,dk,page,start,count,paged", [
    (1, 1, 1, 32, 16, 0, None, False), (3, 1, 4, 64, 32, 31, None, False), (5, 1, 3, 128, 64, [0, 1, 63, 64, 127], None, True),
    (4, 33, 2, 64, 32, 5, [33, 0, 1, 28], True), (2, 100, 5, 32, 16, 0, None, False), (3, 70, 1, 256, 128, [10, 0, 200], [70, 64, 70], True),
    (2, 200, 2, 128, 256, 30, None, False), (4, 7, 12, 64, 16, [-1, 300, 60, 15], [7, 7, 9, 0], True)])
def test_store_rounds_as_defined(dtype, n, T, h, dk, page, start, count, paged):
    per = 2 if page >= 128 else 9
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, paged, seed=5)
    fill(gpu, ref)
    g = torch.Generator().manual_seed(7)
    x = torch.randn((n, T, 3, h, dk), generator=g) * torch.exp2(torch.randint(-9, 6, (n, T, 3, h, 1), generator=g).float())
    x = x.to(dtype)
    xg = x.cuda()
    gpu.store(xg[:, :, 1], xg[:, :, 2], start=ints(start), count=None if count is None else ints(count), table=tab)
    lst = lambda v, d: [d] * n if v is None else [v] * n if isinstance(v, int) else v
    ref.store(x[:, :, 1], x[:, :, 2], lst(start, 0), lst(count, T), rtab, per)
    same_cache(gpu, ref)                                           # every page: what was not written stays


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_pages_of_every_size(dtype, dk, page):
    "a thread keeps as many pieces as the page needs: whole pages, one that has rows in front, one that ends early"
    n, h, per, T = 2, 2, 3, 2 * page - 3
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, False, seed=dk + page)
    g = torch.Generator().manual_seed(page)
    for start, size in ((0, 1.0), (page // 2 + 1, 40.0)):
        k, v = ((torch.randn((n, T, h, dk), generator=g) * size).to(dtype) for _ in range(2))
        gpu.store(k.cuda(), v.cuda(), start=start)
        ref.store(k, v, [start] * n, [T] * n, rtab, per)
        same_cache(gpu, ref)


def test_store_ties_ends_and_what_has_no_code():
    "halves go to the even code; the page's scale at its borders; zeros, denormals, the largest floats, infinities and NaN"
    h, dk, page = 4, 32, 16
    gpu, ref, _, _ = pair(1, 8, h, dk, page, False)
    pos = VALUES[:127]
    mid = torch.cat([(pos[:-1] + pos[1:]) / 2, pos]).float()       # exact in fp32
    x = torch.zeros((1, 8 * page, h, dk))
    flat = x[0, :page].view(page, h * dk)
    for i in range(h):                                             # page 0: every midpoint and value, at three scales
        vals = torch.cat([mid, -mid])[:page * dk - 2]
        blk = torch.zeros(page * dk)
        blk[:len(vals)] = vals
        blk[-1] = 448.0
        flat.view(page, h, dk)[:, i] = blk.view(page, dk) * 2.0 ** (5 * i - 8)
    inf, nan, big, tiny = math.inf, math.nan, 3.4028234663852886e38, 2.0 ** -149
    edge = [[0.0, -0.0], [448.0, 449.0], [tiny, -tiny], [big, -big], [inf, 1.0], [nan, 3.0], [-inf, nan], [448.0001, 1.0], [2.0 ** -100, 2.0 ** -109],
            [1.75 * 2.0 ** 119, 1.0], [2.0 ** -94, 1e-40], [224.0, 224.0001]]
    for j, e in enumerate(edge):                                   # pages 1 ..: one edge a (page, head)
        x[0, (1 + j // h) * page + j % 3, j % h, 5:5 + len(e)] = torch.tensor(e)
    y = -x.flip(1).contiguous()
    gpu.store(x.cuda(), y.cuda())
    ref.store(x, y, [0], [8 * page], None, 8)
    same_cache(gpu, ref)
    k, _ = gpu.load(8 * page)
    assert not bool(torch.isinf(k).any())                          # a cache holds no infinity


@pytest.mark.parametrize("dtype", DTYPES)
def test_appends_one_by_one_rescale_the_page(dtype):
    n, h, dk, page, per = 3, 2, 64, 16, 3
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, True, seed=9)
    g = torch.Generator().manual_seed(11)
    for t in range(40):
        size = 2.0 ** ((t * 5) % 17 - 8)                           # up and down: some tokens raise the page's exponent, some do not
        k, v = (torch.randn((n, 1, h, dk), generator=g) * size).to(dtype), torch.randn((n, 1, h, dk), generator=g).to(dtype)
        start = [t, max(0, t - 3), t] if t % 2 else t
        gpu.store(k.cuda(), v.cuda(), start=ints(start), table=tab)
        ref.store(k, v, start if isinstance(start, list) else [t] * n, [1] * n, rtab, per)
    same_cache(gpu, ref)


def test_store_keeps_rows_behind_and_drops_what_has_no_page():
    n, h, dk, page, per = 3, 2, 32, 16, 2
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, True, seed=13)
    fill(gpu, ref)
    rtab[1, 1], rtab[2, 0] = ref.n_pages + 5, -7
    tab.copy_(rtab.cuda())
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((n, 40, h, dk), generator=g), torch.randn((n, 40, h, dk), generator=g)
    gpu.store(k.cuda(), v.cuda(), start=3, count=ints([40, 20, 40]), table=tab)
    ref.store(k, v, [3] * n, [40, 20, 40], rtab, per)
    same_cache(gpu, ref)


# ---------------------------------------------------------------------------------------------- attend
CASES = [  # n, Lq, h, G, dk, page, per, lens, paged, mask
    (1, 1, 1, 1, 32, 16, 1, [1], False, False),
    (3, 1, 4, 1, 64, 32, 4, 127, False, True),
    (4, 1, 2, 1, 32, 16, 5, [0, 1, 16, 80], True, False),
    (5, 1, 3, 5, 64, 32, 3, [96, 95, 33, 2, 0], True, False),
    (2, 1, 1, 8, 128, 64, 20, [1280, 1], True, False),
    (1, 1, 2, 16, 128, 16, 70, 1101, True, True),
    (2, 1, 1, 17, 64, 32, 5, [160, 77], False, False),
    (2, 3, 2, 1, 64, 32, 4, [100, 2], True, False),
    (3, 7, 1, 3, 256, 128, 2, [250, 7, 3], True, True),
    (2, 33, 2, 2, 128, 32, 6, [190, 40], True, False),
    (1, 70, 1, 1, 32, 16, 5, 75, False, False),
    (2, 5, 2, 4, 256, 16, 3, [48, 31], False, True),
    (2, 20, 1, 8, 64, 256, 1, [256, 19], True, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attend_matches_the_definition(case, dtype):
    n, Lq, h, G, dk, page, per, lens, paged, masked = case
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, paged, seed=17)
    fill(gpu, ref)
    g = torch.Generator().manual_seed(19)
    q = (torch.randn((n, Lq, 2, h * G, dk), generator=g) * 0.2).to(dtype)
    mask = (torch.rand((n, per * page), generator=g) < 0.7) if masked else None
    if masked:
        mask[0] = False                                            # a sequence that sees nothing
        if n > 1:
            mask = mask[:, :per * page - 3]                        # tokens past the mask are not visible
    ll = [lens] * n if isinstance(lens, int) else lens
    for causal in (True, False):
        for scale in (None, 0.03):
            o = gpu.attend(q.cuda()[:, :, 1], ints(lens), table=tab, causal=causal, key_mask=None if mask is None else mask.cuda(), scale=scale)
            want, wv, qk = ref.attend(q[:, :, 1], ll, rtab, per, causal, mask, scale)
            lim = attend_bound(want, wv, qk, dk, per * page, dtype)
            off = (o.cpu().double() - want).abs()
            assert bool((off <= lim).all()), (causal, scale, float((off / lim).max()), (off / lim).argmax())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,h,per,Lq,G,dk,page,splits", [
    (2, 2, 20, 1, 4, 64, 32, 1), (2, 2, 20, 5, 2, 128, 32, 3), (110, 4, 4, 1, 4, 32, 32, 1), (40, 10, 7, 2, 1, 64, 16, 1),
    (3, 1, 5, 3, 1, 256, 64, 2), (70, 2, 8, 1, 1, 32, 16, 1), (9, 2, 3, 1, 1, 64, 128, 1)])
def test_masks_of_runs(n, h, per, Lq, G, dk, page, splits, dtype):
    "runs of masked tokens longer and shorter than what a kernel takes at once, single visible tokens, none; NaN codes behind the masks"
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, True, seed=43)
    fill(gpu, ref)
    W = per * page
    g = torch.Generator().manual_seed(47)
    mask = torch.zeros((n, W + 5), dtype=torch.bool)
    for b in range(n):
        kind = b % 6
        if kind == 0:
            mask[b, W // 2:W // 2 + 40] = True
        elif kind == 1:
            mask[b, int(torch.randint(0, W, (1,), generator=g))] = True
        elif kind == 2:
            mask[b] = True
            mask[b, 16:16 + 48] = False
        elif kind == 3:
            mask[b] = True
            mask[b, 5:min(W - 3, 75)] = False
        elif kind == 4:
            mask[b] = (torch.arange(W + 5) // 16) % 2 == 1
    if n > 50:
        rtab[1, per - 1] = -1
        tab.copy_(rtab.cuda())
    lens = [W - (b * 7) % 23 for b in range(n)]
    q = (torch.randn((n, Lq, h * G, dk), generator=g) * 0.2).to(dtype)
    clean = ref.attend(q, lens, rtab, per, True, mask)
    for b in range(n):
        for i in range(per):
            p = ref.page_of(rtab, per, b, i)
            if p is not None:
                dead = ~mask[b, i * page:(i + 1) * page].cuda()
                gpu.k[p][:, dead] = 127
                gpu.v[p][:, dead] = 255
    o = gpu.attend(q.cuda(), ints(lens), table=tab, key_mask=mask.cuda(), splits=splits)
    lim = attend_bound(*clean, dk, W, dtype)
    assert bool(((o.cpu().double() - clean[0]).abs() <= lim).all())


@pytest.mark.parametrize("Lq,G", [(1, 1), (1, 4), (9, 2)])
def test_what_is_dead_or_masked_never_matters(Lq, G):
    "NaN codes and exponents of 255 in dead rows, masked tokens, pages of nobody; absent pages"
    n, h, dk, page, per = 3, 2, 64, 32, 4
    gpu, ref, tab, rtab = pair(n, per, h, dk, page, True, seed=23)
    fill(gpu, ref)
    lens = [100, 37, 64]
    mask = torch.ones((n, per * page), dtype=torch.uint8)
    mask[0, 10:50] = 0
    rtab[2, 0] = -1
    rtab[1, 3] = 1 << 30
    tab.copy_(rtab.cuda())
    clean = ref.attend(q := torch.randn((n, Lq, h * G, dk), generator=torch.Generator().manual_seed(3)) * 0.2, lens, rtab, per, True, mask)
    used = set()
    for b in range(n):
        for i in range(per):
            p = ref.page_of(rtab, per, b, i)
            if p is None:
                continue
            for t in range(page):
                pos = i * page + t
                if pos >= lens[b] or not mask[b, pos]:
                    gpu.k[p, :, t] = 127
                    gpu.v[p, :, t] = 255
                else:
                    used.add(p)
    for p in range(ref.n_pages):
        if p not in used:
            gpu.k_exp[p] = 255
            gpu.v_exp[p] = 255
    o = gpu.attend(q.cuda(), ints(lens), table=tab, key_mask=mask.cuda())
    assert bool(((o.cpu().double() - clean[0]).abs() <= attend_bound(*clean, dk, per * page, torch.float32)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq,G,dk", [(1, 1, 64), (1, 8, 128), (6, 3, 64), (40, 1, 32), (3, 1, 256)])
def test_a_nan_key_or_value_reaches_the_queries_that_see_it(Lq, G, dk, dtype):
    "causal queries in front of it, masked tokens, pages of masked tokens only (whatever their exponents)"
    n, h, page, per = 2, 2, 16, 6
    gpu, ref, _, _ = pair(n, per, h, dk, page, False)
    fill(gpu, ref)
    L = per * page - 3
    mask = torch.ones((n, L), dtype=torch.bool)
    mask[1, 2 * page:3 * page] = False
    mask[0, 5] = False
    gpu.k[per + 2], gpu.v[per + 2], gpu.k_exp[per + 2], gpu.v_exp[per + 2] = 127, 255, 255, 255
    gpu.v[0, :, 5], gpu.k[0, :, 5] = 127, 127
    q = (torch.randn((n, Lq, h * G, dk), generator=torch.Generator().manual_seed(1)) * 0.2).to(dtype)
    lim = None
    for at in (L - 1, L - 2, L - min(Lq, 20)):                     # seen by the last 1, 2, min(Lq, 20) queries
        page_at, row = divmod(at, page)
        saved = gpu.v[page_at, 1, row, 3].clone()
        gpu.v[page_at, 1, row, 3] = 127
        o = gpu.attend(q.cuda(), L, key_mask=mask.cuda()).cpu()
        gpu.v[page_at, 1, row, 3] = saved
        want, wv, qk = ref.attend(q, [L] * n, None, per, True, mask)
        hit = torch.zeros_like(want, dtype=torch.bool)
        hit[0, at - (L - Lq) if at >= L - Lq else 0:, G:, 3] = True
        assert torch.equal(torch.isnan(o), hit), (at, torch.isnan(o).nonzero()[:5], hit.nonzero()[:5])
        lim = attend_bound(want, wv, qk, dk, L, dtype)
        assert bool((((o.double() - want).abs() <= lim) | hit).all())
        saved = gpu.k[page_at, 0, row, 3].clone()
        gpu.k[page_at, 0, row, 3] = 255
        o = gpu.attend(q.cuda(), L, key_mask=mask.cuda()).cpu()
        gpu.k[page_at, 0, row, 3] = saved
        hit[:] = False
        hit[0, at - (L - Lq) if at >= L - Lq else 0:, :G] = True
        assert torch.equal(torch.isnan(o), hit)
        assert bool((((o.double() - want).abs() <= lim) | hit).all())


def test_values_of_a_visible_nan_reach_their_own_row_only():
    n, h, dk, page = 2, 2, 64, 32
    gpu, ref, _, _ = pair(n, 2, h, dk, page, False)
    fill(gpu, ref)
    gpu.v[0, 1, 3, 7] = 127
    for G in (1, 4):
        o = gpu.attend(torch.randn((n, 1, h * G, dk)).cuda(), 50)
        bad = torch.isnan(o).cpu()
        assert bool(bad[0, 0, G:2 * G, 7].all()) and int(bad.sum()) == G


@pytest.mark.parametrize("Lq,G", [(1, 1), (1, 3), (20, 2)])
def test_scales_of_either_sign_and_out_of_place_or_in_place(Lq, G):
    n, h, dk, page, per = 2, 2, 64, 16, 5
    gpu, ref, _, _ = pair(n, per, h, dk, page, False)
    fill(gpu, ref)
    q = torch.randn((n, Lq, h * G, dk), generator=torch.Generator().manual_seed(1)) * 0.2
    for scale in (-0.125, 0.0, -2.0, 1e-3):
        want = ref.attend(q, [70, 33], None, per, scale=scale)
        o = gpu.attend(q.cuda(), ints([70, 33]), scale=scale)
        lim = attend_bound(want[0], want[1], want[2].abs(), dk, 80, torch.float32)
        assert bool(((o.cpu().double() - want[0]).abs() <= lim).all()), scale
        qq = q.cuda()
        assert torch.equal(gpu.attend(qq, ints([70, 33]), scale=scale, out=qq), o) and torch.equal(qq, o)


def test_no_sequences_no_queries_no_keys():
    from transvae_amd.kv8 import KV8Cache
    c = KV8Cache.empty(4, 2, 64, 32, "cuda:0")
    tab = torch.zeros((0, 3), dtype=torch.int32).cuda()
    assert c.attend(torch.zeros((0, 1, 4, 64)).cuda(), 0, table=tab).shape == (0, 1, 4, 64)
    c.store(torch.zeros((0, 5, 2, 64)).cuda(), torch.zeros((0, 5, 2, 64)).cuda(), table=tab)
    assert c.load(5, table=tab)[0].shape == (0, 5, 2, 64)
    tab = torch.zeros((1, 3), dtype=torch.int32).cuda()
    assert c.attend(torch.zeros((1, 0, 4, 64)).cuda(), 1, table=tab).shape == (1, 0, 4, 64)
    assert float(c.attend(torch.ones((1, 2, 4, 64)).cuda(), 0, table=tab).abs().max()) == 0
    assert float(c.attend(torch.ones((1, 2, 4, 64)).cuda(), 9, table=tab, key_mask=torch.zeros((1, 0), dtype=torch.bool).cuda()).abs().max()) == 0
    before = c.k.clone()
    c.store(torch.ones((1, 0, 2, 64)).cuda(), torch.ones((1, 0, 2, 64)).cuda(), table=tab)
    c.store(torch.ones((1, 3, 2, 64)).cuda(), torch.ones((1, 3, 2, 64)).cuda(), count=0, table=tab)
    assert torch.equal(c.k, before)


@pytest.mark.parametrize("G,Lq", [(1, 1), (4, 1), (2, 9)])
def test_pages_past_four_gigabytes(G, Lq):
    "byte offsets over 2^32: a sequence in the last pages of a large pool reads and writes what it would in a small one"
    from transvae_amd.kv8 import KV8Cache
    h, dk, page = 8, 128, 64
    pages = (1 << 32) // (h * page * dk) + 40
    big = KV8Cache(*[torch.empty((pages, h, page, dk), dtype=torch.uint8, device="cuda:0") for _ in range(2)],
                   *[torch.full((pages, h), 127, dtype=torch.uint8, device="cuda:0") for _ in range(2)])
    small = KV8Cache.empty(40, h, dk, page, "cuda:0")
    tab = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].view(2, 18).to(torch.int32).cuda()
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn((2, 1000, h, dk), generator=g).cuda() for _ in range(2))
    q = torch.randn((2, Lq, h * G, dk), generator=g).cuda()
    out = []
    for c, t in ((big, tab + (pages - 40)), (small, tab)):
        c.store(k, v, start=7, table=t)
        out.append((c.load(1007, table=t)[0][:, 7:], c.load(1007, table=t)[1][:, 7:], c.attend(q, 1007, table=t, key_mask=(torch.arange(1007) >= 7)[None].expand(2, -1).cuda())))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_unaligned_and_strided_arguments():
    n, h, dk, page = 2, 2, 64, 32
    gpu, ref, _, _ = pair(n, 2, h, dk, page, False)
    fill(gpu, ref)
    base = torch.randn(n * 3 * h * dk * 2 + 1).cuda()
    q = base[1:1 + n * 3 * h * dk].view(n, 3, h, dk)               # off the 16-byte border
    want = gpu.attend(q.clone(), 40)
    assert torch.equal(gpu.attend(q, 40), want)
    qt = q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)    # dense in another dimension
    assert torch.equal(gpu.attend(qt, 40), want)
    wide = torch.full((n, 3, h, 2 * dk), 7.0).cuda()
    assert gpu.attend(q, 40, out=wide[..., dk:]) is not None and torch.equal(wide[..., dk:], want) and float(wide[..., :dk].min()) == 7.0
    odd = torch.zeros(n * 3 * h * dk + 1).cuda()[1:].view(n, 3, h, dk)
    assert torch.equal(gpu.attend(q, 40, out=odd), want) and torch.equal(odd, want)
    m = torch.rand((n, 128), generator=torch.Generator().manual_seed(5)).cuda() < 0.5
    assert torch.equal(gpu.attend(q, 40, key_mask=m[:, ::2]), gpu.attend(q, 40, key_mask=m[:, ::2].contiguous()))
    assert torch.equal(gpu.attend(q, 40, key_mask=m[:1].expand(n, -1)), gpu.attend(q, 40, key_mask=m[:1].repeat(n, 1)))
    a, b = gpu.load(64), None
    gpu.store(qt, q, start=9)
    b = gpu.load(64)
    gpu.store(q.clone(), q.clone(), start=9)
    assert all(torch.equal(x, y) for x, y in zip(b, gpu.load(64))) and not torch.equal(a[0], b[0])


@pytest.mark.parametrize("G,Lq,keys", [(1, 1, 3000), (8, 1, 3000), (2, 20, 1500)])
def test_every_number_of_parts_gives_the_same_attention(G, Lq, keys):
    h, dk, page = 2, 64, 32
    per = -(-keys // page)
    gpu, ref, tab, rtab = pair(1, per, h, dk, page, True, seed=29)
    fill(gpu, ref)
    q = torch.randn((1, Lq, h * G, dk), generator=torch.Generator().manual_seed(1)) * 0.2
    want = ref.attend(q, [keys], rtab, per)
    lim = attend_bound(*want, dk, keys, torch.float32)
    for splits in (1, 2, 3, 17, 64, 1000):
        o = gpu.attend(q.cuda(), keys, table=tab, splits=splits)
        assert bool(((o.cpu().double() - want[0]).abs() <= lim).all()), splits


def test_streams_and_replayed_graphs():
    n, h, G, dk, page, per = 4, 2, 2, 64, 32, 40
    gpu, ref, tab, _ = pair(n, per, h, dk, page, True, seed=31)
    fill(gpu, ref)
    g = torch.Generator().manual_seed(1)
    k, v, q = (torch.randn((n, 1, m, dk), generator=g).cuda() for m in (h, h, h * G))
    start, lens = ints([3, 900, 64, 1200]), ints([4, 901, 65, 1201])

    def step():
        gpu.store(k, v, start=start, table=tab)
        return gpu.attend(q, lens, table=tab), gpu.load(5, start=start, table=tab)[0]

    saved = [t.clone() for t in (gpu.k, gpu.v, gpu.k_exp, gpu.v_exp)]
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                             # two graphs of the same cache, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for rep in range(3):
        for gr, out in graphs:
            for t, s in zip((gpu.k, gpu.v, gpu.k_exp, gpu.v_exp), saved):
                t.copy_(s)
            k.normal_(generator=torch.Generator(device="cuda").manual_seed(rep))
            q.mul_(1.01)
            gr.replay()
            got = [t.clone() for t in out]
            torch.cuda.synchronize()
            for t, s in zip((gpu.k, gpu.v, gpu.k_exp, gpu.v_exp), saved):
                t.copy_(s)
            assert all(torch.equal(a, b) for a, b in zip(got, step())), rep
