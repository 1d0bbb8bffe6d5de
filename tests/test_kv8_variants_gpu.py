"""Attention over the 8-bit cache against a vectorised 64-bit form, for what the loops of tests/kv8_reference.py are too slow to reach:
the precision of its parts, and the kernel variants that only many rows select."""
import math

import pytest
import torch

from kv8_reference import VALUES, attend_bound

pytestmark = pytest.mark.gpu


def cache_of(pages, h, dk, page, n_seq, seed):
    "random codes without NaN and exponents around 1, made on the GPU"
    from transvae_amd.kv8 import KV8Cache
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = KV8Cache.empty(pages, h, dk, page, "cuda:0", n_seq=n_seq)
    for name in ("k", "v"):
        codes = torch.randint(0, 256, c.k.shape, generator=gen, device="cuda", dtype=torch.uint8)
        codes[(codes & 127) == 127] = 126
        getattr(c, name).copy_(codes)
        getattr(c, name + "_exp").copy_(torch.randint(117, 122, c.k_exp.shape, generator=gen, device="cuda", dtype=torch.uint8))
    return c


def attend64(c, q, lens, table=None, causal=True, mask=None, scale=None):
    "what tests/kv8_reference.py's Cache.attend gives, on the GPU and some sequences at a time; lens (n,) on the GPU"
    n, Lq, hq, dk = q.shape
    h, page = c.heads, c.page
    per = c.n_pages // c.n_seq if table is None else table.shape[1]
    ids = torch.arange(n * per, device="cuda").view(n, per) if table is None else table.long()
    L, G = per * page, hq // h
    scale = 1 / math.sqrt(dk) if scale is None else scale
    values = VALUES.cuda()
    out = [torch.empty(q.shape, dtype=torch.float64, device="cuda") for _ in range(2)] + [torch.empty((n, Lq, hq), dtype=torch.float64, device="cuda")]
    some = max(1, (1 << 24) // (L * h * max(dk, Lq * G)))
    for a in range(0, n, some):
        b = slice(a, min(n, a + some))
        B = b.stop - a
        there = (ids[b] >= 0) & (ids[b] < c.n_pages)
        at = torch.where(there, ids[b], torch.zeros_like(ids[b]))
        k, v = (torch.where(there[:, :, None, None, None], values[x[at].long()] * torch.exp2(e[at].double() - 127)[..., None, None], 0.0)
                .transpose(1, 2).reshape(B, h, L, dk).contiguous() for x, e in ((c.k, c.k_exp), (c.v, c.v_exp)))
        qh = q[b].double().view(B, Lq, h, G, dk).permute(0, 2, 1, 3, 4).reshape(B, h, Lq * G, dk).contiguous()
        j, i = torch.arange(L, device="cuda"), torch.arange(Lq, device="cuda")
        ll = lens[b].long().clamp(0, L)
        see = j < (ll[:, None, None] - (Lq - 1 - i if causal else 0 * i)[None, :, None])
        see = see & there.repeat_interleave(page, 1)[:, None]
        if mask is not None:
            seen = torch.zeros((B, L), dtype=torch.bool, device="cuda")
            w = min(L, mask.shape[1])
            seen[:, :w] = mask[b, :w] != 0
            see = see & seen[:, None]
        see = see[:, None, :, None].expand(B, h, Lq, G, L).reshape(B, h, Lq * G, L)
        kt = k.transpose(2, 3).contiguous()
        s = (torch.matmul(qh, kt) * scale).masked_fill(~see, -math.inf)
        qk = (torch.matmul(qh.abs(), kt.abs()) * abs(scale)).masked_fill(~see, 0.0).amax(-1)
        w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        back = lambda x: x.view(B, h, Lq, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Lq, hq, -1)
        out[0][b], out[1][b], out[2][b] = back(torch.matmul(w, v)), back(torch.matmul(w, v.abs())), back(qk[..., None])[..., 0]
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,G", [(1, 4), (9, 2), (5, 8)])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_weights_of_16_bit_queries_are_not_rounded_to_16_bits(dk, Lq, G, dtype):
    """Keys in pairs that differ in one dimension, their values in sign only: what is left of a pair is the difference of two close
    weights, a few thousandths of them, so the result's own rounding is as much smaller and shows how the weights were rounded.
    They may be off by 2^-17 relative; the rest is attend_bound's for fp32."""
    n, h, page, per = 2, 2, 32, 3
    c = cache_of(n * per, h, dk, page, n, dk)
    c.k[:, :, 1::2, 1:] = c.k[:, :, ::2, 1:]
    c.v[:, :, 1::2] = c.v[:, :, ::2] ^ 128
    q = (torch.randn((n, Lq, h * G, dk), generator=torch.Generator().manual_seed(Lq)) * 0.05).to(dtype).cuda()
    lens = torch.tensor([96, 70], dtype=torch.int32).cuda()
    want, wv, qk = attend64(c, q, lens, causal=False)
    lim = attend_bound(want, wv, qk, dk, per * page, torch.float32) + 2.0 ** -17 * wv + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
    off = (c.attend(q, lens, causal=False).double() - want).abs()
    assert bool((off <= lim).all()), float((off / lim).max())


@pytest.mark.parametrize("G,Lq", [(1, 1), (4, 3)])
def test_a_million_tokens_and_a_table_of_as_many(G, Lq):
    "the default number of parts stays within what the join takes; a part sums at most 1152 keys, the join 1024 parts"
    h, dk, page, L = 1, 32, 256, (1 << 20) + 256 * 100
    c = cache_of(L // page, h, dk, page, 1, 3)
    q = (torch.randn((1, Lq, G, dk), generator=torch.Generator().manual_seed(1)) * 0.2).cuda()
    for lens in (L, torch.tensor([L - 5], dtype=torch.int32).cuda(), torch.tensor([300], dtype=torch.int32).cuda()):
        want, wv, qk = attend64(c, q, torch.as_tensor([lens]).cuda() if isinstance(lens, int) else lens)
        off = (c.attend(q, lens).double() - want).abs()
        assert bool((off <= attend_bound(want, wv, qk, dk, 1152 + 1024, torch.float32)).all())


@pytest.mark.parametrize("Lq,n", [(0, 1), (1, 0)])
def test_nothing_to_attend_over_long_sequences(Lq, n):
    "no queries or no sequences, where the tokens would be cut into parts"
    c = cache_of(8, 1, 32, 256, None, 5)
    table = torch.arange(8, dtype=torch.int32).cuda().view(1, 8)[:n]
    for splits in (None, 3):
        assert c.attend(torch.zeros((n, Lq, 1, 32)).cuda(), 2048, table=table, splits=splits).shape == (n, Lq, 1, 32)


def test_one_token_out_of_an_odd_width_buffer():
    "one sequence, one token, one head: strides of single elements are no strides"
    c, d = (cache_of(2, 1, 64, 16, 1, 7) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    k, v, q, out = (torch.randn((1, 1, 1, 65), generator=g).cuda()[..., :64] for _ in range(4))
    dense = lambda x: x.clone(memory_format=torch.contiguous_format).view(64).view(1, 1, 1, 64)
    c.store(k, v, start=9)
    d.store(dense(k), dense(v), start=9)
    assert all(torch.equal(getattr(c, x), getattr(d, x)) for x in ("k", "v", "k_exp", "v_exp"))
    want = c.attend(dense(q), 10)
    assert torch.equal(c.attend(q, 10), want) and c.attend(q, 10, out=out) is out and torch.equal(out, want)


def compare(n, h, G, Lq, dk, page, per, dtype, masked, splits=None, causal=True, seed=11):
    """Ragged sequences (none, one token, all of them), scattered pages, an absent one; codes that no query sees are NaN"""
    keys = per * page
    c = cache_of(n * per + 2, h, dk, page, None, seed)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(n * per + 2, generator=g)[:n * per].view(n, per).to(torch.int32)
    table[n // 2, per - 1] = -1
    lens = torch.randint(0, keys + 1, (n,), generator=g, dtype=torch.int32)
    lens[:4] = torch.tensor([0, 1, keys, keys - 1])[:n]
    table, lens = table.cuda(), lens.cuda()
    mask = None
    if masked:
        mask = (torch.rand((n, keys - 3), generator=g) < 0.6).cuda()
        mask[n - 1] = False
        mask[n - 2, 16:80] = False
    q = (torch.randn((n, Lq, h * G, dk), generator=g) * 0.2).to(dtype).cuda()
    want, wv, qk = attend64(c, q, lens, table, causal, mask)
    live = torch.arange(keys, device="cuda")[None] < lens[:, None]
    if masked:
        live[:, :keys - 3] &= mask
        live[:, keys - 3:] = False
    there = (table >= 0) & (table < c.n_pages)
    pages, dead = table[there].long(), ~live.view(n, per, page)[there]
    for x in (c.k, c.v):
        x[pages] = torch.where(dead[:, None, :, None], torch.full((), 255, dtype=torch.uint8, device="cuda"), x[pages])
    off = (c.attend(q, lens, table=table, causal=causal, key_mask=mask, splits=splits).double() - want).abs()
    lim = attend_bound(want, wv, qk, dk, keys, dtype)
    assert bool((off <= lim).all()), (float((off / lim).nan_to_num(nan=math.inf).max()), (~(off <= lim)).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,h,dk,page,per,splits", [
    (257, 4, 32, 16, 8, None), (513, 4, 64, 32, 4, None), (1025, 4, 128, 64, 2, None), (1025, 8, 256, 128, 1, None), (3001, 3, 32, 16, 33, None),
    (400, 3, 32, 16, 16, 2), (700, 3, 64, 256, 1, 3)])
def test_single_query_rows_a_wave_each(n, h, dk, page, per, splits, masked, dtype):
    "so many rows (rows * parts >= keys a part * dk / 4) that a wave takes a row of its own, as in a large decoding step"
    compare(n, h, 1, 1, dk, page, per, dtype, masked, splits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,G", [(1, 4), (5, 5), (35, 2), (1, 33)])
@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_tiles_a_wave_each_and_a_block_each(dk, Lq, G, dtype):
    """One, two and several tiles of 16 to 64 query rows a key head: 384 tiles of at most 128 keys and more take a wave each (at 256
    dimensions 128), fewer a block each; masked and not, whole and in parts"""
    for masked in (False, True):
        compare(129, 3, G, Lq, dk, 32, 4, dtype, masked)
        compare(3, 2, G, Lq, dk, 64, 9, dtype, masked)
    compare(80, 3, G, Lq, dk, 16, 13, dtype, True, splits=2, causal=False)


def test_a_number_of_rows_may_be_any_number():
    "count as a number, in store and load alike: none below zero, all of them beyond what there are, also past 32 bits"
    c, d = (cache_of(4, 2, 64, 16, 2, 7) for _ in range(2))
    rows = torch.randn((2, 5, 2, 64), generator=torch.Generator().manual_seed(3)).cuda()
    for count, n in ((1 << 40, 5), (7, 5), (3, 3), (0, 0), (-1, 0), (-(1 << 40), 0)):
        c.store(rows, rows, start=2, count=count)
        if n:
            d.store(rows[:, :n], rows[:, :n], start=2)
        assert torch.equal(c.k, d.k) and torch.equal(c.v_exp, d.v_exp)
        k, v = c.load(5, start=2, count=count)
        assert torch.equal(k[:, :n], d.load(5, start=2)[0][:, :n]) and float(k[:, n:].abs().sum() + v[:, n:].abs().sum()) == 0
