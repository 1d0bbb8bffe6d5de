"""Token log probabilities, entropies, alternatives and their gradient (transvae_amd/loss.py token_logprobs) against the
formulas in 64 bits (tests/kv8_reference.py) and against differences."""
import math

import pytest
import torch

from kv8_reference import score, score_grad

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (1, 2, 0), (5, 25, 5), (300, 25, 0), (67, 26, 26), (3, 63, 63), (9, 64, 64), (4, 65, 5), (130, 128, 3), (2, 257, 64),
          (17, 1000, 20), (3, 2048, 4), (3, 2049, 8), (6, 5003, 1), (2, 8191, 64), (4, 30001, 20), (1, 70003, 5), (2, 200000, 64)]


def value_bound(x, lp):
    """How far fp32 may be from a log probability x_y - M - ln l: the differences (x - M is exact to 2^-24 relative), exp2 of a
    rounded argument d log2(e): |d| 2^-23 + 2^-22 relative on terms that weigh e^d, at most 2^-22 + 2^-23 (max of |d| e^d <
    0.37) each; a sum of V terms taken in strands of at most V / 64 and then a tree: (V / 64 + 16) 2^-24; the logarithm 2^-22 relative."""
    V = x.shape[1]
    return (V / 64 + 40) * 2.0 ** -24 + 2.0 ** -22 * (4 + lp.abs().nan_to_num(0, 0, 0))


def close(got, want, lim):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    off = torch.where(torch.isfinite(want), (got - want).abs(), torch.zeros_like(want))
    assert bool((off <= lim).all()), float((off / lim).max())


def check(logits, tokens, top, grads=True, seed=0):
    from transvae_amd.loss import token_logprobs
    x = logits.cuda().requires_grad_(grads)
    rows, V = logits.shape
    logp, ent, tl, ti = token_logprobs(x, None if tokens is None else tokens.cuda(), top=top)
    wl, we, wt, wi = score(logits, tokens, top)
    assert torch.equal(ti.cpu(), wi)
    close(logp, wl, value_bound(logits, wl))
    # entropy: ln l - t / l, t a sum of e^d d: the same relative errors on a sum of magnitude sum p |ln p| = H
    close(ent, we, value_bound(logits, we) + (V / 64 + 40) * 2.0 ** -23 * (1 + we.nan_to_num(0, 0, 0)))
    close(tl, wt, value_bound(logits, wt) if top else torch.zeros_like(wt))
    if not grads:
        return
    g = torch.Generator().manual_seed(seed)
    gl, ge, gt = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn((rows, top), generator=g)
    for use in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        if use == (0, 0, 1) and not top:
            continue
        outs = [o for o, u in zip((logp, ent, tl), use) if u]
        got, = torch.autograd.grad(outs, x, [w.cuda() for w, u in zip((gl, ge, gt), use) if u], retain_graph=True)
        a, b, c = (w if u else None for w, u in zip((gl, ge, gt), use))
        want = score_grad(logits, tokens, wi, a, b, c)
        # every factor is off by at most a few 2^-22 of itself, ln p absolutely by value_bound: times p (|pull| + |g_H| (|ln p| + H))
        lp = torch.log_softmax(logits.double(), 1)
        p = lp.exp()
        size = (gl.abs() + gt.abs().sum(1)).double()[:, None] + ge.abs().double()[:, None] * (lp.abs().nan_to_num(0, 0, 0) + we.nan_to_num(0, 0, 0)[:, None] + 1)
        rel = (V / 64 + 40) * 2.0 ** -22 + 2.0 ** -21 * (4 + lp.abs().nan_to_num(0, 0, 0))
        half = torch.finfo(logits.dtype).eps / 2
        lim = (rel * p * size).nan_to_num(0) + 2.0 ** -22 * want.abs().nan_to_num(0) + half * want.abs().nan_to_num(0) + 2.0 ** -22 * size.nan_to_num(0) * (want != 0) * 1e-3 \
            + torch.finfo(logits.dtype).smallest_normal
        extra = (gl.abs() + gt.abs().sum(1)).double()[:, None] * 2.0 ** -23 * torch.zeros_like(p)
        for r in range(rows):                                      # classes whose own gradient is added: the sum of both parts is rounded
            cols = set(wi[r].tolist()) | ({int(tokens[r])} if tokens is not None and 0 <= int(tokens[r]) < V else set())
            for j in cols:
                extra[r, j] = size[r, j].nan_to_num(0) * 2.0 ** -21
        close(got, want, lim + extra)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top", SHAPES)
def test_values_alternatives_and_gradient(rows, V, top, dtype):
    g = torch.Generator().manual_seed(rows * 7 + V)
    x = (torch.randn((rows, V), generator=g) * 3).to(dtype)        # in 16 bits a long row holds many equal values
    y = torch.randint(-2, V + 2, (rows,), generator=g)             # some are padding
    check(x, y, top, grads=rows * V <= 70003)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 25, 100, 3001, 20000])
def test_masked_classes_and_rows_without_any(V, dtype):
    inf = math.inf
    g = torch.Generator().manual_seed(V)
    x = torch.randn((8, V), generator=g)
    x[0] = -inf                                                    # nothing left
    x[1, 1:] = -inf                                                # one class left
    x[2, torch.rand(V, generator=g) < 0.6] = -inf
    x[3] = torch.finfo(torch.float16).min                          # a mask of the type's lowest value everywhere: uniform
    x[4, :-1] = torch.finfo(torch.float16).min
    x[5] = 0.25                                                    # ties throughout
    x[6] = torch.arange(V) * 0.01                                  # ascending: every value enters the list
    x[7] = 1000.0 + x[7]
    y = torch.randint(0, V, (8,), generator=g)
    x[2, 0] = 1.0
    check(x.to(dtype), y, min(V, 5))


@pytest.mark.parametrize("V", [4, 25, 3001, 30000])
def test_nan_and_infinity_stay_in_their_row(V):
    x = torch.randn((6, V), generator=torch.Generator().manual_seed(V))
    x[1, V // 2] = math.nan
    x[2, V - 1] = math.inf
    x[3] = math.nan
    x[4, :] = math.inf
    x[5, 0], x[5, 1] = math.nan, -math.inf
    check(x, torch.tensor([0, 0, V - 1, 1, 2, 1]), 3, grads=False)
    check(x, torch.tensor([-1] * 6), 3, grads=False)


@pytest.mark.parametrize("V", [20, 700, 9001])
def test_masks_of_the_lowest_value_beside_huge_logits(V):
    "differences that leave fp32's range weigh nothing, and nothing becomes NaN"
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        x = torch.randn((5, V), generator=torch.Generator().manual_seed(V)).to(dtype)
        x[0, ::2] = low
        x[1, 1:] = low
        x[1, 0] = 3e38
        x[2, :] = low
        x[3, V // 2:] = low
        x[3, :V // 2] = 2e31
        x[4, 3] = -low
        from transvae_amd.loss import token_logprobs
        xg = x.cuda().requires_grad_()
        logp, ent, tl, ti = token_logprobs(xg, torch.tensor([1, 0, 2, 0, 3]).cuda(), top=2)
        wl, we, wt, wi = score(x, torch.tensor([1, 0, 2, 0, 3]), 2)
        assert torch.equal(ti.cpu(), wi)
        close(logp, wl, value_bound(x, wl))
        close(ent, we, value_bound(x, we) + 1e-6)
        g, = torch.autograd.grad(logp.sum() + ent.sum() + tl.sum(), xg)
        assert bool(torch.isfinite(g).all())


def test_zeros_of_both_signs_tie():
    x = torch.full((2, 40), -1.0)
    x[0, 7], x[0, 3] = 0.0, -0.0
    x[1, 3], x[1, 7] = 0.0, -0.0
    check(x, None, 4)


@pytest.mark.parametrize("rows,V", [(1, 4099), (2, 30001), (1, 100003), (1, 149999)])
@pytest.mark.parametrize("top", [1, 8, 20, 64])
def test_equal_logits_and_bests_in_one_place_of_long_rows(rows, V, top):
    "long rows are cut into parts: more equal values than a block has threads, all the best in one part, in the last one, none at all"
    g = torch.Generator().manual_seed(V + top)
    for kind in range(6):
        x = torch.randn((rows, V), generator=g)
        if kind == 0:
            x[:] = 0.5
        elif kind == 1:
            x[:] = -math.inf
        elif kind == 2:
            x[:, V // 2:V // 2 + 100] += 20.0
        elif kind == 3:
            x[:, -70:] = 9.0
        elif kind == 4:
            x = x.sort(dim=1).values
        else:
            x = (x * 2).round()                                    # few different values
        check(x, torch.arange(rows) * 37 + V // 2, top, grads=False)


def test_strides_phases_and_leading_dimensions():
    from transvae_amd.loss import token_logprobs
    g = torch.Generator().manual_seed(1)
    for dtype in DTYPES:
        base = torch.randn(4 * 777 + 40, generator=g).to(dtype).cuda()
        for off in (0, 1, 3, 7):
            for V, ld in ((301, 301), (304, 304), (300, 777), (25, 25), (25, 31)):
                x = torch.as_strided(base, (4, V), (ld, 1), off)
                y = torch.randint(0, V, (4, 3), generator=g).cuda()[:, 1]             # a strided column of ids
                a = token_logprobs(x, y, top=3)
                b = token_logprobs(x.clone(), y.clone(), top=3)
                for u, w in zip(a, b):                             # the order of the sums depends on the phase
                    assert torch.allclose(u.double(), w.double(), rtol=1e-5, atol=1e-5)
                assert torch.equal(a[3], b[3])
                xs = x.detach().requires_grad_()
                xc = x.clone().requires_grad_()
                ga, = torch.autograd.grad(sum(t.sum() for t in token_logprobs(xs, y, top=3)[:3]), xs)
                gb, = torch.autograd.grad(sum(t.sum() for t in token_logprobs(xc, y, top=3)[:3]), xc)
                assert torch.allclose(ga.double(), gb.double(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
    x = torch.randn((2, 3, 50), generator=g).cuda()
    y = torch.randint(0, 50, (2, 3), generator=g).cuda()
    for t, o in zip(token_logprobs(x, y, top=2), token_logprobs(x.view(6, 50), y.view(6), top=2)):
        assert torch.equal(t.reshape(o.shape), o) and t.shape[:2] == (2, 3)
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)            # classes are not the dense dimension
    assert torch.equal(token_logprobs(xt, y.int())[0], token_logprobs(x, y)[0])
    one = token_logprobs(x[0, 0], y[0, 0], top=1)
    assert one[0].shape == () and one[2].shape == (1,) and torch.equal(one[0], token_logprobs(x, y)[0][0, 0])
    none = token_logprobs(x[:0], y[:0], top=2)
    assert none[0].shape == (0, 3) and none[3].shape == (0, 3, 2)
    wide = x[:1, :1].expand(4, 2, 50)                              # one row for all
    assert torch.equal(token_logprobs(wide, torch.zeros((4, 2), dtype=torch.int64).cuda())[1], token_logprobs(x[0, 0])[1].expand(4, 2))


@pytest.mark.parametrize("rows,V,top", [(3, 9, 2), (2, 70, 3), (1, 9000, 2)])
def test_gradient_against_differences(rows, V, top):
    """Central differences of the 64-bit definition, step 1e-5: off by step^2 / 6 of the third derivative (< 1e-10 |g|) and by
    1e-16 / 1e-5 of the values (< 1e-9); the kernel itself is fp32."""
    from transvae_amd.loss import token_logprobs
    g = torch.Generator().manual_seed(4)
    x = torch.randn((rows, V), generator=g)
    y = torch.randint(0, V, (rows,), generator=g)
    y[0] = int(x[0].argmax())                                      # the token is an alternative too
    w = [torch.randn(s, generator=g) for s in ((rows,), (rows,), (rows, top))]
    xg = x.cuda().requires_grad_()
    out = token_logprobs(xg, y.cuda(), top=top)
    (sum((o * v.cuda()).sum() for o, v in zip(out, w))).backward()

    def f(z):
        lp = torch.log_softmax(z, 1)
        return (lp.gather(1, y[:, None])[:, 0] * w[0]).sum() - ((lp.exp() * lp).sum(1) * w[1]).sum() + (lp.gather(1, out[3].cpu()) * w[2]).sum()

    cols = sorted(set(y.tolist()) | set(out[3].cpu().view(-1).tolist()) | set(range(0, V, max(1, V // 17))))
    for r in range(rows):
        for c in cols:
            z = x.double()
            z[r, c] += 1e-5
            up = f(z)
            z[r, c] -= 2e-5
            diff = float(up - f(z)) / 2e-5
            assert abs(diff - float(xg.grad[r, c])) <= 2e-6 + 1e-5 * abs(diff), (r, c, diff, float(xg.grad[r, c]))


def test_same_row_whatever_stands_beside_it():
    "a row's results do not depend on how many rows a call has beyond the rule for the parts, nor on the run"
    from transvae_amd.loss import token_logprobs
    x = torch.randn((2000, 30000), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    a = token_logprobs(x, None, top=20)
    b = token_logprobs(x, None, top=20)
    few = token_logprobs(x[:3], None, top=20)
    for u, v, w in zip(a, b, few):
        assert torch.equal(u, v) and torch.allclose(u[:3].double(), w.double(), rtol=1e-6, atol=1e-6)


def test_many_rows_a_wave_each():
    "from 4096 rows on a wave has a row of its own: the same values as in small calls, ties and masked classes included"
    from transvae_amd.loss import token_logprobs
    x = torch.randn((4100, 3000), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    x[5] = 1.0
    x[6] = -math.inf
    x[7, 1:] = -math.inf
    x[8, 2999] = math.nan
    x[9] = torch.arange(3000).float() / 16
    y = torch.arange(4100) % 3001 - 1
    a = token_logprobs(x.cuda(), y.cuda(), top=20)
    check(x[:12], y[:12], 20, grads=False)
    b = token_logprobs(x[:64].cuda(), y[:64].cuda(), top=20)
    assert torch.equal(a[3][:64], b[3])
    for u, w in zip(a[:3], b[:3]):
        assert torch.equal(torch.isnan(u[:64]), torch.isnan(w)) and torch.allclose(u[:64].nan_to_num(0, 0, 0), w.nan_to_num(0, 0, 0), rtol=1e-6, atol=2e-6)
    wl, we, wt, wi = score(x[-30:], y[-30:], 20)
    assert torch.equal(a[3][-30:].cpu(), wi)
    close(a[0][-30:], wl, value_bound(x, wl))
    close(a[2][-30:], wt, value_bound(x, wt))


def test_offsets_past_two_gigabytes():
    "rows * V over 2^31 elements: the last rows are those of a small call"
    from transvae_amd.loss import token_logprobs
    V, rows = 131000, 17000
    x = torch.empty((rows, V), dtype=torch.bfloat16, device="cuda")
    x[-64:].normal_()
    x[:-64] = 0
    y = torch.full((rows,), V - 1, device="cuda")
    xs = x[-64:].clone().requires_grad_()
    x.requires_grad_()
    a = token_logprobs(x, y, top=4)
    b = token_logprobs(xs, y[-64:], top=4)
    assert torch.equal(a[3][-64:], b[3])
    ga, = torch.autograd.grad(a[0].sum() + a[1].sum(), x)
    gb, = torch.autograd.grad(b[0].sum() + b[1].sum(), xs)
    for u, w in ((a[0][-64:], b[0]), (a[1][-64:], b[1]), (ga[-64:], gb)):
        assert torch.allclose(u.float(), w.float(), rtol=1e-2, atol=1e-6)


def test_streams_and_replayed_graphs():
    from transvae_amd.loss import token_logprobs
    for rows, V in ((500, 25), (2, 100003), (64, 5000)):
        x = torch.randn((rows, V)).cuda()
        y = torch.randint(0, V, (rows,)).cuda()
        want = [t.clone() for t in token_logprobs(x, y, top=5)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = token_logprobs(x, y, top=5)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(u, w) for u, w in zip(got, want))
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = token_logprobs(x, y, top=5)
            graphs.append((gr, out))
        for rep in range(3):
            for gr, out in graphs:
                x.normal_()
                gr.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(u, w) for u, w in zip(out, token_logprobs(x, y, top=5)))


def test_captured_gradients_replay():
    "the capture comes before any eager gradient of the same leaf is alive, as for every backward pass"
    from transvae_amd.loss import token_logprobs
    for rows, V, dtype in ((500, 25, torch.float32), (3, 30001, torch.float16), (700, 3001, torch.bfloat16)):
        x = torch.randn((rows, V), generator=torch.Generator().manual_seed(V)).to(dtype).cuda().requires_grad_()
        y = (torch.arange(rows) % V).cuda()
        gl, ge, gt = torch.randn(rows).cuda(), torch.randn(rows).cuda(), torch.randn((rows, 3)).cuda()

        def step():
            logp, ent, tl, _ = token_logprobs(x, y, top=3)
            return torch.autograd.grad((logp, ent, tl), x, (gl, ge, gt))[0]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dx = step()
        for rep in range(4):
            with torch.no_grad():
                x.copy_(torch.randn((rows, V), generator=torch.Generator().manual_seed(rep)))
            gl.normal_(), gt.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(dx, step())
