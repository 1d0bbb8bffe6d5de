"""Token log probabilities at the ends of the range of floats, against the formulas in 64 bits."""
import pytest
import torch

from kv8_reference import score, score_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [25, 200, 1000, 40000])
def test_large_gradients_of_the_entropy_pass_masks_of_the_lowest_value(V, dtype):
    """An entropy's gradient scaled by 2^31 (a loss scale) and more: a class of probability 0 gets none of it, though ln p of a class at
    the lowest value times the gradient is beyond fp32.  Bound: p (|ln p| + H) times the gradient, every factor to a few
    2^-21 (ln p absolutely to (V / 64 + 40) 2^-24 + 2^-20), then the result's own half step."""
    from transvae_amd.loss import token_logprobs
    g = torch.Generator().manual_seed(V)
    x = torch.randn((6, V), generator=g).to(dtype)
    x[0, ::2] = torch.finfo(dtype).min
    x[1, 1:] = torch.finfo(dtype).min
    x[2, 3] = -1e30
    x[3] = 1e30
    x[3, 5:] = torch.finfo(dtype).min
    x[4, 2:V - 2] = -torch.inf
    ge = torch.tensor([2.0 ** 31, 1e12, 1e9, 1e20, 3e30, 1e30])
    xg = x.cuda().requires_grad_()
    got, = torch.autograd.grad(token_logprobs(xg)[1], xg, ge.cuda())
    want = score_grad(x, None, torch.zeros((6, 0), dtype=torch.int64), None, ge, None)
    _, H, _, _ = score(x, None, 0)
    top = x.double().amax(1, keepdim=True)
    lp = (x.double() - top) - torch.logsumexp(x.double() - top, 1, keepdim=True)
    p = lp.exp()
    size = p * (lp.abs().clamp(max=1e3) + H[:, None] + 1) * ge.double()[:, None]
    lim = size * ((V / 64 + 40) * 2.0 ** -23 + 2.0 ** -18) + torch.finfo(dtype).eps / 2 * want.abs()
    off = (got.cpu().double() - want).abs()
    assert bool((off <= lim).all()), (float(off.max()), (~(off <= lim)).nonzero()[:4].tolist())
