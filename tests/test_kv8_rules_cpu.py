"""Rules of the 8-bit cache and of the token scores that need no GPU."""
import pytest
import torch


def _cache(heads=1, pages=2):
    from transvae_amd.kv8 import KV8Cache
    k, v = (torch.zeros((pages, heads, 16, 32), dtype=torch.uint8) for _ in range(2))
    return KV8Cache(k, v, *(torch.zeros((pages, heads), dtype=torch.uint8) for _ in range(2)))


@pytest.mark.parametrize("heads", [1, 2, 3, 8, 40])
def test_parts_stay_within_what_the_kernel_takes(heads):
    "1 .. 1024 parts and rows * parts within one launch, whatever the sequences, queries and capacity"
    c = _cache(heads)
    for n in (0, 1, 2, 7, 255, 256, 2047, 70000):
        for rows in (0, 1, 16, 17, 500):
            for keys in (0, 1, 255, 1024, 100000, 1 << 20, (1 << 20) + 16, 1 << 21, (1 << 31) - 1):
                parts = c._splits(n, rows, keys)
                assert 1 <= parts <= 1024, (n, rows, keys, parts)
                assert parts == 1 or n * rows * heads * parts <= 4 * ((1 << 24) - 1), (n, rows, keys, parts)


def test_nothing_to_do_needs_no_workspace():
    "no sequences or no queries, with several parts: a workspace of no elements has no address"
    import ctypes as C
    from transvae_amd import _lib
    P = C.c_void_p(4096)
    for n, Lq in ((0, 1), (2, 0)):
        assert _lib.lib().tvae_kv8_attn(P, 64, 64, 64, P, 64, 64, 64, 0, P, P, P, P, 8, None, 4, None, 5, None, 0, 0, 1, n, 1, 1, Lq, 64, 32, 1.0, 3, None, None) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_have_strides_that_the_kernels_take(dtype):
    "dimensions of one element keep any stride: a slice of one token out of an odd-width buffer too"
    from transvae_amd.kv8 import _rows
    for shape in ((1, 1, 1, 65), (1, 1, 3, 65), (1, 2, 1, 67), (2, 1, 1, 65), (1, 1, 1, 64), (2, 3, 2, 72)):
        base = torch.arange(float(torch.Size(shape).numel())).view(shape).to(dtype)
        t = base[..., :64]
        r, *ld = _rows(t, "t")
        assert all(x * r.element_size() % 16 == 0 for x in ld) and r.data_ptr() % 16 == 0
        assert torch.equal(torch.as_strided(r, r.shape, (*ld, 1), r.storage_offset()), t)


def test_token_logprobs_refuses_forward_mode_derivatives():
    "a tangent would vanish without a word; refused before anything is launched, with and without a gradient asked for"
    import torch.autograd.forward_ad as fwad
    from transvae_amd._lib import TvaeError
    from transvae_amd.loss import token_logprobs
    for needs in (False, True):
        x = torch.zeros(3, 9, requires_grad=needs)
        with fwad.dual_level():
            dual = fwad.make_dual(x, torch.ones(3, 9))
            with pytest.raises(TvaeError, match="forward"):
                token_logprobs(dual)
            with pytest.raises(TvaeError, match="host tensor"):        # no tangent: on to the next check
                token_logprobs(x)
