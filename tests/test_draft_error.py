"""The measure of the draft attention's accuracy tests (draft_error.py), on the CPU: the
kernels' roundings pass it, a lost tile, a lost share of a stream or coarser keys do not."""

import pytest

import draft_error

torch = pytest.importorskip("torch")


def stream(n, dtype, seed, h=2, g=4, d=128, t=3):
    gen = torch.Generator().manual_seed(seed)
    scale = torch.rand((1, h, d), generator=gen) * 0.3 + 0.05
    zp = torch.randn((1, h, d), generator=gen) * 3 + 7.5
    code = torch.randint(0, 16, (n, h, d), generator=gen).float()
    k = (code.double() - zp.double()) * scale.double()
    v = torch.randn((n, h, d), generator=gen).to(dtype)
    q = (torch.randn((t, h, g, d), generator=gen) / d ** 0.5).to(dtype)
    return q, k, v, scale.double().expand(n, h, d)


def rounded(q, k, v, dtype, keys=torch.float16, drop=slice(0, 0), share=1.0):
    """The attention with the kernel's roundings; tokens of `drop` weighted by 1 - share."""
    x = torch.einsum("thgd,nhd->thgn", q.double(), k.to(keys).double() if dtype != torch.float32 else k)
    w = torch.exp(x - x.amax(-1, keepdim=True)).to(dtype).double()
    w[..., drop] *= 1 - share
    out = torch.einsum("thgn,nhd->thgd", w, v.double()) / w.sum(-1, keepdim=True)
    return out.to(dtype)


@pytest.mark.parametrize("n", [1, 2, 100, 1000, 6000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_kernels_roundings_pass(dtype, n):
    for seed in range(3):
        q, k, v, scale = stream(n, dtype, seed)
        want, rms = draft_error.expected(q.double(), k, v.double(), scale, torch.ones(n, dtype=torch.bool),
                                         torch.ones((3, n), dtype=torch.bool), dtype)
        assert draft_error.excess(rounded(q, k, v, dtype), want, rms) < 1


@pytest.mark.parametrize("n", [600, 3000, 6000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_lost_tile_does_not(dtype, n):
    q, k, v, scale = stream(n, dtype, n)
    want, rms = draft_error.expected(q.double(), k, v.double(), scale, torch.ones(n, dtype=torch.bool),
                                     torch.ones((3, n), dtype=torch.bool), dtype)
    for first in range(0, n - 127, 128):
        got = rounded(q, k, v, dtype, drop=slice(first, first + 128))
        assert draft_error.excess(got, want, rms) > 1
    # a share of the stream at a wrong weight, as a merge would leave it
    assert draft_error.excess(rounded(q, k, v, dtype, drop=slice(0, n // 2), share=0.1), want, rms) > 1


def test_coarser_keys_do_not():
    """Keys at 8 bits in place of 11, where the logits are what counts."""
    q, k, v, scale = stream(1000, torch.float16, 5)
    q = q * 4
    want, rms = draft_error.expected(q.double(), k, v.double(), scale, torch.ones(1000, dtype=torch.bool),
                                     torch.ones((3, 1000), dtype=torch.bool), torch.float16)
    assert draft_error.excess(rounded(q, k, v, torch.float16), want, rms) < 1
    assert draft_error.excess(rounded(q, k, v, torch.float16, keys=torch.bfloat16), want, rms) > 1
