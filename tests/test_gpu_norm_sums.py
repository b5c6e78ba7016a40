"""What the sums over rows of channel_norm's vectors lose, in the norm: biases' gradients, which are sums of what came in, unrounded.

4736 rows of 256 channels are one row for each of 592 CTAs' eight warps.  An addition's rounding is 0.42 2^-24 of the sum on average (a step is 1.44 2^-24 of a value, its
rounding even over it: / sqrt 12); a sum of random signs grows like the root of its terms, so that n additions cost 0.42 sqrt(n / 2) 2^-24 of it.  Eight warps in floats, 0.83;
the CTAs in doubles, nothing; the result, 0.42: 0.93 2^-24, twice of which is allowed.  (592 CTAs in floats, eight chains of 74, would cost 2.7.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_biases_of_norms():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200 as plb

    rows, c = 4736, 256
    g = torch.Generator().manual_seed(4)
    x, grad = torch.randn(rows, c, generator=g).cuda(), torch.randn(rows, c, generator=g).cuda()
    for kind in ("layer", "rms"):
        for place in ("after", "before"):
            bias = torch.zeros(c, device="cuda", requires_grad=True)
            (d,) = torch.autograd.grad(plb.channel_norm(x, **{place: plb.Norm(None, bias, kind)}), bias, grad)
            want = grad.double().sum(0)
            off = float((d.double() - want).norm() / want.norm())
            assert off <= 2 * 0.93 * 2.0 ** -24, (kind, place, off)
