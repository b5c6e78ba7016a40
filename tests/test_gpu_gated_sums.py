"""What gated_mix's sums over rows of floats lose, in the norm.

Where the tensor cores add 16 products to a sum they cut it, toward zero: half a step of float32 on average, 0.72 2^-24 of the sum as it is then (a
step is 2^-24 to 2^-23 of a value, 1.44 2^-24 on average).  A sum leaves tensor memory every 256 rows, after 16 such steps.  Sums of random signs grow like the root of
their terms: 16 steps cut 16 (2 / 3) 0.72 2^-24 of it.  The hidden values, the products' terms and the result's rounding are 2^-24 or less each, 2^-23 together.  The CTAs'
sums are added up in doubles."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

OFF = 16 * (2 / 3) * 0.72 * 2.0 ** -24 + 2.0 ** -23


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


# (as many rows as give every CTA of a B200's 148 four tiles, and ragged ones)
@pytest.mark.parametrize("rows,k,h,n", [(75_776, 16, 32, 16), (75_001, 15, 32, 9), (37_888, 32, 64, 32), (9_000, 75, 128, 21)])
def test_gradients_of_weights(plb, rows, k, h, n):
    g = torch.Generator().manual_seed(rows)
    t = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    a = {"x": t(rows, k), "gate_weight": t(k, h) / math.sqrt(k), "up_weight": t(k, h) / math.sqrt(k), "down_weight": t(h, n) / math.sqrt(h),
         "gate_bias": 0.2 * t(h), "up_bias": 0.2 * t(h), "down_bias": 0.2 * t(n)}
    a = {m: v.cuda().requires_grad_(True) for m, v in a.items()}
    grad = t(rows, n).cuda()
    got = torch.autograd.grad(plb.gated_mix(**a), list(a.values()), grad)
    w = {m: v.detach().double().requires_grad_(True) for m, v in a.items()}
    hidden = torch.nn.functional.silu(w["x"] @ w["gate_weight"] + w["gate_bias"]) * (w["x"] @ w["up_weight"] + w["up_bias"])
    want = torch.autograd.grad(hidden @ w["down_weight"] + w["down_bias"], list(w.values()), grad.double())
    for m, v, e in zip(a, got, want):
        off = float((v.double() - e).norm() / e.norm())
        assert off <= OFF, (m, off, OFF)
