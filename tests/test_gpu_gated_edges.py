"""gated_mix where a tile of rows ends, and at the ends of what its types hold."""
import pytest
import torch

import gated_reference as ref
from mix_reference import assert_within

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


@pytest.mark.parametrize("rows", [1, 63, 64, 100, 128, 130, 40_001])
@pytest.mark.parametrize("dtype,large", [(F16, 300.0), (BF16, 2.0 ** 65), (F32, 2.0 ** 65)])
def test_biases_whose_product_is_beyond_the_type(plb, rows, dtype, large):
    """act(gate_bias) up_bias is more than the type holds, but every row's own values take the biases back to some ones: nothing of the rows that a tile
    has behind the last one may be seen in the sums over rows."""
    for k, h, n in ((16, 32, 16), (21, 42, 5), (120, 256, 120)):
        g = torch.Generator().manual_seed(rows + k)
        # (the channel of ones times a weight of -large is the bias taken back, without a rounding; the others' weights are small beside it)
        x = torch.zeros(1, rows, k)
        x[..., 0] = 1
        t = {"x": x, "residual": None, "gate_weight": torch.zeros(k, h), "up_weight": torch.zeros(k, h), "down_weight": torch.randn(h, n, generator=g),
             "gate_bias": torch.full((h,), large), "up_bias": torch.full((h,), large), "down_bias": torch.randn(n, generator=g)}
        t["gate_weight"][0], t["up_weight"][0] = -large, -large
        t = {m: None if v is None else v.to(dtype).cuda() for m, v in t.items()}
        grad = torch.randn(1, rows, n, generator=g).to(dtype).cuda()
        for activation in ("silu", "gelu", "relu"):
            leaves = {m: v.clone().requires_grad_(True) for m, v in t.items() if v is not None}
            out = plb.gated_mix(**{**t, **leaves}, activation=activation)
            d = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)))
            assert bool((out == t["down_bias"]).all())      # hidden values are zeros
            for m in ("gate_weight", "up_weight", "down_weight", "gate_bias", "up_bias", "down_bias"):
                assert bool(torch.isfinite(d[m]).all()), (m, activation, k)
            # a = 0, so dWd is; u = 0, so dg is; du = da act(0) is; what is left is the sum of dout
            assert not any(d[m].any() for m in d if m != "down_bias")
            assert_within(d["down_bias"], *ref.gated(t, activation, 1.0, grad)["down_bias"], "down_bias")
