"""channel_dropout's backward pass makes the gradients that are wanted, and no other tensor."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("wanted", [("x",), ("residual",), ("x", "residual")])
def test_only_what_is_wanted(plb, wanted, dtype):
    g = torch.Generator().manual_seed(1)
    x, residual, grad = (torch.randn(1 << 20, generator=g).to(dtype).cuda() for _ in range(3))
    leaves = {"x": x, "residual": residual}
    for m in wanted:
        leaves[m].requires_grad_(True)
    out = plb.channel_dropout(x, 0.25, (3, 4), residual=residual, residual_scale=0.5)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(out, [leaves[m] for m in wanted], grad)
    assert torch.cuda.max_memory_allocated() - before == len(wanted) * grad.nbytes
    keep = plb.channel_dropout(torch.ones_like(grad), 0.25, (3, 4)) != 0
    for m, t in zip(wanted, got):
        want = (0.5 * grad.float()) if m == "residual" else torch.where(keep, grad.float() * (1 / 0.75), torch.zeros_like(grad, dtype=torch.float32))
        assert torch.equal(t, want.to(dtype))
