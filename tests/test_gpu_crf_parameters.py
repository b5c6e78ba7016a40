"""DenseCRF's learned parameters and its points without any label."""
import pytest
import torch

from test_gpu_crf_training import plb  # noqa: F401

pytestmark = pytest.mark.gpu


def _image_and_unaries(shape=(1, 13, 17), labels=5):
    g = torch.Generator().manual_seed(labels)
    return torch.rand(shape + (3,), generator=g).cuda(), (2.0 * torch.randn(shape + (labels,), generator=g)).cuda()


KINDS = {"cpu": lambda t: t, "cpu, double": lambda t: t.double(), "double": lambda t: t.double().cuda(), "bfloat16": lambda t: t.bfloat16().cuda(),
         "transposed": lambda t: t.cuda().t().contiguous().t() if t.dim() == 2 else t.cuda()[:, None].expand(-1, 2).contiguous()[:, 0]}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("learned", ["bilateral_weight", "spatial_weight", "compatibility", "label_bias"])
def test_learned_parameters_are_followed(plb, learned, kind):
    """After a step of an optimizer the CRF goes on with the new values, whatever device, type or order they are kept in."""
    labels = 5
    image, u = _image_and_unaries(labels=labels)
    g = torch.Generator().manual_seed(1)
    start = torch.rand((labels, labels) if learned == "compatibility" else (labels,), generator=g)
    p = KINDS[kind](start).detach().requires_grad_(True)
    crf = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **{learned: p})
    optimizer = torch.optim.SGD([p], lr=0.5)
    results = []
    for _ in range(2):
        fresh = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **{learned: p.detach().to("cuda", torch.float32).contiguous()})
        with torch.no_grad():
            want = fresh.infer(u, 3)
            # the filters' sums come in any order, and a constant compatibility has a kernel of its own: 1e-5 a filter, as elsewhere
            assert float((crf.infer(u, 3) - want).abs().max()) <= 1e-4
        q = crf.infer(u, 3)
        assert float((q.detach() - want).abs().max()) <= 1e-4
        results.append(q.detach())
        optimizer.zero_grad()
        (q * q).sum().backward()
        assert p.grad is not None and p.grad.dtype == p.dtype and p.grad.device == p.device and float(p.grad.abs().sum()) > 0
        optimizer.step()
        with torch.no_grad():
            p.mul_(1.5)
    assert float((results[0] - results[1]).abs().max()) > 1e-2
    assert float((crf.step(results[1], u).detach() - plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **{
        learned: p.detach().to("cuda", torch.float32).contiguous()}).step(results[1], u)).abs().max()) <= 1e-4
