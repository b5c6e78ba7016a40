"""DenseCRF's learned parameters and its points without any label."""
import math

import pytest
import torch

from test_gpu_crf_training import FULL, PACKED, _assert_near, _Filter, _matrix, _rounded, _Update, plb  # noqa: F401

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


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("learned", ["bilateral_weight", "compatibility", "label_bias"])
def test_parameters_that_are_learned_no_longer(plb, learned, kind):
    """Frozen after the CRF was made: constants from then on, the unaries still have their gradient."""
    labels = 5
    image, u = _image_and_unaries(labels=labels)
    g = torch.Generator().manual_seed(2)
    p = KINDS[kind](torch.rand((labels, labels) if learned == "compatibility" else (labels,), generator=g)).detach().requires_grad_(True)
    crf = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **{learned: p})
    p.requires_grad_(False)
    fresh = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **{learned: p})
    u.requires_grad_(True)
    results = []
    for c in (crf, fresh):
        q = c.infer(u, 2)
        results.append((q.detach(), *torch.autograd.grad((q * q).sum(), [u])))
    for a, b in zip(*results):
        assert float((a - b).abs().max()) <= 1e-4 * max(1.0, float(b.abs().max()))


class _PaddedUpdate(_Update):
    """A step in 64 bits in which a point without a label comes out as zeros (its gradient, through its output, is zero then)."""

    @staticmethod
    def forward(ctx, qb, qs, wb, ws, bias, u, keep):
        z = bias - u + qb @ wb + qs @ ws
        nothing = (z == -math.inf).all(-1, keepdim=True)
        y = torch.softmax(z.masked_fill(nothing, 0.0), -1).masked_fill(nothing, 0.0)
        ctx.save_for_backward(keep(qb), keep(qs), keep(y), wb, ws)
        return y


ITERATIONS = 3


@pytest.mark.parametrize("checkpoint", [None, "8bit"])
@pytest.mark.parametrize("learned", [False, True])
@pytest.mark.parametrize("shape,labels,compatible", [((2, 7, 9), 5, False), ((1, 11, 6), 21, False), ((1, 11, 6), 21, True), ((1, 4, 5, 6), 3, False),
                                                     ((1, 9, 5), 40, False), ((1, 5, 9), 34, True)])
def test_points_without_a_label(plb, shape, labels, compatible, learned, checkpoint):
    """Padding (every label forbidden) comes out as zeros, sends nothing, and takes no gradient; forbidden labels get nothing."""
    g = torch.Generator().manual_seed(sum(shape) + labels)
    image = torch.rand(shape + (3 if len(shape) == 3 else 1,), generator=g).cuda()
    u = 2.0 * torch.randn(shape + (labels,), generator=g)
    u = torch.where(torch.rand(u.shape, generator=g) < 0.2, math.inf, u)
    padding = torch.rand(shape, generator=g) < 0.15
    padding.view(-1)[0] = True
    u[padding] = math.inf
    u, padding = u.cuda(), torch.isinf(u).all(-1).cuda()      # (of three labels some points have all forbidden one by one)
    grad = torch.randn(shape + (labels,), generator=g).cuda()
    compatibility = torch.rand((labels, labels), generator=g) if compatible else 1.0 - torch.eye(labels)
    params = [torch.tensor(1.5), torch.tensor(0.75), compatibility, torch.randn(labels, generator=g) if learned else torch.zeros(labels)]
    if learned:
        leaves = [p.cuda().requires_grad_(True) for p in params]
        crf = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, *leaves, checkpoint=checkpoint)
    else:
        leaves = []
        crf = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, 1.5, 0.75, compatibility if compatible else None, checkpoint=checkpoint)
    with torch.no_grad():
        plain = crf.infer(u, ITERATIONS)
    u.requires_grad_(True)
    out = crf.infer(u, ITERATIONS)
    got = torch.autograd.grad(out, [u] + leaves, grad)

    b, n = crf.bilateral.call.batch, crf.bilateral.call.n
    mats = [[_matrix(lat, labels, r) for r in (False, True)] for lat in (crf.bilateral, crf.spatial)]
    wide = u.detach().double().cpu().view(b, n, labels).requires_grad_(True)
    wp = [p.double().requires_grad_(True) for p in params]
    keep = _rounded if checkpoint else (lambda t: t)
    nothing = torch.isinf(wide.detach()).all(-1, keepdim=True)
    q = torch.softmax(-wide.masked_fill(nothing, 0.0), -1).masked_fill(nothing, 0.0)
    for _ in range(ITERATIONS):
        q = _PaddedUpdate.apply(_Filter.apply(q, *mats[0]), _Filter.apply(q, *mats[1]), -wp[0] * wp[2], -wp[1] * wp[2], wp[3], wide, keep)
    want = torch.autograd.grad(q, [wide] + wp[:len(leaves)], grad.double().cpu().view(b, n, labels))

    for o in (plain, out.detach(), crf.infer(u.detach(), 0), crf.infer(u, 0).detach()):
        assert bool(torch.isfinite(o).all()) and bool((o[padding] == 0).all()) and bool((o[torch.isinf(u.detach())] == 0).all())
        assert float((o.sum(-1) - (~padding).float()).abs().max()) <= 1e-5
    _assert_near(plain, q.detach().reshape(out.shape), FULL, "q")
    _assert_near(out, q.detach().reshape(out.shape), FULL, "q")
    assert bool((got[0][torch.isinf(u.detach())] == 0).all())
    for name, a, w in zip(("unaries", "bilateral_weight", "spatial_weight", "compatibility", "label_bias"), got, want):
        _assert_near(a, w, PACKED if checkpoint else FULL, name)


@pytest.mark.parametrize("labels", [1, 2, 5, 33, 128])
def test_the_start_of_an_inference(plb, labels):
    """The kernel's softmax and its gradient; torch's where torch follows the unaries or the kernel does not take them."""
    g = torch.Generator().manual_seed(labels)
    u = 3.0 * torch.randn((2, 50, labels), generator=g)
    u[torch.rand(u.shape, generator=g) < 0.3] = math.inf
    u[0, 3] = math.inf
    u[:, 7] = 1.0
    grad = torch.randn(u.shape, generator=g)
    nothing = torch.isinf(u).all(-1, keepdim=True)
    wide = u.double().requires_grad_(True)
    want = torch.softmax(-wide.masked_fill(nothing, 0.0), -1).masked_fill(nothing, 0.0)
    (want_du,) = torch.autograd.grad(want, [wide], grad.double())
    for x in (u.cuda(), u, u.cuda().double(), u.cuda().transpose(0, 1).contiguous().transpose(0, 1)):
        leaf = x.clone().requires_grad_(True) if x.is_contiguous() else x.detach().requires_grad_(True)
        q = plb.DenseCRF._start(leaf)
        (du,) = torch.autograd.grad(q, [leaf], grad.to(q))
        # an exponential, a quotient and a sum of up to 128 terms: 1e-6 as elsewhere; the gradient's sum of up to 128 products of
        # values and upstream gradients of up to 5 again
        assert float((q.detach().cpu().double() - want.detach()).abs().max()) <= 1e-6
        assert float((du.cpu().double() - want_du).abs().max()) <= 1e-5
        assert not bool(q.detach().cpu()[nothing.expand(u.shape)].any()) and not bool(du.cpu()[torch.isinf(u)].any())
        with torch.no_grad():
            assert float((plb.DenseCRF._start(leaf) - q).abs().max()) <= 1e-6
    padded = torch.func.vmap(plb.DenseCRF._start)(u.cuda())
    assert float((padded.cpu().double() - want.detach()).abs().max()) <= 1e-6


def test_unaries_that_are_a_parameter_start_in_the_kernel(plb):
    from permutohedral_lattice_b200 import capi
    u = torch.nn.Parameter(torch.randn((1, 30, 5), generator=torch.Generator().manual_seed(1)).cuda())
    want = torch.softmax(-u.detach().double(), -1)
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled):
            before = capi.lib().pl_launch_count()
            q = plb.DenseCRF._start(u)
            assert capi.lib().pl_launch_count() == before + 1 and type(q) is torch.Tensor and q.requires_grad == enabled
            assert float((q.detach() - want).abs().max()) <= 1e-6
    (du,) = torch.autograd.grad((plb.DenseCRF._start(u) ** 2).sum(), [u])
    d = want * (2 * want - (2 * want * want).sum(-1, keepdim=True))
    assert float((du + d).abs().max()) <= 1e-5
