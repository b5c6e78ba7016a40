"""Gradients of DenseCRF against the same inference in 64 bits, with the two filters as matrices (each lattice applied to unit
vectors, forward and in reverse: the filter's gradient is defined as the reverse filter, not as the transpose)."""
import numpy as np
import pytest
import torch

import mix_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


def _matrix(lattice, labels, reverse):
    """[B, N, N] float64: column j of item b is the filter's answer to the j-th unit vector."""
    call = lattice.call
    n = call.n
    cols = []
    for j in range(0, n, labels):
        x = torch.zeros((call.batch, n, labels), device="cuda")
        for c in range(min(labels, n - j)):
            x[:, j + c, c] = 1.0
        out = lattice.apply(x.view((call.batch,) + tuple(call.sdims) + (labels,)), reverse=reverse)
        cols.append(out.view(call.batch, n, labels)[:, :, :min(labels, n - j)])
    return torch.cat(cols, -1).double().cpu()


class _Filter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, there, back):
        ctx.back = back
        return there @ x

    @staticmethod
    def backward(ctx, g):
        return ctx.back @ g, None, None


class _Update(torch.autograd.Function):
    """The update in 64 bits, its backward pass at what `keep` makes of the activations."""

    @staticmethod
    def forward(ctx, qb, qs, wb, ws, bias, u, keep):
        y = torch.softmax(bias - u + qb @ wb + qs @ ws, -1)
        ctx.save_for_backward(keep(qb), keep(qs), keep(y), wb, ws)
        return y

    @staticmethod
    def backward(ctx, g):
        qb, qs, y, wb, ws = ctx.saved_tensors
        dz = y * (g - (y * g).sum(-1, keepdim=True))
        flat = dz.reshape(-1, dz.shape[-1])
        return (dz @ wb.T, dz @ ws.T, qb.reshape(flat.shape).T @ flat, qs.reshape(flat.shape).T @ flat, flat.sum(0), -dz, None)


def _rounded(t):
    return torch.from_numpy(ref.unpack(*ref.pack(t.float().numpy()))).view(t.shape)


SHAPES = [((2, 7, 9), 5), ((1, 11, 6), 21), ((1, 4, 5, 6), 3)]


def _case(plb, shape, labels, **kw):
    g = torch.Generator().manual_seed(sum(shape) + labels)
    channels = 3 if len(shape) == 3 else 1
    image = torch.rand(shape + (channels,), generator=g).cuda()
    u = (2.0 * torch.randn(shape + (labels,), generator=g)).cuda()
    grad = torch.randn(shape + (labels,), generator=g).cuda()
    crf = plb.DenseCRF(image, labels, 4.0, 0.4, 1.5, **kw)
    return crf, u, grad


def _wanted(crf, labels, u, grad, iterations, params, keep):
    """Inference and gradients in 64 bits: of the unaries and of bilateral_weight, spatial_weight, compatibility, label_bias."""
    b, n = crf.bilateral.call.batch, crf.bilateral.call.n
    mats = [[_matrix(lat, labels, r) for r in (False, True)] for lat in (crf.bilateral, crf.spatial)]
    u = u.detach().double().cpu().view(b, n, labels).requires_grad_(True)
    params = [p.detach().double().cpu().requires_grad_(True) for p in params]
    wb, ws = (-params[i].reshape(-1, 1) * params[2] for i in (0, 1))
    q = torch.softmax(-u, -1)
    for _ in range(iterations):
        q = _Update.apply(_Filter.apply(q, *mats[0]), _Filter.apply(q, *mats[1]), wb, ws, params[3], u, keep)
    return q.detach(), torch.autograd.grad(q, [u] + params, grad.double().cpu().view(b, n, labels))


def _assert_near(got, want, tolerance, what):
    got, want = got.detach().double().cpu().reshape(want.shape), want
    off = float((got - want).norm() / want.norm())
    assert off <= tolerance, (what, off)


# The filters are within 1e-5 of their sums a pass (their own tests' bound); a gradient goes through two of them an iteration.
ITERATIONS, FULL = 4, 1e-4
# In 8 bits a value within 1e-5 of a border between codes may get either (some in a thousand values): a step of 2^-8 of one
# value in a norm over at least a hundred of them, a handful of times.
PACKED = 1e-2


@pytest.mark.parametrize("checkpoint", [None, "8bit"])
@pytest.mark.parametrize("shape,labels", SHAPES)
def test_gradient_of_the_unaries_with_constant_parameters(plb, shape, labels, checkpoint):
    for compat in (None, torch.rand((labels, labels), generator=torch.Generator().manual_seed(5))):
        crf, u, grad = _case(plb, shape, labels, bilateral_weight=1.5, spatial_weight=0.75, compatibility=compat,
                             checkpoint=checkpoint)
        with torch.no_grad():
            before = crf.infer(u, ITERATIONS)
        u.requires_grad_(True)
        out = crf.infer(u, ITERATIONS)
        assert float((out - before).abs().max()) <= 1e-5          # the same kernels: sums in another order at most
        (du,) = torch.autograd.grad(out, [u], grad)
        c = 1.0 - torch.eye(labels) if compat is None else compat
        params = [torch.tensor(1.5), torch.tensor(0.75), c, torch.zeros(labels)]
        keep = _rounded if checkpoint else (lambda t: t)
        want_q, want = _wanted(crf, labels, u, grad, ITERATIONS, params, keep)
        _assert_near(out, want_q.reshape(out.shape), FULL, "q")
        _assert_near(du, want[0], PACKED if checkpoint else FULL, "unaries")


@pytest.mark.parametrize("checkpoint", [None, "8bit"])
@pytest.mark.parametrize("shape,labels", SHAPES)
def test_gradients_of_learned_parameters(plb, shape, labels, checkpoint):
    g = torch.Generator().manual_seed(labels)
    r = lambda *s: torch.rand(s, generator=g)   # noqa: E731
    for vector in (False, True):
        params = [0.5 + r(labels) if vector else 0.5 + r(), 0.5 + r(labels) if vector else 0.5 + r(1), r(labels, labels), r(labels) - 0.5]
        leaves = [p.cuda().requires_grad_(True) for p in params]
        crf, u, grad = _case(plb, shape, labels, bilateral_weight=leaves[0], spatial_weight=leaves[1], compatibility=leaves[2],
                             label_bias=leaves[3], checkpoint=checkpoint)
        u.requires_grad_(True)
        out = crf.infer(u, ITERATIONS)
        got = torch.autograd.grad(out, [u] + leaves, grad)
        want_q, want = _wanted(crf, labels, u, grad, ITERATIONS, params, _rounded if checkpoint else (lambda t: t))
        _assert_near(out, want_q.reshape(out.shape), FULL, "q")
        for name, a, b in zip(("unaries", "bilateral_weight", "spatial_weight", "compatibility", "label_bias"), got, want):
            assert a.shape == b.shape or name == "unaries"
            _assert_near(a, b, PACKED if checkpoint else FULL, name)
        with torch.no_grad():
            assert float((crf.infer(u, ITERATIONS) - out).abs().max()) <= 1e-5
            one = crf.step(torch.softmax(-u, -1), u)
        assert one.grad_fn is None and bool(torch.isfinite(one).all())


def test_a_training_step_of_a_network_around_the_filters(plb):
    """Features mapped by channel_mix to unaries and to the guide's space, a bilateral filter, the CRF with learned parameters,
    a loss: every parameter gets a finite gradient that is not zero, the same twice up to the filters' sums, and near that
    without 8 bits."""
    g = torch.Generator().manual_seed(11)
    shape, labels = (2, 24, 31), 7
    image = torch.rand(shape + (3,), generator=g).cuda()
    features = torch.randn(shape + (20,), generator=g).cuda()
    target = torch.randint(0, labels, shape, generator=g).cuda()

    def step(checkpoint):
        gg = torch.Generator().manual_seed(12)
        t = lambda *s: torch.randn(s, generator=gg).cuda()   # noqa: E731
        p = [0.3 * t(20, 12), t(12), 0.3 * t(12, labels), t(labels), 1.0 + 0.1 * t(labels), 1.0 + 0.1 * t(labels),
             1.0 - torch.eye(labels).cuda() + 0.1 * t(labels, labels), 0.1 * t(labels)]
        for q in p:
            q.requires_grad_(True)
        hidden = plb.channel_mix(features, p[0], p[1], activation="relu", checkpoint=checkpoint)
        smooth = plb.lattice_filter(hidden, image, True, 5.0, 0.3, reuse_lattice=True)
        unaries = plb.channel_mix(smooth, p[2], p[3], residual=None, checkpoint=checkpoint)
        crf = plb.DenseCRF(image, labels, 5.0, 0.3, 2.0, *p[4:], checkpoint=checkpoint)
        q = crf.infer(unaries, 3)
        loss = -torch.log(q.gather(-1, target[..., None]) + 1e-6).mean()
        loss.backward()
        return [x.grad for x in p]

    full, packed, again = step(None), step("8bit"), step("8bit")
    for a, b, c in zip(full, packed, again):
        assert bool(torch.isfinite(b).all()) and float(b.norm()) > 0
        # activations are half a step of 2^-8 off at most: a few per cent of a gradient
        assert float((a - b).norm() / a.norm()) <= 0.1
        assert float((b - c).norm() / b.norm()) <= 2e-3          # another order of the filters' sums, next to a border


def test_crf_refuses(plb):
    image = torch.rand((1, 6, 7, 3), device="cuda")
    for kw in ({"bilateral_weight": torch.ones(4)}, {"spatial_weight": torch.ones(5, 1)}, {"label_bias": torch.ones(4)},
               {"compatibility": torch.ones(4, 5)}, {"checkpoint": "4bit"}):
        with pytest.raises(ValueError):
            plb.DenseCRF(image, 5, **kw)
    crf = plb.DenseCRF(image, 5, label_bias=torch.zeros(5))
    u = torch.zeros((1, 6, 7, 5), device="cuda")
    with pytest.raises(ValueError):
        crf.step(u[:, :3], u)
    with pytest.raises(TypeError):
        crf.step(u, u.half())
    assert float((crf.infer(u, 2) - 0.2).abs().max()) <= 1e-6
    u.requires_grad_(True)
    (first,) = torch.autograd.grad(crf.infer(u, 2).square().sum(), [u], create_graph=True)
    if first.requires_grad:
        with pytest.raises(RuntimeError):
            first.sum().backward()


def test_inference_without_gradients_keeps_its_launches(plb):
    from permutohedral_lattice_b200 import capi
    image = torch.rand((1, 40, 50, 3), device="cuda")
    u = torch.randn((1, 40, 50, 21), device="cuda")
    crf = plb.DenseCRF(image, 21, 12.0, 0.1, 2.0)
    crf.infer(u, 1)
    count = []
    for x in (u, u.clone().requires_grad_(True)):
        with torch.no_grad():
            before = capi.lib().pl_launch_count()
            q = crf._start(x.detach())
            for _ in range(3):
                q = crf.step(q, x)
            count.append(capi.lib().pl_launch_count() - before)
    assert count[0] == count[1]
    assert np.isfinite(q.cpu().numpy()).all()
