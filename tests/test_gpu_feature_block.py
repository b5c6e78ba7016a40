"""channel_norm, gated_mix, channel_dropout and channel_mix as a network's block uses them, up to a CRF's unaries, and sizes between those that the
operators' own tests name."""
import math
import random

import pytest
import torch

import gated_reference
import norm_reference
from mix_reference import assert_within
from test_gpu_gated_mix import make, train

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


def parameters(k, h, labels, dtype=F32):
    g = torch.Generator().manual_seed(11)
    t = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    p = {"w1": 1 + 0.1 * t(k), "b1": 0.1 * t(k), "gate": t(k, h) / math.sqrt(k), "up": t(k, h) / math.sqrt(k), "down": t(h, k) / math.sqrt(h),
         "w2": 1 + 0.1 * t(k), "scale": 0.5 + 0.1 * t(k), "w3": 1 + 0.1 * t(k), "head": t(k, labels) / math.sqrt(k), "bias": t(labels)}
    return {m: v.to(dtype).cuda() for m, v in p.items()}


def block(plb, x, p, seed):
    """norm before, feed-forward block, norm after with dropout, gate and residual, and the norm that the labels' map reads."""
    a = plb.channel_norm(x, before=plb.Norm(p["w1"], p["b1"]))
    f = plb.gated_mix(a, p["gate"], p["up"], p["down"])
    _, y = plb.channel_norm(f, x, p["scale"], after=plb.Norm(p["w2"], kind="rms"), before=plb.Norm(p["w3"], kind="rms"), dropout=0.25, seed=seed)
    return plb.channel_mix(plb.channel_dropout(y, 0.1, (5, 6)), p["head"], p["bias"])


def plain(x, p, keep, keep2):
    k = x.shape[-1]
    rms = lambda v, w: v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w   # noqa: E731
    a = torch.nn.functional.layer_norm(x, (k,), p["w1"], p["b1"], 1e-5)
    f = (torch.nn.functional.silu(a @ p["gate"]) * (a @ p["up"])) @ p["down"]
    h = x + p["scale"] * torch.where(keep, rms(f, p["w2"]) / 0.75, 0.0)
    return torch.where(keep2, rms(h, p["w3"]) / 0.9, 0.0) @ p["head"] + p["bias"]


def test_block_and_its_gradients(plb):
    x = torch.randn(2, 33, 45, 32, generator=torch.Generator().manual_seed(3)).cuda()
    p, seed = parameters(32, 96, 21), torch.tensor([3, 4], device="cuda")
    g = torch.randn(2, 33, 45, 21, generator=torch.Generator().manual_seed(4)).cuda()
    leaves = {"x": x.clone().requires_grad_(True), **{m: v.clone().requires_grad_(True) for m, v in p.items()}}
    out = block(plb, leaves["x"], leaves, seed)
    got = torch.autograd.grad(out, list(leaves.values()), g)
    wide = {m: v.detach().double().requires_grad_(True) for m, v in leaves.items()}
    want = plain(wide["x"], wide, norm_reference.kept(x.shape, 0.25, 3, 4), norm_reference.kept(x.shape, 0.1, 5, 6))
    grads = torch.autograd.grad(want, list(wide.values()), g.double())
    # each of the five operators is some 1e-6 off at most, in the norm, and what follows it grows that by less than ten
    near = lambda a, b: float((a.double() - b).norm() / b.norm()) < 5e-5   # noqa: E731
    assert near(out.detach(), want.detach())
    for m, a, b in zip(leaves, got, grads):
        assert near(a, b), m


def test_block_before_a_crf_in_training(plb):
    """Unaries from the block, messages from the lattices: every parameter gets a gradient, the same one again, and the same in a captured graph."""
    g = torch.Generator().manual_seed(9)
    image = torch.rand(1, 24, 31, 3, generator=g).cuda()
    x = torch.randn(1, 24, 31, 16, generator=g).cuda()
    up = torch.randn(1, 24, 31, 5, generator=g).cuda()
    p, seed = parameters(16, 48, 5), torch.tensor([7, 8], device="cuda")

    def step():
        leaves = {m: v.detach().requires_grad_(True) for m, v in p.items()}
        q = plb.DenseCRF(image, 5, 8.0, 0.125).infer(block(plb, x, leaves, seed), 2)
        return (q.detach(),) + torch.autograd.grad(q, list(leaves.values()), up)

    first = step()
    assert all(bool(torch.isfinite(t).all()) and bool((t != 0).any()) for t in first)
    for a, b in zip(first, step()):       # (the filters' sums are not in a fixed order)
        assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max())

    def features():
        leaves = {m: v.detach().requires_grad_(True) for m, v in p.items()}
        out = block(plb, x, leaves, seed)
        return (out.detach(),) + torch.autograd.grad(out, list(leaves.values()), up)

    want = features()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = features()
    for numbers in ((7, 8), (9, 10)):
        seed.copy_(torch.tensor(numbers))
        want = features()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found, want))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gated_mix_of_many_sizes(plb, dtype):
    """Every way to lay out buffers, and rows that come by the TMA beside rows that do not."""
    rng = random.Random(17)
    sizes = [(rng.choice([1, 5, 130, 700]), rng.randint(1, 128), rng.randint(1, 512), rng.randint(1, 128)) for _ in range(16)]
    sizes += [(rng.choice([3, 129, 800]), 8 * rng.randint(1, 16), 8 * rng.randint(1, 64), 8 * rng.randint(1, 16)) for _ in range(16)]
    sizes += [(20_001, 64, 130, 21), (20_001, 21, 64, 64), (19_003, 128, 512, 7), (19_003, 128, 512, 120), (40_000, 64, 64, 64), (38_000, 16, 32, 16)]
    for rows, k, h, n in sizes:
        biases, residual = rng.choice(["", "g", "ud", "gud"]), rng.random() < 0.7
        a, grad = make(rows, k, h, n, dtype, biases, residual)
        out, d = train(plb, a, grad)
        want = gated_reference.gated(a, "silu", 0.75, grad)
        assert_within(out, *want["out"], "out of %s" % ((rows, k, h, n, biases),))
        for m, t in d.items():
            assert_within(t, *want[m], "%s of %s" % (m, (rows, k, h, n, biases)))


@pytest.mark.parametrize("which", ["x", "residual", "grad"])
def test_one_operand_between_16_byte_boundaries(plb, which):
    for dtype in (BF16, F32):
        a, grad = make(700, 64, 96, 32, dtype)
        want, dwant = train(plb, a, grad)

        def moved(t):
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            return flat[1:].view(t.shape).copy_(t)

        b = dict(a)
        if which != "grad":
            b[which] = moved(a[which])
        leaves = {m: (b[m].detach() if m == which else t.clone()).requires_grad_(True) for m, t in b.items() if t is not None}
        out = plb.gated_mix(**{**b, **leaves}, residual_scale=0.75)
        got = torch.autograd.grad(out, list(leaves.values()), moved(grad) if which == "grad" else grad)
        assert torch.equal(out, want)
        for m, t in zip(leaves, got):
            assert torch.equal(t, dwant[m]), m


def test_operands_of_another_device_are_refused(plb):
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    with pytest.raises(ValueError):
        plb.gated_mix(x, w, w, w.cpu())
    with pytest.raises(ValueError):
        plb.gated_mix(x, w, w, w, residual=x.cpu())
    with pytest.raises(ValueError):
        plb.channel_norm(x, after=plb.Norm(torch.ones(8)))
    with pytest.raises(ValueError):
        plb.channel_norm(x, after=plb.Norm(), dropout=0.5, seed=torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        plb.channel_dropout(x, 0.5, torch.tensor([1, 2]))


def test_workspaces_of_calls_that_follow_one_another(plb):
    """Weights of one call laid out where those of the call before were: calls on one stream, forward and backward in turn."""
    a, ga = make(3000, 64, 256, 64, BF16)
    b, gb = make(2000, 64, 256, 64, BF16, seed=1)
    want = [train(plb, a, ga), train(plb, b, gb)]
    torch.cuda.synchronize()
    got = [train(plb, *args) for _ in range(5) for args in ((a, ga), (b, gb))]
    for i, (out, d) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and all(torch.equal(d[m], want[i % 2][1][m]) for m in d)
