"""Gradients of gated_mix in float16 where the upstream gradient is small, as a mean's over many points is: hidden gradients that
float16 does not hold (2^-25 is nothing to it) are still there in the sums over rows.

Bounds.  dout's largest value becomes 2^-6 to 2^-5 by a power of two; dg and du then lose 2^-22 of themselves (rounded once: 2^-11) and 2^-25, which is 2^-19 of that
value.  Sums of one sign over 8192 rows are cut 512 times, 0.72 2^-24 of half the sum on average: 2^-16.  With the result's rounding, 2^-11 of it: 2^-11 + 2^-14 in
the norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16 = torch.float16
NAMES = ("x", "gate_weight", "up_weight", "down_weight", "gate_bias", "up_bias", "down_bias")


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


def make(rows, k, h, n, size):
    """All of one sign, so that sums over rows grow with their number."""
    g = torch.Generator().manual_seed(rows + k)
    t = lambda *s: 0.5 + torch.rand(s, generator=g)   # noqa: E731
    a = {"x": t(rows, k), "gate_weight": t(k, h) / k, "up_weight": t(k, h) / k, "down_weight": t(h, n) / h, "gate_bias": 0.2 * t(h),
         "up_bias": 0.2 * t(h), "down_bias": 0.2 * t(n)}
    return {m: v.to(F16).cuda() for m, v in a.items()}, (t(rows, n) * size).to(F16).cuda()


def gradients(plb, a, grad, **more):
    leaves = [a[m].clone().requires_grad_(True) for m in NAMES]
    out = plb.gated_mix(**dict(zip(NAMES, leaves)), **more)
    return dict(zip(NAMES, torch.autograd.grad(out, leaves, grad)))


def exact(a, grad):
    w = {m: v.double().requires_grad_(True) for m, v in a.items()}
    hidden = torch.nn.functional.silu(w["x"] @ w["gate_weight"] + w["gate_bias"]) * (w["x"] @ w["up_weight"] + w["up_bias"])
    return dict(zip(NAMES, torch.autograd.grad(hidden @ w["down_weight"] + w["down_bias"], [w[m] for m in NAMES], grad.double())))


@pytest.mark.parametrize("round_hidden", [False, True])
@pytest.mark.parametrize("size", [2.0 ** -23, 2.0 ** -20, 2.0 ** -12, 2.0 ** -5, 1.0])
@pytest.mark.parametrize("rows,k,h,n", [(66_000, 64, 256, 64), (70_001, 21, 42, 5), (20_001, 128, 512, 128), (300, 16, 64, 16)])
def test_sums_of_small_gradients(plb, rows, k, h, n, size, round_hidden):
    a, grad = make(rows, k, h, n, size)
    got, want = gradients(plb, a, grad, round_hidden=round_hidden), exact(a, grad)
    for m in NAMES:
        v, e = got[m].double(), want[m]
        held = e.abs() < 65000
        if m == "x":      # what float16 holds of it, half of 2^-24, and of what is above that 2^-11 and what the sums lose
            allowed = 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -14 + (2.0 ** -11 if round_hidden else 0.0)) * e.abs()
            assert bool(((v - e).abs() <= allowed).all()), float(((v - e).abs() / allowed).max())
        elif float(e[held].norm()) > 0:
            # (half a step where the result itself is small)
            floor = 2.0 ** -25 * math.sqrt(int(held.sum()))
            assert float((v - e)[held].norm()) <= floor + (2.0 ** -11 + 2.0 ** -14 + (2.0 ** -11 if round_hidden else 0.0)) * float(e[held].norm()), m


def test_what_is_not_finite_leaves_the_scale_of_other_rows(plb):
    a, grad = make(1000, 32, 96, 24, 2.0 ** -20)
    clean = gradients(plb, a, grad)["x"]
    for bad in (math.inf, -math.inf, math.nan):
        other = grad.clone()
        other[77, 3] = bad
        dx = gradients(plb, a, other)["x"]
        rows = [r for r in range(1000) if r != 77]
        assert torch.equal(dx[rows], clean[rows]) and not bool(torch.isfinite(dx[77]).any())


def test_gradients_of_zeros_and_between_boundaries(plb):
    a, grad = make(777, 21, 42, 5, 2.0 ** -18)
    zeros = gradients(plb, a, torch.zeros_like(grad))
    assert not any(v.any() for v in zeros.values())
    want = gradients(plb, a, grad)
    for off in range(1, 8):
        flat = torch.empty(grad.numel() + off, dtype=F16, device="cuda")
        moved = flat[off:].view(grad.shape).copy_(grad)
        got = gradients(plb, a, moved)
        assert all(torch.equal(got[m], want[m]) for m in NAMES)


@pytest.mark.parametrize("place", [0, 1, 2, 3, 4])
def test_the_largest_one_is_found_wherever_it_is(plb, place):
    """One value of 1 among ones of 2^-20: with it found there is nothing to scale, and a's and da's product of 3e4 stays what float16 holds."""
    a, _ = make(4001, 8, 16, 5, 1.0)
    grad = torch.full((4001, 5), 2.0 ** -20, dtype=F16, device="cuda")
    at = (0, 7, 10_001, grad.numel() - 2, grad.numel() - 1)[place]
    grad.view(-1)[at] = 1.0
    a["up_bias"].fill_(30000.0)
    got, want = gradients(plb, a, grad), exact(a, grad)
    for m in ("gate_weight", "gate_bias", "up_weight"):
        assert bool(torch.isfinite(got[m]).all())
        assert float((got[m].double() - want[m]).norm()) <= 2.0 ** -10 * float(want[m].norm()), m


def test_a_captured_step_scales_by_what_it_finds(plb):
    a, grad = make(3000, 32, 64, 16, 2.0 ** -4)
    gradients(plb, a, grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = gradients(plb, a, grad)
    for size in (1.0, 2.0 ** -10, 2.0 ** -16):
        grad.copy_(make(3000, 32, 64, 16, 2.0 ** -4 * size)[1])
        graph.replay()
        torch.cuda.synchronize()
        want = gradients(plb, a, grad)
        assert all(torch.equal(found[m], want[m]) for m in NAMES)


def test_two_steps_at_once_have_scales_of_their_own(plb):
    calls = [make(5000, 64, 128, 64, size) for size in (2.0 ** -20, 1.0)]
    want = [gradients(plb, *c) for c in calls]
    sides = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        got = []
        for side, c in zip(sides, calls):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(gradients(plb, *c))
        for side in sides:
            torch.cuda.current_stream().wait_stream(side)
        for g, w in zip(got, want):
            assert all(torch.equal(g[m], w[m]) for m in NAMES)


def test_the_largest_one_beyond_2_31(plb):
    """Only the last rows, whose values lie beyond 2^31 of dout, are not zeros: their scale is found there."""
    rows, last, k = (1 << 31) // 16 + 300, 200, 16
    a, few = make(last, k, 32, 16, 2.0 ** -20)
    want = exact(a, few)
    x = torch.zeros(rows, k, dtype=F16, device="cuda")
    grad = torch.zeros(rows, 16, dtype=F16, device="cuda")
    x[-last:], grad[-last:] = a["x"], few
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("gate_weight", "up_weight", "gate_bias", "up_bias")}
    out = plb.gated_mix(x, leaves["gate_weight"], leaves["up_weight"], a["down_weight"], leaves["gate_bias"], leaves["up_bias"], a["down_bias"])
    for (m, leaf), d in zip(leaves.items(), torch.autograd.grad(out, list(leaves.values()), grad)):
        floor = 2.0 ** -25 * math.sqrt(d.numel())
        assert float((d.double() - want[m]).norm()) <= floor + (2.0 ** -11 + 2.0 ** -14) * float(want[m].norm()), m
