"""gated_mix and its gradients against a plain form in 64 bits (gated_reference.py derives the bounds)."""
import math

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


def make(rows, k, h, n, dtype=F32, biases="gud", residual=True, seed=0):
    """biases: which of gate, up, down."""
    g = torch.Generator().manual_seed(1000003 * seed + 131 * rows + 17 * k + 7 * h + n)
    t = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    a = {"x": t(1, rows, k), "residual": t(1, rows, n), "gate_weight": t(k, h) / math.sqrt(k), "up_weight": t(k, h) / math.sqrt(k),
         "down_weight": t(h, n) / math.sqrt(h), "gate_bias": t(h), "up_bias": t(h), "down_bias": t(n)}
    grad = t(1, rows, n).to(dtype).cuda()
    for name in ("gate", "up", "down"):
        if name[0] not in biases:
            a[name + "_bias"] = None
    if not residual:
        a["residual"] = None
    return {m: None if v is None else v.to(dtype).cuda() for m, v in a.items()}, grad


def train(plb, a, grad, activation="silu", scale=0.75, wanted=None):
    leaves = {m: t.clone().requires_grad_(wanted is None or m in wanted) for m, t in a.items() if t is not None}
    out = plb.gated_mix(**{**a, **leaves}, activation=activation, residual_scale=scale)
    names = [m for m, t in leaves.items() if t.requires_grad]
    return out.detach(), dict(zip(names, torch.autograd.grad(out, [leaves[m] for m in names], grad)))


SHAPES = [(1, 16, 64, 16), (1, 1, 1, 1), (5, 8, 8, 8), (128, 16, 32, 16), (129, 32, 128, 32), (130, 64, 256, 64), (300, 21, 42, 21), (257, 75, 128, 21),
          (64, 128, 512, 128), (400, 128, 512, 128), (1000, 7, 33, 5), (777, 100, 300, 90), (130, 128, 64, 8), (130, 8, 64, 128), (2000, 15, 65, 17),
          (513, 120, 200, 127), (200, 112, 160, 112), (40, 96, 96, 96), (300, 3, 512, 3), (260, 127, 511, 1), (260, 1, 129, 127)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,h,n", SHAPES)
def test_forward_and_gradients(plb, rows, k, h, n, dtype):
    for activation, biases, residual in (("silu", "gud", True), ("gelu", "", False), ("sigmoid", "g", True), ("relu", "ud", False)):
        a, grad = make(rows, k, h, n, dtype, biases, residual)
        plain = plb.gated_mix(**a, activation=activation, residual_scale=0.75)
        assert plain.dtype == dtype and plain.shape == (1, rows, n) and plain.grad_fn is None
        want = ref.gated(a, activation, 0.75, grad)
        assert_within(plain, *want["out"], "out of %s" % activation)
        out, d = train(plb, a, grad, activation)
        assert torch.equal(out, plain)
        for m, t in d.items():
            assert t.dtype == dtype and t.shape == a[m].shape
            assert_within(t, *want[m], "%s of %s" % (m, activation))
        _, again = train(plb, a, grad, activation)
        assert all(torch.equal(again[m], d[m]) for m in d)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_each_gradient_by_itself(plb, dtype):
    for rows, k, h, n in ((300, 21, 42, 21), (140, 64, 256, 64)):
        a, grad = make(rows, k, h, n, dtype)
        _, d = train(plb, a, grad)
        for m in d:
            _, one = train(plb, a, grad, wanted=(m,))
            assert torch.equal(one[m], d[m]), m


@pytest.mark.parametrize("rows,k,h,n,dtype", [(150_001, 64, 256, 64, BF16), (100_100, 32, 128, 32, F32), (40_000, 128, 512, 128, F16), (30_003, 128, 96, 128, F32),
                                              (60_007, 75, 128, 21, F32)])
def test_many_tiles_a_cta(plb, rows, k, h, n, dtype):
    a, grad = make(rows, k, h, n, dtype, biases="gd")
    out, d = train(plb, a, grad)
    want = ref.gated(a, "silu", 0.75, grad)
    assert_within(out, *want["out"], "out")
    for m, t in d.items():
        assert_within(t, *want[m], m)
        if dtype == F32:      # in the norm, beside what one rounding of the result makes
            off = float((t.double() - want[m][0]).norm() / want[m][0].norm())
            assert off < 2e-6, (m, off)


def test_gradients_against_differences(plb):
    """Along random directions: (f(t + e v) - f(t - e v)) / 2e of the formula in 64 bits against the kernels' gradient."""
    for activation in ("silu", "gelu", "sigmoid"):
        a, grad = make(65, 7, 33, 6)
        _, d = train(plb, a, grad, activation)

        def f(t):
            return (ref.gated(t, activation, 0.75)["out"][0] * grad.double()).sum()

        wide = {m: t.double() for m, t in a.items()}
        for m, t in d.items():
            v = torch.randn(t.shape, generator=torch.Generator().manual_seed(3)).cuda().double()
            e = 1e-5
            slope = (f({**wide, m: wide[m] + e * v}) - f({**wide, m: wide[m] - e * v})) / (2 * e)
            assert abs(float(slope) - float((t.double() * v).sum())) <= 1e-5 * (float((t.double() * v).abs().sum()) + 1.0), (m, activation)


def test_bad_values_stay_in_their_row(plb):
    for dtype in (F32, BF16):
        a, _ = make(300, 21, 42, 21, dtype)
        clean = plb.gated_mix(**a)
        a["x"][0, 7, 20], a["x"][0, 140, 0], a["residual"][0, 299, 3] = math.nan, math.inf, math.nan
        out = plb.gated_mix(**a)
        rows = [r for r in range(300) if r not in (7, 140, 299)]
        assert torch.equal(out[0, rows], clean[0, rows])
        assert bool(torch.isnan(out[0, 7]).all()) and not bool(torch.isfinite(out[0, 140]).any())
        assert bool(torch.isnan(out[0, 299, 3])) and torch.equal(out[0, 299, 4:], clean[0, 299, 4:])


def test_large_and_small_values(plb):
    """Gates far out either way, and values near the smallest ones."""
    for dtype in (F32, BF16, F16):
        a, grad = make(130, 16, 32, 16, dtype, biases="")
        for factor in (64.0, 2.0 ** -10):
            b = dict(a, x=a["x"] * factor)
            for activation in ("silu", "gelu", "sigmoid"):
                out, d = train(plb, b, grad, activation)
                want = ref.gated(b, activation, 0.75, grad)
                assert_within(out, *want["out"], activation)
                for m, t in d.items():
                    value, bound = want[m]
                    # (sums beyond what float16 holds are its infinity; on the border either is right)
                    most = torch.finfo(dtype).max
                    beyond, border = value.abs() - bound > most * (1 + 2.0 ** -11), value.abs() + bound > most
                    assert bool(torch.isinf(t[beyond]).all())
                    assert_within(t[~border], value[~border], bound[~border], m)


def test_other_orders_streams_and_alignments(plb):
    a, grad = make(200, 24, 64, 16, BF16)
    out, d = train(plb, a, grad)
    b = {}
    for m, t in a.items():      # between 16-byte boundaries
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        b[m] = flat[1:].view(t.shape).copy_(t)
    moved, dm = train(plb, b, grad)
    assert torch.equal(moved, out) and all(torch.equal(dm[m], d[m]) for m in d)
    c = dict(a, x=torch.empty(24, 200, 1, dtype=BF16, device="cuda").permute(2, 1, 0).copy_(a["x"]), gate_weight=a["gate_weight"].t().contiguous().t())
    again, dc = train(plb, c, grad)
    assert torch.equal(again, out) and all(torch.equal(dc[m], d[m]) for m in d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, do = train(plb, a, grad)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, out) and all(torch.equal(do[m], d[m]) for m in d)
    # gate and up the same tensor; an upstream gradient without memory of its own; no second derivative
    w = a["gate_weight"].clone().requires_grad_(True)
    o = plb.gated_mix(a["x"], w, w, a["down_weight"])
    o.sum().backward()
    _, two = train(plb, {**a, "up_weight": a["gate_weight"], "residual": None, "gate_bias": None, "up_bias": None, "down_bias": None}, torch.ones_like(grad))
    assert torch.equal(w.grad, two["gate_weight"] + two["up_weight"])
    x = a["x"].clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(plb.gated_mix(x, w, w, a["down_weight"]).sum(), x, create_graph=True)[0].sum().backward()


def test_two_calls_at_once_and_a_captured_one(plb):
    a, grad = make(3000, 64, 256, 64, BF16)
    b, grad_b = make(2000, 32, 128, 32, F32)
    want, want_b = train(plb, a, grad), train(plb, b, grad_b)
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for side, args in zip(sides, ((a, grad), (b, grad_b))):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(train(plb, *args))
        for side in sides:
            torch.cuda.current_stream().wait_stream(side)
        for g, w in zip(got, (want, want_b)):
            assert torch.equal(g[0], w[0]) and all(torch.equal(g[1][m], w[1][m]) for m in w[1])
    torch.cuda.synchronize()
    graphs = []
    for args in ((a, grad), (b, grad_b)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            found = train(plb, *args)
        graphs.append((graph, found))
    a["x"].neg_()
    want = train(plb, a, grad)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for (_, g), w in zip(graphs, (want, want_b)):
        assert torch.equal(g[0], w[0]) and all(torch.equal(g[1][m], w[1][m]) for m in w[1])


def test_empty_tensors(plb):
    a, _ = make(0, 21, 42, 5)
    out, d = train(plb, a, torch.zeros(1, 0, 5, device="cuda"))
    assert out.shape == (1, 0, 5) and d["x"].shape == (1, 0, 21) and all(bool((d[m] == 0).all()) for m in d)


@pytest.mark.parametrize("k", [1, 16, 75, 128])
def test_biases_far_above_the_products_cost_the_sums_nothing(plb, k):
    """out = relu(x Wg + 1000) times one: the bias is added once, with a part in 2^23 cut at most, and not to every one of up to 48 products."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(300, k, generator=g).cuda()
    gate = torch.randn(k, 1, generator=g).cuda()
    up, down = torch.zeros(k, 1, device="cuda"), torch.ones(1, 1, device="cuda")
    out = plb.gated_mix(x, gate, up, down, torch.full((1,), 1000.0, device="cuda"), torch.ones(1, device="cuda"), activation="relu")
    want = x.double() @ gate.double() + 1000.0
    # cut: the bias's step, and the two steps of 16 hidden channels of the second product; rounded: on the way out.  u is 1, a its three terms to 2^-27;
    # the eight steps of the products' first terms, whose sums are some 30 here, cut a quarter of such a part.
    assert ((out.double() - want).abs() / want).max().item() <= 4 * 2.0 ** -23


@pytest.mark.parametrize("k", [16, 15])     # by boxes, value by value
def test_values_beyond_2_31(plb, k):
    """Rows whose values lie beyond 2^31 of their tensors, forward and backward, against those rows by themselves."""
    rows, last = (1 << 31) // k + 300, 500
    a, grad = make(last, k, 32, k, BF16, "gud", True)
    far = {m: torch.zeros(1, rows, k, dtype=BF16, device="cuda") for m in ("x", "residual")}
    for m, t in far.items():
        t[:, -last:] = a[m]
    far_grad = torch.zeros_like(far["x"])
    far_grad[:, -last:] = grad
    want = ref.gated(a, "silu", 0.75, grad)
    out, d = train(plb, {**a, **far}, far_grad, wanted=("x", "residual"))
    assert_within(out[:, -last:], *want["out"], "out")
    assert_within(d["x"][:, -last:], *want["x"], "dx")
    assert_within(d["residual"][:, -last:], *want["residual"], "dresidual")
    assert not d["x"][:, :-last].any() and not d["residual"][:, :-last].any()
