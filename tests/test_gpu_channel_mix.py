"""channel_mix, its gradients and the 8-bit activations against plain forms in 64 bits (mix_reference.py derives the bounds)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import mix_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


def make(rows, k, k2, n, dtype=F32, weight_dtype=None, bias=True, residual=True, masked=False, seed=0):
    """x, weight, bias, residual, x2, weight2 and an upstream gradient; shape [1, rows, *]."""
    g = torch.Generator().manual_seed(1000003 * seed + 131 * rows + 17 * k + 7 * k2 + n)
    wd = dtype if weight_dtype is None else weight_dtype
    t = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    r = 2.0 * t(1, rows, n)
    if masked:
        r = torch.where(torch.rand((1, rows, n), generator=g) < 0.3, math.inf, r)
        r = torch.where(torch.rand((1, rows, 1), generator=g) < 0.2, math.inf, r)
        r[0, 0] = math.inf
    a = {"x": t(1, rows, k).to(dtype), "weight": (t(k, n) / math.sqrt(k)).to(wd),
         "bias": t(n).to(wd) if bias else None, "residual": r.to(dtype) if residual else None,
         "x2": t(1, rows, k2).to(dtype) if k2 else None, "weight2": (t(k2, n) / math.sqrt(k2)).to(wd) if k2 else None}
    return {m: v.cuda() if v is not None else None for m, v in a.items()}, t(1, rows, n).to(dtype).cuda()


def needs_of(a):
    return tuple(m for m, v in a.items() if v is not None)


SHAPES = [(1, 1, 0, 1), (1, 21, 21, 21), (2, 2, 2, 2), (31, 3, 1, 5), (32, 8, 8, 8), (33, 75, 0, 16), (257, 21, 21, 21),
          (1000, 33, 17, 40), (64, 128, 128, 128), (63, 127, 1, 128), (130, 128, 0, 1), (129, 1, 128, 127), (500, 64, 64, 64),
          (4099, 9, 7, 24), (20011, 21, 21, 21), (12345, 2, 2, 2), (3001, 64, 0, 96), (777, 16, 32, 48), (2051, 100, 100, 10),
          (900, 32, 32, 32), (333, 4, 4, 4), (70, 4, 0, 3), (5000, 16, 16, 16), (257, 40, 40, 24), (260, 24, 56, 32), (100, 72, 8, 8)]


@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("rows,k,k2,n", SHAPES)
def test_forward(plb, rows, k, k2, n, dtype, weight_dtype):
    for activation, scale, bias, residual in ((None, 1.0, False, False), ("relu", 0.5, True, True), ("softmax", -1.0, True, True),
                                              ("softmax", 1.0, False, False)):
        a, _ = make(rows, k, k2, n, dtype, weight_dtype, bias, residual)
        out = plb.channel_mix(**a, activation=activation, residual_scale=scale)
        assert out.dtype == dtype and out.shape == (1, rows, n) and out.grad_fn is None
        want, bound = ref.forward(a["x"], a["weight"], a["bias"], a["residual"], a["x2"], a["weight2"], activation, scale)
        ref.assert_within(out, want, bound, "%s %s" % (activation, scale))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,k,k2,n", [(1, 5, 5, 5), (77, 21, 21, 21), (300, 128, 128, 128), (1025, 2, 2, 2), (640, 1, 0, 1)])
def test_rows_whose_labels_are_forbidden(plb, rows, k, k2, n, dtype):
    """Forbidden labels get exactly nothing, rows without any label zeros, and neither a gradient."""
    a, g = make(rows, k, k2, n, dtype, masked=True)
    out, saved = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0)
    want, bound = ref.forward(a["x"], a["weight"], a["bias"], a["residual"], a["x2"], a["weight2"], "softmax", -1.0)
    ref.assert_within(out, want, bound)
    forbidden = torch.isinf(a["residual"])
    assert bool((out[forbidden] == 0).all()) and bool((out[0, 0] == 0).all())
    needs = needs_of(a)
    d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "softmax", -1.0, needs)
    assert bool((d.residual[forbidden] == 0).all()) and bool((d.x[0, 0] == 0).all())
    for m, (w, b) in ref.gradients(g, out, a["x"], a["weight"], a["x2"], a["weight2"], "softmax", -1.0).items():
        if m in needs:
            ref.assert_within(getattr(d, m), w, b, m)
    big = torch.where(forbidden, torch.tensor(torch.finfo(dtype).max, dtype=dtype, device="cuda"), a["residual"])
    again = plb.channel_mix(**{**a, "residual": big}, activation="softmax", residual_scale=-1.0)   # the type's largest value
    some = ~forbidden.all(-1)
    assert bool(torch.isfinite(again).all()) and torch.equal(again[some], out[some])


def test_bad_values_stay_in_their_row(plb):
    for dtype in (F32, BF16):
        a, _ = make(200, 21, 21, 21, dtype)
        clean = plb.channel_mix(**a, activation="softmax", residual_scale=-1.0)
        a["x"][0, 7, 20] = math.nan
        a["x2"][0, 40, 0] = math.inf
        a["residual"][0, 199, 3] = math.nan
        a["residual"][0, 100, 3] = -math.inf          # a logit of +infinity
        for activation in ("softmax", None, "relu"):
            out = plb.channel_mix(**a, activation=activation, residual_scale=-1.0)
            assert bool(torch.isnan(out[0, 7]).all()) and bool(torch.isnan(out[0, 199, 3]))
            if activation == "softmax":
                assert all(bool(torch.isnan(out[0, r]).all()) for r in (7, 40, 199, 100))
                keep = [r for r in range(200) if r not in (7, 40, 199, 100)]
                assert torch.equal(out[0, keep], clean[0, keep])
            else:
                assert not bool(torch.isfinite(out[0, 40]).any()) or activation == "relu"
                assert bool(torch.isinf(out[0, 100, 3]))


@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,k,k2,n", SHAPES)
def test_gradients(plb, rows, k, k2, n, dtype, weight_dtype):
    for activation, scale in ((None, 0.25), ("relu", 1.0), ("softmax", -1.0)):
        a, g = make(rows, k, k2, n, dtype, weight_dtype)
        out, saved = plb.channel_mix_raw(**a, activation=activation, residual_scale=scale)
        needs = needs_of(a)
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, needs)
        want = ref.gradients(g, out, a["x"], a["weight"], a["x2"], a["weight2"], activation, scale)
        for m in needs:
            assert getattr(d, m).dtype == a[m].dtype and getattr(d, m).shape == a[m].shape
            ref.assert_within(getattr(d, m), *want[m], "%s of %s" % (m, activation))
        again = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, needs)
        assert all(torch.equal(getattr(d, m), getattr(again, m)) for m in needs)
        for m in needs:   # each by itself
            one = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, (m,))
            assert torch.equal(getattr(one, m), getattr(d, m)) and sum(t is not None for t in one) == 1


def test_gradients_against_differences(plb):
    """Along random directions: (f(t + h v) - f(t - h v)) / 2h of the formula in 64 bits against the kernels' gradient."""
    for activation, scale in ((None, 0.5), ("softmax", -1.0)):
        a, g = make(65, 7, 5, 6)
        leaves = {m: t.clone().requires_grad_(True) for m, t in a.items()}
        grads = torch.autograd.grad(plb.channel_mix(**leaves, activation=activation, residual_scale=scale), list(leaves.values()), g)

        def f(t):
            return (ref.forward(t["x"], t["weight"], t["bias"], t["residual"], t["x2"], t["weight2"], activation, scale)[0]
                    * g.double()).sum()

        for (m, t), grad in zip(a.items(), grads):
            v = torch.randn(t.shape, generator=torch.Generator().manual_seed(3)).cuda().double()
            h = 1e-5
            wide = {name: u.double() for name, u in a.items()}
            slope = (f({**wide, m: wide[m] + h * v}) - f({**wide, m: wide[m] - h * v})) / (2 * h)
            # third order: h^2; float gradients: some 1e-6 of the terms' magnitudes
            scale_of = float((grad.double() * v).abs().sum()) + 1.0
            assert abs(float(slope) - float((grad.double() * v).sum())) <= 1e-5 * scale_of, (m, activation)


def test_autograd_routes(plb):
    a, g = make(300, 21, 21, 21)
    raw, saved = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0)
    want = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "softmax", -1.0, needs_of(a))
    leaves = {m: t.clone().requires_grad_(True) for m, t in a.items()}
    out = plb.channel_mix(**leaves, activation="softmax", residual_scale=-1.0)
    assert torch.equal(out, raw)
    out.backward(g)
    for m, t in leaves.items():
        assert torch.equal(t.grad, getattr(want, m)), m
    # one tensor in both places, one weight for both: the gradients add up
    x, w = a["x"].clone().requires_grad_(True), a["weight"].clone().requires_grad_(True)
    out, saved = plb.channel_mix_raw(x, w, x2=x, weight2=w, activation="softmax")
    d = plb.channel_mix_backward(g, saved, w, w, "softmax", 1.0, ("x", "weight", "x2", "weight2"))
    plb.channel_mix(x, w, x2=x, weight2=w, activation="softmax").backward(g)
    assert torch.equal(x.grad, d.x + d.x2) and torch.equal(w.grad, d.weight + d.weight2)
    # an upstream gradient without memory of its own, tensors in other orders, and no second derivative
    leaves = {m: t.clone().requires_grad_(True) for m, t in a.items()}
    strided = {m: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t for m, t in leaves.items()}
    out = plb.channel_mix(**strided, activation="softmax", residual_scale=-1.0)
    assert torch.equal(out, raw)
    first = torch.autograd.grad(out.sum(), list(leaves.values()), create_graph=True)
    ones = plb.channel_mix_backward(torch.ones_like(g), plb.MixSaved(a["x"], a["x2"], raw), a["weight"], a["weight2"], "softmax",
                                    -1.0, needs_of(a))
    assert all(torch.equal(t, getattr(ones, m)) for m, t in zip(leaves, first))
    with pytest.raises(RuntimeError):
        first[0].sum().backward()
    with torch.no_grad():
        assert plb.channel_mix(**leaves, activation="softmax").grad_fn is None
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: plb.channel_mix(t, a["weight"]))(a["x"][None])


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_addresses_of_any_alignment(plb, offset, dtype):
    """Contiguous views that start between 16-byte boundaries."""
    a, g = make(1000, 21, 21, 21, dtype)
    moved = {}
    for m, t in {**a, "g": g}.items():
        flat = torch.empty(t.numel() + offset, dtype=dtype, device="cuda")
        moved[m] = flat[offset:].view(t.shape)
        moved[m].copy_(t)
    gm = moved.pop("g")
    for checkpoint in (None, "8bit"):
        out, saved = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0, checkpoint=checkpoint)
        other, kept = plb.channel_mix_raw(**moved, activation="softmax", residual_scale=-1.0, checkpoint=checkpoint)
        assert torch.equal(out, other)
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "softmax", -1.0, needs_of(a))
        e = plb.channel_mix_backward(gm, kept, moved["weight"], moved["weight2"], "softmax", -1.0, needs_of(a))
        assert all(torch.equal(getattr(d, m), getattr(e, m)) for m in needs_of(a))


def test_no_rows(plb):
    for shape in ((0,), (2, 0, 3)):
        x = torch.zeros(shape + (5,), device="cuda", requires_grad=True)
        w = torch.ones(5, 4, device="cuda", requires_grad=True)
        b = torch.ones(4, device="cuda", requires_grad=True)
        for checkpoint in (None, "8bit"):
            out = plb.channel_mix(x, w, b, activation="softmax", checkpoint=checkpoint)
            assert out.shape == shape + (4,)
            gx, gw, gb = torch.autograd.grad(out.sum(), (x, w, b))
            assert gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any())
    p = plb.pack_activations(torch.zeros((0, 3), device="cuda"))
    assert p.codes.numel() == 0 and p.scales.numel() == 0 and plb.unpack_activations(p).shape == (0, 3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 1000, 4096, 100003])
def test_8_bit_blocks(plb, dtype, count):
    g = torch.Generator().manual_seed(count)
    v = torch.randn(count, generator=g) * 10.0 ** torch.randint(-6, 4, (count,), generator=g)
    v[: count // 2] = v[: count // 2].abs()
    v = v.to(dtype)
    for offset in (0, 1, 3):
        flat = torch.zeros(count + offset, dtype=dtype, device="cuda")
        flat[offset:] = v.cuda()
        p = plb.pack_activations(flat[offset:])
        codes, headers = ref.pack(v.float().numpy())
        assert np.array_equal(p.codes.cpu().numpy(), codes) and np.array_equal(p.scales.cpu().numpy(), headers)
        want = torch.from_numpy(ref.unpack(codes, headers))
        for to in (F32, BF16):
            assert torch.equal(plb.unpack_activations(p, to).cpu().double(), want)
        assert torch.equal(plb.unpack_activations(p, F16).cpu(), want.to(F16))
        assert plb.unpack_activations(p).dtype == dtype


def test_8_bit_blocks_of_extreme_values(plb):
    big, tiny = 3.4028234663852886e38, 2.0 ** -149
    rows = [[0.0], [-0.0], [big], [-big, big], [tiny], [-tiny], [255 * 2.0 ** -126, 2.0 ** -126], [2.0 ** -127, 2.0 ** -126],
            [255.0, 254.5, 0.5, 1.5, 2.5], [255.00002, 1.0], [127.0, -127.0, 0.5, -0.5, 1.5], [127.00001, -1.0], [-128.0],
            [math.inf, 1.0], [1.0, -math.inf], [math.nan, 2.0], [1.9921875], [1.9921876], [255 * 2.0 ** 120, 1.0],
            [2.0 ** k for k in range(-3, 6)], [-(2.0 ** k) for k in range(-3, 6)]]
    v = np.zeros((len(rows), 32), np.float32)
    for i, r in enumerate(rows):
        v[i, :len(r)] = np.array(r, np.float64).astype(np.float32)
    p = plb.pack_activations(torch.from_numpy(v).cuda())
    codes, headers = ref.pack(v)
    assert np.array_equal(p.scales.cpu().numpy(), headers)
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    back = plb.unpack_activations(p).cpu().double().numpy().reshape(-1)
    assert np.array_equal(back, ref.unpack(codes, headers), equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,k2,n", [(1, 1, 0, 1), (33, 21, 21, 21), (1000, 75, 0, 16), (257, 128, 128, 128), (4099, 2, 2, 2),
                                         (515, 5, 9, 31), (100, 128, 7, 3), (512, 64, 64, 64), (300, 32, 16, 64), (4097, 16, 0, 8),
                                         (1600, 32, 32, 32), (95, 8, 8, 16), (1, 64, 0, 64)])
def test_activations_in_8_bits(plb, rows, k, k2, n, dtype):
    """What the forward pass keeps is what pack_activations makes of the same tensors, and the gradients are those at the
    values that the codes stand for."""
    for activation, scale in (("softmax", -1.0), ("relu", 1.0), (None, 1.0)):
        a, g = make(rows, k, k2, n, dtype)
        plain, _ = plb.channel_mix_raw(**a, activation=activation, residual_scale=scale)
        out, saved = plb.channel_mix_raw(**a, activation=activation, residual_scale=scale, checkpoint="8bit")
        assert torch.equal(out, plain)
        for kept, t in ((saved.x, a["x"]), (saved.x2, a["x2"])):
            if t is None:
                assert kept is None
                continue
            codes, headers = ref.pack(t.float().cpu().numpy())
            assert np.array_equal(kept.codes.cpu().numpy(), codes) and np.array_equal(kept.scales.cpu().numpy(), headers)
        y = None
        if activation:
            codes, headers = ref.pack(out.float().cpu().numpy(), activation == "relu")
            assert np.array_equal(saved.out.codes.cpu().numpy(), codes) and np.array_equal(saved.out.scales.cpu().numpy(), headers)
            y = plb.unpack_activations(saved.out, F32)
            if activation == "relu":
                assert torch.equal(y > 0, out > 0)
        else:
            assert saved.out is None
        needs = needs_of(a)
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, needs)
        x2 = None if saved.x2 is None else plb.unpack_activations(saved.x2, F32)
        want = ref.gradients(g, y, plb.unpack_activations(saved.x, F32), a["weight"], x2, a["weight2"], activation, scale)
        for m in needs:
            ref.assert_within(getattr(d, m), *want[m], "%s of %s" % (m, activation))
        leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
        o = plb.channel_mix(**leaves, activation=activation, residual_scale=scale, checkpoint="8bit")
        for m, t in zip(leaves, torch.autograd.grad(o, list(leaves.values()), g)):
            assert torch.equal(t, getattr(d, m))


def test_8_bits_hold_the_memory_that_they_say(plb):
    rows, n = 1 << 18, 21
    x = torch.rand((1, rows, n), device="cuda")
    w = torch.eye(n, device="cuda", requires_grad=True)

    def held(checkpoint):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = plb.channel_mix(x.clone(), w, x2=x.clone(), weight2=w, activation="softmax", checkpoint=checkpoint)
        out = out.sum()                                  # the output itself may go
        return torch.cuda.memory_allocated() - before, out

    full, kept = held(None)[0], held("8bit")[0]
    assert kept <= 0.28 * full and kept >= 3 * rows * n


def test_mixed_kinds_of_activations(plb):
    """Some in 8 bits, some as they were; and an output kept for an activation that does not read it."""
    a, g = make(700, 21, 10, 21)
    out, full = plb.channel_mix_raw(**a, activation="softmax")
    _, small = plb.channel_mix_raw(**a, activation="softmax", checkpoint="8bit")
    wide = lambda p: plb.unpack_activations(p)   # noqa: E731
    for x, x2, y in ((small.x, full.x2, small.out), (full.x, small.x2, full.out), (small.x, full.x2, full.out)):
        d = plb.channel_mix_backward(g, plb.MixSaved(x, x2, y), a["weight"], a["weight2"], "softmax", 1.0, needs_of(a))
        v = [t if isinstance(t, torch.Tensor) else wide(t) for t in (x, x2, y)]
        e = plb.channel_mix_backward(g, plb.MixSaved(*v), a["weight"], a["weight2"], "softmax", 1.0, needs_of(a))
        want = ref.gradients(g, v[2], v[0], a["weight"], v[1], a["weight2"], "softmax", 1.0)
        for m in needs_of(a):
            ref.assert_within(getattr(d, m), *want[m], m)
            ref.assert_within(getattr(e, m), *want[m], m)


def test_streams_and_graphs(plb):
    """On a stream of the caller's, and captured: two graphs replayed in turn with other inputs, beside eager calls."""
    cases = []
    for seed, (rows, k, k2, n) in enumerate([(3000, 21, 21, 21), (500, 64, 0, 32)]):
        a, g = make(rows, k, k2, n, seed=seed)
        cases.append((a, g))

    def work(a, g):
        out, saved = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0, checkpoint="8bit")
        return [out] + [t for t in plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "softmax", -1.0, needs_of(a))
                        if t is not None]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = [work(a, g) for a, g in cases]
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for a, g in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(a, g)
        graphs.append((graph, outs))
    for round_ in range(3):
        for (a, g), (graph, _) in zip(cases, graphs):
            a["x"].copy_(torch.randn_like(a["x"]) if round_ else a["x"])
            graph.replay()
        eager = [work(a, g) for a, g in cases]
        torch.cuda.synchronize()
        for (_, outs), want in zip(graphs, eager):
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
        if round_ == 0:
            for one, want in zip(beside, eager):
                assert all(torch.equal(o, w) for o, w in zip(one, want))


def test_backward_in_a_graph_of_its_own(plb):
    """Forward and backward through autograd, captured with leaves of the capture's own."""
    a, g = make(900, 21, 21, 21)
    static = {m: t.clone() for m, t in a.items()}

    def step():
        leaves = {m: t.detach().requires_grad_(True) for m, t in static.items()}
        out = plb.channel_mix(**leaves, activation="softmax", residual_scale=-1.0, checkpoint="8bit")
        return [out.detach()] + list(torch.autograd.grad(out, list(leaves.values()), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    static["x"].copy_(torch.randn_like(static["x"]))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("rows,k,k2,n", [(1, 3, 0, 5), (37, 21, 21, 21), (129, 75, 0, 16), (200, 128, 128, 128)])
def test_nothing_is_written_beside_the_outputs(plb, rows, k, k2, n):
    """Every output inside a larger buffer whose other bytes keep what they held."""
    from permutohedral_lattice_b200 import capi
    L = capi.lib()
    a, g = make(rows, k, k2, n)
    stream = torch.cuda.current_stream().cuda_stream
    for pad in (16, 13):
        buffers = {}

        def room(name, count, dtype):
            t = torch.empty(count + 2 * pad, dtype=dtype, device="cuda")
            t.view(torch.uint8).fill_(0xA5)
            buffers[name] = (t, pad, count)
            return t[pad:].data_ptr()

        def packed(name, count):
            return capi.PlPacked(room(name + "c", count, torch.uint8), room(name + "s", -(-count // 32), torch.int16))

        m = capi.PlMix(rows, k, k2, n, capi.PL_ACT_SOFTMAX, 0, 0, -1.0)
        p = lambda t: 0 if t is None else t.data_ptr()   # noqa: E731
        keep = [packed("kx", rows * k), packed("kx2", rows * k2) if k2 else capi.PlPacked(0, 0), packed("ko", rows * n)]
        out = room("out", rows * n, F32)
        assert L.pl_channel_mix(ctypes.byref(m), out, p(a["x"]), p(a["x2"]), p(a["weight"]), p(a["weight2"]), p(a["bias"]),
                                p(a["residual"]), *keep, stream) == 0
        size = ctypes.c_size_t(0)
        assert L.pl_channel_mix_workspace_bytes(ctypes.byref(m), ctypes.byref(size)) == 0
        d = capi.PlMixGradients(room("dx", rows * k, F32), room("dx2", rows * k2, F32) if k2 else 0, room("dw", k * n, F32),
                                room("dw2", k2 * n, F32) if k2 else 0, room("db", n, F32), room("dr", rows * n, F32))
        ws = torch.full((size.value + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        none = capi.PlPacked(0, 0)
        assert L.pl_channel_mix_backward(ctypes.byref(m), g.data_ptr(), capi.PlKept(out, none), capi.PlKept(0, keep[0]),
                                         capi.PlKept(0, keep[1]), p(a["weight"]), p(a["weight2"]), d, ws.data_ptr(), size.value,
                                         stream) == 0
        torch.cuda.synchronize()
        assert bool((ws[size.value:] == 0xA5).all())
        for name, (t, before, count) in buffers.items():
            assert bool((t[:before].view(torch.uint8) == 0xA5).all()), name
            assert bool((t[before + count:].view(torch.uint8) == 0xA5).all()), name
        want, _ = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0)
        t, before, count = buffers["out"]
        assert torch.equal(t[before:before + count], want.flatten())


def test_values_beyond_32_bit_offsets(plb):
    """2.2 billion values in 16 bits: rows behind the 2^31st."""
    rows, k, n = 34_000_003, 64, 2
    x = torch.zeros((rows, k), dtype=BF16, device="cuda")
    w = torch.randn((k, n), generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    tail = torch.randn((1000, k), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    x[-1000:] = tail
    out, saved = plb.channel_mix_raw(x, w, activation="softmax", checkpoint="8bit")
    want, bound = ref.forward(tail, w, None, None, None, None, "softmax", 1.0)
    ref.assert_within(out[-1000:], want, bound)
    assert bool((out[:-1000] == 0.5).all())
    g = torch.zeros_like(out)
    g[-1000:] = torch.randn((1000, n), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    d = plb.channel_mix_backward(g, saved, w, activation="softmax", needs=("x", "weight"))
    assert not bool(d.x[:-1000].any())
    y = plb.unpack_activations(saved.out)[-1000:]
    kept = plb.unpack_activations(saved.x)[-1000:]
    grads = ref.gradients(g[-1000:], y, kept, w, None, None, "softmax", 1.0)
    ref.assert_within(d.x[-1000:], *grads["x"])
    ref.assert_within(d.weight, *grads["weight"])


def test_wide_rows_beyond_32_bit_offsets(plb):
    """2.15 billion floats: rows behind the 2^31st value in the kernels of wide rows, forward and backward."""
    rows, k, n = 16_800_001, 128, 128
    x = torch.zeros((rows, k), device="cuda")
    w = torch.randn((k, n), generator=torch.Generator().manual_seed(0)).cuda()
    tail = torch.randn((50, k), generator=torch.Generator().manual_seed(1)).cuda()
    x[-50:] = tail
    out, saved = plb.channel_mix_raw(x, w, activation="softmax")
    want, bound = ref.forward(tail, w, None, None, None, None, "softmax", 1.0)
    ref.assert_within(out[-50:], want, bound)
    assert bool((out[-51] == 1 / 128).all())
    g = torch.zeros_like(out)
    g[-50:] = torch.randn((50, n), generator=torch.Generator().manual_seed(2)).cuda()
    d = plb.channel_mix_backward(g, saved, w, activation="softmax", needs=("x", "weight"))
    assert not bool(d.x[:-50].any())
    grads = ref.gradients(g[-50:], out[-50:], tail, w, None, None, "softmax", 1.0)
    ref.assert_within(d.x[-50:], *grads["x"])
    ref.assert_within(d.weight, *grads["weight"])


def test_a_single_row_without_other_dimensions(plb):
    a, g = make(1, 9, 4, 6)
    flat = {m: (t[0, 0] if t is not None and t.dim() == 3 else t) for m, t in a.items()}
    out, saved = plb.channel_mix_raw(**flat, activation="softmax", checkpoint="8bit")
    assert out.shape == (6,) and torch.equal(out, plb.channel_mix(**a, activation="softmax")[0, 0])
    d = plb.channel_mix_backward(g[0, 0], saved, a["weight"], a["weight2"], "softmax", 1.0, needs_of(a))
    assert d.x.shape == (9,) and d.x2.shape == (4,) and d.residual.shape == (6,)
    assert plb.channel_mix_backward(g[0, 0], saved, a["weight"], a["weight2"], "softmax", needs=()) == plb.MixGradients()


def test_two_host_threads_on_streams_of_their_own(plb):
    import threading
    cases = [make(4000 + 37 * i, 21 + i, 10, 21, seed=i) for i in range(4)]

    def work(a, g):
        out, saved = plb.channel_mix_raw(**a, activation="softmax", checkpoint="8bit")
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "softmax", 1.0, needs_of(a))
        return [out] + [getattr(d, m) for m in needs_of(a)]

    want = [work(*c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * len(cases)

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = work(*cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for one, other in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(one, other))


def test_the_largest_finite_values(plb):
    """Values up to 3.4e38 and down to the least ones: nothing becomes NaN that is not."""
    for dtype in (F32, BF16, F16):
        big = torch.finfo(dtype).max * 0.99
        x = torch.tensor([[big, 0, 0], [0, big, -big], [torch.finfo(dtype).tiny, 1, 0], [0, 0, 0]], dtype=dtype, device="cuda")
        w = torch.tensor([[0.5, 0.0], [0.25, 0.25], [0.25, -0.125]], dtype=dtype, device="cuda")
        out = plb.channel_mix(x, w)
        want = x.double() @ w.double()
        assert bool(torch.isfinite(out).all())
        assert float(((out.double() - want).abs() / (x.double().abs() @ w.double().abs() + 1e-30)).max()) <= ref.PRODUCT + ref.half_step(dtype)


@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rows,k,k2,n", [(1, 64, 0, 68), (127, 67, 67, 68), (128, 32, 32, 100), (129, 61, 3, 128), (20011, 128, 4, 128),
                                         (38000, 97, 31, 72), (19000, 33, 31, 67), (257, 63, 0, 128), (500, 68, 128, 21)])
def test_many_labels(plb, rows, k, k2, n, dtype, weight_dtype):
    """One tile a CTA and several, widths of whole float4 and others, as many channels in as the tensor-memory kernel takes and fewer."""
    for activation in ("softmax", "relu"):
        a, g = make(rows, k, k2, n, dtype, weight_dtype)
        out, saved = plb.channel_mix_raw(**a, activation=activation, residual_scale=-1.0)
        want, bound = ref.forward(a["x"], a["weight"], a["bias"], a["residual"], a["x2"], a["weight2"], activation, -1.0)
        ref.assert_within(out, want, bound, activation)
        needs = needs_of(a)
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, -1.0, needs)
        gradients = ref.gradients(g, out, a["x"], a["weight"], a["x2"], a["weight2"], activation, -1.0)
        for m in needs:
            ref.assert_within(getattr(d, m), *gradients[m], "%s of %s" % (m, activation))


@pytest.mark.parametrize("moved", ["x", "x2", "weight", "weight2", "bias", "residual"])
def test_many_labels_at_addresses_of_any_alignment(plb, moved):
    a, _ = make(700, 128, 64, 128)
    want, bound = ref.forward(a["x"], a["weight"], a["bias"], a["residual"], a["x2"], a["weight2"], "softmax", -1.0)
    t = a[moved]
    store = torch.empty(t.numel() + 1, device="cuda")
    a[moved] = store[1:].view(t.shape).copy_(t)
    assert a[moved].data_ptr() % 16 == 4
    out = plb.channel_mix(**a, activation="softmax", residual_scale=-1.0)
    ref.assert_within(out, want, bound, moved)
    assert torch.equal(out, plb.channel_mix(**{**a, moved: t}, activation="softmax", residual_scale=-1.0))


def test_bad_values_of_many_labels_stay_in_their_row(plb):
    a, _ = make(300, 128, 70, 128)
    clean = plb.channel_mix(**a, activation="softmax", residual_scale=-1.0)
    a["x"][0, 7, 127] = math.nan
    a["x2"][0, 129, 69] = math.inf
    a["residual"][0, 299, 127] = math.nan
    out = plb.channel_mix(**a, activation="softmax", residual_scale=-1.0)
    bad = [7, 129, 299]
    assert bool(torch.isnan(out[0, bad]).all())
    keep = [r for r in range(300) if r not in bad]
    assert torch.equal(out[0, keep], clean[0, keep])


def test_many_labels_on_several_streams_and_in_graphs(plb):
    """Kernels that take all of an SM's tensor memory, on four streams at once and replayed beside each other, with a library product
    on a fifth."""
    cases = [make(40000 + 131 * i, 128, 0, 128, seed=i)[0] for i in range(4)]
    want = [plb.channel_mix(**a, activation="softmax") for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, results = [], []
    for s, a in zip(streams, cases):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            results.append(plb.channel_mix(**a, activation="softmax"))
        graphs.append(graph)
    square = torch.randn((2048, 2048), device="cuda", dtype=BF16)
    torch.cuda.synchronize()
    for _ in range(5):
        torch.cuda.synchronize()
        eager = []
        for s, a, graph in zip(streams, cases, graphs):
            with torch.cuda.stream(s):
                graph.replay()
                eager.append(plb.channel_mix(**a, activation="softmax"))
        square @ square
        torch.cuda.synchronize()
        assert all(torch.equal(r, w) for r, w in zip(results, want)) and all(torch.equal(r, w) for r, w in zip(eager, want))
