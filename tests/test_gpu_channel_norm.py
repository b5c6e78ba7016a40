"""channel_norm and channel_dropout against plain forms in 64 bits (norm_reference.py derives the bounds)."""
import math

import pytest
import torch

import norm_reference as ref
from mix_reference import assert_within

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
KEY, OFFSET = 0x9ABCDEF012345678, 0x1122334455667788


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


# after, before, residual, gate, p, biases
FORMS = [("layer", "", False, "", 0.0, True), ("", "rms", False, "", 0.0, False), ("", "layer", True, "", 0.0, True),
         ("rms", "", True, "channel", 0.25, True), ("layer", "rms", True, "full", 0.1, True), ("rms", "layer", True, "channel", 0.4, False),
         ("", "", True, "full", 0.5, False), ("", "", False, "channel", 0.0, False), ("layer", "layer", False, "", 0.0, True)]
SHAPES = [(1, 1), (1, 21), (1, 512), (7, 2), (33, 3), (100, 4), (65, 5), (257, 8), (1000, 21), (130, 32), (77, 64), (501, 75),
          (64, 128), (19, 255), (40, 256), (9, 300), (11, 511), (13, 512), (20011, 16), (5000, 24), (6001, 7)]


def make(rows, c, form, dtype, vector_dtype=None, seed=0):
    after, before, residual, gate, p, biases = form
    g = torch.Generator().manual_seed(1000003 * seed + 131 * rows + 17 * c)
    vd = dtype if vector_dtype is None else vector_dtype
    t = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    a = {"x": (1.5 * t(1, rows, c) + 0.3).to(dtype), "residual": t(1, rows, c).to(dtype) if residual else None,
         "gate": {"": None, "channel": t(c).to(vd), "full": t(1, rows, c).to(dtype)}[gate]}
    for place, kind in (("after", after), ("before", before)):
        a[place + "_weight"] = (1 + 0.3 * t(c)).to(vd) if kind else None
        a[place + "_bias"] = t(c).to(vd) if kind and biases else None
    grads = [t(1, rows, c).to(dtype).cuda() for _ in range(2)]
    return {m: v.cuda() if v is not None else None for m, v in a.items()}, grads


def call(plb, a, form, seed=(KEY, OFFSET), **more):
    after, before, _, _, p, _ = form
    norms = {place: plb.Norm(a[place + "_weight"], a[place + "_bias"], kind, 1e-4) for place, kind in (("after", after), ("before", before))
             if kind}
    return plb.channel_norm(a["x"], a["residual"], a["gate"], **norms, residual_scale=-0.75, dropout=p, seed=seed if p else None, **more)


def want_of(a, form, grads=None, out=None):
    after, before, _, _, p, _ = form
    keep = ref.kept(tuple(a["x"].shape), p, KEY, OFFSET) if p else None
    norms = [(a[place + "_weight"], a[place + "_bias"], kind, 1e-4) if kind else None for place, kind in (("after", after), ("before", before))]
    return ref.norm(a["x"], a["residual"], a["gate"], *norms, -0.75, p, keep, grads)


def outputs_of(got, form):
    """{name: tensor} of what the call returned."""
    after, before, residual, gate, p, _ = form
    if not before:
        return {"h": got}
    if not (after or residual or gate or p):
        return {"y": got}
    return dict(zip(("h", "y"), got))


@pytest.mark.parametrize("dtype,vector_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_forward_and_gradients(plb, rows, c, dtype, vector_dtype):
    for form in FORMS:
        a, grads = make(rows, c, form, dtype, vector_dtype)
        outs = outputs_of(call(plb, a, form), form)
        want = want_of(a, form, (grads[0] if "h" in outs else None, grads[1] if "y" in outs else None))
        for m, t in outs.items():
            assert t.dtype == dtype and t.shape == a["x"].shape and t.grad_fn is None
            assert_within(t, *want[m], "%s of %s" % (m, form))
        leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
        again = outputs_of(call(plb, {**a, **leaves}, form), form)
        assert all(torch.equal(again[m], outs[m]) for m in outs)
        up = [grads[0 if m == "h" else 1] for m in outs]
        got = dict(zip(leaves, torch.autograd.grad(list(again.values()), list(leaves.values()), up, retain_graph=True)))
        for m, t in got.items():
            assert t.dtype == a[m].dtype and t.shape == a[m].shape
            assert_within(t, *want[m], "d %s of %s" % (m, form))
        # the same bits again, and each by itself
        for m, leaf in leaves.items():
            (one,) = torch.autograd.grad(list(again.values()), [leaf], up, retain_graph=True)
            assert torch.equal(one, got[m]), (m, form)


def test_many_rows_share_a_cta(plb):
    """Threads with several rows each, and a last piece that is not whole."""
    for rows, c, dtype in ((400_003, 21, F32), (700_001, 8, BF16), (90_001, 128, F16)):
        for form in (FORMS[4], FORMS[3]):
            a, grads = make(rows, c, form, dtype)
            leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
            outs = outputs_of(call(plb, {**a, **leaves}, form), form)
            up = [grads[0 if m == "h" else 1] for m in outs]
            want = want_of(a, form, (grads[0], grads[1] if "y" in outs else None))
            got = dict(zip(leaves, torch.autograd.grad(list(outs.values()), list(leaves.values()), up)))
            for m, t in list(outs.items()) + list(got.items()):
                assert_within(t, *want[m], "%s of %s" % (m, form))


def test_only_one_output_is_used(plb):
    form = FORMS[4]
    a, grads = make(300, 21, form, F32)
    for used in ("h", "y"):
        leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
        outs = outputs_of(call(plb, {**a, **leaves}, form), form)
        up = grads[0] if used == "h" else grads[1]
        got = torch.autograd.grad(outs[used], list(leaves.values()), up)
        want = want_of(a, form, (up, torch.zeros_like(up)) if used == "h" else (None, up))
        for m, t in zip(leaves, got):
            assert_within(t, *want[m], "%s from %s" % (m, used))


def test_gradients_against_differences(plb):
    """Along random directions: (f(t + e v) - f(t - e v)) / 2e of the formula in 64 bits against the kernels' gradient."""
    for form in (FORMS[4], FORMS[5], FORMS[2]):
        a, grads = make(65, 7, form, F32)
        leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
        outs = outputs_of(call(plb, {**a, **leaves}, form), form)
        got = torch.autograd.grad(list(outs.values()), list(leaves.values()), [grads[0 if m == "h" else 1] for m in outs])

        def f(t):
            want = want_of({**a, **t}, form)
            return sum((want[m][0] * grads[0 if m == "h" else 1].double()).sum() for m in outs)

        for (m, leaf), grad in zip(leaves.items(), got):
            v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(3)).cuda().double()
            e, wide = 1e-5, {name: t.detach().double() for name, t in leaves.items()}
            slope = (f({**wide, m: wide[m] + e * v}) - f({**wide, m: wide[m] - e * v})) / (2 * e)
            assert abs(float(slope) - float((grad.double() * v).sum())) <= 1e-5 * (float((grad.double() * v).abs().sum()) + 1.0), (m, form)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_dropout(plb, dtype):
    for shape in ((1,), (3,), (4,), (5, 7), (2, 33, 21), (1000, 64), (0, 4), ()):
        for p in (0.0, 0.1, 0.999, 2.0 ** -40):
            x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
            residual = torch.randn(shape, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
            keep = ref.kept(shape, p, 7, 9)
            for offset in (0, 1):     # also between 16-byte boundaries
                flat = torch.empty(x.numel() + offset, dtype=dtype, device="cuda")
                leaf = flat[offset:].view(shape).copy_(x).requires_grad_(True)
                other = residual.clone().requires_grad_(True)
                out = plb.channel_dropout(leaf, p, (7, 9), other, 0.5)
                want = torch.where(keep, x.double() / (1 - p), torch.zeros_like(x, dtype=torch.float64)) + 0.5 * residual.double()
                assert_within(out, want, 4 * ref.U * (want.abs() + residual.double().abs()))
                g = torch.randn(shape, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
                dx, dr = torch.autograd.grad(out, [leaf, other], g)
                want = torch.where(keep, g.double() / (1 - p), torch.zeros_like(g, dtype=torch.float64))
                assert_within(dx, want, 3 * ref.U * want.abs())
                assert torch.equal(dr, (0.5 * g.float()).to(dtype))
                alone = plb.channel_dropout(x, p, torch.tensor([7, 9], device="cuda"))
                assert torch.equal(alone == 0, ~keep | (x == 0))


def test_dropped_share_and_words(plb):
    """The mask is the generator's: seeds as numbers, as a tensor, negative as the same 64 bits; other seeds, other masks."""
    x = torch.ones(1000, 100, device="cuda")
    one = plb.channel_dropout(x, 0.3, (KEY, OFFSET))
    assert abs(float((one == 0).float().mean()) - 0.3) < 6 * math.sqrt(0.21 / x.numel())
    assert torch.equal(one != 0, ref.kept((1000, 100), 0.3, KEY, OFFSET))
    tensor = torch.tensor([KEY - (1 << 64), OFFSET], device="cuda")
    assert torch.equal(plb.channel_dropout(x, 0.3, tensor), one)
    assert torch.equal(plb.channel_dropout(x, 0.3, (KEY - (1 << 64), OFFSET)), one)
    assert torch.equal(plb.channel_dropout(x, 0.3, 5), plb.channel_dropout(x, 0.3, (5, 0)))
    assert not torch.equal(plb.channel_dropout(x, 0.3, (KEY, OFFSET + 1)), one)
    assert not torch.equal(plb.channel_dropout(x, 0.3, (KEY + 1, OFFSET)), one)
    assert torch.equal(plb.channel_norm(x, dropout=0.3, seed=(KEY, OFFSET)), one)
    for c in (3, 21, 33):     # rows of single values by way of shared memory
        x = torch.ones(257, c, device="cuda")
        assert torch.equal(plb.channel_norm(x, dropout=0.3, seed=tensor), plb.channel_dropout(x, 0.3, tensor))


def test_bad_values_stay_in_their_row(plb):
    form = FORMS[4]
    a, grads = make(200, 21, form, F32)
    clean = outputs_of(call(plb, a, form), form)
    keep = ref.kept((1, 200, 21), 0.1, KEY, OFFSET)
    a["x"][0, 7, 20], a["residual"][0, 40, 0], a["gate"][0, 199, 3] = math.nan, math.inf, math.nan
    outs = outputs_of(call(plb, a, form), form)
    rows = [r for r in range(200) if r not in (7, 40, 199)]
    for m in outs:
        assert torch.equal(outs[m][0, rows], clean[m][0, rows])
    assert bool(torch.isnan(outs["h"][0, 7][keep[0, 7]]).all()) and bool(torch.isnan(outs["y"][0, 7]).all())
    # a row with an infinity has no deviation to speak of: what is finite in it is nothing beside it (rms)
    assert bool(torch.isnan(outs["y"][0, 40, 0])) and torch.equal(outs["y"][0, 40, 1:], a["before_bias"][1:])
    assert bool(torch.isfinite(outs["h"][0, 40, 1:]).all())
    x = torch.full((4, 8), math.nan, device="cuda")
    dropped = plb.channel_dropout(x, 0.5, 3)
    assert torch.equal(torch.isnan(dropped), ref.kept((4, 8), 0.5, 3, 0)) and bool((dropped[~torch.isnan(dropped)] == 0).all())


def test_constant_and_extreme_rows(plb):
    for dtype in (F32, BF16, F16):
        x = torch.stack([torch.zeros(64), torch.full((64,), 3.0), torch.full((64,), -1e4), 1e-4 * torch.arange(64.0)]).to(dtype).cuda()
        for kind in ("layer", "rms"):
            y = plb.channel_norm(x, after=plb.Norm(kind=kind, eps=1e-5))
            want, bound = ref.norm(x, None, None, (None, None, kind, 1e-5), None, 1.0, 0.0, None)["h"]
            assert_within(y, want, bound, kind)
            assert bool((y[0] == 0).all())


def test_other_orders_devices_and_streams(plb):
    form = FORMS[4]
    a, grads = make(96, 24, form, F32)
    want = outputs_of(call(plb, a, form), form)
    b = dict(a)
    b["x"] = torch.empty(24, 96, 1, device="cuda").permute(2, 1, 0).copy_(a["x"])
    b["residual"] = torch.stack([a["residual"], a["residual"]], -1)[..., 0]
    b["gate"] = a["gate"].expand_as(a["gate"])
    got = outputs_of(call(plb, b, form), form)
    assert all(torch.equal(got[m], want[m]) and got[m].is_contiguous() for m in want)
    # an upstream gradient without memory of its own
    leaf = a["x"].clone().requires_grad_(True)
    plb.channel_norm(leaf, after=plb.Norm()).sum().backward()
    full = a["x"].clone().requires_grad_(True)
    plb.channel_norm(full, after=plb.Norm()).backward(torch.ones_like(full))
    assert torch.equal(leaf.grad, full.grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = outputs_of(call(plb, a, form), form)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[m], want[m]) for m in want)
    with pytest.raises(RuntimeError):     # no second derivative
        d = torch.autograd.grad(plb.channel_norm(leaf, after=plb.Norm()).sum(), leaf, create_graph=True)[0]
        d.sum().backward()


def test_captured_graph_follows_its_seed(plb):
    """Forward and backward in a graph, replayed with another seed in the tensor; two graphs side by side."""
    form = FORMS[5]
    a, grads = make(500, 32, form, F32)
    seed = torch.tensor([1, 2], device="cuda")
    call(plb, a, form, seed=seed)

    def step():
        leaves = {m: t.detach().requires_grad_(True) for m, t in a.items() if t is not None}
        outs = outputs_of(call(plb, {**a, **leaves}, form, seed=seed), form)
        return list(outs.values()) + list(torch.autograd.grad(list(outs.values()), list(leaves.values()), [grads[0], grads[1]]))

    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            found = step()
        graphs.append((graph, found))
    for numbers in ((1, 2), (5, 6)):
        seed.copy_(torch.tensor(numbers))
        want = [t.clone() for t in step()]
        for graph, found in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, found in graphs:
            assert all(torch.equal(f, w) for f, w in zip(found, want))


def test_a_seed_that_changed_before_the_backward_pass_is_an_error(plb):
    x, seed = torch.randn(8, 4, device="cuda", requires_grad=True), torch.tensor([1, 2], device="cuda")
    for out in (plb.channel_dropout(x, 0.5, seed), plb.channel_norm(x, after=plb.Norm(), dropout=0.5, seed=seed)):
        seed.add_(1)
        with pytest.raises(RuntimeError):
            out.sum().backward()


def test_empty_tensors(plb):
    for c in (1, 21):
        x = torch.zeros(2, 0, c, device="cuda", requires_grad=True)
        w = torch.ones(c, device="cuda", requires_grad=True)
        h, y = plb.channel_norm(x, x, w, plb.Norm(w), plb.Norm(w, w), dropout=0.5, seed=1)
        assert h.shape == y.shape == x.shape
        d = torch.autograd.grad(h.sum() + y.sum(), [x, w])
        assert d[0].shape == x.shape and bool((d[1] == 0).all())


def test_values_beyond_2_31(plb):
    """Rows whose first value's number does not fit 32 bits, and the dropout's words there."""
    rows, c = (1 << 31) // 64 + 300, 64
    x = torch.zeros(rows, c, dtype=BF16, device="cuda")
    x[-200:] = torch.randn(200, c, generator=torch.Generator().manual_seed(1)).to(BF16)
    h = plb.channel_norm(x, after=plb.Norm(kind="rms"), dropout=0.25, seed=(3, 4))
    want, bound = ref.norm(x[-200:], None, None, (None, None, "rms", 1e-5), None, 1.0, 0.0, None)["h"]
    last = plb.channel_dropout(torch.ones_like(x), 0.25, (3, 4))[-200:] != 0
    assert torch.equal(h[-200:] != 0, last & (x[-200:] != 0)) and 0.7 < float(last.float().mean()) < 0.8
    assert_within(h[-200:][last], want[last] / 0.75, bound[last] / 0.75 + 3 * ref.U * want[last].abs() / 0.75)
    # the words of the last quads, one by one
    first = (rows - 200) * c
    words = []
    for quad in range(first // 4, first // 4 + 4):
        words += _quad(quad, 3, 4)
    assert torch.equal(last.flatten()[:16].cpu(), torch.tensor([w >= 1 << 30 for w in words]))


def _quad(quad, key, offset):
    c, k = [quad & 0xFFFFFFFF, quad >> 32, offset & 0xFFFFFFFF, offset >> 32], [key & 0xFFFFFFFF, key >> 32]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c
