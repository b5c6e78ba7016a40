"""gated_mix of 16-bit types: hidden values as two terms of the type, however many rows there are, or (round_hidden) rounded once.

Bounds: gated_reference.py's, with what a hidden value loses on its way to the next product in place of half a step: the second term
is the rounded rest of the first, so what is left is half a step of half a step, 2^-16 of a value in bfloat16 and 2^-22 in float16 (and
2^-25 where that is less than its least step holds).  Of GELU's Phi the smaller of it and 1 - Phi may be off by 2^-18 of it, beside float arithmetic."""
import math

import pytest
import torch

import gated_reference as ref
from mix_reference import assert_within
from test_gpu_gated_mix import SHAPES, make, train

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
REST = {BF16: 2.0 ** -16, F16: 2.0 ** -22, F32: 0.0}
FORMS = [("silu", "gud", True), ("gelu", "u", False), ("sigmoid", "g", True), ("relu", "ud", False)]


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


@pytest.fixture
def two_terms(monkeypatch):
    plain = ref._act

    def act(g, eg, kind):
        a, ea, d, ed = plain(g, eg, kind)
        if kind == "gelu":
            off = 2.0 ** -18 * 0.5 * torch.erfc(g.abs() / math.sqrt(2))
            ea, ed = ea + g.abs() * off, ed + off
        return a, ea, d, ed

    monkeypatch.setattr(ref, "half_step", REST.__getitem__)
    monkeypatch.setattr(ref, "_act", act)


def check(plb, a, grad, activation, label=None, **more):
    leaves = {m: t.clone().requires_grad_(True) for m, t in a.items() if t is not None}
    out = plb.gated_mix(**{**a, **leaves}, activation=activation, residual_scale=0.75, **more)
    want = ref.gated(a, activation, 0.75, grad)
    assert_within(out, *want["out"], "out of %s" % (label,))
    d = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)))
    for m, t in d.items():
        assert_within(t, *want[m], "%s of %s" % (m, label))
    return out.detach(), d


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,h,n", SHAPES)
def test_small_calls(plb, two_terms, rows, k, h, n, dtype):
    for activation, biases, residual in FORMS:
        check(plb, *make(rows, k, h, n, dtype, biases, residual), activation, activation)


LARGE = [(65_536, 64, 256, 64), (65_537, 64, 256, 64), (80_001, 128, 512, 128), (70_001, 21, 42, 5), (70_003, 75, 128, 21), (66_001, 120, 200, 127),
         (66_000, 128, 96, 7), (70_000, 8, 96, 128), (150_001, 16, 64, 16)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,h,n", LARGE)
def test_large_calls(plb, two_terms, rows, k, h, n, dtype):
    for activation, biases, residual in FORMS:
        check(plb, *make(rows, k, h, n, dtype, biases, residual), activation, activation)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,h,n", SHAPES)
def test_rounded_once_small(plb, rows, k, h, n, dtype):
    for activation, biases, residual in FORMS:
        check(plb, *make(rows, k, h, n, dtype, biases, residual), activation, activation, round_hidden=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,h,n", LARGE)
def test_rounded_once_large(plb, rows, k, h, n, dtype):
    for activation, biases, residual in FORMS:
        a, grad = make(rows, k, h, n, dtype, biases, residual)
        out, d = check(plb, a, grad, activation, activation, round_hidden=True)
        again, da = check(plb, a, grad, activation, activation, round_hidden=True)
        assert torch.equal(out, again) and all(torch.equal(d[m], da[m]) for m in d)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("k,h,n", [(64, 256, 64), (21, 42, 5), (128, 512, 128)])
def test_a_row_has_the_same_bits_in_calls_of_any_size(plb, k, h, n, dtype):
    a, grad = make(70_000, k, h, n, dtype)
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("x", "residual")}
    out = plb.gated_mix(**{**a, **leaves})
    dx, dr = torch.autograd.grad(out, list(leaves.values()), grad)
    for at, rows in ((0, 1), (128, 500), (300, 65_536)):
        part = {m: a[m][:, at:at + rows].contiguous().requires_grad_(True) for m in ("x", "residual")}
        few = plb.gated_mix(**{**a, **part})
        dx_few, dr_few = torch.autograd.grad(few, list(part.values()), grad[:, at:at + rows])
        for whole, one in ((out, few), (dx, dx_few), (dr, dr_few)):
            assert torch.equal(whole[:, at:at + rows], one)


def test_floats_take_all_terms_either_way(plb):
    a, grad = make(777, 32, 96, 32, F32)
    for m in (False, True):
        leaves = {name: t.clone().requires_grad_(True) for name, t in a.items()}
        out = plb.gated_mix(**leaves, residual_scale=0.75, round_hidden=m)
        want, d = train(plb, a, grad)
        assert torch.equal(out, want)
        assert all(torch.equal(t, d[name]) for name, t in zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)))


def test_what_rounding_once_costs(plb):
    """One output channel per hidden one (weights of ones on the diagonal, u of ones, relu): out is the hidden value as it arrived."""
    for dtype, terms in ((BF16, 8), (F16, 11)):
        x = (1 + torch.rand(300, 64, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
        eye, up = torch.eye(64, dtype=dtype, device="cuda"), torch.ones(64, dtype=dtype, device="cuda")
        gate = eye * 1.2109375                                  # (8 bits, so that products have more than the type holds)
        minus = -(x.float() * 1.2109375).to(dtype)               # what is left after it is what the hidden value keeps beyond one rounding
        call = dict(up_bias=up, residual=minus, activation="relu")
        exact = x.double() * 1.2109375 + minus.double()
        out = plb.gated_mix(x, gate, eye * 0, eye, **call)
        assert_within(out, exact, 2.0 ** (-2 * terms) * (exact + -minus.double()) + 2.0 ** -20, "two terms")
        assert bool((exact != 0).any()) and not plb.gated_mix(x, gate, eye * 0, eye, **call, round_hidden=True).any()
