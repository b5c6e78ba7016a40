"""Activations of gated_mix far from zero, value by value: one channel in, between and out, so that nothing but the activation's own error is left.

Bounds.  u = 2^-24.  Of e = exp(-|g|) the exponent's rounding is off by |g| u twice over (the product and its constant) and the instruction by 2^-22; sums, products and
the quotient of 16-bit types (one reciprocal, three products) add a few u: (2 |g| + 12) u of either sigmoid(g) or 1 - sigmoid(g), where g is held
to u.  On the way out: two terms of the type, 2^-16 (bfloat16) or 2^-22 (float16), and what float16 cannot hold, 2^-25."""
import math

import pytest
import torch

from mix_reference import assert_within

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
REST = {F32: 2.0 ** -25, F16: 2.0 ** -22, BF16: 2.0 ** -16}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}


@pytest.fixture(scope="module")
def plb():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    import permutohedral_lattice_b200
    return permutohedral_lattice_b200


def alone(plb, g, up, activation):
    """act(g) up and its gradient by g, row by row."""
    x = g.view(-1, 1).clone().requires_grad_(True)
    one = torch.ones(1, 1, dtype=g.dtype, device="cuda")
    out = plb.gated_mix(x, one, 0 * one, one, up_bias=up * one[0], activation=activation)
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    return out.detach()[:, 0], dx[:, 0]


def points(dtype, least, most):
    """Both sides, closely between -most and most, and around those values that the type has."""
    g = torch.cat([torch.linspace(-most, most, 4001, dtype=torch.float64), torch.linspace(-least, least, 801, dtype=torch.float64)])
    return g.to(dtype).cuda()


def sigmoid_forms(g, activation):
    """act, act' and what either may be off, in 64 bits."""
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    off = (2 * g.abs() + 12) * U
    if activation == "sigmoid":
        return s, off * s, s * r, (2 * off + U) * s * r
    return g * s, (off + U) * (g * s).abs(), s * (1 + g * r), off * s + (2 * off + 3 * U) * (g * s * r).abs()


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_shut_and_open_gates(plb, dtype, activation):
    for up in (1.0, 2000.0):
        g = points(dtype, 3.0, 30.0 if dtype == F16 else 60.0)
        out, dx = alone(plb, g, up, activation)
        act, eact, slope, eslope = (up * v for v in sigmoid_forms(g.double(), activation))
        assert_within(out, act, eact + REST[dtype] * act.abs() + TINY[dtype], "act")
        assert_within(dx, slope, eslope + (REST[dtype] + U) * slope.abs() + TINY[dtype], "slope")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gates_shut_far_out(plb, dtype):
    """silu's products with large values of the other side: nothing of a gate that is shut comes through."""
    for g, up in ((-200.0, 100.0), (-2000.0, 2000.0), (-30000.0, 30000.0)):
        out, dx = alone(plb, torch.full((130,), g, dtype=dtype, device="cuda"), up, "silu")
        assert not out.any() and not dx.any(), (g, out[0], dx[0])
        out, dx = alone(plb, torch.full((130,), -g, dtype=dtype, device="cuda"), 1.0, "silu")
        assert bool((out == torch.tensor(-g, dtype=dtype)).all()) and bool((dx == 1).all())


def gelu_forms(g, own):
    """act, act' and what either may be off.  own: of the smaller of Phi and 1 - Phi, its polynomial of t = 1 / (1 + p |g|), whose relative slope in t is at
    most 1, beside t's own 3 u; it is times exp(-g^2 / 2), (1.5 g^2 + 8) u off, from three roundings of its exponent and an instruction of 2^-22."""
    small = 0.5 * torch.erfc(g.abs() / math.sqrt(2))
    cdf = torch.where(g < 0, small, 1 - small)
    density = g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    ecdf = ((1.5 * g * g + 12) * U + own) * small + U * cdf
    return g * cdf, g.abs() * ecdf + U * (g * cdf).abs(), cdf + density, ecdf + (1.5 * g * g + 10) * U * density.abs() + U * (cdf + density).abs()


def test_gelu_of_floats(plb):
    """To some u of the value, in the tails too."""
    g = points(F32, 1.0, 10.0)
    out, dx = alone(plb, g, 1.0, "gelu")
    act, eact, slope, eslope = gelu_forms(g.double(), 6 * U)
    assert_within(out, act, eact + REST[F32] * act.abs(), "act")
    assert_within(dx, slope, eslope + REST[F32] * slope.abs(), "slope")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gelu_of_16_bit_types(plb, dtype):
    """To 2^-18 of the smaller of Phi and 1 - Phi, in the tails too, where either type holds more of it than an absolute 1e-7."""
    for up in (1.0, 30000.0):
        g = points(dtype, 3.0, 6.5 if dtype == F16 else 12.0)
        out, dx = alone(plb, g, up, "gelu")
        held = float(torch.tensor(up, dtype=dtype))      # (29 952 in bfloat16, whose numbers are 128 apart there)
        act, eact, slope, eslope = (held * v for v in gelu_forms(g.double(), 2.0 ** -18 + 6 * U))
        if dtype == F16 and up > 1.0:      # (what it holds)
            keep = (act.abs() < 60000.0) & (slope.abs() < 60000.0)
            out, dx, act, eact, slope, eslope = (v[keep] for v in (out, dx, act, eact, slope, eslope))
        assert_within(out, act, eact + (REST[dtype] + U) * act.abs() + TINY[dtype], "act")
        assert_within(dx, slope, eslope + (REST[dtype] + U) * slope.abs() + TINY[dtype], "slope")
