"""channel_mix where tiles, widths and values meet in ways that ordinary calls do not reach (bounds: mix_reference.py)."""
import math

import pytest
import torch

import mix_reference as ref
from test_gpu_channel_mix import BF16, F16, F32, make, needs_of, plb  # noqa: F401

pytestmark = pytest.mark.gpu


def _moved(t, offset):
    """The same values, contiguous, `offset` elements behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)
    return flat[offset:].view(t.shape).copy_(t)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,k,k2,n", [(400_045, 8, 0, 4), (400_045, 5, 0, 1), (123_457, 2, 0, 5), (400_063, 3, 2, 5), (38_007, 6, 0, 5)])
def test_residuals_of_tiles_of_several_blocks(plb, rows, k, k2, n, offset):
    """Narrow float rows, several blocks of 32 in a tile: a last tile that is not whole, or a residual between 16-byte boundaries,
    is copied by the lanes, and is there before its first block is finished."""
    a, _ = make(rows, k, k2, n)
    a["residual"] = _moved(a["residual"], offset)
    for activation in (None, "softmax"):
        want, bound = ref.forward(a["x"], a["weight"], a["bias"], a["residual"], a["x2"], a["weight2"], activation, -1.0)
        for checkpoint in (None, "8bit"):
            out, saved = plb.channel_mix_raw(**a, activation=activation, residual_scale=-1.0, checkpoint=checkpoint)
            ref.assert_within(out, want, bound, "%s %s" % (activation, checkpoint))
            for kept, t in ((saved.x, a["x"]), (saved.x2, a["x2"]), (saved.out, out)) if checkpoint else ():
                if kept is not None:
                    alone = plb.pack_activations(t)
                    assert torch.equal(kept.codes, alone.codes) and torch.equal(kept.scales, alone.scales)


@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,k,k2,n", [(700, 3, 100, 3), (701, 100, 2, 4), (130, 4, 73, 2), (1025, 128, 4, 4), (33, 2, 128, 2)])
def test_gradients_of_a_narrow_input_beside_a_wide_one(plb, rows, k, k2, n, dtype, weight_dtype):
    """Up to four channels of one input and of the output, and another input too wide for one pass."""
    for activation, scale in ((None, 0.25), ("relu", 1.0), ("softmax", -1.0)):
        a, g = make(rows, k, k2, n, dtype, weight_dtype)
        for checkpoint in (None, "8bit"):
            out, saved = plb.channel_mix_raw(**a, activation=activation, residual_scale=scale, checkpoint=checkpoint)
            y, x, x2 = (plb.unpack_activations(t, F32) if isinstance(t, plb.PackedActivations) else t
                        for t in (saved.out, saved.x, saved.x2))
            want = ref.gradients(g, y, x, a["weight"], x2, a["weight2"], activation, scale)
            d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, needs_of(a))
            for m in needs_of(a):
                ref.assert_within(getattr(d, m), *want[m], "%s of %s" % (m, activation))
                one = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], activation, scale, (m,))
                assert torch.equal(getattr(one, m), getattr(d, m))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("checkpoint", [None, "8bit"])
@pytest.mark.parametrize("rows,k,k2,n", [(700, 21, 21, 21), (1001, 2, 2, 2), (333, 3, 0, 4), (97, 8, 8, 8), (300, 75, 0, 16), (130, 64, 64, 64),
                                         (257, 128, 128, 128), (41, 100, 5, 33)])
def test_rows_of_zeros_have_no_gradient_whatever_comes_from_above(plb, rows, k, k2, n, dtype, checkpoint):
    """The gradient of a logarithm of the output is infinite, or NaN, in a row without a label: nothing of it goes further."""
    a, g = make(rows, k, k2, n, dtype, masked=True)
    out, saved = plb.channel_mix_raw(**a, activation="softmax", residual_scale=-1.0, checkpoint=checkpoint)
    empty = torch.isinf(a["residual"]).all(-1)
    assert bool(empty[0, 0]) and not bool(empty.all())
    bad = torch.tensor([math.nan, math.inf, -math.inf, 1.0], dtype=dtype, device="cuda")
    place = torch.arange(rows * n, device="cuda").view(1, rows, n)
    above = torch.where(empty[..., None], bad[place % 4], g)
    needs = needs_of(a)
    d = plb.channel_mix_backward(above, saved, a["weight"], a["weight2"], "softmax", -1.0, needs)
    y, x, x2 = (plb.unpack_activations(t, F32) if isinstance(t, plb.PackedActivations) else t for t in (saved.out, saved.x, saved.x2))
    want = ref.gradients(torch.where(empty[..., None], torch.zeros_like(g), g), y, x, a["weight"], x2, a["weight2"], "softmax", -1.0)
    for m in needs:
        ref.assert_within(getattr(d, m), *want[m], m)
    assert not bool(d.residual[empty].any()) and not bool(d.x[empty].any())
    # a row with a label passes on what is not finite
    row = int((~empty[0]).nonzero()[0])
    above = g.clone()
    above[0, row] = math.nan
    d = plb.channel_mix_backward(above, saved, a["weight"], a["weight2"], "softmax", -1.0, ("x", "residual"))
    assert bool(torch.isnan(d.x[0, row]).all()) and bool(torch.isfinite(d.x[0, row + 1:]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,k2,n", [(300, 21, 21, 21), (301, 2, 2, 2), (95, 3, 0, 4), (130, 64, 0, 70), (260, 8, 8, 8)])
def test_relu_of_what_is_not_finite(plb, rows, k, k2, n, dtype):
    """An infinite output passes its gradient on; as a block in 8 bits, which comes back as NaN, the block's gradients are NaN:
    no zeros that would pass for a mask.  A row that is NaN has gradients that are."""
    a, g = make(rows, k, k2, n, dtype)
    a["residual"][0, 40, 1] = math.inf
    a["x"][0, 90, 0] = math.nan
    for checkpoint in (None, "8bit"):
        out, saved = plb.channel_mix_raw(**a, activation="relu", checkpoint=checkpoint)
        assert bool(torch.isinf(out[0, 40, 1])) and bool(torch.isnan(out[0, 90]).all())
        d = plb.channel_mix_backward(g, saved, a["weight"], a["weight2"], "relu", 1.0, ("x", "residual"))
        y = out if checkpoint is None else plb.unpack_activations(saved.out, dtype)
        bad = torch.isnan(y)
        assert bool(bad[0, 90].all()) and bool(bad[0, 40, 1]) == (checkpoint is not None)
        assert torch.equal(torch.isnan(d.residual), bad)
        assert torch.equal(d.residual[~bad], torch.where(out > 0, g, torch.zeros_like(g))[~bad])
        rows_bad = bad.any(-1)
        assert torch.equal(torch.isnan(d.x).any(-1), rows_bad)


@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("rows,k,k2,n", [(200, 2, 2, 2), (200, 3, 0, 4), (200, 4, 1, 3), (200, 21, 21, 21), (200, 64, 0, 16), (200, 40, 40, 40),
                                         (200, 33, 0, 67), (200, 64, 64, 128)])
def test_rows_that_are_not_finite(plb, rows, k, k2, n, dtype, weight_dtype):
    """NaN in a row of x: all of its output is NaN, of relu too.  An infinity: each value is NaN or what the formula gives.
    Other rows have the same bits."""
    a, _ = make(rows, k, k2, n, dtype, weight_dtype)
    bad = {7: math.nan, 40: math.inf, 41: -math.inf}
    other = [r for r in range(rows) if r not in bad]
    for activation in (None, "relu", "softmax"):
        clean = plb.channel_mix(**a, activation=activation)
        for name in ("x", "x2") if k2 else ("x",):
            dirty = {**a, name: a[name].clone()}
            for row, value in bad.items():
                dirty[name][0, row, -1] = value
            out = plb.channel_mix(**dirty, activation=activation)
            assert torch.equal(out[0, other], clean[0, other])
            assert bool(torch.isnan(out[0, 7]).all())
            want, _ = ref.forward(dirty["x"], a["weight"], a["bias"], a["residual"], dirty["x2"], a["weight2"], activation, 1.0)
            for row in (40, 41):
                nan = torch.isnan(out[0, row])
                assert torch.equal(out[0, row].double()[~nan], want[0, row][~nan]), (activation, name, row)
