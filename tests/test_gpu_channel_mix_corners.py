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
            out, _ = plb.channel_mix_raw(**a, activation=activation, residual_scale=-1.0, checkpoint=checkpoint)
            ref.assert_within(out, want, bound, "%s %s" % (activation, checkpoint))
