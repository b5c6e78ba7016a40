"""What channel_norm and channel_dropout refuse, on the CPU: types and shapes are looked at before the device."""
import ctypes

import numpy as np
import pytest
import torch

import permutohedral_lattice_b200 as plb
from permutohedral_lattice_b200 import capi

X = torch.zeros(2, 4, 3)


@pytest.mark.parametrize("args,error", [
    ({"after": plb.Norm()}, ValueError),                                            # a CPU tensor
    ({}, ValueError),                                                               # nothing to do
    ({"x": [1.0], "after": plb.Norm()}, TypeError),
    ({"x": X.double(), "after": plb.Norm()}, TypeError),
    ({"x": torch.zeros(()), "after": plb.Norm()}, ValueError),
    ({"x": torch.zeros(2, 0), "after": plb.Norm()}, ValueError),
    ({"x": torch.zeros(2, 513), "after": plb.Norm()}, ValueError),
    ({"after": (None, None)}, TypeError),
    ({"after": plb.Norm(kind="batch")}, ValueError),
    ({"after": plb.Norm(eps=0.0)}, ValueError),
    ({"after": plb.Norm(eps=float("nan"))}, ValueError),
    ({"after": plb.Norm(eps=1e-60)}, ValueError),                                   # zero as a float
    ({"before": plb.Norm(torch.ones(4))}, ValueError),
    ({"before": plb.Norm(torch.ones(3), torch.zeros(3, 1))}, ValueError),
    ({"before": plb.Norm(torch.ones(3).half())}, TypeError),
    ({"x": X.half(), "after": plb.Norm(torch.ones(3)), "before": plb.Norm(torch.ones(3).half())}, TypeError),
    ({"residual": torch.zeros(4, 3)}, ValueError),
    ({"residual": X.half()}, TypeError),
    ({"gate": torch.zeros(2, 4, 1)}, ValueError),
    ({"gate": X.half()}, TypeError),
    ({"after": plb.Norm(), "dropout": 1.0, "seed": 1}, ValueError),
    ({"after": plb.Norm(), "dropout": -0.1, "seed": 1}, ValueError),
    ({"after": plb.Norm(), "dropout": float("nan"), "seed": 1}, ValueError),
    ({"after": plb.Norm(), "dropout": 0.1}, ValueError),                            # without a seed
    ({"after": plb.Norm(), "dropout": 0.1, "seed": 1 << 64}, ValueError),
    ({"after": plb.Norm(), "dropout": 0.1, "seed": (1, 2, 3)}, ValueError),
    ({"after": plb.Norm(), "dropout": 0.1, "seed": torch.zeros(2)}, ValueError),
    ({"after": plb.Norm(), "dropout": 0.1, "seed": torch.zeros(3, dtype=torch.int64)}, ValueError),
])
def test_channel_norm_refuses(args, error):
    with pytest.raises(error):
        plb.channel_norm(**{"x": X, **args})


def test_channel_dropout_refuses():
    for args, error in [((X, 0.1, 1), ValueError), ((X, 1.5, 1), ValueError), ((X, 0.1, None), ValueError), ((X.int(), 0.1, 1), TypeError),
                        ((X, 0.1, 1, X[0]), ValueError), ((X, 0.1, 1, X.half()), TypeError), ((X, 0.1, "1"), ValueError)]:
        with pytest.raises(error):
            plb.channel_dropout(*args)


def test_c_entries_refuse_before_any_launch():
    L = capi.lib()
    none = capi.PlNorm(0, 0.0)
    rms = capi.PlNorm(2, 1e-5)

    def shape(**kw):
        fields = dict(rows=4, channels=3, dtype=0, vector_dtype=0, gate_of_values=0, residual_scale=1.0, after=none, before=rms,
                      dropout=capi.PlDropout(0.0, 0, 0))
        return ctypes.byref(capi.PlChannelNorm(**{**fields, **kw}))

    def forward(m, h=0, y=16, x=16):
        return L.pl_channel_norm(m, h, y, x, 0, 0, 0, 0, 0, 0, 0, 0)

    assert forward(None) == capi.PL_INVALID_ARGUMENT
    for bad in ({"rows": -1}, {"rows": (1 << 40) + 1}, {"channels": 0}, {"dtype": 3}, {"vector_dtype": 1}, {"after": capi.PlNorm(3, 1.0)},
                {"before": capi.PlNorm(1, 0.0)}, {"before": capi.PlNorm(1, float("nan"))}, {"dropout": capi.PlDropout(1.0, 0, 0)},
                {"dropout": capi.PlDropout(float("nan"), 0, 0)}):
        assert forward(shape(**bad)) == capi.PL_INVALID_ARGUMENT, bad
    assert forward(shape(channels=513)) == capi.PL_UNSUPPORTED_DIMS
    assert forward(shape(), x=0) == capi.PL_INVALID_ARGUMENT
    assert forward(shape(), y=0) == capi.PL_INVALID_ARGUMENT
    assert forward(shape(before=none), y=16) == capi.PL_INVALID_ARGUMENT
    assert forward(shape(rows=0), 0, 0, 0) == capi.PL_OK

    def back(m, dh=0, dy=16, x=16, d=None, ws=16, nbytes=1 << 30):
        return L.pl_channel_norm_backward(m, dh, dy, x, 0, 0, 0, 0, 0, 0, capi.PlNormGradients(**(d or {"x": 16})), ws, nbytes, 0)

    assert back(shape(), dy=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), dh=16, dy=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(before=none), dy=16) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), d={"after_weight": 16}) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), x=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), nbytes=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(), ws=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(), ws=20) == capi.PL_INVALID_ARGUMENT
    p = ctypes.byref(capi.PlDropout(0.5, 0, 0))
    assert L.pl_channel_dropout(16, 0, 16, 0, -1, 0, 1.0, p, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_channel_dropout(16, 0, 16, 0, 4, 3, 1.0, p, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_channel_dropout(0, 0, 16, 0, 4, 0, 1.0, p, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_channel_dropout(16, 0, 16, 0, 4, 0, 1.0, None, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_channel_dropout(0, 0, 0, 0, 0, 0, 1.0, p, 0, 0) == capi.PL_OK


def test_the_reference_generator():
    """The tests' own form of it: the published words of a counter and key of zeros, and of ones (Random123's known answers)."""
    from norm_reference import philox_words
    assert [hex(int(w)) for w in philox_words(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    assert np.array_equal(philox_words(9, 3, 1 << 40)[:4], philox_words(4, 3, 1 << 40))
