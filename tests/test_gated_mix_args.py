"""What gated_mix refuses, on the CPU: types and shapes are looked at before the device."""
import ctypes

import pytest
import torch

import permutohedral_lattice_b200 as plb
from permutohedral_lattice_b200 import capi


def _args(**change):
    a = {"x": torch.zeros(1, 4, 3), "gate_weight": torch.zeros(3, 5), "up_weight": torch.zeros(3, 5), "down_weight": torch.zeros(5, 2)}
    return {**a, **change}


@pytest.mark.parametrize("change,error", [
    ({}, ValueError),                                                      # CPU tensors
    ({"x": [1.0]}, TypeError),
    ({"x": torch.zeros(1, 4, 3).double()}, TypeError),
    ({"x": torch.zeros(())}, ValueError),
    ({"x": torch.zeros(1, 4, 2)}, ValueError),
    ({"gate_weight": None}, TypeError),
    ({"gate_weight": torch.zeros(3, 5).half()}, TypeError),
    ({"gate_weight": torch.zeros(15)}, ValueError),
    ({"up_weight": torch.zeros(3, 4)}, ValueError),
    ({"down_weight": torch.zeros(4, 2)}, ValueError),
    ({"down_weight": torch.zeros(5)}, ValueError),
    ({"down_weight": torch.zeros(5, 0)}, ValueError),
    ({"down_weight": torch.zeros(5, 129)}, ValueError),
    ({"x": torch.zeros(4, 129), "gate_weight": torch.zeros(129, 5), "up_weight": torch.zeros(129, 5)}, ValueError),
    ({"gate_weight": torch.zeros(3, 513), "up_weight": torch.zeros(3, 513), "down_weight": torch.zeros(513, 2)}, ValueError),
    ({"gate_bias": torch.zeros(4)}, ValueError),
    ({"up_bias": torch.zeros(5).half()}, TypeError),
    ({"down_bias": torch.zeros(5)}, ValueError),
    ({"residual": torch.zeros(1, 4, 3)}, ValueError),
    ({"residual": torch.zeros(1, 4, 2).half()}, TypeError),
    ({"activation": "tanh"}, ValueError),
    ({"activation": None}, ValueError),
])
def test_gated_mix_refuses(change, error):
    with pytest.raises(error):
        plb.gated_mix(**_args(**change))


def test_c_entries_refuse_before_any_launch():
    L = capi.lib()

    def shape(**kw):
        fields = dict(rows=4, k=3, h=5, n=2, activation=0, dtype=0, residual_scale=1.0)
        return ctypes.byref(capi.PlGated(**{**fields, **kw}))

    def forward(m, out=16, x=16, w=(16, 16, 16), ws=16, nbytes=1 << 40):
        return L.pl_gated_mix(m, out, x, *w, 0, 0, 0, 0, ws, nbytes, 0)

    assert forward(None) == capi.PL_INVALID_ARGUMENT
    for bad in ({"rows": -1}, {"rows": (1 << 40) + 1}, {"k": 0}, {"h": 0}, {"n": 0}, {"activation": 4}, {"activation": -1}, {"dtype": 3}):
        assert forward(shape(**bad)) == capi.PL_INVALID_ARGUMENT, bad
    for bad in ({"k": 129}, {"h": 513}, {"n": 129}):
        assert forward(shape(**bad)) == capi.PL_UNSUPPORTED_DIMS, bad
    for bad in ({"out": 0}, {"x": 0}, {"w": (0, 16, 16)}, {"w": (16, 16, 0)}):
        assert forward(shape(), **bad) == capi.PL_INVALID_ARGUMENT, bad
    assert forward(shape(rows=0), 0, 0, (0, 0, 0), 0, 0) == capi.PL_OK
    assert forward(shape(), ws=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert forward(shape(), nbytes=100) == capi.PL_WORKSPACE_TOO_SMALL
    assert forward(shape(), ws=24) == capi.PL_INVALID_ARGUMENT

    def back(m, grad=16, x=16, d=None, ws=16, nbytes=1 << 40):
        d = capi.PlGatedGradients(**({"gate_weight": 16} if d is None else d))
        return L.pl_gated_mix_backward(m, grad, x, 16, 16, 16, 0, 0, d, ws, nbytes, 0)

    assert back(shape(), grad=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), x=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), nbytes=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(), ws=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(), ws=24) == capi.PL_INVALID_ARGUMENT
    assert back(shape(h=513)) == capi.PL_UNSUPPORTED_DIMS
    assert L.pl_gated_mix_workspace_bytes(shape(), 1, None) == capi.PL_INVALID_ARGUMENT
