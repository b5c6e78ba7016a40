"""What channel_mix and the 8-bit activations refuse, on the CPU: types and shapes are looked at before the device."""
import ctypes

import pytest
import torch

import permutohedral_lattice_b200 as plb
from permutohedral_lattice_b200 import capi


def _args(k=3, n=2, k2=0, dtype=torch.float32):
    a = {"x": torch.zeros(1, 4, k, dtype=dtype), "weight": torch.zeros(k, n, dtype=dtype)}
    if k2:
        a.update(x2=torch.zeros(1, 4, k2, dtype=dtype), weight2=torch.zeros(k2, n, dtype=dtype))
    return a


@pytest.mark.parametrize("change,error", [
    ({}, ValueError),                                                     # a CPU tensor
    ({"x": [1.0]}, TypeError),
    ({"x": torch.zeros(1, 4, 3, dtype=torch.float64)}, TypeError),
    ({"x": torch.zeros((), dtype=torch.float32)}, ValueError),
    ({"x": torch.zeros(1, 4, 5)}, ValueError),
    ({"weight": torch.zeros(3, 2, dtype=torch.bfloat16)}, TypeError),     # float32 values take float32 weights
    ({"weight": torch.zeros(3)}, ValueError),
    ({"weight": torch.zeros(3, 0)}, ValueError),
    ({"weight": torch.zeros(3, 129)}, ValueError),
    ({"x": torch.zeros(4, 129), "weight": torch.zeros(129, 2)}, ValueError),
    ({"x2": torch.zeros(1, 4, 3)}, ValueError),                           # without its weight
    ({"x2": torch.zeros(1, 5, 3), "weight2": torch.zeros(3, 2)}, ValueError),
    ({"x2": torch.zeros(1, 4, 3), "weight2": torch.zeros(3, 3)}, ValueError),
    ({"x2": torch.zeros(1, 4, 3, dtype=torch.float16), "weight2": torch.zeros(3, 2)}, TypeError),
    ({"bias": torch.zeros(3)}, ValueError),
    ({"bias": torch.zeros(2, dtype=torch.float16)}, TypeError),
    ({"residual": torch.zeros(1, 4, 3)}, ValueError),
    ({"residual": torch.zeros(2)}, ValueError),                           # no broadcasting
    ({"activation": "gelu"}, ValueError),
    ({"checkpoint": "4bit"}, ValueError),
])
def test_channel_mix_refuses(change, error):
    with pytest.raises(error):
        plb.channel_mix(**{**_args(), **change})
    with pytest.raises(error):
        plb.channel_mix_raw(**{**_args(), **change})


def test_backward_refuses():
    g, w = torch.zeros(1, 4, 2), torch.zeros(3, 2)
    saved = plb.MixSaved(torch.zeros(1, 4, 3), None, torch.zeros(1, 4, 2))
    for args, kw, error in [
        ((g, saved, w), {}, ValueError),                                   # CPU tensors
        ((g, saved, w), {"needs": ("y",)}, ValueError),
        ((g, tuple(saved), w), {}, TypeError),
        ((g, saved, w), {"needs": ("x2",)}, ValueError),
        ((g, saved, w.double()), {}, TypeError),
        ((g, saved._replace(x=None), w), {}, TypeError),
        ((g, saved._replace(out=None), w), {"activation": "softmax"}, TypeError),
        ((g, saved._replace(x=torch.zeros(1, 5, 3)), w), {}, ValueError),
        ((g, saved._replace(x=torch.zeros(1, 4, 3).half()), w), {}, TypeError),
        ((g, saved, w), {"activation": "tanh"}, ValueError),
    ]:
        with pytest.raises(error):
            plb.channel_mix_backward(*args, **kw)


def test_packed_activations_refuse():
    with pytest.raises(ValueError):
        plb.pack_activations(torch.zeros(3))
    with pytest.raises(TypeError):
        plb.pack_activations(torch.zeros(3, dtype=torch.int32))
    codes, scales = torch.zeros(33, dtype=torch.uint8), torch.zeros(2, dtype=torch.int16)
    for p, error in [
        (plb.PackedActivations(codes, scales, (33,), torch.float32), ValueError),   # CPU tensors
        (plb.PackedActivations(codes, scales[:1], (33,), torch.float32), ValueError),
        (plb.PackedActivations(codes, scales, (3, 10), torch.float32), ValueError),
        (plb.PackedActivations(codes.to(torch.int8), scales, (33,), torch.float32), TypeError),
        (plb.PackedActivations(codes, scales, (33,), torch.int32), TypeError),
        (plb.PackedActivations(torch.zeros(66, dtype=torch.uint8)[::2], scales, (33,), torch.float32), ValueError),
        ((codes, scales), TypeError),
    ]:
        with pytest.raises(error):
            plb.unpack_activations(p)


def test_c_entries_refuse_before_any_launch():
    L, none = capi.lib(), capi.PlPacked(0, 0)

    def shape(**kw):
        fields = dict(rows=4, k=3, k2=0, n=2, activation=0, dtype=0, weight_dtype=0, residual_scale=1.0)
        return ctypes.byref(capi.PlMix(**{**fields, **kw}))

    def mix(m, out=16, x=16, x2=0, w=16, w2=0, keep=none, keep2=none):
        return L.pl_channel_mix(m, out, x, x2, w, w2, 0, 0, keep, keep2, none, 0)

    assert mix(None) == capi.PL_INVALID_ARGUMENT
    for bad in ({"rows": -1}, {"rows": (1 << 40) + 1}, {"k": 0}, {"k2": -1}, {"n": 0}, {"activation": 3}, {"activation": -1},
                {"dtype": 3}, {"weight_dtype": 1}):
        assert mix(shape(**bad)) == capi.PL_INVALID_ARGUMENT, bad
    for bad in ({"k": 129}, {"n": 129}, {"k2": 129}):
        assert mix(shape(**bad)) == capi.PL_UNSUPPORTED_DIMS, bad
    for bad in ({"out": 0}, {"x": 0}, {"w": 0}, {"keep": capi.PlPacked(16, 0)}, {"keep2": capi.PlPacked(16, 16)}):
        assert mix(shape(), **bad) == capi.PL_INVALID_ARGUMENT, bad
    assert mix(shape(k2=1)) == capi.PL_INVALID_ARGUMENT
    assert mix(shape(rows=0), 0, 0, 0, 0) == capi.PL_OK

    def back(m, grad=16, out=0, x=16, w=16, d=None, ws=16, nbytes=1 << 30):
        kept = lambda p: capi.PlKept(p, none)   # noqa: E731
        d = {"x": 16} if d is None else d
        return L.pl_channel_mix_backward(m, grad, kept(out), kept(x), kept(0), w, 0, capi.PlMixGradients(**d), ws, nbytes, 0)

    assert back(shape(), grad=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(activation=2)) == capi.PL_INVALID_ARGUMENT              # without its output
    assert back(shape(), x=0, d={"weight": 16}) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), w=0) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), d={"x2": 16}) == capi.PL_INVALID_ARGUMENT
    assert back(shape(), nbytes=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(), ws=0) == capi.PL_WORKSPACE_TOO_SMALL
    assert back(shape(k=129)) == capi.PL_UNSUPPORTED_DIMS
    assert L.pl_channel_mix_workspace_bytes(shape(), None) == capi.PL_INVALID_ARGUMENT
    p = capi.PlPacked(16, 16)
    assert L.pl_pack_activations(p, 16, -1, 0, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_pack_activations(p, 16, 4, 3, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_pack_activations(none, 16, 4, 0, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_unpack_activations(0, p, 4, 0, 0) == capi.PL_INVALID_ARGUMENT
    assert L.pl_unpack_activations(0, none, 0, 0, 0) == capi.PL_OK


def test_the_reference_form_of_the_8_bit_blocks():
    """The tests' own form: half a step off at most, whole steps exact, and what the header says."""
    import numpy as np
    from mix_reference import pack, unpack
    rng = np.random.default_rng(0)
    v = (rng.standard_normal(1000) * 10.0 ** rng.integers(-30, 30, 1000)).astype(np.float32)
    v[64:96] = np.abs(v[64:96])
    codes, headers = pack(v)
    back = unpack(codes, headers)
    step = np.repeat(2.0 ** ((headers & 255) - 127.0), 32)[:1000]
    assert (np.abs(back - v) <= step / 2).all() and (headers[2] & 256) == 0 and (headers[3] & 256) == 256
    again, same = pack(back.astype(np.float32))
    assert np.array_equal(unpack(again, same), back)
