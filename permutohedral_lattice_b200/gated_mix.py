"""A gated feed-forward block of points' features, the nonlinear map beside `channel_mix`'s linear one:

    out = (act(x @ gate_weight + gate_bias) * (x @ up_weight + up_bias)) @ down_weight + down_bias + residual_scale * residual

over channels-last tensors [*, K], in one kernel after one that lays out the weights: the hidden channels' values are neither written nor kept, the
backward pass makes them again from x.  The reference ships no such operator; networks that make a CRF's features or unaries of points have it.
"""
import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import capi
from .channel_mix import MOST_CHANNELS, _DTYPES, _check_device, _check_values, _contiguous, _ptr
from .channel_norm import _follows
from .lattice_filter import _OnDevice, _stream_handle

MOST_HIDDEN = 512
_ACTIVATIONS = {"silu": capi.PL_GATE_SILU, "gelu": capi.PL_GATE_GELU, "sigmoid": capi.PL_GATE_SIGMOID, "relu": capi.PL_GATE_RELU}
# What _GatedMix takes gradients of, in its order; the weights in that of the C structure.
_WEIGHTS = ("gate_weight", "up_weight", "down_weight", "gate_bias", "up_bias", "down_bias")
_NAMES = ("x", "residual") + _WEIGHTS


@functools.lru_cache(maxsize=1024)
def _structure(rows, k, h, n, activation, dtype, residual_scale, round_hidden):
    """The C structure of a call, which the library only reads, and the bytes of workspace that it takes, forward and backward."""
    m = ctypes.byref(capi.PlGated(rows, k, h, n, _ACTIVATIONS[activation], _DTYPES[dtype], residual_scale, int(round_hidden)))
    nbytes = ctypes.c_size_t(0)
    sizes = []
    for backward in (0, 1):
        capi.check(capi.lib().pl_gated_mix_workspace_bytes(m, backward, ctypes.byref(nbytes)), "pl_gated_mix_workspace_bytes")
        sizes.append(nbytes.value)
    return m, sizes[0], sizes[1]


def _check(x, residual, weights, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError('activation must be "silu", "gelu", "sigmoid" or "relu"')
    _check_values(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [*, channels]")
    gate, up, down = weights[:3]
    for name, w in zip(_WEIGHTS, weights):
        if w is None and name.endswith("bias"):
            continue
        _check_values(w, name, x.dtype)
    k = x.shape[-1]
    if gate.dim() != 2 or gate.shape[0] != k:
        raise ValueError("gate_weight must be [channels of x, hidden channels]")
    if up.shape != gate.shape:
        raise ValueError("up_weight must have gate_weight's shape")
    h = gate.shape[1]
    if down.dim() != 2 or down.shape[0] != h:
        raise ValueError("down_weight must be [hidden channels, channels of the output]")
    n = down.shape[1]
    if not 1 <= k <= MOST_CHANNELS or not 1 <= n <= MOST_CHANNELS or not 1 <= h <= MOST_HIDDEN:
        raise ValueError("1 to %d channels in and out, and 1 to %d in between, are supported" % (MOST_CHANNELS, MOST_HIDDEN))
    for name, b, size in zip(_WEIGHTS[3:], weights[3:], (h, h, n)):
        if b is not None and tuple(b.shape) != (size,):
            raise ValueError("%s must be [%d]" % (name, size))
    if residual is not None:
        _check_values(residual, "residual", x.dtype)
        if tuple(residual.shape) != tuple(x.shape[:-1]) + (n,):
            raise ValueError("residual must have the output's shape")
    index = x.get_device()
    if index < 0 or (residual is not None and residual.get_device() != index) or any(w is not None and w.get_device() != index for w in weights):
        _check_device((("x", x), ("residual", residual)) + tuple(zip(_WEIGHTS, weights)))
    return h, n


def _forward(device, s, n, x, residual, gate, up, down, gate_bias, up_bias, down_bias):
    out = x.new_empty(x.shape[:-1] + (n,))
    with _OnDevice(device):
        workspace = torch.empty(s[1], dtype=torch.uint8, device=device)
        rc = capi.lib().pl_gated_mix(s[0], out.data_ptr(), x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), _ptr(gate_bias), _ptr(up_bias),
                                     _ptr(down_bias), _ptr(residual), workspace.data_ptr(), s[1], _stream_handle(device))
        if rc != capi.PL_OK:
            capi.check(rc, "pl_gated_mix")
    return out


class _GatedMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, s, n, x, residual, *weights):
        ctx.args = device, s
        ctx.save_for_backward(x, *weights)
        return _forward(device, s, n, x, residual, *weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, *weights = ctx.saved_tensors
        device, s = ctx.args
        grad = grad.contiguous()
        made = {name: torch.empty_like(t) for name, t, wanted in zip(_NAMES, (x, grad, *weights), ctx.needs_input_grad[3:]) if wanted}
        with _OnDevice(device):
            workspace = torch.empty(s[2], dtype=torch.uint8, device=device)
            capi.check(capi.lib().pl_gated_mix_backward(
                s[0], grad.data_ptr(), x.data_ptr(), *map(_ptr, weights[:5]),
                capi.PlGatedGradients(**{name: t.data_ptr() for name, t in made.items()}), workspace.data_ptr(), s[2], _stream_handle(device)),
                "pl_gated_mix_backward")
        return (None, None, None) + tuple(made.get(name) for name in _NAMES)


def gated_mix(x, gate_weight, up_weight, down_weight, gate_bias=None, up_bias=None, down_bias=None, residual=None, activation="silu",
              residual_scale=1.0, round_hidden=False):
    """(act(x @ gate_weight + gate_bias) * (x @ up_weight + up_bias)) @ down_weight + down_bias + residual_scale * residual, with
    gradients for all tensors.

    x [*, K], gate_weight and up_weight [K, H], down_weight [H, N], biases [H], [H], [N], residual and the output [*, N]: all of one type,
    float32, float16 or bfloat16; up to 128 channels in and out and 512 in between.  activation: "silu", "gelu" (of the normal distribution
    itself, to 2^-18 of it in 16-bit types), "sigmoid" or "relu".

    Products of floats are off by 2^-25, sums are float32, cut on the tensor cores: results of floats are 3e-7 to 6e-7 off in the norm.  Of
    16-bit types the hidden values (and, in the backward pass, their gradients) go on to the next product as two terms of that type, so that
    results are off by their own rounding.  round_hidden: rounded once to it, as between layers of their own; results are then 1.4 times as
    far off, and large calls faster (forward by an eighth, a training step by up to a third).  Gradients' sums over rows have a fixed order.

    x, the weights and hidden values have to be finite, and below 3.38e38 (of float16 all of them below 65504): of a row that is not, values
    come out infinite or NaN, other rows are as they would be; the weights' gradients are then not finite.  Hidden values of float16 below
    2^-25 are zeros.  So are their gradients, but where all of the upstream gradient is below 2^-6 they are scaled: zeros below 2^-19 of its
    largest value, and to stay below 2^22 of it.

    In a CUDA graph: one ordinary call of the same sizes before the capture, forward and backward, which sets the kernels up; forward and
    backward together, on leaves made inside it."""
    weights = (gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias)
    h, n = _check(x, residual, weights, activation)
    k = x.shape[-1]
    s = _structure(x.numel() // k, k, h, n, activation, x.dtype, float(residual_scale), bool(round_hidden))
    tensors = (x.contiguous(), _contiguous(residual), gate_weight.contiguous(), up_weight.contiguous(), down_weight.contiguous(), _contiguous(gate_bias),
               _contiguous(up_bias), _contiguous(down_bias))
    if not _follows(tensors):
        return _forward(x.device, s, n, *tensors)
    return _GatedMix.apply(x.device, s, n, *tensors)
