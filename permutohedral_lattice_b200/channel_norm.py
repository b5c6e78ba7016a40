"""What a network's blocks of features take beside their products: norms over the channels, and dropout.

    u = after(x)                              the norm after the block that gave x
    h = residual_scale * residual + gate * dropout(u)
    y = before(h)                             the norm before the next block

over channels-last tensors [*, C] of points, in one pass, and their gradients in one more, from what came in: neither the
normed values nor the dropout's mask are kept (`channel_norm`).  `channel_dropout` is dropout by itself, with the residual.
The reference ships no such operators; networks that make a CRF's features or unaries of points have them.
"""
import ctypes
import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import capi
from .channel_mix import _DTYPES, _check_device, _check_values, _contiguous, _ptr
from .lattice_filter import _OnDevice, _stream_handle, _watched_by_torch

MOST_NORM_CHANNELS = 512
_KINDS = {"layer": capi.PL_NORM_LAYER, "rms": capi.PL_NORM_RMS}


class Norm(NamedTuple):
    """A norm over the channels: kind "layer", (x - mean) / sqrt(variance + eps), or "rms", x / sqrt(mean of squares + eps); times
    weight [C], plus bias [C], where they are given."""
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    kind: str = "layer"
    eps: float = 1e-5


def _check_share(p, seed):
    """p as a number, and seed as a tensor or a pair of numbers below 2^64."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError("the share of dropped values must be at least 0 and below 1")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or tuple(seed.shape) != (2,):
            raise ValueError("a seed on the GPU must be int64 [2]: the generator's key, and an offset")
        return p, seed
    if seed is None:
        if p > 0.0:
            raise ValueError("dropout takes a seed")
        return p, (0, 0)
    pair = (seed, 0) if isinstance(seed, int) else tuple(seed)
    if len(pair) != 2 or not all(isinstance(v, int) and -(1 << 63) <= v < (1 << 64) for v in pair):
        raise ValueError("seed must be a whole number of 64 bits, two of them (key, offset), or an int64 tensor of both")
    return p, tuple(v % (1 << 64) for v in pair)


def _check_norm(norm, name, channels):
    if not isinstance(norm, Norm):
        raise TypeError("%s must be a Norm" % name)
    if norm.kind not in _KINDS:
        raise ValueError('%s: kind must be "layer" or "rms"' % name)
    if not 0.0 < float(norm.eps) <= 3.402e38 or ctypes.c_float(norm.eps).value == 0.0:
        raise ValueError("%s: eps must be positive" % name)
    for part, t in (("weight", norm.weight), ("bias", norm.bias)):
        if t is not None:
            _check_values(t, "%s.%s" % (name, part))
            if tuple(t.shape) != (channels,):
                raise ValueError("%s.%s must be [channels]" % (name, part))


def _named(residual, gate, after, before):
    """The vectors of the channels among the arguments, with their names."""
    found = [(place + part, t) for place, norm in (("after", after), ("before", before)) if norm is not None
             for part, t in ((".weight", norm.weight), (".bias", norm.bias)) if t is not None]
    return found if gate is None or gate.dim() > 1 else found + [("gate", gate)]


def _check(x, residual, gate, after, before, p, seed):
    """Returns the device and the type of the channels' vectors."""
    _check_values(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [*, channels]")
    channels = x.shape[-1]
    if not 1 <= channels <= MOST_NORM_CHANNELS:
        raise ValueError("x: 1 to %d channels are supported" % MOST_NORM_CHANNELS)
    if after is not None:
        _check_norm(after, "after", channels)
    if before is not None:
        _check_norm(before, "before", channels)
    if after is None and before is None and residual is None and gate is None and not p:
        raise ValueError("nothing to do: a norm, a residual, a gate or dropout is needed")
    if residual is not None:
        _check_values(residual, "residual", x.dtype)
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
    if gate is not None:
        _check_values(gate, "gate")
        if gate.shape == x.shape and gate.dim() > 1:
            _check_values(gate, "gate", x.dtype)
        elif tuple(gate.shape) != (channels,):
            raise ValueError("gate must be [channels], or of x's shape")
    vectors = _named(residual, gate, after, before)
    vector_dtype = vectors[0][1].dtype if vectors else x.dtype
    index = x.get_device()
    same = index >= 0 and (residual is None or residual.get_device() == index) and (gate is None or gate.get_device() == index) and (
        not p or not isinstance(seed, torch.Tensor) or seed.get_device() == index)
    for name, t in vectors:
        if t.dtype is not vector_dtype or (vector_dtype is not x.dtype and vector_dtype is not torch.float32):
            raise TypeError("%s must be float32 or of x's dtype, like all vectors of the channels" % name)
        same = same and t.get_device() == index
    if not same:
        _check_device([("x", x), ("residual", residual), ("gate", gate)] + vectors + [("seed", seed if p and isinstance(seed, torch.Tensor) else None)])
    return x.device, vector_dtype


@functools.lru_cache(maxsize=1024)
def _dropout_of(p, key, offset):
    return ctypes.byref(capi.PlDropout(p, key, offset))


@functools.lru_cache(maxsize=1024)
def _structure(rows, channels, dtype, vector_dtype, gate_of_values, residual_scale, after, after_eps, before, before_eps, p, key, offset):
    """The C structure of a call, which the library only reads: sizes and numbers, no addresses."""
    def norm(kind, eps):
        return capi.PlNorm(_KINDS[kind], eps) if kind else capi.PlNorm(capi.PL_NORM_NONE, 0.0)

    return ctypes.byref(capi.PlChannelNorm(rows, channels, _DTYPES[dtype], _DTYPES[vector_dtype], int(gate_of_values), residual_scale,
                                           norm(after, after_eps), norm(before, before_eps), capi.PlDropout(p, key, offset)))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(channels):
    nbytes = ctypes.c_size_t(0)
    m = _structure(0, channels, torch.float32, torch.float32, False, 1.0, None, 0.0, None, 0.0, 0.0, 0, 0)
    capi.check(capi.lib().pl_channel_norm_workspace_bytes(m, ctypes.byref(nbytes)), "pl_channel_norm_workspace_bytes")
    return nbytes.value


def _forward(device, m, wants_h, wants_y, seed, x, residual, gate, after_weight, after_bias, before_weight, before_bias):
    h = torch.empty_like(x) if wants_h else None
    y = torch.empty_like(x) if wants_y else None
    with _OnDevice(device):
        rc = capi.lib().pl_channel_norm(m, _ptr(h), _ptr(y), x.data_ptr(), _ptr(residual), _ptr(gate), _ptr(after_weight), _ptr(after_bias),
                                        _ptr(before_weight), _ptr(before_bias), _ptr(seed), _stream_handle(device))
        if rc != capi.PL_OK:
            capi.check(rc, "pl_channel_norm")
    return h, y


# What _ChannelNorm takes gradients of, in its order.
_NAMES = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")


class _ChannelNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, m, has_after, wants_h, wants_y, seed, x, residual, gate, *weights):
        h, y = _forward(device, m, wants_h, wants_y, seed, x, residual, gate, *weights)
        ctx.set_materialize_grads(False)
        ctx.device, ctx.m, ctx.outputs = device, m, (wants_h, wants_y)
        keep_x = has_after or wants_y or ctx.needs_input_grad[8]
        ctx.save_for_backward(x if keep_x else None, residual if wants_y else None, gate, seed, *weights)
        return (h, y) if wants_h and wants_y else (y if h is None else h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, residual, gate, seed, *weights = ctx.saved_tensors
        m, device = ctx.m, ctx.device
        with_h, with_y = ctx.outputs
        dh, dy = grads if with_h and with_y else (grads[0], None) if with_h else (None, grads[0])
        if dh is None and dy is None:
            return (None,) * (6 + len(_NAMES))
        if with_y and dy is None:       # nobody used y
            dy = torch.zeros_like(dh)
        dh, dy = _contiguous(dh), _contiguous(dy)
        like = dh if dy is None else dy
        made = {name: torch.empty_like(t) for name, t, wanted in zip(_NAMES, (like, like, gate, *weights), ctx.needs_input_grad[6:]) if wanted}
        with _OnDevice(device):
            workspace = torch.empty(_workspace_bytes(like.shape[-1]), dtype=torch.uint8, device=device)
            d = capi.PlNormGradients(**{name: t.data_ptr() for name, t in made.items()})
            capi.check(capi.lib().pl_channel_norm_backward(
                m, _ptr(dh), _ptr(dy), _ptr(x), _ptr(residual), _ptr(gate), _ptr(weights[0]), _ptr(weights[1]), _ptr(weights[2]), _ptr(seed),
                d, workspace.data_ptr(), workspace.numel(), _stream_handle(device)), "pl_channel_norm_backward")
        return (None,) * 6 + tuple(made.get(name) for name in _NAMES)


def _follows(tensors):
    """Whether autograd, or something else that follows tensors, has to know of a call."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return _watched_by_torch()


def channel_norm(x, residual=None, gate=None, after=None, before=None, residual_scale=1.0, dropout=0.0, seed=None):
    """h = residual_scale * residual + gate * dropout(after(x)) and y = before(h), in one pass, with gradients.

    x [*, C] in float32, float16 or bfloat16, 1 to 512 channels; residual like x; gate [C], or like x; after, before: `Norm`s;
    each may be missing.  Norms' weights and biases and a gate [C]: float32 or x's dtype, all the same.  Returns h without
    `before`, (h, y) with it, and y alone where h is x itself (`before` and nothing else).  Statistics and sums are
    float32, and h on its way to y; each result is rounded once.

    dropout: the share of values that become zero (whatever they were), others are divided by 1 - dropout.  seed: a whole number, two
    (key, offset), or both as an int64 tensor on the GPU, read when the kernel runs: a captured CUDA graph drops other
    values once that tensor holds other numbers.  The same seed drops the same values of a tensor of the same size; the backward pass
    makes the mask again from it (pl_dropout in include/pl_lattice.h defines it).

    Gradients' sums over rows have a fixed order.  A value that is not finite makes its row, and the gradients of the vectors, not
    finite.  In a CUDA graph: forward and backward together, on leaves made inside it."""
    p, seed = _check_share(dropout, seed)
    device, vector_dtype = _check(x, residual, gate, after, before, p, seed)
    on_gpu = isinstance(seed, torch.Tensor)
    key, offset = (0, 0) if on_gpu else seed
    channels = x.shape[-1]
    kind_a, eps_a, wa, ba = (None, 0.0, None, None) if after is None else (after.kind, float(after.eps), after.weight, after.bias)
    kind_b, eps_b, wb, bb = (None, 0.0, None, None) if before is None else (before.kind, float(before.eps), before.weight, before.bias)
    m = _structure(x.numel() // channels, channels, x.dtype, vector_dtype, gate is not None and gate.dim() > 1, float(residual_scale),
                   kind_a, eps_a, kind_b, eps_b, p, key, offset)
    wants_h = before is None or after is not None or residual is not None or gate is not None or p > 0.0
    tensors = (x.contiguous(), _contiguous(residual), _contiguous(gate), _contiguous(wa), _contiguous(ba), _contiguous(wb), _contiguous(bb))
    seed = seed.contiguous() if on_gpu and p else None
    if not _follows(tensors):
        h, y = _forward(device, m, wants_h, before is not None, seed, *tensors)
        return (h, y) if wants_h and y is not None else (y if h is None else h)
    return _ChannelNorm.apply(device, m, after is not None, wants_h, before is not None, seed, *tensors)


def _drop(device, x, residual, share, seed, residual_scale, wants_out, wants_scaled):
    out = torch.empty_like(x) if wants_out else None
    scaled = torch.empty_like(x) if wants_scaled else None
    with _OnDevice(device):
        rc = capi.lib().pl_channel_dropout(_ptr(out), _ptr(scaled), x.data_ptr(), _ptr(residual), x.numel(), _DTYPES[x.dtype],
                                           residual_scale, share, _ptr(seed), _stream_handle(device))
        if rc != capi.PL_OK:
            capi.check(rc, "pl_channel_dropout")
    return out, scaled


class _ChannelDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, share, residual_scale, seed, x, residual):
        ctx.args = device, share, residual_scale
        ctx.save_for_backward(seed)
        return _drop(device, x, residual, share, seed, residual_scale, True, False)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (seed,) = ctx.saved_tensors
        device, share, residual_scale = ctx.args
        return (None, None, None, None) + _drop(device, grad.contiguous(), None, share, seed, residual_scale, *ctx.needs_input_grad[4:])


def channel_dropout(x, p, seed, residual=None, residual_scale=1.0):
    """residual_scale * residual + dropout(x): x of any shape, residual like it, float32, float16 or bfloat16, with gradients for both.
    p, seed: see `channel_norm`, whose dropout of a tensor drops the same values.  No mask is kept: the backward pass makes it again."""
    _check_values(x, "x")
    p, seed = _check_share(p, seed)
    if residual is not None:
        _check_values(residual, "residual", x.dtype)
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
    on_gpu = isinstance(seed, torch.Tensor)
    tensor = seed if on_gpu and p else None
    index = x.get_device()
    if index < 0 or (residual is not None and residual.get_device() != index) or (tensor is not None and tensor.get_device() != index):
        _check_device((("x", x), ("residual", residual), ("seed", tensor)))
    share = _dropout_of(p, 0, 0) if on_gpu else _dropout_of(p, *seed)
    x, residual, tensor = x.contiguous(), _contiguous(residual), _contiguous(tensor)
    if not _follows((x, residual)):
        return _drop(x.device, x, residual, share, tensor, float(residual_scale), True, False)[0]
    return _ChannelDropout.apply(x.device, share, float(residual_scale), tensor, x, residual)
