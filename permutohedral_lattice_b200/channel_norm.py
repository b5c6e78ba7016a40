"""What a network's blocks of features take beside their products: norms over the channels, and dropout.

    u = after(x)                              the norm after the block that gave x
    h = residual_scale * residual + gate * dropout(u)
    y = before(h)                             the norm before the next block

over channels-last tensors [*, C] of points, in one pass, and their gradients in one more, from what came in: neither the
normed values nor the dropout's mask are kept (`channel_norm`).  `channel_dropout` is dropout by itself, with the residual.
The reference ships no such operators; the networks that give CRF-as-RNN (its README.md:15-16) its unaries do.
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


class _Shape(NamedTuple):
    """What a call's C structure holds besides pointers."""
    rows: int
    channels: int
    dtype: torch.dtype
    vector_dtype: torch.dtype
    gate_of_values: bool
    residual_scale: float
    after: Optional[tuple]       # kind, eps
    before: Optional[tuple]
    p: float
    seed: Optional[tuple]        # key, offset, where they are numbers


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
    if norm is None:
        return
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


def _check(x, residual, gate, after, before, dropout, seed):
    """Returns the device, p, the seed, and the type of the channels' vectors."""
    _check_values(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [*, channels]")
    channels = x.shape[-1]
    if not 1 <= channels <= MOST_NORM_CHANNELS:
        raise ValueError("x: 1 to %d channels are supported" % MOST_NORM_CHANNELS)
    _check_norm(after, "after", channels)
    _check_norm(before, "before", channels)
    p, seed = _check_share(dropout, seed)
    if after is None and before is None and residual is None and gate is None and not p:
        raise ValueError("nothing to do: a norm, a residual, a gate or dropout is needed")
    vectors = [(name, t) for name, norm in (("after", after), ("before", before)) if norm is not None
               for name, t in ((name + ".weight", norm.weight), (name + ".bias", norm.bias)) if t is not None]
    if residual is not None:
        _check_values(residual, "residual", x.dtype)
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
    if gate is not None:
        _check_values(gate, "gate")
        if gate.shape == x.shape and gate.dim() > 1:
            _check_values(gate, "gate", x.dtype)
        elif tuple(gate.shape) == (channels,):
            vectors.append(("gate", gate))
        else:
            raise ValueError("gate must be [channels], or of x's shape")
    vector_dtype = vectors[0][1].dtype if vectors else x.dtype
    for name, t in vectors:
        if t.dtype not in (torch.float32, x.dtype):
            raise TypeError("%s must be float32 or of x's dtype" % name)
        if t.dtype != vector_dtype:
            raise TypeError("%s must have dtype %s like the other vectors of the channels" % (name, vector_dtype))
    on = [("x", x), ("residual", residual), ("gate", gate)] + vectors
    if p and isinstance(seed, torch.Tensor):
        on.append(("seed", seed))
    return _check_device(on), p, seed, vector_dtype


def _dropout_of(p, seed):
    if isinstance(seed, torch.Tensor):
        return capi.PlDropout(p, 0, 0, seed.data_ptr() if p else 0)
    return capi.PlDropout(p, *(seed or (0, 0)), 0)


def _structure(s, weights, seed):
    """weights: after's weight and bias, before's weight and bias."""
    def norm(of, weight, bias):
        return capi.PlNorm(_KINDS[of[0]], of[1], _ptr(weight), _ptr(bias)) if of else capi.PlNorm(capi.PL_NORM_NONE, 0.0, 0, 0)

    return ctypes.byref(capi.PlChannelNorm(
        s.rows, s.channels, _DTYPES[s.dtype], _DTYPES[s.vector_dtype], int(s.gate_of_values), s.residual_scale,
        norm(s.after, *weights[:2]), norm(s.before, *weights[2:]), _dropout_of(s.p, s.seed if seed is None else seed)))


def _forward(device, s, x, residual, gate, weights, seed, wants_h):
    h = torch.empty_like(x) if wants_h else None
    y = torch.empty_like(x) if s.before else None
    with _OnDevice(device):
        capi.check(capi.lib().pl_channel_norm(_structure(s, weights, seed), _ptr(h), _ptr(y), x.data_ptr(), _ptr(residual), _ptr(gate),
                                              _stream_handle(device)), "pl_channel_norm")
    return h, y


@functools.lru_cache(maxsize=256)
def _workspace_bytes(s):
    nbytes = ctypes.c_size_t(0)
    capi.check(capi.lib().pl_channel_norm_workspace_bytes(_structure(s, (None,) * 4, None), ctypes.byref(nbytes)),
               "pl_channel_norm_workspace_bytes")
    return nbytes.value


# What _ChannelNorm takes gradients of, in its order.
_NAMES = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")


class _ChannelNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, s, wants_h, seed, x, residual, gate, *weights):
        h, y = _forward(device, s, x, residual, gate, weights, seed, wants_h)
        ctx.set_materialize_grads(False)
        ctx.device, ctx.s, ctx.outputs = device, s, (wants_h, y is not None)
        needs = dict(zip(_NAMES, ctx.needs_input_grad[4:]))
        keep_x = s.after is not None or s.before is not None or needs["gate"]
        ctx.save_for_backward(x if keep_x else None, residual if s.before else None, gate, seed, *weights)
        return (h, y) if wants_h and y is not None else (y if h is None else h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, residual, gate, seed, *weights = ctx.saved_tensors
        s, device = ctx.s, ctx.device
        needs = [name for name, wanted in zip(_NAMES, ctx.needs_input_grad[4:]) if wanted]
        with_h, with_y = ctx.outputs
        dh, dy = grads if with_h and with_y else (grads[0], None) if with_h else (None, grads[0])
        if dh is None and dy is None:
            return (None,) * (4 + len(_NAMES))
        if with_y and dy is None:       # nobody used y
            dy = torch.zeros_like(dh)
        dh, dy = _contiguous(dh), _contiguous(dy)
        like = dh if dy is None else dy
        shapes = {"x": like, "residual": like, "gate": gate, "after_weight": weights[0], "after_bias": weights[1],
                  "before_weight": weights[2], "before_bias": weights[3]}
        made = {name: torch.empty(shapes[name].shape, dtype=shapes[name].dtype, device=device) for name in needs}
        with _OnDevice(device):
            workspace = torch.empty(_workspace_bytes(s._replace(rows=0, p=0.0, seed=(0, 0))), dtype=torch.uint8, device=device)
            d = capi.PlNormGradients(**{name: t.data_ptr() for name, t in made.items()})
            capi.check(capi.lib().pl_channel_norm_backward(
                _structure(s, weights, seed), _ptr(dh), _ptr(dy), _ptr(x), _ptr(residual), _ptr(gate), d, workspace.data_ptr(),
                workspace.numel(), _stream_handle(device)), "pl_channel_norm_backward")
        return (None,) * 4 + tuple(made.get(name) for name in _NAMES)


def _follows(tensors):
    return _watched_by_torch() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


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
    device, p, seed, vector_dtype = _check(x, residual, gate, after, before, dropout, seed)
    on_gpu = isinstance(seed, torch.Tensor)
    channels = x.shape[-1]
    of_values = gate is not None and gate.dim() > 1
    shape = _Shape(x.numel() // channels, channels, x.dtype, vector_dtype, of_values, float(residual_scale),
                   None if after is None else (after.kind, float(after.eps)), None if before is None else (before.kind, float(before.eps)),
                   p, None if on_gpu else seed)
    wants_h = before is None or after is not None or residual is not None or gate is not None or p > 0.0
    weights = tuple(t for norm in (after, before) for t in ((None, None) if norm is None else (norm.weight, norm.bias)))
    tensors = tuple(_contiguous(t) for t in (x, residual, gate) + weights)
    seed = seed.contiguous() if on_gpu and p else None
    if not _follows(tensors):
        h, y = _forward(device, shape, *tensors[:3], tensors[3:], seed, wants_h)
        return (h, y) if wants_h and y is not None else (y if h is None else h)
    return _ChannelNorm.apply(device, shape, wants_h, seed, *tensors)


def _drop(device, x, residual, p, seed, residual_scale, wants_scaled):
    out = torch.empty_like(x)
    scaled = torch.empty_like(x) if wants_scaled else None
    with _OnDevice(device):
        capi.check(capi.lib().pl_channel_dropout(out.data_ptr(), _ptr(scaled), x.data_ptr(), _ptr(residual), x.numel(), _DTYPES[x.dtype],
                                                 residual_scale, ctypes.byref(_dropout_of(p, seed)), _stream_handle(device)),
                   "pl_channel_dropout")
    return out, scaled


class _ChannelDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, p, numbers, residual_scale, seed, x, residual):
        ctx.args = device, p, numbers, residual_scale
        ctx.save_for_backward(seed)
        return _drop(device, x, residual, p, numbers if seed is None else seed, residual_scale, False)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (seed,) = ctx.saved_tensors
        device, p, numbers, residual_scale = ctx.args
        dx, dresidual = _drop(device, grad.contiguous(), None, p, numbers if seed is None else seed, residual_scale, ctx.needs_input_grad[6])
        return None, None, None, None, None, dx if ctx.needs_input_grad[5] else None, dresidual


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
    device = _check_device((("x", x), ("residual", residual), ("seed", seed if on_gpu and p else None)))
    x, residual = x.contiguous(), _contiguous(residual)
    tensor = seed.contiguous() if on_gpu and p else None
    numbers = (0, 0) if on_gpu else seed
    if not _follows((x, residual)):
        return _drop(device, x, residual, p, numbers if tensor is None else tensor, float(residual_scale), False)[0]
    return _ChannelDropout.apply(device, p, numbers, float(residual_scale), tensor, x, residual)
