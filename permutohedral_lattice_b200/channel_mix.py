"""Training beside the lattice filter: products of channels with an epilogue, and activations kept in 8 bits.

    out = act(x @ weight [+ x2 @ weight2] [+ bias] [+ residual_scale * residual])

over channels-last tensors [*, K] (a point's channels are its row), act the identity, "relu" or "softmax" over the output's
channels.  In a dense CRF x and x2 are the two filtered label distributions, the weights the kernels' weights times the
labels' compatibility, the residual the unaries (`DenseCRF` calls it for learned parameters); beside the filter it is the
1x1 map between a network's features and the lattice's.  The reference ships no such operator: README.md:15-16 names
CRF-as-RNN, which trains these parameters, as its user.

`checkpoint="8bit"` keeps what the backward pass needs in 8 bits (`PackedActivations`): blocks of 32 consecutive values
that share a power of two, a quarter of float32's memory, half a step (1/510 to 1/255 of the block's largest value, with
negative values in the block 1/254 to 1/127) off at most.
"""
import ctypes
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import capi
from .lattice_filter import _OnDevice, _stream_handle, _watched_by_torch

MOST_CHANNELS = 128   # of an input, and of the output
BLOCK = 32            # values that share an exponent
_DTYPES = {torch.float32: capi.PL_F32, torch.float16: capi.PL_F16, torch.bfloat16: capi.PL_BF16}
_ACTIVATIONS = {None: capi.PL_ACT_NONE, "relu": capi.PL_ACT_RELU, "softmax": capi.PL_ACT_SOFTMAX}
_NAMES = ("x", "weight", "bias", "residual", "x2", "weight2")


class PackedActivations(NamedTuple):
    """A tensor in 8 bits: `codes` uint8, one a value, and `scales` int16, the header of every 32 consecutive values:
    (e + 127) | signed << 8 for codes in steps of 2^e (in two's complement if signed), 255 for a block of NaN."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype          # of the tensor that was packed


class MixSaved(NamedTuple):
    """What the backward pass of a `channel_mix` reads: tensors, or the same in 8 bits.  out: None without activation."""
    x: Union[torch.Tensor, PackedActivations, None]
    x2: Union[torch.Tensor, PackedActivations, None]
    out: Union[torch.Tensor, PackedActivations, None]


class MixGradients(NamedTuple):
    x: Optional[torch.Tensor] = None
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    residual: Optional[torch.Tensor] = None
    x2: Optional[torch.Tensor] = None
    weight2: Optional[torch.Tensor] = None


def _check_values(t, name, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if dtype is None:
        if t.dtype not in _DTYPES:
            raise TypeError("%s must be float32, float16 or bfloat16" % name)
    elif t.dtype is not dtype:
        raise TypeError("%s must have dtype %s like the other operand" % (name, dtype))


def _check_device(tensors):
    """All on one GPU, which is returned."""
    index = None
    for name, t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("%s must be a CUDA tensor (there is no CPU path in this package)" % name)
        at = t.get_device()
        if index is not None and at != index:
            raise ValueError("%s is on device %d, the other operands are on %d" % (name, at, index))
        index, device_of = at, t
    return device_of.device


def _check_weight(w, name, x_dtype, dtype, k, n):
    _check_values(w, name, dtype)
    if w.dtype is not torch.float32 and w.dtype is not x_dtype:
        raise TypeError("%s must be float32 or of the input's dtype" % name)
    shape = w.shape
    if len(shape) != 2 or (k is not None and shape[0] != k) or (n is not None and shape[1] != n):
        raise ValueError("%s must be [channels of its input, channels of the output]" % name)
    if not 1 <= shape[0] <= MOST_CHANNELS or not 1 <= shape[1] <= MOST_CHANNELS:
        raise ValueError("%s: 1 to %d channels are supported" % (name, MOST_CHANNELS))


def _check_activation(activation):
    if activation not in _ACTIVATIONS:
        raise ValueError('activation must be None, "relu" or "softmax"')


def _check_mix(x, weight, bias, residual, x2, weight2, activation, checkpoint):
    _check_activation(activation)
    if checkpoint not in (None, "8bit"):
        raise ValueError('checkpoint must be None or "8bit"')
    _check_values(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [*, channels]")
    _check_weight(weight, "weight", x.dtype, None, x.shape[-1], None)
    n = weight.shape[1]
    if (x2 is None) != (weight2 is None):
        raise ValueError("x2 and weight2 come together")
    if x2 is not None:
        _check_values(x2, "x2", x.dtype)
        if x2.shape[:-1] != x.shape[:-1] or x2.dim() != x.dim():
            raise ValueError("x2 must match x in all dimensions but the channels")
        _check_weight(weight2, "weight2", x.dtype, weight.dtype, x2.shape[-1], n)
    if bias is not None:
        _check_values(bias, "bias", weight.dtype)
        if tuple(bias.shape) != (n,):
            raise ValueError("bias must be [channels of the output]")
    if residual is not None:
        _check_values(residual, "residual", x.dtype)
        if tuple(residual.shape) != tuple(x.shape[:-1]) + (n,):
            raise ValueError("residual must have the output's shape")
    return _check_device((("x", x), ("weight", weight), ("x2", x2), ("weight2", weight2), ("bias", bias),
                          ("residual", residual)))


def _ptr(t):
    return 0 if t is None else t.data_ptr()


_NOT_PACKED = capi.PlPacked(0, 0)


def _packed(p):
    return _NOT_PACKED if p is None else capi.PlPacked(p.codes.data_ptr(), p.scales.data_ptr())


def _kept(a):
    if isinstance(a, PackedActivations):
        return capi.PlKept(0, _packed(a))
    return capi.PlKept(_ptr(a), _NOT_PACKED)


def _contiguous(t):
    return None if t is None else t.contiguous()


def _empty_packed(shape, dtype, device):
    count = 1
    for s in shape:
        count *= int(s)
    return PackedActivations(torch.empty(count, dtype=torch.uint8, device=device),
                             torch.empty(-(-count // BLOCK), dtype=torch.int16, device=device), tuple(shape), dtype)


@functools.lru_cache(maxsize=1024)
def _shape_of(rows, k, k2, n, activation, dtype, weight_dtype, residual_scale):
    """The C structure of a call, which the library only reads (building it takes a tenth of a small call's time on the host)."""
    return ctypes.byref(capi.PlMix(rows, k, k2, n, _ACTIVATIONS[activation], _DTYPES[dtype], _DTYPES[weight_dtype], residual_scale))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*shape):
    nbytes = ctypes.c_size_t(0)
    capi.check(capi.lib().pl_channel_mix_workspace_bytes(_shape_of(*shape), ctypes.byref(nbytes)), "pl_channel_mix_workspace_bytes")
    return max(1, nbytes.value)


def pack_activations(x):
    """x (float32, float16 or bfloat16) in 8 bits: see PackedActivations.  Not followed by autograd."""
    _check_values(x, "x")
    device = _check_device((("x", x),))
    x = x.detach().contiguous()
    p = _empty_packed(x.shape, x.dtype, device)
    with _OnDevice(device):
        capi.check(capi.lib().pl_pack_activations(_packed(p), x.data_ptr(), x.numel(), _DTYPES[x.dtype], 0,
                                                  _stream_handle(device)), "pl_pack_activations")
    return p


def _check_packed(p, name):
    if not isinstance(p, PackedActivations):
        raise TypeError("%s must be PackedActivations" % name)
    count = 1
    for s in p.shape:
        count *= int(s)
    if p.codes.dtype != torch.uint8 or p.scales.dtype != torch.int16:
        raise TypeError("%s must have codes in uint8 and scales in int16" % name)
    if p.codes.numel() != count or p.scales.numel() != -(-count // BLOCK):
        raise ValueError("%s must have a code for each of its %d values and a scale for every %d" % (name, count, BLOCK))
    if not p.codes.is_contiguous() or not p.scales.is_contiguous():
        raise ValueError("%s must have contiguous codes and scales" % name)
    if p.dtype not in _DTYPES:
        raise TypeError("%s must be of float32, float16 or bfloat16 values" % name)
    return count


def unpack_activations(packed, dtype=None):
    """The values of a PackedActivations, in `dtype` (default: that of the tensor that was packed).  float32 and bfloat16
    hold each exactly; float16 rounds, and takes those beyond 65504 for infinities."""
    count = _check_packed(packed, "packed")
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    device = _check_device((("codes", packed.codes), ("scales", packed.scales)))
    x = torch.empty(packed.shape, dtype=dtype, device=device)
    with _OnDevice(device):
        capi.check(capi.lib().pl_unpack_activations(x.data_ptr(), _packed(packed), count, _DTYPES[dtype],
                                                    _stream_handle(device)), "pl_unpack_activations")
    return x


def _forward(device, x, weight, bias, residual, x2, weight2, activation, residual_scale, keep):
    """The call itself on checked arguments; keep: which of "x", "x2" and "out" to put into 8 bits too.
    Returns out and {name: PackedActivations}."""
    x, weight = x.contiguous(), weight.contiguous()
    bias, residual, x2, weight2 = _contiguous(bias), _contiguous(residual), _contiguous(x2), _contiguous(weight2)
    k, k2, n = x.shape[-1], 0 if x2 is None else x2.shape[-1], weight.shape[1]
    out = x.new_empty(x.shape[:-1] + (n,)) if residual is None else torch.empty_like(residual)
    packs = {}
    if keep:
        like = {"x": x, "x2": x2, "out": out}
        packs = {name: _empty_packed(like[name].shape, x.dtype, device) for name in keep if like[name] is not None}
    m = _shape_of(out.numel() // n, k, k2, n, activation, x.dtype, weight.dtype, residual_scale)
    with _OnDevice(device):
        rc = capi.lib().pl_channel_mix(
            m, out.data_ptr(), x.data_ptr(), _ptr(x2), weight.data_ptr(), _ptr(weight2), _ptr(bias), _ptr(residual),
            _packed(packs.get("x")), _packed(packs.get("x2")), _packed(packs.get("out")), _stream_handle(device))
        if rc != capi.PL_OK:
            capi.check(rc, "pl_channel_mix")
    return out, packs


def channel_mix_raw(x, weight, bias=None, residual=None, x2=None, weight2=None, activation=None, residual_scale=1.0,
                    checkpoint=None):
    """channel_mix without autograd.  Returns (out, MixSaved): what channel_mix_backward takes, tensors or, with
    checkpoint="8bit", PackedActivations."""
    device = _check_mix(x, weight, bias, residual, x2, weight2, activation, checkpoint)
    x, weight, bias, residual, x2, weight2 = (None if t is None else t.detach()
                                              for t in (x, weight, bias, residual, x2, weight2))
    names = ("x", "x2") + (("out",) if activation else ())
    out, packs = _forward(device, x, weight, bias, residual, x2, weight2, activation, float(residual_scale),
                          names if checkpoint else ())
    kept = packs if checkpoint else {"x": x, "x2": x2, "out": out if activation else None}
    return out, MixSaved(kept.get("x"), kept.get("x2"), kept.get("out"))


def _check_saved(a, name, rows_shape, channels, dtype):
    if isinstance(a, PackedActivations):
        _check_packed(a, name)
        shape, kind = tuple(a.shape), a.dtype
    else:
        _check_values(a, name)
        shape, kind = tuple(a.shape), a.dtype
    if kind != dtype:
        raise TypeError("%s must have dtype %s like grad_out" % (name, dtype))
    if shape != tuple(rows_shape) + (channels,):
        raise ValueError("%s must be %s" % (name, tuple(rows_shape) + (channels,)))


def _saved_tensors(name, a):
    return ((name + ".codes", a.codes), (name + ".scales", a.scales)) if isinstance(a, PackedActivations) else ((name, a),)


def channel_mix_backward(grad_out, saved, weight, weight2=None, activation=None, residual_scale=1.0,
                         needs=("x", "weight")):
    """The gradients of channel_mix named in `needs` ("x", "weight", "bias", "residual", "x2", "weight2"), from that of
    its output and what its forward pass kept: saved.out with an activation, saved.x for "weight", saved.x2 for "weight2".
    Sums over rows have a fixed order: the same inputs give the same bits."""
    _check_activation(activation)
    needs = tuple(needs)
    for name in needs:
        if name not in _NAMES:
            raise ValueError("needs: unknown gradient %r" % (name,))
    if not isinstance(saved, MixSaved):
        raise TypeError("saved must be MixSaved")
    _check_values(grad_out, "grad_out")
    if grad_out.dim() < 1:
        raise ValueError("grad_out must be [*, channels]")
    dtype, head, n = grad_out.dtype, grad_out.shape[:-1], grad_out.shape[-1]
    _check_weight(weight, "weight", dtype, None, None, n)
    k, k2 = weight.shape[0], 0
    if weight2 is not None:
        _check_weight(weight2, "weight2", dtype, weight.dtype, None, n)
        k2 = weight2.shape[0]
    elif "x2" in needs or "weight2" in needs:
        raise ValueError("the gradients of x2 and weight2 take weight2")
    out = saved.out if activation else None
    x = saved.x if "weight" in needs else None
    x2 = saved.x2 if "weight2" in needs else None
    if activation:
        _check_saved(out, "saved.out", head, n, dtype)
    if "weight" in needs:
        _check_saved(x, "saved.x", head, k, dtype)
    if "weight2" in needs:
        _check_saved(x2, "saved.x2", head, k2, dtype)
    device = _check_device((("grad_out", grad_out), ("weight", weight), ("weight2", weight2)) + tuple(
        t for name, a in (("saved.out", out), ("saved.x", x), ("saved.x2", x2)) for t in _saved_tensors(name, a)))
    return _backward(device, grad_out, out, x, x2, weight, weight2, activation, float(residual_scale), needs)


def _backward(device, grad_out, out, x, x2, weight, weight2, activation, residual_scale, needs):
    grad_out, weight, weight2 = grad_out.contiguous(), weight.contiguous(), _contiguous(weight2)
    out, x, x2 = (a if a is None or isinstance(a, PackedActivations) else a.contiguous() for a in (out, x, x2))
    head, n = tuple(grad_out.shape[:-1]), grad_out.shape[-1]
    k, k2 = weight.shape[0], 0 if weight2 is None else weight2.shape[0]
    shapes = {"x": (head + (k,), grad_out.dtype), "x2": (head + (k2,), grad_out.dtype),
              "residual": (head + (n,), grad_out.dtype), "weight": ((k, n), weight.dtype),
              "weight2": ((k2, n), weight.dtype), "bias": ((n,), weight.dtype)}
    made = {name: torch.empty(shapes[name][0], dtype=shapes[name][1], device=device) for name in needs}
    shape = (grad_out.numel() // n, k, k2, n, activation, grad_out.dtype, weight.dtype, residual_scale)
    with _OnDevice(device):
        workspace = torch.empty(_workspace_bytes(*shape), dtype=torch.uint8, device=device)
        d = capi.PlMixGradients(**{name: t.data_ptr() for name, t in made.items()})
        rc = capi.lib().pl_channel_mix_backward(
            _shape_of(*shape), grad_out.data_ptr(), _kept(out), _kept(x), _kept(x2), weight.data_ptr(), _ptr(weight2), d,
            workspace.data_ptr(), workspace.numel(), _stream_handle(device))
        if rc != capi.PL_OK:
            capi.check(rc, "pl_channel_mix_backward")
    return MixGradients(**made)


class _ChannelMixFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, device, x, weight, bias, residual, x2, weight2, activation, residual_scale, checkpoint):
        needed = dict(zip(_NAMES, ctx.needs_input_grad[1:7]))
        keep = [name for name, wanted in (("x", needed["weight"]), ("x2", needed["weight2"]), ("out", activation))
                if wanted and any(needed.values())]
        out, packs = _forward(device, x, weight, bias, residual, x2, weight2, activation, residual_scale,
                              keep if checkpoint else ())
        kept = packs if checkpoint else {"x": x, "x2": x2, "out": out}
        ctx.meta, tensors = {}, [weight, weight2]
        for name in keep:
            if checkpoint:
                ctx.meta[name] = (len(tensors), kept[name].shape, kept[name].dtype)
                tensors += [kept[name].codes, kept[name].scales]
            else:
                ctx.meta[name] = (len(tensors), None, None)
                tensors.append(kept[name])
        ctx.save_for_backward(*tensors)
        ctx.args = (device, activation, residual_scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        tensors = ctx.saved_tensors
        needs = [name for name, wanted in zip(_NAMES, ctx.needs_input_grad[1:7]) if wanted]

        def saved(name):
            if name not in ctx.meta:
                return None
            at, shape, dtype = ctx.meta[name]
            return tensors[at] if shape is None else PackedActivations(tensors[at], tensors[at + 1], shape, dtype)

        device, activation, residual_scale = ctx.args
        g = _backward(device, grad, saved("out"), saved("x"), saved("x2"), tensors[0], tensors[1], activation,
                      residual_scale, needs)
        return (None, g.x, g.weight, g.bias, g.residual, g.x2, g.weight2, None, None, None)


def channel_mix(x, weight, bias=None, residual=None, x2=None, weight2=None, activation=None, residual_scale=1.0,
                checkpoint=None):
    """act(x @ weight [+ x2 @ weight2] [+ bias] [+ residual_scale * residual]), with gradients for all six tensors.

    x [*, K], x2 [*, K2], residual [*, N] and the output [*, N] in float32, float16 or bfloat16; weight [K, N],
    weight2 [K2, N] and bias [N] in float32 or the input's dtype; up to 128 channels each.  activation: None, "relu" or
    "softmax" over the channels; a row whose channels are all forbidden by an infinite residual gives zeros and has no
    gradient.  checkpoint="8bit" keeps the activations that the backward pass needs in 8 bits: their gradients are those
    at the rounded activations, and x, x2 and the output may be freed in between.  x, x2 and the weights have to be finite
    (of a row that is not, each value comes out NaN or as the formula gives it; other rows are as they would be).  In a CUDA
    graph: one ordinary call before the capture, which sets the kernel up; forward and backward together, on leaves made inside
    it."""
    device = _check_mix(x, weight, bias, residual, x2, weight2, activation, checkpoint)
    args = (x, weight, bias, residual, x2, weight2)
    if not _watched_by_torch() and not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)):
        return _forward(device, *args, activation, float(residual_scale), ())[0]
    return _ChannelMixFunction.apply(device, *args, activation, float(residual_scale), checkpoint)
