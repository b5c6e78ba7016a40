"""Training operators around the lattice filter, as timed cases: what a dense CRF's mean-field step and a learned map
of features need besides the filter.

The product of channels with bias, residual and activation (`channel_mix`), forward and with its gradients; activations
kept in 8 bits (`pack_activations`, `unpack_activations`), written by the forward pass and read by the backward pass.
Where `own` is false, `run` computes them with elementary torch operations, else by the package's entry points.

Inputs are synthetic, made on the GPU from a seed: filtered label distributions, negative log-likelihoods, patch
features in [0, 1].  In "masked" cases a part of the labels is forbidden (an infinite unary), and some rows are padding
(all of them are): such a row comes out as zeros.
"""
import math

import torch

own = False

BLOCK = 32                       # values that share an exponent
MOST_ROWS = 16 * 512 * 512       # the largest listed call: 16 images of 512 x 512 with 21 labels
MOST_VALUES = MOST_ROWS * 21
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _case(what, shape, k, k2=0, n=0, activation="", bias=False, residual=False, masked=False, dtype="float32",
          name=None):
    """what: "mix" (forward), "train" (forward and gradients), "train_8bit" (the same with its input kept in 8 bits),
    "mix_8bit" (forward that also writes its activations in 8 bits), "gradients_8bit" (the backward pass from them),
    "pack" or "unpack".  shape: batch and spatial sizes.  k, k2: channels of the one or two inputs.  n: of the output."""
    case = {"what": what, "shape": shape, "k": k, "k2": k2, "n": n, "activation": activation, "bias": bias,
            "residual": residual, "masked": masked, "dtype": dtype}
    if name is not None:
        case["name"] = name
    return case


def _update(what, shape, labels, **kw):
    """The step after the two filters of a CRF: both filtered distributions, unaries, softmax."""
    return _case(what, shape, labels, labels, labels, "softmax", residual=True, **kw)


def listed():
    return [
        # one small image, 21 labels: latency of a call
        _update("mix", "1x33x45", 21, name="update_thumbnail"),
        # a photograph of ragged size whose unaries forbid labels, with a learned prior of the labels
        _update("mix", "1x375x500", 21, bias=True, masked=True, name="update_photo"),
        # a training batch of the benchmark's size: forward, and the gradients of inputs, weights, prior and unaries
        _update("train", "16x512x512", 21, bias=True, name="update_train_batch"),
        # volumes with two classes, in training
        _update("train", "2x111x128x120", 2, name="update_train_volumes"),
        # as many labels as an update takes, ragged image, in training
        _update("train", "1x321x481", 128, bias=True, name="update_train_many_labels"),
        # 64 labels in 16 bits
        _update("mix", "4x512x512", 64, dtype="bfloat16", masked=True, name="update_half"),
        # the forward pass of a training step that keeps its activations in 8 bits, and the backward pass that reads them
        _update("mix_8bit", "8x512x512", 21, name="update_keeps_8bit"),
        _update("gradients_8bit", "16x512x512", 21, bias=True, name="gradients_from_8bit"),
        # patch features of 5 x 5 colours mapped to a lattice's 16 dimensions, as they are and in training
        _case("mix", "2x1024x1024", 75, 0, 16, bias=True, name="features"),
        _case("train_8bit", "2x1024x1024", 75, 0, 16, name="features_train_8bit"),
        # label distributions of a batch to 8 bits, and of a small image back
        _case("pack", "16x512x512", 21, name="pack_batch"),
        _case("unpack", "1x33x45", 21, dtype="bfloat16", name="unpack_thumbnail"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["mix", "train", "train_8bit", "mix_8bit", "gradients_8bit", "pack", "unpack"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    if what in ("pack", "unpack"):
        k, k2, n, activation = _log_uniform(rng, 1, 128), 0, 0, ""
    elif what == "train_8bit" or rng.random() < 0.3:
        k, k2, n = _log_uniform(rng, 1, 128), 0, _log_uniform(rng, 1, 128)
        activation = "" if what == "train_8bit" else rng.choice(["", "softmax", "relu"] if what == "mix" else ["", "softmax"])
    else:
        k = k2 = n = _log_uniform(rng, 2, 128)
        activation = "softmax"
    residual = activation == "softmax" and (k2 > 0 or rng.random() < 0.5)
    # a pass costs no more than the largest listed one: of its values, or of its products where there are many channels
    most = min(MOST_ROWS, MOST_VALUES // max(k, n), MOST_ROWS * 21 * 42 // max(1, n * (k + k2)))
    return _case(what, "1x%d" % _log_uniform(rng, 1, most), k, k2, n, activation, n > 0 and rng.random() < 0.5, residual,
                 residual and rng.random() < 0.3, dtype)


def _shape(case):
    return tuple(int(s) for s in case["shape"].split("x"))


def work(case):
    rows = math.prod(_shape(case))
    size = 4 if case["dtype"] == "float32" else 2
    k, n, what = case["k"] + case["k2"], case["n"], case["what"]
    kept = 1 + 2 / BLOCK                                     # bytes of a value in 8 bits
    weights = k * n * size
    residual = n if case["residual"] else 0
    y = n if case["activation"] else 0                       # the gradient of a plain product does not read its output
    forward = rows * size * (k + n + residual) + weights
    products = 2 * rows * n * k
    if what == "mix":
        return {"bytes": forward, "flops": products}
    if what == "mix_8bit":
        return {"bytes": forward + rows * kept * (k + y), "flops": products}
    gradients = rows * size * (n + k + residual) + 2 * weights
    if what == "train":
        # the step as a whole: x, residual and g read once, out and the gradients written once
        return {"bytes": rows * size * (k + residual + n) + rows * size * (n + k + residual) + 2 * weights,
                "flops": 3 * products}
    if what == "train_8bit":
        return {"bytes": forward + gradients, "flops": 3 * products}
    if what == "gradients_8bit":
        return {"bytes": gradients + rows * kept * (k + y), "flops": 2 * products}
    return {"bytes": rows * k * (size + kept), "flops": 0}


def _made_weights(g, k, n, dtype, crf):
    if crf and k == n:                                       # minus a kernel's weight times a learned compatibility
        w = 1.0 - torch.eye(n, device="cuda") + 0.1 * torch.randn((k, n), generator=g, device="cuda")
        return (-1.5 * w).to(dtype)
    return (torch.randn((k, n), generator=g, device="cuda") / math.sqrt(k)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape, dtype, what = _shape(case), DTYPES[case["dtype"]], case["what"]
    k, k2, n = case["k"], case["k2"], case["n"]

    def randn(*size):
        return torch.randn(size, generator=g, device="cuda")

    def distributions(channels):
        return torch.softmax(2.0 * randn(*shape, channels), -1)

    s = {"case": dict(case)}
    if what in ("pack", "unpack"):
        x = distributions(k) if case["dtype"] == "float32" else randn(*shape, k)
        if what == "pack":
            s["x"] = x.to(dtype)
        else:
            s["codes"], s["scales"] = _encode(x.to(dtype))
        return s
    crf = case["activation"] == "softmax"
    s["x"] = (distributions(k) if crf else torch.rand((*shape, k), generator=g, device="cuda")).to(dtype)
    s["x2"] = distributions(k2).to(dtype) if k2 else None
    s["weight"] = _made_weights(g, k, n, dtype, crf)
    s["weight2"] = _made_weights(g, k2, n, dtype, crf) if k2 else None
    s["bias"] = (0.5 * randn(n)).to(dtype) if case["bias"] else None
    s["residual"] = None
    if case["residual"]:
        u = -torch.log(distributions(n) + 1e-6)
        if case["masked"]:
            u = torch.where(torch.rand((*shape, n), generator=g, device="cuda") < 0.2, math.inf, u)
            padding = torch.rand((*shape, 1), generator=g, device="cuda") < 0.02
            u = torch.where(padding, math.inf, u)
        s["residual"] = u.to(dtype)
    if what in ("train", "train_8bit", "gradients_8bit"):
        s["grad"] = randn(*shape, n).to(dtype)
    if what == "gradients_8bit":
        s["out"] = (_encode(distributions(n).to(dtype)) if case["activation"] else None)
        s["x"] = _encode(s["x"])
        s["x2"] = _encode(s["x2"]) if k2 else None
        s["residual"] = None
    elif what != "mix" and what != "mix_8bit":
        for name in ("x", "x2", "weight", "weight2", "bias", "residual"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _power(e):
    """2^e for whole -126 <= e <= 127, to the bit: the GPU's pow is not."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x):
    """codes [values] uint8 and headers [blocks] int16 of a tensor: blocks of 32 consecutive values that share the exponent e,
    the least one >= -126 at which the largest magnitude is at most 255 (no value negative) or 127 steps of 2^e."""
    flat = x.float().reshape(-1)
    count = flat.numel()
    v = torch.nn.functional.pad(flat, (0, -count % BLOCK)).view(-1, BLOCK)
    signed = (v < 0).any(1)
    most = v.abs().amax(1)
    bad = ~torch.isfinite(v).all(1)
    steps = torch.where(signed, 127.0, 255.0)
    mantissa, exponent = torch.frexp(torch.where(bad, torch.ones_like(most), most))
    e = exponent - torch.where(signed, 7, 8) + (mantissa > steps / (steps + 1)).to(exponent.dtype)
    e = torch.where(most == 0, torch.full_like(e, -126), e).clamp(min=-126)
    codes = torch.round((v * _power(-e)[:, None]).nan_to_num(0.0, 0.0, 0.0)).to(torch.int16)
    codes = torch.where(bad[:, None], torch.zeros_like(codes), codes)
    header = torch.where(bad, torch.full_like(e, 255), (e + 127) + 256 * signed.to(e.dtype))
    return codes.reshape(-1)[:count].to(torch.uint8), header.to(torch.int16)


def _decode(codes, header, shape):
    """The values, float32."""
    count = codes.numel()
    v = torch.nn.functional.pad(codes, (0, -count % BLOCK)).view(-1, BLOCK).to(torch.int32)
    header = header.to(torch.int32)[:, None]
    v = torch.where(((header & 256) != 0) & (v > 127), v - 256, v)
    x = v.float() * _power(torch.clamp((header & 255) - 127, max=127))
    x = torch.where((header & 255) == 255, torch.full_like(x, math.nan), x)
    return x.reshape(-1)[:count].view(shape)


def _plain_forward(s):
    """The output in 32 bits, not yet rounded."""
    z = s["x"].detach().float() @ s["weight"].detach().float()
    if s["x2"] is not None:
        z = z + s["x2"].detach().float() @ s["weight2"].detach().float()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    if s["residual"] is not None:
        z = z - s["residual"].detach().float()
    if s["case"]["activation"] == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if s["case"]["activation"] == "softmax":
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
        return e / torch.where(top == -math.inf, torch.ones_like(top), e.sum(-1, keepdim=True))
    return z


def _plain_gradients(s, y, x, x2):
    """From the upstream gradient and what the forward pass kept (32 bits)."""
    g, dtype = s["grad"].float(), s["grad"].dtype
    dz = g if y is None else y * (g - (g * y).sum(-1, keepdim=True))
    out = {"x": (dz @ s["weight"].detach().float().t()).to(dtype)}
    long = dz.reshape(-1, dz.shape[-1]).double()
    out["weight"] = (x.reshape(-1, x.shape[-1]).t().double() @ long).to(dtype)
    if x2 is not None:
        out["x2"] = (dz @ s["weight2"].detach().float().t()).to(dtype)
        out["weight2"] = (x2.reshape(-1, x2.shape[-1]).t().double() @ long).to(dtype)
    if s["bias"] is not None:
        out["bias"] = long.sum(0).to(dtype)
    if s["case"]["residual"]:
        out["residual"] = (-dz).to(dtype)
    return out


def _run_plain(s):
    case, what = s["case"], s["case"]["what"]
    dtype, shape = DTYPES[case["dtype"]], _shape(case)
    if what == "pack":
        codes, header = _encode(s["x"])
        return {"codes": codes, "scales": header}
    if what == "unpack":
        return {"x": _decode(s["codes"], s["scales"], (*shape, case["k"])).to(dtype)}
    if what == "gradients_8bit":
        y = _decode(*s["out"], (*shape, case["n"])) if s["out"] is not None else None
        x2 = _decode(*s["x2"], (*shape, case["k2"])) if s["x2"] is not None else None
        return _plain_gradients(s, y, _decode(*s["x"], (*shape, case["k"])), x2)
    out = _plain_forward(s).to(dtype)
    kept = {}
    if what == "mix_8bit":     # in bfloat16, which holds every value of 8 bits and an exponent
        names = ["x"] + (["x2"] if s["x2"] is not None else []) + (["y"] if case["activation"] else [])
        tensors = {"x": s["x"], "x2": s["x2"], "y": out}
        kept = {"kept_" + m: _decode(*_encode(tensors[m]), tensors[m].shape).bfloat16() for m in names}
    if what in ("mix", "mix_8bit"):
        return {"out": out, **kept}
    x, x2 = s["x"].detach(), s["x2"].detach() if s["x2"] is not None else None
    if what == "train_8bit":
        x = _decode(*_encode(x), x.shape)
        x2 = _decode(*_encode(x2), x2.shape) if x2 is not None else None
    y = out.float() if case["activation"] else None
    return {"out": out, **_plain_gradients(s, y, x.float(), x2.float() if x2 is not None else None)}


def _run_own(s):
    import permutohedral_lattice_b200 as plb

    case, what = s["case"], s["case"]["what"]
    dtype, shape = DTYPES[case["dtype"]], _shape(case)
    activation = case["activation"] or None
    if what == "pack":
        p = plb.pack_activations(s["x"])
        return {"codes": p.codes, "scales": p.scales}
    if what == "unpack":
        return {"x": plb.unpack_activations(plb.PackedActivations(s["codes"], s["scales"], (*shape, case["k"]), dtype))}
    if what == "gradients_8bit":
        def kept(name, channels):
            return None if s[name] is None else plb.PackedActivations(*s[name], (*shape, channels), dtype)

        saved = plb.MixSaved(kept("x", case["k"]), kept("x2", case["k2"]), kept("out", case["n"]))
        needs = ["x", "weight"] + (["x2", "weight2"] if case["k2"] else []) + (["bias"] if case["bias"] else []) + (
            ["residual"] if case["residual"] else [])
        grads = plb.channel_mix_backward(s["grad"], saved, s["weight"], s["weight2"], activation=activation,
                                         residual_scale=-1.0, needs=needs)
        return {m: getattr(grads, m) for m in needs}
    given = {"x2": s["x2"], "weight2": s["weight2"], "activation": activation, "residual_scale": -1.0}
    if what == "mix_8bit":
        out, saved = plb.channel_mix_raw(s["x"], s["weight"], s["bias"], s["residual"], checkpoint="8bit", **given)
        kept = {"x": saved.x, "x2": saved.x2, "y": saved.out if activation else None}
        return {"out": out, **{"kept_" + m: plb.unpack_activations(p, torch.bfloat16) for m, p in kept.items()
                               if p is not None}}
    checkpoint = "8bit" if what == "train_8bit" else None
    out = plb.channel_mix(s["x"], s["weight"], s["bias"], s["residual"], checkpoint=checkpoint, **given)
    if what == "mix":
        return {"out": out}
    leaves = {m: s[m] for m in ("x", "weight", "x2", "weight2", "bias", "residual") if s[m] is not None}
    grads = torch.autograd.grad(out, list(leaves.values()), s["grad"])
    return {"out": out.detach(), **dict(zip(leaves, grads))}


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _values_64(codes, header):
    """What a block's codes stand for, float64: its own reading of the format."""
    h = header.long().repeat_interleave(BLOCK)[: codes.numel()]
    c = codes.long()
    c = c - 256 * ((h >= 256) & (c >= 128)).long()
    return c.double() * ((h % 256 - 127 + 1023) << 52).view(torch.float64)


def _kept_64(x):
    """Values after a round trip through 8 bits, float64, blocks that are all finite: from the definition, by trying exponents."""
    flat = x.double().reshape(-1)
    pad = (-flat.numel()) % BLOCK
    v = torch.cat([flat, flat.new_zeros(pad)]).reshape(-1, BLOCK)
    top = v.abs().max(dim=1, keepdim=True).values
    limit = torch.where((v < 0).any(dim=1, keepdim=True), 127.0, 255.0).to(top)
    step = torch.full_like(top, 2.0 ** -126)
    e = torch.ceil(torch.log2(torch.clamp(top / limit, min=2.0 ** -126))).long()
    for near in (1, 0, -1):      # the least exponent that holds the block, wherever the logarithm's rounding put it
        candidate = ((torch.clamp(e + near, min=-126) + 1023) << 52).view(torch.float64)
        step = torch.where(top <= limit * candidate, candidate, step)
    return (torch.round(v / step) * step).reshape(-1)[: flat.numel()].reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    what, shape = case["what"], _shape(case)
    k, k2, n = case["k"], case["k2"], case["n"]
    if what == "pack":
        return None                                          # whole numbers, equal on both sides
    if what == "unpack":
        return {"x": _values_64(s["codes"], s["scales"]).reshape(*shape, k)}
    wide = {m: s[m].detach().double() for m in ("weight", "weight2", "bias", "residual") if s[m] is not None}
    result = {}
    if what == "gradients_8bit":
        x = _values_64(*s["x"]).reshape(-1, k)
        x2 = _values_64(*s["x2"]).reshape(-1, k2) if k2 else None
        y = _values_64(*s["out"]).reshape(-1, n) if case["activation"] else None
    else:
        x, x2 = s["x"].detach().double().reshape(-1, k), s["x2"].detach().double().reshape(-1, k2) if k2 else None
        logits = torch.einsum("rk,kn->rn", x, wide["weight"])
        if k2:
            logits += torch.einsum("rk,kn->rn", x2, wide["weight2"])
        if "bias" in wide:
            logits += wide["bias"]
        if "residual" in wide:
            logits -= wide["residual"].reshape(-1, n)
        y = logits
        if case["activation"] == "softmax":
            y = torch.nan_to_num(torch.softmax(logits, dim=-1), nan=0.0)      # rows with nothing allowed: zeros
        elif case["activation"] == "relu":
            y = logits.clamp(min=0.0)
        result["out"] = y.reshape(*shape, n)
        if what == "mix":
            return result
        if what == "mix_8bit":
            result["kept_x"] = _kept_64(s["x"])
            if k2:
                result["kept_x2"] = _kept_64(s["x2"])
            if case["activation"]:
                result["kept_y"] = None                      # a rounding of computed values: next to a border it goes either way
            return result
        if what == "train_8bit":
            x, x2 = _kept_64(s["x"]).reshape(-1, k), _kept_64(s["x2"]).reshape(-1, k2) if k2 else None
        if not case["activation"]:
            y = None
    d = s["grad"].double().reshape(-1, n)
    if y is not None:
        d = y * d - y * (y * d).sum(dim=1, keepdim=True)
    result["x"] = torch.einsum("rn,kn->rk", d, wide["weight"]).reshape(*shape, k)
    result["weight"] = torch.einsum("rk,rn->kn", x, d)
    if k2:
        result["x2"] = torch.einsum("rn,kn->rk", d, wide["weight2"]).reshape(*shape, k2)
        result["weight2"] = torch.einsum("rk,rn->kn", x2, d)
    if case["bias"]:
        result["bias"] = d.sum(dim=0)
    if case["residual"]:
        result["residual"] = -d.reshape(*shape, n)
    return result
