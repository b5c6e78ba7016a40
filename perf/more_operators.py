"""Operators of a learned block of features, as timed cases: what the networks around the lattice filter, which give a dense
CRF its features and unaries, need between two products of channels.

`channel_norm`: norms after and before a block, with dropout, gate and scaled residual between them.  `channel_dropout`:
dropout from a counter-based generator, no mask stored.  `gated_mix`: a gated feed-forward block.  Each forward, and in
training with its gradients.  Where `own` is false, `run` computes them with elementary torch operations, else by the
package's entry points.

Inputs are synthetic, made on the GPU from a seed: features and gradients of unit size, weights as a network's are after
its initialisation, norms' weights near one.
"""
import math

import torch

own = False

MOST_ROWS = 16 * 512 * 512              # the largest listed call of rows: 16 images of 512 x 512
MOST_VALUES = MOST_ROWS * 32            # of a norm or dropout
MOST_HIDDEN = 8 * 512 * 512 * 256       # hidden values of a feed-forward block
MOST_PRODUCTS = MOST_HIDDEN * 3 * 64    # its multiplications
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = {"layer": 1e-5, "rms": 1e-6}
RESIDUAL_SCALE = 0.75


def _case(what, shape, k, h=0, n=0, train=False, dtype="float32", residual=False, bias=True, activation="silu", after="",
          before="", gate="", p=0.0, name=None):
    """what: "dropout", "norm" or "gated".  shape: batch and spatial sizes, as text.  k: channels; h, n: hidden and output channels
    of a gated block.  train: forward and gradients.  after, before: "", "layer" or "rms".  gate: "", "channel" (a value a channel)
    or "full" (a value for each of x).  p: share of dropped values."""
    case = {"what": what, "shape": shape, "k": k, "h": h, "n": n, "train": train, "dtype": dtype, "residual": residual,
            "bias": bias, "activation": activation, "after": after, "before": before, "gate": gate, "p": p}
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # a thumbnail's label features: latency of a call
        _case("dropout", "1x33x45", 21, p=0.1, name="dropout_thumbnail"),
        # a training batch of the benchmark's size: a block's output dropped and added to its input, and the gradients
        _case("dropout", "16x512x512", 21, train=True, dtype="bfloat16", residual=True, p=0.2, name="dropout_train_batch"),
        # the norm before a block on a photograph's features
        _case("norm", "1x375x500", 64, before="layer", name="norm_photo"),
        # between two blocks of a training batch: norm after, dropout, learned gate of the channels, residual, norm before
        _case("norm", "16x512x512", 32, train=True, dtype="bfloat16", residual=True, bias=False, after="rms", before="rms",
              gate="channel", p=0.1, name="norm_between_blocks_train"),
        # volumes with an odd number of channels, gated value by value, in training
        _case("norm", "2x111x128x120", 21, train=True, residual=True, after="layer", gate="full", name="norm_gated_volumes_train"),
        # wide features: residual and norm in inference
        _case("norm", "4x321x481", 256, dtype="float16", residual=True, bias=False, before="rms", name="norm_wide"),
        # the features of one point: latency of a feed-forward block
        _case("gated", "1x1", 64, 256, 64, dtype="bfloat16", residual=True, bias=False, name="gated_point"),
        # patch features of 5 x 5 colours to 21 labels' unaries on a photograph of ragged size
        _case("gated", "1x375x500", 75, 128, 21, name="gated_unaries_photo"),
        # a batch of images in inference
        _case("gated", "4x512x512", 64, 256, 64, dtype="bfloat16", residual=True, bias=False, name="gated_batch"),
        # the same block in training
        _case("gated", "8x512x512", 64, 256, 64, train=True, dtype="bfloat16", residual=True, bias=False, name="gated_train_batch"),
        # volumes in training, in float32
        _case("gated", "2x111x128x120", 32, 128, 32, train=True, residual=True, name="gated_train_volumes"),
        # as many channels as a product takes, ragged image, in training
        _case("gated", "1x321x481", 128, 512, 128, train=True, dtype="float16", activation="gelu", name="gated_train_wide"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["dropout", "norm", "norm", "gated", "gated", "gated"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    train, residual, bias = rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5
    if what == "gated":
        k, h, n = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 512), _log_uniform(rng, 1, 128)
        if rng.random() < 0.4:      # sizes as networks have them
            k, h, n = (max(8, 8 * round(v / 8)) for v in (k, h, n))
        most = min(MOST_ROWS, MOST_HIDDEN // h, MOST_PRODUCTS // (h * (2 * k + n)), MOST_VALUES // max(k, n))
        return _case(what, "1x%d" % _log_uniform(rng, 1, most), k, h, n, train, dtype, residual, bias,
                     rng.choice(["silu", "silu", "gelu", "sigmoid"]))
    k = _log_uniform(rng, 2, 512)
    if rng.random() < 0.4:
        k = max(8, 8 * round(k / 8))
    shape = "1x%d" % _log_uniform(rng, 1, min(MOST_ROWS, MOST_VALUES // k))
    if what == "dropout":
        return _case(what, shape, k, train=train, dtype=dtype, residual=residual, p=round(rng.uniform(0.05, 0.6), 3))
    after, before = rng.choice([("", "layer"), ("", "rms"), ("layer", ""), ("rms", ""), ("rms", "rms"), ("layer", "layer")])
    plain = not after and not residual
    return _case(what, shape, k, train=train, dtype=dtype, residual=residual, bias=bias, after=after, before=before,
                 gate="" if plain else rng.choice(["", "channel", "full"]),
                 p=0.0 if plain or rng.random() < 0.5 else round(rng.uniform(0.05, 0.6), 3))


def _shape(case):
    return tuple(int(s) for s in case["shape"].split("x"))


def _only_before(case):
    """Whether h is x itself, so that the call gives y alone."""
    return not (case["after"] or case["residual"] or case["gate"] or case["p"])


def work(case):
    rows, size = math.prod(_shape(case)), 4 if case["dtype"] == "float32" else 2
    k, h, n, train, residual = case["k"], case["h"], case["n"], case["train"], case["residual"]
    if case["what"] == "gated":
        weights = (h * (2 * k + n)) * size
        values = k + n + (n if residual else 0)
        products = 2 * rows * h * (2 * k + n)
        if not train:
            return {"bytes": rows * values * size + weights, "flops": products}
        # the step as a whole: x, residual and the gradient of out once, out and the other gradients once
        return {"bytes": rows * size * (2 * values) + 2 * weights, "flops": 3 * products}
    if case["what"] == "dropout":
        once = 2 + (1 if residual else 0)
        return {"bytes": rows * k * size * (2 * once if train else once), "flops": 0}
    inputs = 1 + (1 if residual else 0) + (1 if case["gate"] == "full" else 0)
    outputs = (0 if _only_before(case) else 1) + (1 if case["before"] else 0)
    return {"bytes": rows * k * size * (2 * (inputs + outputs) if train else inputs + outputs), "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape, dtype = _shape(case), DTYPES[case["dtype"]]
    k, h, n = case["k"], case["h"], case["n"]

    def randn(*size):
        return torch.randn(size, generator=g, device="cuda", dtype=torch.float32 if case["dtype"] == "float32" else dtype)

    def weight(rows, columns):
        return (torch.randn((rows, columns), generator=g, device="cuda") / math.sqrt(rows)).to(dtype)

    def vector(size, about, spread):
        return (about + spread * torch.randn(size, generator=g, device="cuda")).to(dtype)

    s = {"case": dict(case), "leaves": {"x": randn(*shape, k)}}
    leaves = s["leaves"]
    width = n if case["what"] == "gated" else k
    if case["residual"]:
        leaves["residual"] = randn(*shape, width)
    if case["what"] == "gated":
        leaves["gate_weight"], leaves["up_weight"], leaves["down_weight"] = weight(k, h), weight(k, h), weight(h, n)
        if case["bias"]:
            leaves["gate_bias"], leaves["up_bias"], leaves["down_bias"] = vector(h, 0.0, 0.2), vector(h, 0.0, 0.2), vector(n, 0.0, 0.2)
    elif case["what"] == "norm":
        for place in ("after", "before"):
            if case[place]:
                leaves[place + "_weight"] = vector(k, 1.0, 0.1)
                if case["bias"]:
                    leaves[place + "_bias"] = vector(k, 0.0, 0.2)
        if case["gate"] == "channel":
            leaves["gate"] = vector(k, 0.5, 0.2)
        elif case["gate"] == "full":
            leaves["gate"] = torch.sigmoid(randn(*shape, k).float()).to(dtype)
    if case["p"]:
        s["seed"] = torch.randint(0, 1 << 40, (2,), generator=g, device="cuda")     # the generator's key, and its offset
    if case["train"]:
        for leaf in leaves.values():
            leaf.requires_grad_(True)
        s["grads"] = [randn(*shape, width) for _ in range(2 if case["before"] and not _only_before(case) else 1)]
    return s


def _philox(seed, count):
    """Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): the words of `count` values, word i % 4 of
    counter (i / 4, offset) under the key, as int64."""
    low = 0xFFFFFFFF
    quads = torch.arange((count + 3) // 4, device="cuda")
    c0, c1 = quads & low, quads >> 32
    c2, c3 = (seed[1] & low).expand_as(c0), ((seed[1] >> 32) & low).expand_as(c0)
    k0, k1 = seed[0] & low, (seed[0] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), -1).reshape(-1)[:count]


def _threshold(p):
    return min(int(p * 4294967296.0 + 0.5), 0xFFFFFFFF)


def _dropped(v, s):
    """v / (1 - p) where the generator keeps it, zero elsewhere."""
    p = s["case"]["p"]
    if not p:
        return v
    keep = (_philox(s["seed"], v.numel()) >= _threshold(p)).view(v.shape)
    return torch.where(keep, v * (1.0 / (1.0 - p)), torch.zeros_like(v))


def _norm(x, kind):
    """The values without weight and bias, and the reciprocal deviation."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS[kind])
    return x * rstd, rstd


def _norm_gradient(d, xhat, rstd, kind):
    inner = d - xhat * (d * xhat).mean(-1, keepdim=True)
    if kind == "layer":
        inner = inner - d.mean(-1, keepdim=True)
    return inner * rstd


def _over_rows(v):
    return v.reshape(-1, v.shape[-1]).double().sum(0)


def _plain_norm(s, f):
    case = s["case"]
    u, xhat, rstd = f["x"], None, None
    if case["after"]:
        xhat, rstd = _norm(f["x"], case["after"])
        u = xhat * f["after_weight"] + f.get("after_bias", 0.0)
    v = _dropped(u, s)
    h = v * f["gate"] if case["gate"] else v
    if case["residual"]:
        h = h + RESIDUAL_SCALE * f["residual"]
    outs = {} if _only_before(case) else {"h": h}
    hhat, hrstd = None, None
    if case["before"]:
        hhat, hrstd = _norm(h, case["before"])
        outs["y"] = hhat * f["before_weight"] + f.get("before_bias", 0.0)
    if not case["train"]:
        return outs
    grads = dict(zip(outs, (g.float() for g in s["grads"])))
    found, dh = {}, grads.get("h", 0.0)
    if case["before"]:
        dy = grads["y"]
        found["before_weight"] = _over_rows(dy * hhat)
        if case["bias"]:
            found["before_bias"] = _over_rows(dy)
        dh = dh + _norm_gradient(dy * f["before_weight"], hhat, hrstd, case["before"])
    if case["residual"]:
        found["residual"] = RESIDUAL_SCALE * dh
    dv = dh
    if case["gate"]:
        found["gate"] = dh * v if case["gate"] == "full" else _over_rows(dh * v)
        dv = dh * f["gate"]
    du = _dropped(dv, s)
    if case["after"]:
        found["after_weight"] = _over_rows(du * xhat)
        if case["bias"]:
            found["after_bias"] = _over_rows(du)
        du = _norm_gradient(du * f["after_weight"], xhat, rstd, case["after"])
    found["x"] = du
    return {**outs, **{"d_" + m: found[m] for m in f}}


def _activated(g, kind):
    """act(g) and act'(g)."""
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-g))
    if kind == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _plain_gated(s, f):
    case = s["case"]
    x = f["x"].reshape(-1, case["k"])
    g, u = x @ f["gate_weight"] + f.get("gate_bias", 0.0), x @ f["up_weight"] + f.get("up_bias", 0.0)
    act, slope = _activated(g, case["activation"])
    a = act * u
    out = a @ f["down_weight"] + f.get("down_bias", 0.0)
    if case["residual"]:
        out = out + RESIDUAL_SCALE * f["residual"].reshape(out.shape)
    outs = {"out": out.reshape(*_shape(case), case["n"])}
    if not case["train"]:
        return outs
    d = s["grads"][0].float().reshape(-1, case["n"])
    found = {"down_weight": a.t().double() @ d.double(), "down_bias": _over_rows(d)}
    da = d @ f["down_weight"].t()
    dg, du = da * u * slope, da * act
    long = x.t().double()
    found["gate_weight"], found["up_weight"] = long @ dg.double(), long @ du.double()
    found["gate_bias"], found["up_bias"] = _over_rows(dg), _over_rows(du)
    found["x"] = (dg @ f["gate_weight"].t() + du @ f["up_weight"].t()).reshape(f["x"].shape)
    if case["residual"]:
        found["residual"] = (RESIDUAL_SCALE * d).reshape(f["residual"].shape)
    return {**outs, **{"d_" + m: found[m] for m in f}}


def _run_plain(s):
    case = s["case"]
    f = {m: leaf.detach().float() for m, leaf in s["leaves"].items()}
    if case["what"] == "norm":
        outs = _plain_norm(s, f)
    elif case["what"] == "gated":
        outs = _plain_gated(s, f)
    else:
        outs = {"out": _dropped(f["x"], s) + (RESIDUAL_SCALE * f["residual"] if case["residual"] else 0.0)}
        if case["train"]:
            g = s["grads"][0].float()
            outs["d_x"] = _dropped(g, s)
            if case["residual"]:
                outs["d_residual"] = RESIDUAL_SCALE * g
    return {m: t.to(DTYPES[case["dtype"]]) for m, t in outs.items()}


def _run_own(s):
    import permutohedral_lattice_b200 as plb

    case, leaves = s["case"], s["leaves"]
    if case["what"] == "dropout":
        outs = {"out": plb.channel_dropout(leaves["x"], case["p"], s["seed"], residual=leaves.get("residual"),
                                           residual_scale=RESIDUAL_SCALE)}
    elif case["what"] == "gated":
        outs = {"out": plb.gated_mix(**leaves, activation=case["activation"], residual_scale=RESIDUAL_SCALE)}
    else:
        norms = {place: plb.Norm(leaves[place + "_weight"], leaves.get(place + "_bias"), case[place], EPS[case[place]])
                 for place in ("after", "before") if case[place]}
        got = plb.channel_norm(leaves["x"], leaves.get("residual"), leaves.get("gate"), **norms,
                               residual_scale=RESIDUAL_SCALE, dropout=case["p"], seed=s.get("seed"))
        names = ([] if _only_before(case) else ["h"]) + (["y"] if case["before"] else [])
        outs = dict(zip(names, got if len(names) == 2 else (got,)))
    if not case["train"]:
        return outs
    grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), s["grads"])
    return {**{m: t.detach() for m, t in outs.items()}, **{"d_" + m: g for m, g in zip(leaves, grads)}}


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _keep_64(seed, shape, p):
    """Which values are kept: the generator from its definition, 64-bit products from 16-bit pieces."""
    count = math.prod(shape)
    key, offset = (int(v) for v in seed.tolist())
    index = torch.arange(count, device="cuda")
    block, which = index.div(4, rounding_mode="floor"), index.remainder(4)
    block = block[::4].contiguous()
    word = [block % 2 ** 32, block // 2 ** 32, torch.full_like(block, offset % 2 ** 32), torch.full_like(block, offset // 2 ** 32 % 2 ** 32)]

    def product(v, by):
        low, high = v * (by % 65536), v * (by // 65536)            # each below 2^48
        total = low + (high % 65536) * 65536                       # below 2^49
        return (total // 2 ** 32 + high // 65536) % 2 ** 32, total % 2 ** 32

    for r in range(10):
        high0, low0 = product(word[0], 0xD2511F53)
        high2, low2 = product(word[2], 0xCD9E8D57)
        word = [high2 ^ word[1] ^ ((key + r * 0x9E3779B9) % 2 ** 32), low2,
                high0 ^ word[3] ^ ((key // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32), low0]
    return (torch.cat([w[:, None] for w in word], 1).flatten()[:count] >= min(round(p * 2 ** 32), 2 ** 32 - 1)).reshape(shape)


def _rows_64(case, t, keep):
    """The outputs of some rows, in 64 bits, followed by autograd."""
    k = case["k"]
    scaled = RESIDUAL_SCALE * t["residual"] if case["residual"] else 0.0

    def drop(v):
        return v if keep is None else torch.where(keep, v / (1.0 - case["p"]), 0.0)

    def norm(v, place):
        if case[place] == "layer":
            return torch.nn.functional.layer_norm(v, (k,), t[place + "_weight"], t.get(place + "_bias"), EPS["layer"])
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS["rms"]) * t[place + "_weight"]
        return v + t[place + "_bias"] if case["bias"] else v

    if case["what"] == "dropout":
        return {"out": drop(t["x"]) + scaled}
    if case["what"] == "gated":
        linear = lambda v, m: torch.einsum("rk,kn->rn", v, t[m + "_weight"]) + (t[m + "_bias"] if case["bias"] else 0.0)   # noqa: E731
        act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[case["activation"]]
        return {"out": linear(act(linear(t["x"], "gate")) * linear(t["x"], "up"), "down") + scaled}
    h = drop(norm(t["x"], "after") if case["after"] else t["x"])
    if case["gate"]:
        h = h * t["gate"]
    h = h + scaled
    outs = {} if _only_before(case) else {"h": h}
    return {**outs, "y": norm(h, "before")} if case["before"] else outs


def exact(case, seed):
    s = prepare(case, seed)
    shape, rows = _shape(case), math.prod(_shape(case))
    width = case["n"] or case["k"]
    keep = _keep_64(s["seed"], (rows, case["k"]), case["p"]) if case["p"] else None
    of_rows = {m for m in s["leaves"] if m in ("x", "residual") or (m == "gate" and case["gate"] == "full")}
    wide = {m: leaf.detach().double().reshape(rows, -1) if m in of_rows else leaf.detach().double() for m, leaf in s["leaves"].items()}
    parts, sums = {}, {}
    step = max(1, (1 << 28) // max(case["k"], case["h"], width))         # some gigabytes at a time
    for lo in range(0, rows, step):
        t = {m: (v[lo:lo + step] if m in of_rows else v).detach().requires_grad_(case["train"]) for m, v in wide.items()}
        outs = _rows_64(case, t, None if keep is None else keep[lo:lo + step])
        for m, v in outs.items():
            parts.setdefault(m, []).append(v.detach())
        if case["train"]:
            up = [g.double().reshape(rows, width)[lo:lo + step] for g in s["grads"]]
            for m, d in zip(t, torch.autograd.grad(list(outs.values()), list(t.values()), up)):
                if m in of_rows:
                    parts.setdefault("d_" + m, []).append(d)
                else:
                    sums["d_" + m] = sums.get("d_" + m, 0.0) + d
        del outs, t
    result = {m: torch.cat(v).reshape(*shape, -1) for m, v in parts.items()}
    return {**result, **sums}
