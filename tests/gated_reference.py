"""Plain 64-bit form of gated_mix and its gradients, with bounds on what the kernels' arithmetic may be off.

u = 2^-24.  Products.  A float as three bfloat16 terms, each the nearest to what is left: 2^-9, 2^-18 and 2^-27 of it remain; of nine
products the six largest are taken: two operands cut at 2^-27 and two products of 2^-27 left out, 2^-25 in all.  16-bit values multiply exactly.
Sums.  n terms, each addition rounded or cut by at most 2 u of the terms' magnitudes; the small terms' products, 2^-8 of the others,
five times as many: 2.2 (n + 3) u.  Sums over rows: chains of at most 8192 rows (float32: 256), their ends added up as floats.
Hidden values, of 16-bit types, are rounded once more on their way to a product: half a step.
Activations: their slope (at most 1.13) times what g is off, and 8 u (1 + |g|) for the exponential (or erf) and the quotient."""
import math

import torch

U = 2.0 ** -24
PRODUCT = 2.0 ** -25


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _act(g, eg, kind):
    """act, its bound, act', its bound."""
    fe = 8 * U * (1 + g.abs())
    s = torch.sigmoid(g)
    if kind == "silu":
        a, d, curve = g * s, s * (1 + g * (1 - s)), 0.5
    elif kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        a, d, curve = g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 0.8
    elif kind == "sigmoid":
        a, d, curve = s, s * (1 - s), 0.1
    else:
        a, d = g.clamp(min=0), (g > 0).double()
        return a, eg, d, (g.abs() <= eg).double()
    return a, 1.13 * eg + fe, d, curve * eg + fe


def _mul(a, ea, b, eb):
    return a * b, a.abs() * eb + b.abs() * ea + ea * eb + U * (a * b).abs()


def _product(a, ea, b, chain=None):
    n = a.shape[-1] if chain is None else chain
    return a @ b, ea @ b.abs() + (PRODUCT + 2.2 * (n + 3) * U) * (a.abs() @ b.abs())


def gated(t, activation, scale, grad=None):
    """t: {name: tensor or None}.  {name: (value, bound)}, float64, before the rounding to the type: out and, with grad, the gradients."""
    dtype = t["x"].dtype
    hs, tiny = half_step(dtype), 2.0 ** -25 if dtype == torch.float16 else 0.0
    w = {m: None if v is None else v.detach().double() for m, v in t.items()}
    x = w["x"].reshape(-1, w["x"].shape[-1])
    shape = t["x"].shape[:-1]
    zero = torch.zeros_like(x)

    def linear(weight, bias):
        z, e = _product(x, zero, weight)
        if bias is not None:
            e = e + 2.2 * U * (z.abs() + bias.abs())
            z = z + bias
        return z, e

    def rounded(v, e):
        return v, e + hs * (v.abs() + e) + tiny

    g, eg = linear(w["gate_weight"], w["gate_bias"])
    u, eu = linear(w["up_weight"], w["up_bias"])
    act, eact, slope, eslope = _act(g, eg, activation)
    a, ea = rounded(*_mul(act, eact, u, eu))
    out, eo = _product(a, ea, w["down_weight"])
    if w["down_bias"] is not None:
        out = out + w["down_bias"]
        eo = eo + 2 * U * (out.abs() + w["down_bias"].abs())
    if w["residual"] is not None:
        r = scale * w["residual"].reshape(out.shape)
        out = out + r
        eo = eo + 2 * U * (out.abs() + r.abs())
    n = out.shape[-1]
    found = {"out": (out.reshape(*shape, n), eo.reshape(*shape, n))}
    if grad is None:
        return found
    d = grad.detach().double().reshape(-1, n)
    da, eda = _product(d, torch.zeros_like(d), w["down_weight"].t())
    dg, edg = rounded(*_mul(*_mul(da, eda, u, eu), slope, eslope))
    du, edu = rounded(*_mul(da, eda, act, eact))
    dxg, exg = _product(dg, edg, w["gate_weight"].t())
    dxu, exu = _product(du, edu, w["up_weight"].t())
    found["x"] = ((dxg + dxu).reshape(t["x"].shape), (exg + exu + 2.2 * dg.shape[-1] * U * (dg.abs() @ w["gate_weight"].t().abs()
                                                                                        + du.abs() @ w["up_weight"].t().abs())).reshape(t["x"].shape))
    found["residual"] = (scale * grad.detach().double(), 2 * U * (scale * grad.detach().double()).abs())
    chain = min(x.shape[0], 256 if dtype == torch.float32 else 8192) + 300

    def over_rows(a, ea, b, eb):
        return a.t() @ b, ea.t() @ b.abs() + (a.abs() + ea).t() @ eb + (PRODUCT + 2.2 * chain * U) * (a.abs().t() @ b.abs())

    ones = torch.ones_like(x[:, :1])
    none = torch.zeros_like(ones)
    zd = torch.zeros_like(d)
    found["gate_weight"], found["up_weight"] = over_rows(x, zero, dg, edg), over_rows(x, zero, du, edu)
    found["down_weight"] = over_rows(a, ea, d, zd)
    for name, v, e in (("gate_bias", dg, edg), ("up_bias", du, edu), ("down_bias", d, zd)):
        value, bound = over_rows(ones, none, v, e)
        found[name] = (value[0], bound[0])
    return found
