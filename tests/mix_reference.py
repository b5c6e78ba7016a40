"""Plain 64-bit forms of channel_mix, its gradients and the 8-bit blocks, with bounds on what float arithmetic may be off.

Units: u = 2^-24, half a step of float32 relative to the value.  A product of two floats that are each taken as two terms of
11 bits is off by at most 2^-21 for either operand's cut and 2^-22 for the product of the low terms, 2^-20 in all; a sum
of n terms rounded (or cut) at every step by at most 2 n u of the terms' magnitudes.  Other ways to compute it (FMA in
float32) are within that."""
import numpy as np
import torch

U = 2.0 ** -24
PRODUCT = 2.0 ** -20


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def forward(x, w, bias, residual, x2, w2, activation, scale):
    """out and a bound for each of its elements, before the rounding to the output's type; all float64."""
    d = lambda t: None if t is None else t.detach().double()   # noqa: E731
    x, w, bias, residual, x2, w2 = map(d, (x, w, bias, residual, x2, w2))
    z, mag, terms = x @ w, x.abs() @ w.abs(), x.shape[-1]
    if x2 is not None:
        z, mag, terms = z + x2 @ w2, mag + x2.abs() @ w2.abs(), terms + x2.shape[-1]
    if bias is not None:
        z, mag = z + bias, mag + bias.abs()
    if residual is not None:
        z = z + scale * residual
        mag = mag + torch.where(torch.isinf(residual), torch.zeros_like(residual), (scale * residual).abs())
    off = (PRODUCT + 2 * (terms + 3) * U) * mag
    if activation == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), off
    if activation == "softmax":
        top = z.amax(-1, keepdim=True)
        empty = top == -np.inf
        e = torch.exp(z - torch.where(empty, torch.zeros_like(top), top))
        y = e / torch.where(empty, torch.ones_like(top), e.sum(-1, keepdim=True))
        # each logit is off by `off` (one that is forbidden not at all) and again by the subtraction of the largest, the
        # exponential by 2 steps, the sum and quotient by a step a term
        n = z.shape[-1]
        live = torch.where(z == -np.inf, torch.zeros_like(off), off).amax(-1, keepdim=True)
        shift = torch.where(y > 0, (z - torch.where(empty, torch.zeros_like(top), top)).abs(), torch.zeros_like(z))
        return y, y * (torch.expm1(2 * live + 2 * U * shift) + (2 * n + 12) * U) + 1e-37
    return z, off


def gradients(g, y, x, w, x2, w2, activation, scale):
    """{name: (gradient, bound)} in float64, before the rounding to its type; y, x and x2: what the forward pass kept."""
    d = lambda t: None if t is None else t.detach().double()   # noqa: E731
    g, y, x, w, x2, w2 = map(d, (g, y, x, w, x2, w2))
    n = g.shape[-1]
    dz, off = g, torch.zeros_like(g)
    if activation == "relu":
        dz = torch.where(y > 0, g, torch.zeros_like(g))
    elif activation == "softmax":
        s, mag = (y * g).sum(-1, keepdim=True), (y * g).abs().sum(-1, keepdim=True)
        dz = y * (g - s)
        off = y * (2 * (n + 1) * U * mag + 4 * U * (g.abs() + s.abs()))
    dz, off = dz.reshape(-1, n), off.reshape(-1, n)
    a = dz.abs()
    result = {"residual": ((scale * dz).reshape(g.shape), abs(scale) * (off + U * a).reshape(g.shape) * 2)}
    result["bias"] = (dz.sum(0), off.sum(0) + 128 * U * a.sum(0))
    for name, inp, weight in (("", x, w), ("2", x2, w2)):
        if weight is None:
            continue
        k = weight.shape[0]
        result["x" + name] = ((dz @ weight.t()).reshape(g.shape[:-1] + (k,)),
                              (off @ weight.abs().t() + (PRODUCT + 2 * n * U) * (a @ weight.abs().t())).reshape(
                                  g.shape[:-1] + (k,)))
        if inp is not None:
            m = inp.reshape(-1, k)
            # chains of at most 64 rounded additions, their ends summed more exactly
            result["weight" + name] = (m.t() @ dz, m.abs().t() @ off + (PRODUCT + 128 * U) * (m.abs().t() @ a))
    return result


def assert_within(got, want, bound, what=""):
    """Element by element: the bound and the rounding to got's type, of the value and of whatever is off already."""
    g = got.detach().double()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    assert bool(torch.isfinite(g).all()), what + ": not finite"
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37   # half the least step
    allowed = bound + half_step(got.dtype) * (want.abs() + bound) + tiny
    over = (g - want).abs() - allowed
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, "%s: %g over what is allowed, %g off at a value of %g" % (
        what, worst, float((g - want).abs().flatten()[over.argmax()]), float(want.flatten()[over.argmax()]))


def pack(values, keep_nonzero=False):
    """codes and headers of a flat float32 array, block by block as the format is defined."""
    v = np.asarray(values, np.float32).reshape(-1)
    codes, headers = np.zeros(v.size, np.uint8), np.zeros(-(-v.size // 32), np.int16)
    for b in range(headers.size):
        block = v[32 * b:32 * b + 32].astype(np.float64)
        if not np.isfinite(block).all():
            headers[b] = 255
            continue
        signed = bool((block < 0).any())
        limit = 127.0 if signed else 255.0
        e = -126
        while np.abs(block).max() > limit * 2.0 ** e and e < (121 if signed else 120):
            e += 1
        c = np.clip(np.rint(block / 2.0 ** e), -127 if signed else 0, limit)
        if keep_nonzero:
            c = np.where((c == 0) & (block != 0), np.sign(block), c)
        codes[32 * b:32 * b + 32] = c.astype(np.int64).astype(np.uint8)
        headers[b] = (e + 127) | (256 if signed else 0)
    return codes, headers


def unpack(codes, headers):
    h = np.repeat(np.asarray(headers, np.int64), 32)[:codes.size]
    c = codes.astype(np.int64)
    c = np.where((h & 256) != 0, codes.view(np.int8).astype(np.int64), c)
    return np.where((h & 255) == 255, np.nan, c * 2.0 ** ((h & 255) - 127.0))
