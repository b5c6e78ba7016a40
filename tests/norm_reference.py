"""Plain 64-bit forms of channel_norm, its gradients and the dropout's mask, with bounds on what float arithmetic may be off.

u = 2^-24, half a step of float32 relative to the value.  Each quantity goes with a bound on its error: a product's is
|a| eb + |b| ea + ea eb + u |ab|, a sum's of n terms the terms' errors and n u of their magnitudes whatever the order, a
reciprocal root's half the relative error of what is under it (all of it is allowed) and 2 steps, 4 u."""
import numpy as np
import torch

U = 2.0 ** -24
CHAIN = 256   # rounded additions of a sum over rows: some of a thread's rows, 5 of lanes, 8 of warps, 80 of shares


def philox_words(count, key, offset):
    """Words of `count` values: Philox4x32-10 as its paper defines it, in numpy's 64-bit integers."""
    quads = np.arange(-(-count // 4), dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    full = lambda v: np.full_like(quads, v & 0xFFFFFFFF)   # noqa: E731
    c = [quads & low, quads >> shift, full(offset), full(offset >> 32)]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> shift) ^ c[1] ^ np.uint64(k0), q & low, (p >> shift) ^ c[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:count]


def kept(shape, p, key, offset, device="cuda"):
    words = philox_words(int(np.prod(shape)), key, offset)
    threshold = min(int(p * 4294967296.0 + 0.5), 0xFFFFFFFF)
    return torch.from_numpy((words >= threshold).reshape(shape)).to(device)


def _mul(a, ea, b, eb):
    return a * b, a.abs() * eb + b.abs() * ea + ea * eb + U * (a * b).abs()


def _mean(a, ea):
    n = a.shape[-1]
    return a.mean(-1, keepdim=True), ea.mean(-1, keepdim=True) + (n + 2) * U * a.abs().mean(-1, keepdim=True)


def _norm(x, ex, kind, eps):
    """hat, its bound, reciprocal deviation, its relative bound."""
    d, ed = x, ex
    if kind == "layer":
        m, em = _mean(x, ex)
        d = x - m
        ed = ex + em + U * d.abs()
    q, eq = _mean(d * d, 2 * d.abs() * ed + ed * ed + U * d * d)
    rel = eq / (q + eps) + 6 * U
    rstd = 1.0 / torch.sqrt(q + eps)
    hat = d * rstd
    return hat, ed * rstd * (1 + rel) + hat.abs() * (rel + 2 * U), rstd, rel


def _back(t, et, hat, ehat, rstd, rel, kind):
    q, eq = _mean(*_mul(t, et, hat, ehat))
    inner, ei = t - hat * q, et + hat.abs() * eq + ehat * (q.abs() + eq) + 3 * U * (t.abs() + (hat * q).abs())
    if kind == "layer":
        s, es = _mean(t, et)
        inner, ei = inner - s, ei + es + 3 * U * s.abs()
    d = rstd * inner
    return d, rstd * ei * (1 + rel) + d.abs() * (rel + 2 * U)


def _rows(v, e):
    n = v.shape[-1]
    return v.reshape(-1, n).sum(0), (e + CHAIN * U * v.abs()).reshape(-1, n).sum(0)


def norm(x, residual, gate, after, before, scale, p, keep, grads=None):
    """{name: (value, bound)} of h, y and, with grads = (dh or None, dy or None), the gradients, in float64, before the rounding to
    their types.  after, before: None or (weight, bias, kind, eps)."""
    wide = lambda t: None if t is None else t.detach().double()   # noqa: E731
    x, residual, gate = wide(x), wide(residual), wide(gate)
    after, before = (None if n is None else (wide(n[0]), wide(n[1]), n[2], n[3]) for n in (after, before))
    zero = torch.zeros_like(x)
    v, ev = x, zero
    if after:
        hat_a, ehat_a, rstd_a, rel_a = _norm(x, zero, after[2], after[3])
        v, ev = hat_a, ehat_a
        if after[0] is not None:
            v, ev = _mul(v, ev, after[0], zero)
        if after[1] is not None:
            v = v + after[1]
            ev = ev + U * v.abs()

    def drop(v, ev):
        if keep is None:
            return v, ev
        return torch.where(keep, v / (1 - p), zero), torch.where(keep, ev / (1 - p) + 3 * U * v.abs() / (1 - p), zero)

    v, ev = drop(v, ev)
    h, eh = (v, ev) if gate is None else _mul(v, ev, gate, zero)
    if residual is not None:
        h = h + scale * residual
        eh = eh + 2 * U * ((scale * residual).abs() + h.abs())
    found = {"h": (h, eh)}
    if before:
        hat_b, ehat_b, rstd_b, rel_b = _norm(h, eh, before[2], before[3])
        y, ey = hat_b, ehat_b
        if before[0] is not None:
            y, ey = _mul(y, ey, before[0], zero)
        if before[1] is not None:
            y = y + before[1]
            ey = ey + U * y.abs()
        found["y"] = (y, ey)
    if grads is None:
        return found
    d, ed = (zero, zero) if grads[0] is None else (wide(grads[0]), zero)
    if before:
        t, et = wide(grads[1]), zero
        found["before_weight"] = _rows(*_mul(t, et, hat_b, ehat_b))
        found["before_bias"] = _rows(t, et)
        if before[0] is not None:
            t, et = _mul(t, et, before[0], zero)
        b, eb = _back(t, et, hat_b, ehat_b, rstd_b, rel_b, before[2])
        d = d + b
        ed = ed + eb + U * d.abs()
    found["residual"] = (scale * d, abs(scale) * (ed + 2 * U * d.abs()))
    dg = _mul(d, ed, v, ev)
    if gate is not None:
        found["gate"] = dg if gate.dim() > 1 else _rows(*dg)
        d, ed = _mul(d, ed, gate, zero)
    d, ed = drop(d, ed)
    if after:
        found["after_weight"] = _rows(*_mul(d, ed, hat_a, ehat_a))
        found["after_bias"] = _rows(d, ed)
        if after[0] is not None:
            d, ed = _mul(d, ed, after[0], zero)
        d, ed = _back(d, ed, hat_a, ehat_a, rstd_a, rel_a, after[2])
    found["x"] = (d, ed)
    return found
