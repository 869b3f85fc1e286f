"""CPU oracle of the rotary positions, the short causal convolution and the selective scan, in 64 bits.

TEST INFRASTRUCTURE ONLY.  The formulas are written out, forward and backward, token by token, and are
checked against autograd and against differences.  All of them are sums of products, so the same
functions called with ``absolute=True`` bound the size of what is summed: the magnitude that rounding
errors are relative to (``bounds`` below turns it into a tolerance).
"""
from __future__ import annotations

import torch

U = 2.0 ** -24                      # one fp32 rounding, relative


def rotary(x, freqs, positions, factor, interleaved, axes=1, inverse=False, absolute=False):
    """x (..., L, D); positions broadcastable to (..., L) (axes > 1: (..., L, axes))."""
    x = x.detach().double()
    P = freqs.numel()
    pos = positions.double()
    pos = pos.repeat_interleave(P // axes, -1) if axes > 1 else pos[..., None]
    ang = pos * freqs.double() * (-1.0 if inverse else 1.0)
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor
    out = x.clone()
    for i in range(P):
        m, n = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
        a, b = x[..., m], x[..., n]
        if absolute:
            out[..., m] = out[..., n] = (a.abs() + b.abs()) * factor
        else:
            out[..., m], out[..., n] = a * c[..., i] - b * s[..., i], a * s[..., i] + b * c[..., i]
    return out


def _spans(T, cu):
    if cu is None:
        return [(0, T)]
    b = cu.tolist()
    return list(zip(b[:-1], b[1:]))


def conv(x, w, bias=None, silu=False, init=None, dy=None, dfin=None, cu=None, absolute=False):
    """x (B, T, C) (packed: B = 1).  Dict of y, final and, with dy, dx, dw, db, dinit."""
    ab = (lambda v: v.abs()) if absolute else (lambda v: v)
    x, w = ab(x.detach().double()), ab(w.detach().double())
    bias = w.new_zeros(w.shape[0]) if bias is None else ab(bias.detach().double())
    B, T, C = x.shape
    W = w.shape[1]
    spans = _spans(T, cu)
    S = B if cu is None else len(spans)
    hist = x.new_zeros(S, W - 1, C) if init is None else ab(init.detach().double())
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    final, dinit = torch.zeros_like(hist), torch.zeros_like(hist)
    dw, db = torch.zeros_like(w), torch.zeros_like(bias)
    for r, (lo, hi) in enumerate(spans):
        of = slice(None) if cu is None else slice(r, r + 1)
        n = hi - lo
        f = torch.cat((hist[of], x[:, lo:hi]), 1)
        p = sum(f[:, j:j + n] * w[:, j] for j in range(W)) + bias
        sg = torch.sigmoid(p)
        if absolute:                # |silu| <= |p|, |silu'| <= 1.1, |silu''| <= 0.5
            y[:, lo:hi], slope = p, 1.1 + 0.5 * p
        else:
            y[:, lo:hi], slope = p * sg, sg * (1 + p * (1 - sg))
        if not silu:
            y[:, lo:hi], slope = p, torch.ones_like(p)
        final[of] = f[:, n:]
        if dy is None:
            continue
        g = ab(dy.detach().double())[:, lo:hi] * slope
        df = torch.zeros_like(f)
        if dfin is not None:
            df[:, n:] += ab(dfin.detach().double())[of]
        for j in range(W):
            df[:, j:j + n] += g * w[:, j]
            dw[:, j] += (g * f[:, j:j + n]).sum((0, 1))
        db += g.sum((0, 1))
        dx[:, lo:hi], dinit[of] = df[:, W - 1:], df[:, :W - 1]
    out = {"y": y, "final": final}
    return out if dy is None else dict(out, dx=dx, dw=dw, db=db, dinit=dinit)


def scan(x, dt, A, Bm, Cm, D=None, z=None, bias=None, softplus=False, init=None, dy=None, dfin=None, cu=None,
         absolute=False):
    """x, dt, z, dy (B, T, C), Bm, Cm (B, T, G, N) (packed: B = 1).  Dict of y, final and, with dy, dx, ddt,
    dA, dB, dC, dD, dz, dbias, dinit."""
    ab = (lambda v: v.abs()) if absolute else (lambda v: v)
    d64 = lambda v: v.detach().double()                                             # noqa: E731
    raw, A0 = d64(dt), d64(A)
    if bias is not None:
        raw = raw + d64(bias)
    d = torch.nn.functional.softplus(raw) if softplus else raw
    slope = torch.where(raw > 20, torch.ones_like(raw), torch.sigmoid(raw)) if softplus else torch.ones_like(raw)
    x, Bm, Cm, Aa, da = ab(d64(x)), ab(d64(Bm)), ab(d64(Cm)), ab(A0), ab(d)
    D = x.new_zeros(x.shape[2]) if D is None else ab(d64(D))
    B, T, C = x.shape
    G, N = Bm.shape[2:]
    if z is None:
        gate, gslope = torch.ones_like(x), torch.zeros_like(x)
    else:
        zz = d64(z)
        sg = torch.sigmoid(zz)
        # the slope of silu is a sum of two terms of opposite sign for z < 0 (they cancel at z = -1.28): what
        # its roundings are relative to is the sum of their sizes, not of the slope itself
        gate, gslope = ab(zz * sg), sg * (1 + (zz.abs() if absolute else zz) * (1 - sg))
    wide = lambda v: v.repeat_interleave(C // G, 1)                                 # noqa: E731
    tight = lambda v: v.unflatten(1, (G, C // G)).sum(2)                            # noqa: E731
    spans = _spans(T, cu)
    S = B if cu is None else len(spans)
    start = x.new_zeros(S, C, N) if init is None else ab(d64(init))
    final, dinit = start.clone(), torch.zeros_like(start)
    s = torch.zeros_like(x)
    inside = torch.zeros(T, dtype=torch.bool)
    keep = []
    for r, (lo, hi) in enumerate(spans):
        of = slice(None) if cu is None else slice(r, r + 1)
        inside[lo:hi] = True
        h = start[of]
        for t in range(lo, hi):
            a = torch.exp(d[:, t, :, None] * A0)
            before, h = h, a * h + (da[:, t] * x[:, t])[..., None] * wide(Bm[:, t])
            keep.append((before, h, a))
            s[:, t] = (h * wide(Cm[:, t])).sum(-1)
        final[of] = h
    out = {"y": (s + D * x) * gate * inside[:, None], "final": final}
    if dy is None:
        return out
    dy = ab(d64(dy)) * inside[:, None]
    e = dy * gate
    g = {k: torch.zeros_like(v) for k, v in dict(dx=x, ddt=x, dA=A0, dB=Bm, dC=Cm).items()}
    at = sum(hi - lo for lo, hi in spans)
    for r, (lo, hi) in reversed(list(enumerate(spans))):
        of = slice(None) if cu is None else slice(r, r + 1)
        back = torch.zeros_like(start[of]) if dfin is None else ab(d64(dfin))[of]
        for t in range(hi - 1, lo - 1, -1):
            at -= 1
            before, h, a = keep[at]
            grad = back + e[:, t, :, None] * wide(Cm[:, t])
            g["dC"][:, t] = tight(e[:, t, :, None] * h)
            g["dB"][:, t] = tight((da[:, t] * x[:, t])[..., None] * grad)
            gB = (grad * wide(Bm[:, t])).sum(-1)
            back = grad * a
            r_ = back * before
            g["dx"][:, t] = da[:, t] * gB + D * e[:, t]
            g["ddt"][:, t] = ((r_ * Aa).sum(-1) + x[:, t] * gB) * slope[:, t]
            g["dA"] += (r_ * da[:, t, :, None]).sum(0)
        dinit[of] = back
    return dict(out, **g, dD=(e * x).sum((0, 1)), dz=dy * (s + D * x) * gslope, dbias=g["ddt"].sum((0, 1)), dinit=dinit)


def bounds(ref, major, dtype, roundings):
    """Largest allowed error, elementwise: one rounding to ``dtype`` of the exact value (half a step), plus
    ``roundings`` roundings of fp32 relative to what is summed."""
    half = torch.finfo(dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -126}[dtype]
    return half * ref.abs() + (1 + half) * roundings * U * major.abs() + tiny
