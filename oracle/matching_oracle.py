"""Plain 64-bit forms of the matching-transformer operators, and elementwise bounds on what the
kernels may be off by, from the roundings that their types force.

u(t) = eps(t) / 2 is the relative error of one rounding to type t (bf16 2^-8, fp16 2^-11, fp32 2^-24).
"""
import math
from fractions import Fraction

import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the type's subnormals: the absolute error of rounding a value below its range."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def allowed(b, lq, lk, band=None, lengths=None, mask=None):
    ok = torch.ones(b, lq, lk, dtype=torch.bool)
    i, j = torch.arange(lq)[:, None], torch.arange(lk)[None]
    if band is not None:
        ok &= (i - j >= 0) & (i - j < band)
    if lengths is not None:
        ok &= j[None] < lengths.cpu().long().clamp(0, lk)[:, None, None]
    if mask is not None:
        ok &= mask.cpu()[:, None, :]
    return ok


def attention(q, k, v, scale, ok, dout=None, raised=0):
    """(out, lse), with ``dout`` also (dq, dk, dv), and bounds of the same shapes, as two dicts.

    Bounds, elementwise with p the weights, L keys, D values, u the type's unit, f = 2^-24:
      score s:   (D + 2) f scale sum |q||k|                                          =: es
      weight p:  relative rp = 2 max_j es + (L + 64) f  (sum of weights; exponential within 2^-22),
                 and u more where it is rounded as an operand (16-bit types)
      out:       (u + rp + L f) sum p|v| + u |out|
      ds = p (g.v - delta):  p (D f sum |g||v| + sum |g| bound(out)) + |ds| (u + rp + 4 f)
      dq:        scale (sum bound(ds) |k| + L f sum |ds||k|) + u |dq|, dk and dv alike over the rows
    fp16 adds half a subnormal step for operands below the type's range: weights (times 2^14 in dv),
    ds of rows brought to |g| <= 1 (dq) and of key heads brought to |g| <= 1 (dk), there times 2^raised
    (dq) and 2^(raised - 1) (dk): 0 is an upper bound where the range is not passed, which takes 8.
    """
    t = q.dtype
    low = t != torch.float32
    u, uw, sub = unit(t), unit(t) if low else 0.0, tiny(t)
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    g = h // kv
    bad = ~ok.any(1)  # (b, lk): nobody looks there, and its values may be anything
    k, v = (torch.where(bad[:, :, None, None], torch.zeros(()).double(), x) for x in (k, v))
    ke, ve = (x.repeat_interleave(g, 2).permute(0, 2, 1, 3) for x in (k, v))
    qe = q.permute(0, 2, 1, 3)
    s = scale * (qe @ ke.transpose(2, 3))
    es = scale * (d + 2) * F32 * (qe.abs() @ ke.abs().transpose(2, 3))
    s = s.masked_fill(~ok[:, None], -math.inf)
    es = es.masked_fill(~ok[:, None], 0.0)
    lse = torch.logsumexp(s, -1) if lk else torch.full(s.shape[:3], -math.inf, dtype=torch.float64)
    p = torch.where(ok[:, None], torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None]), 0.0)
    worst = es.amax(-1, keepdim=True) if lk else es.sum(-1, keepdim=True)
    rp = 2 * worst + (lk + 64) * F32
    out = p @ ve
    eo = (uw + rp + lk * F32) * (p @ ve.abs()) + u * out.abs() + sub * (ok[:, None].double() @ ve.abs()) + tiny(t)
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    val = {"out": back(out), "lse": lse.permute(0, 2, 1)}
    tol = {"out": back(eo), "lse": (rp[..., 0] + 4 * F32 * lse.abs().nan_to_num(posinf=0.0)).permute(0, 2, 1)}
    if dout is None:
        return val, tol
    ge = dout.detach().cpu().double().permute(0, 2, 1, 3)
    dp = ge @ ve.transpose(2, 3)
    delta = (ge * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eds = (p * (d * F32 * (ge.abs() @ ve.abs().transpose(2, 3)) + (ge.abs() * eo).sum(-1, keepdim=True))
           + ds.abs() * (uw + rp + 4 * F32))
    gmax = ge.abs().amax(-1, keepdim=True)
    kmax = ge.abs().reshape(b, kv, -1).amax(-1) if ge.numel() else ge.new_zeros(b, kv)
    kmax = kmax.repeat_interleave(g, 1)[:, :, None, None]
    some = ok[:, None].double()
    lower = 2.0 ** -raised
    eq = scale * ((eds + sub * 2 * lower * gmax * some) @ ke.abs() + (lk + 8) * F32 * (ds.abs() @ ke.abs()))
    ek = scale * ((eds + sub * (4 if raised else 2) * lower * kmax * some).transpose(2, 3) @ qe.abs()
                  + (lq * g + 8) * F32 * (ds.abs().transpose(2, 3) @ qe.abs()))
    ev = ((p * (uw + rp + (lq * g + 8) * F32) + sub * 2.0 ** -14 * some).transpose(2, 3) @ ge.abs())
    heads = lambda x: x.reshape(b, kv, g, lk, d).sum(2).permute(0, 2, 1, 3)  # noqa: E731
    dq, dk, dv = back(scale * (ds @ ke)), heads(scale * (ds.transpose(2, 3) @ qe)), heads(p.transpose(2, 3) @ ge)
    val.update(dq=dq, dk=dk, dv=dv)
    tol.update(dq=back(eq) + u * dq.abs() + tiny(t), dk=heads(ek) + u * dk.abs() + tiny(t),
               dv=heads(ev) + u * dv.abs() + tiny(t))
    return val, tol


def _pi(bits):
    """pi as a fraction, within 2^-(bits - 8): 16 atan(1/5) - 4 atan(1/239) (Machin)."""
    def atan(n):
        x = total = (1 << bits) // n
        k = 1
        while x:
            x, k = x // (n * n), k + 2
            total += x // k if k % 4 == 1 else -(x // k)
        return total
    return Fraction(16 * atan(5) - 4 * atan(239), 1 << bits)


def wrapped(positions, frequencies):
    """positions * frequencies modulo 2 pi, in [-pi, pi], exact up to the one rounding to 64 bits: both are
    whole multiples of powers of two, and their product is formed as a fraction."""
    turn = 2 * _pi(300)

    def one(p, f):
        a = Fraction(p) * Fraction(f)
        return float(a - turn * round(a / turn))
    rows = [[one(p, f) for f in frequencies.tolist()] for p in positions.reshape(-1).tolist()]
    return torch.tensor(rows, dtype=torch.float64).view(*positions.shape, -1)


def rotary(x, positions, frequencies, layout, amplitude=1.0, inverse=False, exact=False):
    """(y, bound): the turn in 64 bits; off by one rounding of y, and 2^-22 of the pair's length for
    the fp32 angle (in turns, within 2^-26 of 1), its sine and the two products.  ``exact``: the angle is
    formed exactly (the product in 64 bits else), at whatever position."""
    r = 2 * frequencies.numel()
    a = x.detach().cpu().double()
    angle = positions.cpu().double().reshape(-1, positions.shape[-1])[:, :, None] * frequencies.cpu()
    if exact:
        angle = wrapped(positions.reshape(-1, positions.shape[-1]), frequencies)
    z = torch.polar(torch.full_like(angle, amplitude), -angle if inverse else angle)[:, :, None]
    one, two = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    w = torch.complex(a[..., one].contiguous(), a[..., two].contiguous())
    y, tol = a.clone(), torch.zeros_like(a)
    turned = w * z
    y[..., one], y[..., two] = turned.real, turned.imag
    far = 4.0 * F32 * abs(amplitude) * w.abs()
    # |t f / 2 pi| carries a relative error of 2 * 2^-53 in 64 bits
    far = far + abs(amplitude) * w.abs() * (angle.abs() * 2.0 ** -51)[:, :, None]
    tol[..., one] = tol[..., two] = far
    return y, tol + unit(x.dtype) * y.abs() * (tol > 0) + tiny(x.dtype) * (tol > 0)


def rms_norm(x, weight, residual, eps, dy=None, dsummed=None):
    """({y, summed, dx, dweight}, bounds): with C values a row and R rows
      n = s / sqrt(mean s^2 + eps): (C / 2 + 8) f relative
      y: (C / 2 + 10) f |y| + u |y|
      dx: (h + |n| mean |h n|) / rms times (3 C + 32) f, + u |dx|
      dw: sum |g n| times (R + C / 2 + 16) f, + u |dw|
    """
    t, w = x.dtype, weight.detach().cpu().double()
    s = x.detach().cpu().double()
    if residual is not None:
        s = (s + residual.detach().cpu().double()).to(residual.dtype).double()
    c = s.shape[-1]
    inv = 1.0 / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    n = s * inv
    y = n * w
    val = {"y": y, "summed": s}
    tol = {"y": ((c / 2 + 10) * F32 + unit(t)) * y.abs() + tiny(t), "summed": torch.zeros_like(s)}
    if dy is not None:
        g = dy.detach().cpu().double()
        hw = g * w
        ds = inv * (hw - n * (hw * n).mean(-1, keepdim=True))
        eds = inv * (hw.abs() + n.abs() * (hw * n).abs().mean(-1, keepdim=True)) * (3 * c + 32) * F32
        if dsummed is not None:
            z = dsummed.detach().cpu().double()
            ds, eds = ds + z, eds + 2 * F32 * (z.abs() + ds.abs())
        dw = (g * n).reshape(-1, c).sum(0)
        edw = (g * n).abs().reshape(-1, c).sum(0) * (n.numel() // c + c / 2 + 16) * F32
        val.update(dx=ds, dweight=dw)
        tol.update(dx=eds, dweight=edw + unit(weight.dtype) * dw.abs() + tiny(weight.dtype))
    return val, tol
