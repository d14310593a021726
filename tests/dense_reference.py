"""Plain 64-bit forms of the dense feed-forward operators, each with a bound of how far a result may be off.

The bounds are elementwise and worst-case.  ``unit`` is half a step of the 16-bit type (one rounding); a sum of K products in FP32 is
off by at most ``K * 2**-23`` of the sum of their magnitudes, in whatever order and with truncated or rounded steps; the activation's
elementary functions are good to 2**-20 of the magnitudes they combine.  What a formula amplifies follows its derivatives:
``|silu'| <= 1.1``, ``|silu''| <= 0.5``, ``|silu(g)| <= |g|``.
"""

import math

import torch

FUNC = 2.0 ** -20


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_step(dtype):
    """Half of the distance between the smallest numbers of the type: what a rounding may cost there."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def acc(k):
    return (k + 8) * 2.0 ** -23


class Block:
    """Forward and gradients of the gated block in 64 bits: ``y, dx, dw13, dw2`` and bounds under the same names in ``off``."""

    def __init__(self, x, w13, w2, clamp, dy=None):
        dtype = x.dtype
        u, tiny = half_step(dtype), floor_step(dtype)
        c = math.inf if clamp is None else clamp
        x, w13, w2 = (t.detach().double() for t in (x, w13, w2))
        m, hidden = x.shape
        inter = w2.shape[1]
        wg, wu = w13[:inter], w13[inter:]
        g, up = x @ wg.T, x @ wu.T
        eg, eu = acc(hidden) * (x.abs() @ wg.abs().T), acc(hidden) * (x.abs() @ wu.abs().T)
        gc, uc = g.clamp(max=c), up.clamp(-c, c)
        s = torch.sigmoid(gc)
        silu = gc * s
        h = silu * uc
        dh_off = 1.1 * uc.abs() * eg + silu.abs() * eu + 1.1 * eg * eu + FUNC * h.abs() + u * h.abs() + tiny
        self.y = h @ w2.T
        self.off = {"y": (dh_off + acc(inter) * h.abs()) @ w2.abs().T * (1 + acc(inter)) + u * self.y.abs() + tiny}
        if dy is None:
            return
        dy = dy.double()
        dh = dy @ w2
        e_dh = acc(hidden) * (dy.abs() @ w2.abs())
        slope = s * (1 + gc * (1 - s))
        dg = dh * uc * slope * (g <= c)
        du = dh * silu * (up.abs() <= c)
        near_g, near_u = (g - c).abs() <= eg, (up.abs() - c).abs() <= eu
        off_g = 1.1 * uc.abs() * e_dh + (dh.abs() + e_dh) * (1.1 * eu + 0.5 * uc.abs() * eg + FUNC * uc.abs()) + u * dg.abs() + tiny
        off_u = silu.abs() * e_dh + (dh.abs() + e_dh) * (1.1 * eg + FUNC * silu.abs()) + u * du.abs() + tiny
        off_g = off_g + near_g * 1.1 * dh.abs() * uc.abs()
        off_u = off_u + near_u * dh.abs() * silu.abs()
        d, off_d = torch.cat((dg, du), 1), torch.cat((off_g, off_u), 1)
        self.dx, self.dw13, self.dw2 = d @ w13, d.T @ x, dy.T @ h
        self.off["dx"] = (off_d + acc(2 * inter) * d.abs()) @ w13.abs() * (1 + acc(2 * inter)) + u * self.dx.abs() + tiny
        self.off["dw13"] = (off_d + acc(m) * d.abs()).T @ x.abs() * (1 + acc(m)) + u * self.dw13.abs() + tiny
        self.off["dw2"] = dy.abs().T @ (dh_off + acc(m) * h.abs()) * (1 + acc(m)) + u * self.dw2.abs() + tiny


def quantize(x):
    """Whole numbers and FP32 scales, exactly."""
    x = x.double()
    amax = x.abs().amax(-1)
    scale = torch.where(amax == 0, 1.0, (amax / 127).float().double())
    q = torch.round(x / scale[..., None])
    bad = ~torch.isfinite(amax)
    scale = torch.where(bad, math.nan, scale)
    return torch.where(bad[..., None], 0.0, q).to(torch.int8), scale.float()


def _scaled(x, sx, w, sw):
    return (x.double() @ w.double().T) * sx.double()[:, None] * sw.double()


def projection(x, sx, w, sw, bias, out_dtype):
    """Value and bound: the sums are exact but for their conversion to FP32, then two products, an addition and a rounding."""
    y = _scaled(x, sx, w, sw)
    off = 4 * 2.0 ** -24 * y.abs()
    if bias is not None:
        off = off + 2.0 ** -24 * (y.abs() + bias.double().abs())
        y = y + bias.double()
    return y, off + half_step(out_dtype) * y.abs() + floor_step(out_dtype)


def gated_projection(x, sx, w13, sw, clamp, out_dtype):
    c = math.inf if clamp is None else clamp
    inter = w13.shape[0] // 2
    v = _scaled(x, sx, w13, sw)
    g, u = v[:, :inter], v[:, inter:]
    eg, eu = 4 * 2.0 ** -24 * g.abs(), 4 * 2.0 ** -24 * u.abs()
    gc, uc = g.clamp(max=c), u.clamp(-c, c)
    silu = gc * torch.sigmoid(gc)
    h = silu * uc
    off = 1.1 * uc.abs() * eg + silu.abs() * eu + 1.1 * eg * eu + FUNC * h.abs()
    return h, off + half_step(out_dtype) * h.abs() + floor_step(out_dtype)


def check(name, got, want, off):
    """Everywhere within its bound (NaN and infinity where the plain form has them)."""
    got = got.double().to(want.device)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), name
    wrong = finite & ~((got - want).abs() <= off)
    if bool(wrong.any()):
        at = tuple(torch.nonzero(wrong)[0].tolist())
        raise AssertionError(f"{name}: {int(wrong.sum())} of {wrong.numel()} off, first at {at}: {float(got[at])} for {float(want[at])}, "
                             f"bound {float(off[at])}")
