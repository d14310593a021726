"""Plain 64-bit forms of the experts' products, each with a bound of how far a result may be off (see ``dense_reference``).

Products in 8-bit floating point: a value of 8 bits times another is exact in FP32.  A sum over K of them in the tensor core and over its groups
in FP32 is off by at most ``K * 2**-23`` of the sum of the magnitudes of what is added, as there; the product of the two scales and its use by one
fused multiply-add cost ``2**-24`` each for every group, which ``acc`` has room for.
"""

import math

import torch

import dense_reference as R

BLOCK = 128


def pieces(ends, rows):
    """(expert, first row, row behind the last); none where the ends are not in order."""
    ends = ends.tolist()
    if any(b < a for a, b in zip([0] + ends, ends)) or ends[-1] > rows:
        return []
    return [(e, a, b) for e, (a, b) in enumerate(zip([0] + ends, ends)) if b > a]


class Projection:
    """``y, dx, dw`` and bounds under the same names in ``off``."""

    def __init__(self, x, w, ends, dy=None):
        u, tiny = R.half_step(x.dtype), R.floor_step(x.dtype)
        x, w = x.detach().double(), w.detach().double()
        rows, (experts, channels, width) = x.shape[0], w.shape
        self.y = torch.zeros((rows, channels), dtype=torch.float64, device=x.device)
        self.off = {"y": torch.zeros_like(self.y)}
        if dy is not None:
            dy = dy.double()
            self.dx, self.dw = torch.zeros_like(x), torch.zeros_like(w)
            self.off.update(dx=torch.zeros_like(x), dw=torch.zeros_like(w))
        for e, a, b in pieces(ends, rows):
            self.y[a:b] = x[a:b] @ w[e].T
            self.off["y"][a:b] = R.acc(width) * (x[a:b].abs() @ w[e].abs().T) + u * self.y[a:b].abs() + tiny
            if dy is not None:
                self.dx[a:b], self.dw[e] = dy[a:b] @ w[e], dy[a:b].T @ x[a:b]
                self.off["dx"][a:b] = R.acc(channels) * (dy[a:b].abs() @ w[e].abs()) + u * self.dx[a:b].abs() + tiny
                self.off["dw"][e] = R.acc(b - a) * (dy[a:b].abs().T @ x[a:b].abs()) + u * self.dw[e].abs() + tiny


class Block:
    """``y, dx, dw13, dw2`` of the gated block with each row's expert."""

    def __init__(self, x, w13, w2, ends, clamp, dy=None):
        names = ("y",) if dy is None else ("y", "dx", "dw13", "dw2")
        like = {"y": x, "dx": x, "dw13": w13, "dw2": w2}
        for n in names:
            setattr(self, n, torch.zeros(like[n].shape, dtype=torch.float64, device=x.device))
        self.off = {n: torch.zeros_like(getattr(self, n)) for n in names}
        for e, a, b in pieces(ends, x.shape[0]):
            one = R.Block(x[a:b], w13[e], w2[e], clamp, None if dy is None else dy[a:b])
            for n in names:
                at = slice(a, b) if n in ("y", "dx") else e
                getattr(self, n)[at] = getattr(one, n)
                self.off[n][at] = one.off[n]


def quantize(x):
    """E4M3 values and FP32 scales, exactly: the nearest of the type's 253 finite numbers, on a border the one whose last bit is 0."""
    x = x.double()
    lead, width = x.shape[:-1], x.shape[-1]
    groups = torch.nn.functional.pad(x, (0, -width % BLOCK)).reshape(*lead, -(-width // BLOCK), BLOCK)
    amax = groups.abs().amax(-1)
    scale = torch.where(amax == 0, 1.0, (amax / 448).float().double())
    bad = ~torch.isfinite(amax)
    scale = torch.where(bad, math.nan, scale)
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().to(x.device)
    borders = (codes[1:] + codes[:-1]) / 2
    ratio = torch.where(bad[..., None], 0.0, groups / scale[..., None])
    low, high = torch.bucketize(ratio.abs(), borders), torch.bucketize(ratio.abs(), borders, right=True)
    q = codes[torch.where(low % 2 == 0, low, high)] * torch.where(ratio.signbit(), -1.0, 1.0)
    return q.flatten(-2)[..., :width], scale.float()


def spread(scales, rows, cols, parts=0):
    """A scale for each value: of groups of 128 columns, and (``parts``) of 128 rows of each part."""
    s = scales.double().repeat_interleave(BLOCK, -1)[..., :cols]
    if parts:
        s = torch.cat([p.repeat_interleave(BLOCK, -2)[..., :rows // parts, :] for p in s.chunk(parts, -2)], -2)
    return s


def fp8_product(x, sx, w, sw, ends, out_dtype, gated=False, clamp=None):
    """Value and bound; x ``(T, K)``, w ``(E, N, K)``."""
    rows, (experts, channels, width) = x.shape[0], w.shape
    xs = x.double() * spread(sx, 0, width)
    ends = torch.tensor([rows]) if ends is None else ends
    shape = (rows, channels // 2 if gated else channels)
    value, off = torch.zeros(shape, dtype=torch.float64, device=x.device), torch.zeros(shape, dtype=torch.float64, device=x.device)
    u, tiny, c = R.half_step(out_dtype), R.floor_step(out_dtype), math.inf if clamp is None else clamp
    for e, a, b in pieces(ends, rows):
        ws = w[e].double() * spread(sw[e], channels, width, 2 if gated else 1)
        y, far = xs[a:b] @ ws.T, R.acc(width) * (xs[a:b].abs() @ ws.abs().T)
        if not gated:
            value[a:b], off[a:b] = y, far + u * y.abs() + tiny
            continue
        (g, up), (eg, eu) = y.chunk(2, 1), far.chunk(2, 1)
        gc, uc = g.clamp(max=c), up.clamp(-c, c)
        silu = gc * torch.sigmoid(gc)
        h = silu * uc
        value[a:b] = h
        off[a:b] = (1.1 * uc.abs() * eg + silu.abs() * eu + 1.1 * eg * eu + R.FUNC * h.abs()) * (1 + u) + u * h.abs() + tiny
    # past the type's largest number (by half a step, u of it) a value rounds to an infinity; within its bound of there it may be either
    top = torch.finfo(out_dtype).max * (1 + u)
    value, off = torch.where(value.abs() - off > top, value.sign() * math.inf, value), torch.where((value.abs() - top).abs() <= off, math.inf, off)
    return value, off
