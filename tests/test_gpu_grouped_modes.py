"""Products of a layer's experts: strides, values that are no numbers, ends out of order, streams, graphs, sizes, and runs of them together."""

import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import dense_reference as R
import grouped_reference as G
from helpers import ROOT
from test_gpu_fp8 import E4M3, _case
from test_gpu_grouped import DEV, _ends, _rand

pytestmark = pytest.mark.gpu


def _api():
    from vllm_plugin_b200 import api
    return api


def _block(seed, rows, experts, hidden, inter, dtype=torch.bfloat16, grad=False):
    t = (_rand(seed, rows, hidden, dtype=dtype), _rand(seed + 100, experts, 2 * inter, hidden, std=0.1, dtype=dtype),
         _rand(seed + 200, experts, hidden, inter, std=0.1, dtype=dtype))
    return [a.requires_grad_(grad) for a in t] + [_rand(seed + 300, rows, hidden, dtype=dtype)]


def _check_block(x, w13, w2, ends, clamp, dy, got):
    want = G.Block(x, w13, w2, ends, clamp, dy)
    for name, g in zip(("y", "dx", "dw13", "dw2"), got):
        R.check(name, g.detach(), getattr(want, name), want.off[name])


# ---------------------------------------------------------------------------------------------------------------------
# strides and values
# ---------------------------------------------------------------------------------------------------------------------
def test_rows_of_any_stride():
    api = _api()
    x, w13, w2, _ = _block(1, 60, 3, 128, 72)
    wide = torch.zeros((60, 320), dtype=x.dtype, device=DEV)
    for view in (x[::2], x.T.contiguous().T, x[4:5].expand(12, 128), wide[:, 64:192].copy_(x), wide[:, 3:131].copy_(x), x[:0],
                 torch.cat((x.new_zeros(1), x.flatten()))[1:].view(60, 128)):
        rows = view.shape[0]
        ends = _ends([rows // 3, 0, rows // 2])
        many = torch.stack((ends, ends + 1), 1)[:, 0]                          # ends of any stride
        leaves = [t.detach().clone().requires_grad_(True) if i else t.detach().requires_grad_(True) for i, t in enumerate((view, w13, w2))]
        y = api.grouped_feed_forward(*leaves, many, activation_clamp=2.0)
        up = _rand(9, rows, 128)
        for dy in (up, up.T.contiguous().T, torch.cat((up.new_zeros(3), up.flatten()))[3:].view(rows, 128)):
            grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            _check_block(view, w13, w2, ends, 2.0, dy, (y, *grads))
        w = w13.detach().clone().requires_grad_(True)
        y = api.grouped_projection(leaves[0], w, many)
        grads = torch.autograd.grad(y, (leaves[0], w), torch.ones((), dtype=y.dtype, device=DEV).expand(y.shape))
        want = G.Projection(view, w, ends, torch.ones_like(y))
        for name, g in zip(("y", "dx", "dw"), (y, *grads)):
            R.check(name, g.detach(), getattr(want, name), want.off[name])


@pytest.mark.parametrize("rows", [5, 90, 700])
def test_parts_of_the_gradients(rows):
    api = _api()
    x, w13, w2, dy = _block(2, rows, 3, 64, 40)
    ends = _ends([rows // 2, 0, rows - rows // 2 - 1])
    want = G.Block(x, w13, w2, ends, None, dy)
    for mask in range(1, 8):
        leaves = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w13, w2))]
        api.grouped_feed_forward(*leaves, ends).backward(dy)
        for i, name in enumerate(("dx", "dw13", "dw2")):
            if mask >> i & 1:
                R.check(name, leaves[i].grad, getattr(want, name), want.off[name])
            else:
                assert leaves[i].grad is None
    one = G.Projection(x, w13, ends, torch.cat((dy, dy[:, :16]), 1))
    for mask in range(1, 4):
        leaves = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w13))]
        api.grouped_projection(*leaves, ends).backward(torch.cat((dy, dy[:, :16]), 1))
        for i, name in enumerate(("dx", "dw")):
            if mask >> i & 1:
                R.check(name, leaves[i].grad, getattr(one, name), one.off[name])
            else:
                assert leaves[i].grad is None


def test_shared_leaves_accumulate():
    api = _api()
    x, w13, w2, dy = _block(6, 33, 2, 64, 32, torch.float16, True)
    ends, other = _ends([20, 13]), _ends([3, 30])
    got = torch.autograd.grad(api.grouped_feed_forward(x, w13, w2, ends) + api.grouped_feed_forward(x, w13, w2, other, activation_clamp=0.5), (x, w13, w2), dy)
    one = torch.autograd.grad(api.grouped_feed_forward(x, w13, w2, ends), (x, w13, w2), dy)
    two = torch.autograd.grad(api.grouped_feed_forward(x, w13, w2, other, activation_clamp=0.5), (x, w13, w2), dy)
    assert all(torch.equal(g, p + q) for g, p, q in zip(got, one, two))


def test_backward_twice_and_changes_noticed():
    api = _api()
    x, w13, w2, dy = _block(3, 9, 2, 64, 32, grad=True)
    ends = _ends([4, 5])
    y = api.grouped_feed_forward(x, w13, w2, ends)
    first = torch.autograd.grad(y, (x, w13, w2), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, w13, w2), dy)))
    y = api.grouped_projection(x, w13, ends)
    (dx,) = torch.autograd.grad(y, (x,), torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    for change in (x, w13, ends):
        y, z = api.grouped_feed_forward(x, w13, w2, ends), api.grouped_projection(x, w13, ends)
        with torch.no_grad():
            change.add_(0)
        for out in (y, z):
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()




@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_no_numbers_stay_with_their_expert(bad):
    """In rows of another expert, in rows of none, in another expert's weights: the neighbours' last tiles and stages end with them."""
    api = _api()
    counts = [33, 40, 0, 70, 65, 12]
    ends, spare = _ends(counts), 21
    rows = sum(counts) + spare
    hidden, inter = 72, 40                                  # not whole stages: the next expert's weights follow
    x, w13, w2, dy = _block(11, rows, 6, hidden, inter)
    spoilt = (1, 4)
    good = torch.ones(rows, dtype=torch.bool, device=DEV)
    for e, a, b in G.pieces(ends, rows):
        if e in spoilt:
            good[a:b] = False
    good[sum(counts):] = False
    x2, dy2, w13b, w2b = x.clone(), dy.clone(), w13.clone(), w2.clone()
    x2[~good], dy2[~good] = bad, bad
    for e in (*spoilt, 2):
        w13b[e], w2b[e] = bad, bad
    clean = torch.tensor([e not in spoilt for e in range(6)], device=DEV)
    leaves = [t.requires_grad_(True) for t in (x2, w13b, w2b)]
    y = api.grouped_feed_forward(*leaves, ends, activation_clamp=2.0)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy2))
    want = G.Block(x, w13, w2, ends, 2.0, dy)
    for name, g, keep in zip(("y", "dx", "dw13", "dw2"), got, (good, good, clean, clean)):
        R.check(name, g[keep], getattr(want, name)[keep], want.off[name][keep])
    assert not got[0][sum(counts):].any() and not got[1][sum(counts):].any() and not got[2][2].any() and not got[3][2].any()
    y = api.grouped_projection(leaves[0], leaves[1], ends)
    up = torch.cat((dy2, dy2[:, :8]), 1)
    got = (y.detach(), *torch.autograd.grad(y, leaves[:2], up))
    one = G.Projection(x, w13, ends, torch.cat((dy, dy[:, :8]), 1))
    for name, g, keep in zip(("y", "dx", "dw"), got, (good, good, clean)):
        R.check(name, g[keep], getattr(one, name)[keep], one.off[name][keep])
    # few rows: the other kernel
    few = _ends([2, 3, 0, 1])
    y = api.grouped_projection(x2.detach()[:9], w13b.detach()[[0, 1, 2, 3]].contiguous(), few)
    xs = x.clone()[:9]
    R.check("few", y[[0, 1, 5]], G.Projection(xs, w13[:4], few).y[[0, 1, 5]], G.Projection(xs, w13[:4], few).off["y"][[0, 1, 5]])
    assert not y[6:].any()


def test_fp8_values_that_are_no_numbers_stay_in_their_row():
    """A scale that is no number, a value that is none: their row, or their channels, alone."""
    api = _api()
    for rows in (5, 40, 300):
        x, sx, w, sw = _case(rows, 1, 260, 400, 1)
        want, off = G.fp8_product(x, sx, w, sw, None, torch.float32)
        bad = sx.clone()
        bad[rows // 2, 3] = math.nan
        xb = x.clone()
        xb.view(torch.uint8)[0, 7] = 0x7F                                     # NaN in E4M3
        got = api.fp8_projection(xb, bad, w[0], sw[0], out_dtype=torch.float32)
        keep = torch.ones(rows, dtype=torch.bool, device=DEV)
        keep[0] = keep[rows // 2] = False
        assert torch.isnan(got[~keep]).all()
        R.check("others", got[keep], want[keep], off[keep])
        wrong = sw.clone()
        wrong[0, 1, 0] = math.inf                                             # channels 128 to 255
        got = api.fp8_projection(x, sx, w[0], wrong[0], out_dtype=torch.float32)
        assert not torch.isfinite(got[:, 128:256]).any()
        keep = torch.tensor([c < 128 or c >= 256 for c in range(260)], device=DEV)
        R.check("other channels", got[:, keep], want[:, keep], off[:, keep])


def test_fp8_strides_and_shapes():
    api = _api()
    x, sx, w, sw = _case(60, 1, 72, 144, 1)
    want, off = G.fp8_product(x, sx, w, sw, None, torch.bfloat16)
    wide = torch.zeros((60, 320), dtype=torch.uint8, device=DEV)
    wide[:, 16:160] = x.view(torch.uint8)
    odd = torch.zeros((60, 320), dtype=torch.uint8, device=DEV)
    odd[:, 3:147] = x.view(torch.uint8)
    turned = sx.T.contiguous().T
    for xv, sv in ((x, sx), (wide.view(E4M3)[:, 16:160], turned), (odd.view(E4M3)[:, 3:147], sx), (x.view(torch.uint8).T.contiguous().T.view(E4M3), turned)):
        R.check("y", api.fp8_projection(xv, sv, w[0], sw[0].T.contiguous().T), want, off)
    y = api.fp8_projection(x.view(3, 4, 5, 144), sx.view(3, 4, 5, 2), w[0], sw[0])
    assert y.shape == (3, 4, 5, 72)
    R.check("y", y.view(60, 72), want, off)
    y = api.fp8_projection(x[7], sx[7], w[0], sw[0])
    assert y.shape == (72,)
    R.check("y", y[None], want[7:8], off[7:8])
    assert api.fp8_projection(x[:0], sx[:0], w[0], sw[0]).shape == (0, 72)
    assert api.fp8_gated_projection(x[:0], sx[:0], w[0][:64], sw[0].expand(2, 2).contiguous()).shape == (0, 32)
    assert api.fp8_projection(x[:0], sx[:0], w, sw, ends=_ends([0])).shape == (0, 72)
    R.check("steps", api.fp8_projection(x[::3], sx[::3], w[0], sw[0]), want[::3], off[::3])


@pytest.mark.parametrize("channels", [1, 2, 3, 129, 255, 1000])
@pytest.mark.parametrize("rows", [1, 30, 260])
def test_fp8_rows_that_start_anywhere(rows, channels):
    api = _api()
    x, sx, w, sw = _case(rows, 1, channels, 272, 1)
    for dtype in (torch.bfloat16, torch.float32):
        want, off = G.fp8_product(x, sx, w, sw, None, dtype)
        R.check("y", api.fp8_projection(x, sx, w[0], sw[0], out_dtype=dtype), want, off)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [257, 256 + 64, 256 + 65, 777, 1030])
def test_fp8_rows_beyond_the_last_tile(rows, gated):
    """5120 wide: a few rows beyond a tile of 256 go by themselves where that saves a turn, and the results are the same rows."""
    api = _api()
    channels = 4608 if gated else 5003
    x, sx, w, sw = _case(rows, 1, channels, 5120, 1 + gated)
    want, off = G.fp8_product(x, sx, w, sw, None, torch.float32, gated, 3.0 if gated else None)
    got = api.fp8_gated_projection(x, sx, w[0], sw[0], activation_clamp=3.0, out_dtype=torch.float32) if gated else api.fp8_projection(
        x, sx, w[0], sw[0], out_dtype=torch.float32)
    R.check("y", got, want, off)


# ---------------------------------------------------------------------------------------------------------------------
# quantiser
# ---------------------------------------------------------------------------------------------------------------------
def test_quantiser_borders():
    """Every multiple of a half step up to the largest value, for scales of which quotients are exact or nearly so; the smallest numbers of the types;
    groups of zeros; infinities and NaN."""
    api = _api()
    for dtype in (torch.bfloat16, torch.float16):
        rows = []
        codes = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
        borders = (codes[1:] + codes[:-1]) / 2
        for scale in (1.0, 2.0 ** -5, 3.0, 7.0 * 2 ** -6, 2.0 ** -12, 5.0 * 2 ** -3, 1.4142):
            some = torch.cat((borders, codes)) * scale
            some = torch.cat((some, -some)).float().to(dtype)
            for part in some.split(127):
                rows.append(torch.cat((part, part.new_full((1,), 448 * scale), part.new_zeros(127 - part.numel()))))
        tiny = torch.arange(128).double() * (2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -24)
        rows += [tiny.to(dtype), (tiny / 8).to(dtype), torch.zeros(128, dtype=dtype), torch.full((128,), torch.finfo(dtype).max, dtype=dtype),
                 (torch.arange(128).double() * 2.0 ** -66).to(dtype)]
        for bad in (math.inf, -math.inf, math.nan):
            r = torch.ones(128, dtype=dtype)
            r[17] = bad
            rows.append(r)
        x = torch.stack(rows).to(DEV)
        x = torch.cat((x, -x, x.flip(1)))
        for shape in (x.shape, (x.shape[0] // 3, 384)):
            q, s = api.prepare_fp8_inputs(x.view(shape))
            want_q, want_s = G.quantize(x.view(shape))
            assert torch.equal(s.view(torch.int32), want_s.view(torch.int32)) or torch.equal(torch.nan_to_num(s, -1.0), torch.nan_to_num(want_s, -1.0))
            assert torch.equal(q.double(), want_q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantiser_of_many_values(dtype):
    """A million of them at random, of which some are next to a border: every one is the nearest."""
    api = _api()
    x = _rand(5, 2000, 640, dtype=torch.float32).to(dtype)
    q, s = api.prepare_fp8_inputs(x)
    want_q, want_s = G.quantize(x)
    assert torch.equal(s, want_s) and torch.equal(q.double(), want_q)


def test_quantiser_strides_shapes_and_out():
    api = _api()
    x = _rand(3, 60, 320)
    for view in (x, x.view(3, 4, 5, 320), x[7], x[::2], x[:, 3:203], x[:, 8:264], x.T.contiguous().T, x[4:5].expand(6, 320), x[:0], x[:, :1],
                 torch.cat((x.new_zeros(1), x.flatten()))[1:].view(60, 320)):
        q, s = api.prepare_fp8_inputs(view)
        groups = -(-view.shape[-1] // 128)
        assert q.shape == view.shape and s.shape == (*view.shape[:-1], groups)
        want_q, want_s = G.quantize(view.contiguous())
        assert torch.equal(s, want_s) and torch.equal(q.double(), want_q)
        out = (torch.empty_like(q), torch.empty_like(s))
        back = api.prepare_fp8_inputs(view, out)
        assert back[0] is out[0] and back[1] is out[1] and torch.equal(out[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(out[1], s)
    q, s = api.prepare_fp8_inputs(x)
    for out in ((q, s[:, :2]), (q.view(torch.uint8), s), (q[:5], s), (q, s.double()), (q.T, s)):
        with pytest.raises(ValueError):
            api.prepare_fp8_inputs(x, out)
    for bad in (x.float(), x[:, :0], x.to(torch.int8)):
        with pytest.raises(ValueError):
            api.prepare_fp8_inputs(bad)
    with pytest.raises(NotImplementedError):
        api.prepare_fp8_inputs(x.clone().requires_grad_(True))


# ---------------------------------------------------------------------------------------------------------------------
# ends
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("values", [[5, 3, 9], [-1, 4, 9], [2, 4, 11], [2**31 - 1, 2**31 - 1, 2**31 - 1], [-2**31, 0, 5], [0, -3, 9]])
@pytest.mark.parametrize("rows", [10, 400])
def test_ends_out_of_order(values, rows):
    """No row is an expert's then: zeros, a report, and nothing that lasts."""
    api = _api()
    if rows == 400:
        values = [v * 40 if abs(v) < 20 else v for v in values]
    bad, good = torch.tensor(values, dtype=torch.int32, device=DEV), _ends([rows // 2, 0, rows // 2])
    x, w13, w2, dy = _block(4, rows, 3, 64, 32, grad=True)
    q, sx, w, sw = _case(rows, 3, 64, 64, 2)
    api.read_dense_status()
    interval = api.get_kernel_options().status_poll_interval
    try:
        api.set_kernel_options(status_poll_interval=0)
        y = api.grouped_feed_forward(x, w13, w2, bad)
        z = api.grouped_projection(x, w13, bad)
        results = [y, z, *torch.autograd.grad(y, (x, w13, w2), dy), *torch.autograd.grad(z, (x, w13), torch.ones_like(z)),
                   api.fp8_projection(q, sx, w, sw[:, :1], ends=bad), api.fp8_gated_projection(q, sx, w, sw, ends=bad, out_dtype=torch.float32)]
        assert not any(r.any() for r in results)
        with pytest.raises(AssertionError, match="ends"):
            api.read_dense_status()
        api.read_dense_status()
    finally:
        api.set_kernel_options(status_poll_interval=interval)
    y = api.grouped_feed_forward(x, w13, w2, good)
    _check_block(x, w13, w2, good, None, dy, (y, *torch.autograd.grad(y, (x, w13, w2), dy)))
    api.read_dense_status()


def test_later_calls_report_ends_out_of_order():
    api = _api()
    x, w13, _, _ = _block(4, 10, 2, 64, 32)
    api.read_dense_status()
    bad, good = torch.tensor([6, 4], dtype=torch.int32, device=DEV), _ends([6, 4])
    interval = api.get_kernel_options().status_poll_interval
    try:
        api.set_kernel_options(status_poll_interval=1)
        raised = 0
        api.grouped_projection(x, w13, bad)
        for _ in range(6):
            torch.cuda.synchronize()
            try:
                api.grouped_projection(x, w13, good)
            except AssertionError as e:
                raised += 1
                assert "ends" in str(e)
        assert raised == 1
    finally:
        api.set_kernel_options(status_poll_interval=interval)
    api.read_dense_status()


# ---------------------------------------------------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------------------------------------------------
def test_no_rows():
    api = _api()
    x, w13, w2, dy = _block(4, 0, 3, 64, 32, grad=True)
    ends = _ends([0, 0, 0])
    y = api.grouped_feed_forward(x, w13, w2, ends)
    z = api.grouped_projection(x, w13, ends)
    assert y.shape == (0, 64) and z.shape == (0, 64)
    for g, like in zip((*torch.autograd.grad(y, (x, w13, w2), dy), *torch.autograd.grad(z, (x, w13), z.detach())), (x, w13, w2, x, w13)):
        assert g.shape == like.shape and not g.any()


@pytest.mark.parametrize("experts", [257, 1000, 1024])
def test_many_experts(experts):
    """Most with a row or none, one with many."""
    api = _api()
    counts = [(e * 7 + 3) % 4 // 2 for e in range(experts)]
    counts[experts // 2], counts[-1] = 300, 5
    ends, rows = _ends(counts), sum(counts) + 3
    x, w, dy = _rand(1, rows, 64), _rand(2, experts, 24, 64, std=0.1), _rand(3, rows, 24)
    x.requires_grad_(True), w.requires_grad_(True)
    want = G.Projection(x, w, ends, dy)
    y = api.grouped_projection(x, w, ends)
    for name, g in zip(("y", "dx", "dw"), (y, *torch.autograd.grad(y, (x, w), dy))):
        R.check(name, g.detach(), getattr(want, name), want.off[name])
    q, sx, w8, sw = _case(rows, experts, 24, 64, 1)
    value, off = G.fp8_product(q, sx, w8, sw, ends, torch.bfloat16)
    R.check("fp8", api.fp8_projection(q, sx, w8, sw, ends=ends), value, off)


@pytest.mark.parametrize("counts", [[64], [65], [16] * 4, [64] * 7 + [1], [64] * 8, [65] * 8, [1] * 32 + [500], [40] * 5 + [8], [41] * 5 + [8], [1024] + [0] * 20, [2] * 90])
def test_either_side_of_the_lines_between_the_kernels(counts):
    """Few rows and pairs, 16 bits and 8, tiles that do and do not fit at once, K split and not."""
    api = _api()
    ends, rows = _ends(counts), sum(counts)
    for width, channels in ((1032, 136), (264, 5128)):
        x, w = _rand(1, rows, width), _rand(2, len(counts), channels, width, std=0.1)
        want = G.Projection(x, w, ends)
        R.check("y", api.grouped_projection(x, w, ends), want.y, want.off["y"])
    x, w13, w2, _ = _block(5, rows, len(counts), 520, 72)
    want = G.Block(x, w13, w2, ends, 1.0)
    R.check("block", api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=1.0), want.y, want.off["y"])
    for gated in (False, True):
        q, sx, w8, sw = _case(rows, len(counts), 272, 1168, 1 + gated)
        value, off = G.fp8_product(q, sx, w8, sw, ends, torch.bfloat16, gated)
        got = (api.fp8_gated_projection if gated else api.fp8_projection)(q, sx, w8, sw, ends=ends)
        R.check("fp8", got, value, off)
    api.read_dense_status()


def test_more_tiles_than_pairs():
    api = _api()
    counts = [700, 0, 1300, 255, 257, 64]
    ends, rows = _ends(counts), sum(counts) + 5
    x, w13, w2, dy = _block(8, rows, 6, 1032, 776, grad=True)
    y = api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=4.0)
    _check_block(x, w13, w2, ends, 4.0, dy, (y, *torch.autograd.grad(y, (x, w13, w2), dy)))
    for gated in (False, True):
        q, sx, w8, sw = _case(rows, 6, 3000 - 56 * gated, 400, 1 + gated)
        value, off = G.fp8_product(q, sx, w8, sw, ends, torch.float16, gated, 1.0 if gated else None)
        got = api.fp8_gated_projection(q, sx, w8, sw, ends=ends, activation_clamp=1.0, out_dtype=torch.float16) if gated else api.fp8_projection(
            q, sx, w8, sw, ends=ends, out_dtype=torch.float16)
        R.check("fp8", got, value, off)


def test_outputs_past_32_bit_offsets():
    """More than 2^31 values: the last rows, by few and by many."""
    api = _api()
    rows, width, channels = 70000, 64, 32768
    x, w = _rand(1, rows, width), _rand(2, 2, channels, width, std=0.1)
    ends = _ends([rows - 40, 40])
    y = api.grouped_projection(x, w, ends)
    want = G.Projection(x[-60:], w, _ends([20, 40]))
    R.check("y", y[-60:], want.y, want.off["y"])
    del y, w
    q, sx, w8, sw = _case(rows, 1, channels, width, 1)
    y = api.fp8_projection(q, sx, w8[0], sw[0])
    value, off = G.fp8_product(q[-30:], sx[-30:], w8, sw, None, torch.bfloat16)
    R.check("fp8", y[-30:], value, off)


def test_c_interface_leaves_what_is_around_the_output():
    """Rows in front of and behind the output's, and with 8 bits and no ends nothing but the rows."""
    from vllm_plugin_b200.backend import _native as N, dense as D
    api = _api()
    x, w13, _, _ = _block(4, 50, 2, 64, 32)
    api.grouped_projection(x, w13, _ends([20, 20]))
    lib, status, stream = N.load(), D._on_device(0).status_ptr, torch.cuda.current_stream().cuda_stream
    for rows in (50, 700):
        x = _rand(1, rows, 64)
        ends = _ends([rows // 2, rows // 3])
        room = torch.full((rows + 16, 64), 7.0, dtype=x.dtype, device=DEV)
        a = N.MmoeGroupedProduct(0, rows, 2, 64, 64, 0, 64, x.data_ptr(), w13.data_ptr(), ends.data_ptr(), room[8:].data_ptr(), status)
        N.check(lib.mmoe_grouped_projection(ctypes.byref(a), stream))
        want = G.Projection(x, w13, ends)
        R.check("y", room[8:-8], want.y, want.off["y"])
        assert (room[:8] == 7).all() and (room[-8:] == 7).all()
        q, sx, w8, sw = _case(rows, 1, 67, 80, 1)
        room = torch.full((rows * 67 + 512,), 7.0, device=DEV)
        b = N.MmoeFp8Product(rows, 1, 80, 67, 3, math.inf, 0, 0, 80, q.data_ptr(), sx.data_ptr(), w8.data_ptr(), sw.data_ptr(), None, room[256:].data_ptr(), status)
        N.check(lib.mmoe_fp8_projection(ctypes.byref(b), stream))
        value, off = G.fp8_product(q, sx, w8, sw, None, torch.float32)
        R.check("fp8", room[256:-256].view(rows, 67), value, off)
        assert (room[:256] == 7).all() and (room[-256:] == 7).all()


# ---------------------------------------------------------------------------------------------------------------------
# gradients against differences, repeats, streams, graphs
# ---------------------------------------------------------------------------------------------------------------------
def test_gradients_against_differences():
    """Central differences of the operators' own outputs along their gradients, in FP16 with a step of 2^-3.  They are off by the third-order term
    (below 1 % here) and by the rounding of the outputs, 2^-11 of each value's share of the sum."""
    api = _api()
    ends = _ends([9, 0, 15])
    x, w13, w2, dy = _block(21, 26, 3, 64, 48, torch.float16, True)
    up = _rand(22, 26, 96, dtype=torch.float16)
    for run, args, dy in ((lambda *a: api.grouped_feed_forward(*a, ends), (x, w13, w2), dy), (lambda *a: api.grouped_projection(*a, ends), (x, w13), up)):
        y = run(*args)
        grads = torch.autograd.grad(y, args, dy)
        noise = 2.0 ** -11 * float((y.detach().double() * dy.double()).norm())
        for i, g in enumerate(grads):
            d = g.double() / g.double().norm()
            values = []
            for sign in (1, -1):
                moved = [t.detach() for t in args]
                moved[i] = (moved[i].double() + sign * 2.0 ** -3 * d).half()
                values.append((moved[i].double(), float((run(*moved).double() * dy.double()).sum())))
            got, want = values[0][1] - values[1][1], float(((values[0][0] - values[1][0]) * g.double()).sum())
            assert abs(got - want) <= 0.01 * abs(want) + 8 * noise, (i, got, want, noise)


def test_calls_repeat_bit_for_bit():
    api = _api()
    for counts in ([1, 0, 2], [40, 3, 90], [500, 300, 7]):
        rows, ends = sum(counts), _ends(counts)
        x, w13, w2, dy = _block(rows, rows, 3, 1024, 520, grad=True)
        q, sx, w8, sw = _case(rows, 3, 528, 1040, 2)
        runs = []
        for _ in range(3):
            y = api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=1.0)
            runs.append((y.detach(), *torch.autograd.grad(y, (x, w13, w2), dy), api.fp8_gated_projection(q, sx, w8, sw, ends=ends),
                         api.fp8_projection(q, sx, w8, sw[:, :5].contiguous(), ends=ends)))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_two_streams_at_once():
    api = _api()
    work = []
    for i, counts in enumerate(([1, 2], [200, 100], [30, 34], [600, 3])):
        rows, ends = sum(counts), _ends(counts)
        x, w13, w2, dy = _block(i, rows, 2, 512, 264, grad=True)
        q, sx, w8, sw = _case(rows, 2, 264, 512, 1)

        def calls(x=x, w13=w13, w2=w2, dy=dy, ends=ends, q=q, sx=sx, w8=w8, sw=sw):
            y = api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=1.5)
            return (y.detach(), *torch.autograd.grad(y, (x, w13, w2), dy), api.fp8_projection(q, sx, w8, sw, ends=ends), *api.prepare_fp8_inputs(x.detach()))
        work.append(calls)
    want = [c() for c in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(6):
        for i, c in enumerate(work):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, c()))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(r, want[i]))
    api.read_dense_status()


def test_a_captured_call_goes_by_the_ends_at_its_replay():
    api = _api()
    rows = 600
    x, w13, w2, _ = _block(3, rows, 4, 256, 136)
    q, sx, w8, sw = _case(rows, 4, 144, 256, 2)
    ends = _ends([0, 0, 0, 0])

    def calls():
        return (api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=2.0), api.grouped_projection(x, w13, ends), api.fp8_gated_projection(q, sx, w8, sw, ends=ends),
                api.fp8_projection(q, sx, w8, sw, ends=ends))

    calls()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls()
        graphs.append((graph, out))
    for counts in ([600, 0, 0, 0], [1, 2, 3, 4], [0, 0, 0, 0], [150, 151, 149, 150], [0, 300, 0, 299]):
        ends.copy_(_ends(counts))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        eager = calls()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        want = G.Block(x, w13, w2, ends, 2.0)
        R.check("y", eager[0], want.y, want.off["y"])
    api.read_dense_status()


def test_a_training_step_in_a_graph():
    api = _api()
    x, w13, w2, dy = _block(7, 90, 3, 128, 64, grad=True)
    ends = _ends([30, 30, 30])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        api.grouped_feed_forward(x, w13, w2, ends).backward(dy)
        for t in (x, w13, w2):
            t.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = api.grouped_feed_forward(x, w13, w2, ends)
        y.backward(dy)
    captured = [t.grad for t in (x, w13, w2)]
    for counts in ([1, 0, 80], [89, 1, 0]):
        with torch.no_grad():
            x.copy_(_rand(sum(counts), 90, 128))
            dy.copy_(_rand(sum(counts) + 1, 90, 128))
        ends.copy_(_ends(counts))
        graph.replay()
        torch.cuda.synchronize()
        _check_block(x, w13, w2, ends, None, dy, (y, *captured))


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """A graph of any of the operators that train stands against a capture of any other with the same leaves."""
    api = _api()
    x, w13, w2, dy = _block(3, 5, 2, 64, 32, grad=True)
    ends = _ends([2, 3])
    for eager in (lambda: api.grouped_feed_forward(x, w13, w2, ends), lambda: api.grouped_projection(x, w13, ends), lambda: api.gated_feed_forward(x, w13[0], w2[0])):
        eager()                                                 # (first calls, outside the capture)
        alive = eager()
        refused = 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for run in (lambda: api.grouped_feed_forward(x, w13, w2, ends), lambda: api.grouped_projection(x, w13, ends)):
                try:
                    run()
                except RuntimeError:
                    refused += 1
            with torch.no_grad():
                y = api.grouped_projection(x, w13, ends)
        assert refused == 2
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, api.grouped_projection(x, w13, ends))
        alive.sum().backward()
        del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        api.grouped_feed_forward(x, w13, w2, ends)


def test_first_calls():
    """In inference mode, then training; inside a capture (the quantiser alone); from another thread."""
    program = """
import threading
import torch
from vllm_plugin_b200 import api
x, w13, w2 = (torch.randn(s, device="cuda").bfloat16() for s in ((5, 64), (2, 64, 64), (2, 64, 32)))
ends = torch.tensor([2, 5], dtype=torch.int32, device="cuda")
refused = 0
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s = api.prepare_fp8_inputs(x)
    try:
        api.grouped_projection(x, w13, ends)
    except RuntimeError:
        refused += 1
graph.replay()
torch.cuda.synchronize()
again = api.prepare_fp8_inputs(x)
assert refused == 1 and torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(s, again[1])
with torch.inference_mode():
    want = api.grouped_feed_forward(x, w13, w2, ends).clone()
got = []
def other():
    for _ in range(40):
        got.append(api.grouped_feed_forward(x, w13, w2, ends))
    torch.cuda.synchronize()
t = threading.Thread(target=other)
t.start()
t.join()
assert len(got) == 40 and all(torch.equal(y, want) for y in got)
w13.requires_grad_(True)
for _ in range(80):
    api.grouped_feed_forward(x, w13, w2, ends).sum().backward()
    torch.cuda.synchronize()
api.read_dense_status()
print("ok")
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr


def test_refusals():
    api = _api()
    x, w13, w2, _ = _block(3, 5, 2, 64, 32)
    ends = _ends([2, 3])
    q, sx, w, pairs = _case(5, 2, 64, 64, 2)
    sw = pairs[:, :1].contiguous()
    api.fp8_projection(q, sx, w, sw, ends=ends)
    api.fp8_gated_projection(q, sx, w, pairs, ends=ends)
    for bad in (ends.cpu(), ends.long(), ends[:1]):
        for call in (lambda: api.grouped_projection(x, w13, bad), lambda: api.grouped_feed_forward(x, w13, w2, bad), lambda: api.fp8_projection(q, sx, w, sw, ends=bad)):
            with pytest.raises(AssertionError, match="ends"):
                call()
    for call in (lambda: api.grouped_projection(x.float(), w13, ends), lambda: api.grouped_projection(x[None], w13, ends), lambda: api.grouped_projection(x, w13.half(), ends),
                 lambda: api.grouped_projection(x, w13.cpu(), ends), lambda: api.grouped_feed_forward(x, w13, w13, ends),
                 lambda: api.fp8_projection(q, sx[:, :0], w, sw, ends=ends), lambda: api.fp8_projection(q, sx.double(), w, sw, ends=ends),
                 lambda: api.fp8_projection(q, sx, w, pairs, ends=ends), lambda: api.fp8_gated_projection(q, sx, w, sw, ends=ends), lambda: api.fp8_projection(q, sx, w, sw), lambda: api.fp8_projection(q[None], sx[None], w, sw, ends=ends),
                 lambda: api.fp8_projection(x, sx, w, sw, ends=ends), lambda: api.fp8_projection(q, sx, w13, sw, ends=ends),
                 lambda: api.fp8_projection(q, sx, w, sw, ends=ends, out_dtype=torch.float64), lambda: api.fp8_projection(q, sx, w, sw, ends=ends, out_dtype=E4M3),
                 lambda: api.fp8_gated_projection(q, sx, w[:, :24].contiguous(), pairs, ends=ends), lambda: api.fp8_gated_projection(q, sx, w, pairs, ends=ends, activation_clamp=-1.0),
                 lambda: api.fp8_projection(q[:, :40], sx, w[:, :, :40].contiguous(), sw, ends=ends)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: api.fp8_projection(q, sx.clone().requires_grad_(True), w, sw, ends=ends), lambda: api.fp8_projection(q, sx, w, sw.clone().requires_grad_(True), ends=ends)):
        with pytest.raises(NotImplementedError):
            call()
    with torch.no_grad():
        api.fp8_projection(q, sx.clone().requires_grad_(True), w, sw, ends=ends)


def test_tangents_and_traces_are_refused():
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    api = _api()
    x, w13, w2, _ = _block(3, 5, 2, 64, 32)
    ends = _ends([2, 3])
    q, sx, w, sw = _case(5, 2, 64, 64, 1)
    with fwd.dual_level():
        for call in (lambda d: api.grouped_feed_forward(d, w13, w2, ends), lambda d: api.grouped_projection(d, w13, ends), lambda d: api.prepare_fp8_inputs(d)):
            with pytest.raises(NotImplementedError):
                call(fwd.make_dual(x, torch.ones_like(x)))
        with pytest.raises(NotImplementedError):
            api.fp8_projection(q, fwd.make_dual(sx, torch.ones_like(sx)), w, sw, ends=ends)
    for run, args in ((lambda a, b, c, d: api.grouped_feed_forward(a, b, c, d), (x, w13, w2, ends)), (lambda a, b, c: api.grouped_projection(a, b, c), (x, w13, ends)),
                      (lambda a: api.prepare_fp8_inputs(a), (x,)),
                      (lambda a, b, c, d, e: api.fp8_projection(a, b, c, d, ends=e), (q, sx, w, sw, ends))):
        run(*args)
        with pytest.raises(NotImplementedError):
            make_fx(run)(*args)
        with pytest.raises(NotImplementedError):
            torch.jit.trace(run, args, check_trace=False)


# ---------------------------------------------------------------------------------------------------------------------
# runs of them together
# ---------------------------------------------------------------------------------------------------------------------
def _route(logits, top):
    """Weights and experts of each token, and its routes in the order of the experts."""
    weights, experts = torch.softmax(logits.float(), -1).topk(top, -1)
    order = torch.argsort(experts.flatten(), stable=True)
    counts = torch.zeros(logits.shape[1], dtype=torch.int64, device=logits.device).scatter_add_(0, experts.flatten(), torch.ones_like(experts.flatten()))
    return weights, order, counts.cumsum(0).to(torch.int32)


@pytest.mark.parametrize("tokens", [1, 37, 400])
def test_a_layer_of_experts_that_is_trained(tokens):
    """Routing, the experts' block over the sorted rows, the weighted sum of a token's routes, and the gradients through all of it, against the same layer
    with each expert's block computed in 64 bits.  The bounds are those of the block; a token's sum has two of its rows, whose weights are below one."""
    api = _api()
    top, experts, hidden, inter = 2, 6, 128, 72
    x, w13, w2, _ = _block(5, tokens, experts, hidden, inter)
    logits = _rand(77, tokens, experts, dtype=torch.float32)
    weights, order, ends = _route(logits, top)
    dy = _rand(78, tokens, hidden, dtype=torch.float32)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w13, w2)]
    rows = leaves[0][order // top]
    out = api.grouped_feed_forward(rows, leaves[1], leaves[2], ends, activation_clamp=3.0)
    y = torch.zeros(tokens, hidden, device=DEV).index_add_(0, order // top, out.float() * weights.flatten()[order, None])
    y.backward(dy)
    up = (dy[order // top] * weights.flatten()[order, None]).to(x.dtype)
    want = G.Block(rows.detach(), w13, w2, ends, 3.0, up)
    total, off = torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV), torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV)
    w = weights.double().flatten()[order, None]
    total.index_add_(0, order // top, want.y * w)
    off.index_add_(0, order // top, (want.off["y"] + 2.0 ** -22 * want.y.abs()) * w)
    R.check("y", y.detach(), total, off + 2.0 ** -22 * total.abs())
    R.check("dw13", leaves[1].grad, want.dw13, want.off["dw13"])
    R.check("dw2", leaves[2].grad, want.dw2, want.off["dw2"])
    dx, dx_off = torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV), torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV)
    dx.index_add_(0, order // top, want.dx)
    # two values of 16 bits added in 16 bits
    dx_off.index_add_(0, order // top, want.off["dx"] + 2.0 ** -8 * want.dx.abs())
    R.check("dx", leaves[0].grad, dx, 1.01 * dx_off)


@pytest.mark.parametrize("tokens", [3, 300])
def test_experts_in_8_bits_from_end_to_end(tokens):
    """Quantiser, gated product, quantiser, second product, over sorted rows and in one graph; a shared expert in the same form beside them.  Each step's inputs
    are those that the step before left, so that each is held to its own bound."""
    api = _api()
    top, experts, hidden, inter = 2, 5, 256, 144
    _, order, ends = _route(_rand(7, tokens, experts, dtype=torch.float32), top)
    x = _rand(8, tokens, hidden)
    _, _, w13, s13 = _case(1, experts, 2 * inter, hidden, 2)
    _, _, w2, s2 = _case(1, experts, hidden, inter, 1)
    s13, s2 = s13 * 0.01, s2 * 0.01

    def step():
        q, s = api.prepare_fp8_inputs(x)
        rows, scales = q.view(torch.uint8)[order // top].view(E4M3), s[order // top]
        h = api.fp8_gated_projection(rows, scales, w13, s13, ends=ends, activation_clamp=5.0)
        hq, hs = api.prepare_fp8_inputs(h)
        y = api.fp8_projection(hq, hs, w2, s2, ends=ends, out_dtype=torch.float32)
        shared = api.fp8_gated_projection(q, s, w13[0], s13[0], activation_clamp=5.0)
        return rows, scales, h, hq, hs, y, shared, q, s

    eager = step()
    rows, scales, h, hq, hs, y, shared, q, s = eager
    want_q, want_s = G.quantize(x)
    assert torch.equal(q.double(), want_q) and torch.equal(s, want_s)
    R.check("h", h, *G.fp8_product(rows, scales, w13, s13, ends, torch.bfloat16, True, 5.0))
    want_q, want_s = G.quantize(h)
    assert torch.equal(hq.double(), want_q) and torch.equal(hs, want_s)
    R.check("y", y, *G.fp8_product(hq, hs, w2, s2, ends, torch.float32))
    R.check("shared", shared, *G.fp8_product(q, s, w13[:1], s13[:1], None, torch.bfloat16, True, 5.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, eager))


def test_beside_the_layer():
    """A shared expert with block scales beside the MXFP8 x MXFP4 experts: its output as the layer's residual."""
    import helpers as H
    from oracle import mmoe_oracle as O
    api = _api()
    layer = H.make_layer(512, 256, 8, 2, False, seed=0)
    m = 33
    hid = O.make_hidden(m, layer.hidden, 1)
    ids, w = O.make_routing(m, layer.num_experts, layer.num_topk, 2)
    want, buf = H.run_layer(layer, hid, ids, w)
    weights = H.kernel_weights(layer, torch.device(DEV))
    x, ids, w = hid.to(DEV), ids.to(DEV), w.to(DEV)
    _, _, w13, s13 = _case(1, 1, 512, 512, 2)
    _, _, w2, s2 = _case(1, 1, 512, 256, 1)
    s13, s2 = s13 * 0.01, s2 * 0.01
    y = torch.empty_like(x)
    api.stage_inputs_for_mega_moe(buf, x, ids, w)
    h = api.fp8_gated_projection(*api.prepare_fp8_inputs(x), w13[0], s13[0], activation_clamp=10.0)
    shared = api.fp8_projection(*api.prepare_fp8_inputs(h), w2[0], s2[0])
    api.fp8_fp4_mega_moe(y, weights[0], weights[1], buf, activation_clamp=10.0, residual=shared)
    assert torch.equal(y, want + shared)
