"""Dense feed-forward operators on the GPU against plain 64-bit forms (``dense_reference.py``)."""

import ctypes
import math

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _api():
    from vllm_plugin_b200 import api
    return api


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _block_inputs(m, hidden, inter, dtype, seed=0, grad=False):
    gen = _gen(seed)
    # g and u of unit size whatever the width
    x = _randn(gen, m, hidden, dtype=dtype)
    w13 = _randn(gen, 2 * inter, hidden, dtype=dtype, std=hidden ** -0.5)
    w2 = _randn(gen, hidden, inter, dtype=dtype, std=inter ** -0.5)
    dy = _randn(gen, m, hidden, dtype=dtype)
    for t in (x, w13, w2):
        t.requires_grad_(grad)
    return x, w13, w2, dy


def _int8(gen, rows, k):
    q = torch.randint(-127, 128, (rows, k), generator=gen, device=DEV, dtype=torch.int32).to(torch.int8)
    return q, torch.rand(rows, generator=gen, device=DEV) * 0.02 + 1e-3


# ---------------------------------------------------------------------------------------------------------------------
# quantiser
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 5120), (3, 7), (2, 8), (5, 100), (7, 2304), (33, 264), (130, 4099), (4, 20001), (3, 32768)])
def test_quantiser_is_exact(m, k, dtype):
    gen = _gen(m * 7 + k)
    x = _randn(gen, m, k, dtype=dtype)
    x[:, :: 97] *= 30
    q, s = _api().prepare_int8_inputs(x)
    want_q, want_s = R.quantize(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (m,)
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("m,k", [(511, 264), (512, 8), (513, 264), (1001, 1280), (600, 1288), (520, 5120), (700, 24), (530, 33), (516, 21000)])
def test_quantiser_of_many_tokens(m, k):
    """From 512 tokens on fewer threads take a row, down to a warp of a block of eight rows; the last block has rows that are none."""
    gen = _gen(m + k)
    x = _randn(gen, m, k, dtype=torch.bfloat16)
    x[m // 3, 1 % k] = math.inf
    x[m // 2] = 0
    room = torch.full((m + 9, k), 55, dtype=torch.int8, device=DEV), torch.full((m + 9,), 55.0, device=DEV)
    _api().prepare_int8_inputs(x, out=(room[0][:m], room[1][:m]))
    want_q, want_s = R.quantize(x)
    assert torch.equal(room[0][:m], want_q) and torch.equal(room[1][:m].nan_to_num(-1), want_s.nan_to_num(-1))
    assert bool((room[0][m:] == 55).all()) and bool((room[1][m:] == 55).all())


def test_quantiser_borders():
    """Values halfway between two whole numbers go to the even one, neighbours of the border to their own side; rows of zeros, of
    the type's smallest and largest numbers, with infinities and NaN."""
    api = _api()
    k = 264
    x = torch.zeros((12, k), device=DEV)
    x[0, 0], x[0, 1:255] = 127, torch.arange(254, device=DEV) - 126.5        # scale 1: every half
    x[1] = x[0] * 2 ** -20
    x[2, :] = 0
    x[3, 5] = -3.0
    x[4, 0] = math.inf
    x[5, 17], x[5, 3] = math.nan, 5.0
    x[6, 0], x[6, 1] = -math.inf, math.nan
    x[7, :] = torch.linspace(-1, 1, k, device=DEV)
    x[8, 0], x[8, 1:] = 1.0, 0.5 / 127
    for dtype in (torch.bfloat16, torch.float16):
        t = x.to(dtype)
        info = torch.finfo(dtype)
        t[9, :] = info.smallest_normal * info.eps                             # the smallest number there is
        t[9, 7] *= 100
        t[10, :] = info.max
        t[10, 9] = -info.max
        t[11, :] = info.smallest_normal * torch.linspace(-3, 3, k, device=DEV).to(dtype)
        q, s = api.prepare_int8_inputs(t)
        want_q, want_s = R.quantize(t)
        assert torch.equal(q, want_q) and torch.equal(s.nan_to_num(-1), want_s.nan_to_num(-1))
        assert torch.isnan(s[4:7]).all() and not q[4:7].any() and s[2] == 1


def test_quantiser_strides_shapes_and_out():
    api = _api()
    gen = _gen(5)
    big = _randn(gen, 40, 200, dtype=torch.bfloat16)
    for x in (big[:, 8:72], big[:, 3:70], big[::2], big.T, big[:, ::3], big.reshape(5, 8, 200), big[:0], big[7], big[3:4].expand(6, 200),
              big.flatten()[1:1 + 64 * 16].view(64, 16)):
        q, s = api.prepare_int8_inputs(x)
        want_q, want_s = R.quantize(x)
        assert torch.equal(q, want_q) and torch.equal(s, want_s) and q.shape == x.shape and s.shape == x.shape[:-1]
    room_q = torch.full((50, 200), 77, dtype=torch.int8, device=DEV)
    room_s = torch.full((50,), 77.0, device=DEV)
    q, s = api.prepare_int8_inputs(big, out=(room_q[:40], room_s[:40]))
    assert q.data_ptr() == room_q.data_ptr() and torch.equal(q, R.quantize(big)[0])
    assert bool((room_q[40:] == 77).all()) and bool((room_s[40:] == 77).all())        # rows behind the last stay as they were
    off = torch.empty(40 * 200 + 1, dtype=torch.int8, device=DEV)[1:].view(40, 200)   # a place that allows no wide stores
    api.prepare_int8_inputs(big, out=(off, room_s[:40]))
    assert torch.equal(off, q)


# ---------------------------------------------------------------------------------------------------------------------
# products of 8-bit integers
# ---------------------------------------------------------------------------------------------------------------------
INT8_SHAPES = [(1, 16, 1), (1, 5120, 257), (2, 32, 8), (3, 2304, 5120), (7, 48, 130), (8, 144, 24), (16, 1008, 129), (17, 272, 520), (33, 128, 64),
               (64, 2304, 1000), (65, 400, 333), (100, 4112, 72), (129, 256, 256), (200, 1040, 1111), (256, 512, 128), (257, 128, 2304), (300, 5120, 264),
               (513, 96, 777), (1021, 1024, 640), (2000, 272, 2049)]


@pytest.mark.parametrize("m,k,n", INT8_SHAPES)
def test_int8_projection(m, k, n):
    gen = _gen(m + 3 * k + 7 * n)
    (x, sx), (w, sw) = _int8(gen, m, k), _int8(gen, n, k)
    bias = _randn(gen, n)
    for out_dtype, b in ((torch.bfloat16, None), (torch.float16, bias), (torch.float32, bias), (torch.float32, None)):
        y = _api().int8_projection(x, sx, w, sw, bias=b, out_dtype=out_dtype)
        assert y.dtype == out_dtype and y.shape == (m, n)
        R.check(f"{out_dtype}", y, *R.projection(x, sx, w, sw, b, out_dtype))


@pytest.mark.parametrize("m,k,n", INT8_SHAPES)
def test_int8_gated_projection(m, k, n):
    gen = _gen(m + 5 * k + 11 * n)
    (x, sx), (w, sw) = _int8(gen, m, k), _int8(gen, 2 * n, k)
    sx, sw = sx * k ** -0.25, sw * k ** -0.25
    for out_dtype, clamp in ((torch.bfloat16, 10.0), (torch.float16, 0.75), (torch.float32, None)):
        h = _api().int8_gated_projection(x, sx, w, sw, activation_clamp=clamp, out_dtype=out_dtype)
        assert h.dtype == out_dtype and h.shape == (m, n)
        R.check(f"{out_dtype}", h, *R.gated_projection(x, sx, w, sw, clamp, out_dtype))


def test_int8_sums_are_exact_at_the_largest_width():
    """Sums up to 127 * 128 * 131056, just below 2^31, where 32-bit floats have long lost whole numbers."""
    k = 131056
    x = torch.full((3, k), 127, dtype=torch.int8, device=DEV)
    w = torch.full((130, k), -128, dtype=torch.int8, device=DEV)
    x[1, ::2] = -127
    x[2, 5] = 126
    one = torch.ones(3, device=DEV), torch.ones(130, device=DEV)
    y = _api().int8_projection(x, one[0], w, one[1], out_dtype=torch.float32)
    want = torch.tensor([-127 * 128 * k, 0, -127 * 128 * k + 128], dtype=torch.float64, device=DEV)
    assert torch.equal(y, want.float()[:, None].expand(3, 130))


def test_int8_scales_that_are_no_numbers_stay_in_their_row():
    gen = _gen(3)
    for m in (1, 20, 300):
        (x, sx), (w, sw) = _int8(gen, m, 256), _int8(gen, 96, 256)
        sx[m // 2], sw[5] = math.nan, math.inf
        y = _api().int8_projection(x, sx, w, sw, out_dtype=torch.float32)
        R.check("nan", y, *R.projection(x, sx, w, sw, None, torch.float32))
        h = _api().int8_gated_projection(x, sx, w, torch.ones_like(sw))
        assert torch.isnan(h[m // 2]).all() and (m == 1 or torch.isfinite(h[0]).all())


def test_int8_strides_and_shapes():
    api = _api()
    gen = _gen(11)
    (big, sx), (w, sw) = _int8(gen, 60, 320), _int8(gen, 40, 128)
    flat = big.flatten()
    for x, s in ((big[:, :128], sx), (big[:, 16:144], sx), (big[:, 3:131], sx), (big[::3, 32:160], sx[::3]), (big[:, :128].reshape(3, 20, 128), sx.view(3, 20)),
                 (big[:0, :128], sx[:0]), (big[4, :128], sx[4]), (big[2:3, :128].expand(9, 128), sx[2:3].expand(9)), (flat[1:1 + 50 * 128].view(50, 128), sx[:50]),
                 (big[:, :256:2], sx)):
        y = api.int8_projection(x, s, w, sw, out_dtype=torch.float32)
        want, off = R.projection(x.reshape(-1, 128), s.reshape(-1), w, sw, None, torch.float32)
        assert y.shape == (*x.shape[:-1], 40)
        R.check("strides", y.reshape(-1, 40), want, off)
    y = api.int8_projection(big[:, :128], sx[:, None], w, sw[:, None])          # scales as columns
    assert torch.equal(y, api.int8_projection(big[:, :128], sx, w, sw))


def test_outputs_past_32_bit_offsets():
    m, n, k = 140000, 16384, 16
    gen = _gen(2)
    (x, sx), (w, sw) = _int8(gen, m, k), _int8(gen, n, k)
    y = _api().int8_projection(x, sx, w, sw)
    rows = torch.tensor([0, 1, 131071, 131072, 131073, m - 1], device=DEV)
    R.check("far", y[rows], *R.projection(x[rows], sx[rows], w, sw, None, torch.bfloat16))


def test_c_interface_leaves_rows_behind_the_last():
    from vllm_plugin_b200.backend import _native as N, dense as D
    api = _api()
    gen = _gen(8)
    for m in (1, 5, 40, 200, 700):
        (x, sx), (w, sw) = _int8(gen, m, 128), _int8(gen, 200, 128)
        api.int8_projection(x, sx, w, sw)                    # prepares the device
        for gated in (False, True):
            n = 100 if gated else 200
            room = torch.full((m + 300, n), 7.0, dtype=torch.bfloat16, device=DEV)
            a = N.MmoeInt8Product(m, 128, n, N.MMOE_BF16, math.inf, 0, 128, x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), None,
                                  room.data_ptr(), D._on_device(0).status_ptr)
            run = N.load().mmoe_int8_gated_projection if gated else N.load().mmoe_int8_projection
            N.check(run(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
            want = api.int8_gated_projection(x, sx, w, sw) if gated else api.int8_projection(x, sx, w, sw)
            assert torch.equal(room[:m], want) and bool((room[m:] == 7).all())


# ---------------------------------------------------------------------------------------------------------------------
# gated block
# ---------------------------------------------------------------------------------------------------------------------
BLOCK_SHAPES = [(1, 8, 8), (1, 5120, 2304), (2, 64, 24), (3, 136, 72), (8, 520, 264), (16, 256, 128), (17, 1000, 688), (31, 128, 4104), (33, 72, 1032),
                (64, 512, 256), (100, 2048, 136), (128, 264, 520), (129, 640, 384), (255, 128, 640), (257, 1032, 264), (300, 512, 1288), (600, 256, 256),
                (1021, 776, 520), (2100, 136, 264)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,hidden,inter", BLOCK_SHAPES)
def test_block_and_gradients(m, hidden, inter, dtype):
    x, w13, w2, dy = _block_inputs(m, hidden, inter, dtype, seed=m + hidden, grad=True)
    for clamp in (None, 1.25):
        y = _api().gated_feed_forward(x, w13, w2, activation_clamp=clamp)
        grads = torch.autograd.grad(y, (x, w13, w2), dy)
        ref = R.Block(x, w13, w2, clamp, dy)
        assert y.dtype == dtype
        R.check("y", y.detach(), ref.y, ref.off["y"])
        for name, got in zip(("dx", "dw13", "dw2"), grads):
            assert got.dtype == dtype
            R.check(name, got, getattr(ref, name), ref.off[name])
        with torch.no_grad():
            assert torch.equal(_api().gated_feed_forward(x, w13, w2, activation_clamp=clamp), y)


def test_gradients_against_differences():
    """Directional derivatives of the operator's own output, which owe nothing to the formulas of the gradients.  A step of 2^-3 along
    a random direction, in FP16: the central difference of sum(y * dy) is off by its third-order term (here below 1 %) and by the
    rounding of y, 2^-11 of each of y's values: sum over n values of variance ~ (2^-11 |y dy|)^2 / 3, over the step's length."""
    api = _api()
    gen = _gen(21)
    m, hidden, inter = 24, 64, 48
    x, w13, w2, dy = _block_inputs(m, hidden, inter, torch.float16, seed=4, grad=True)
    y = api.gated_feed_forward(x, w13, w2)
    grads = torch.autograd.grad(y, (x, w13, w2), dy)
    noise = 2.0 ** -11 * float((y.detach().double() * dy.double()).norm())
    for i, g in enumerate(grads):
        d = g.detach().double() / g.double().norm()                   # along the gradient itself: the largest signal there is
        step = 2.0 ** -3
        ends = []
        for sign in (1, -1):
            args = [t.detach() for t in (x, w13, w2)]
            moved = (args[i].double() + sign * step * d).half()
            args[i] = moved
            ends.append((moved.double(), float((api.gated_feed_forward(*args).double() * dy.double()).sum())))
        got = ends[0][1] - ends[1][1]
        want = float(((ends[0][0] - ends[1][0]) * g.double()).sum())
        assert abs(got - want) <= 0.01 * abs(want) + 8 * noise, (i, got, want, noise)


def test_block_shapes_and_strides():
    api = _api()
    x, w13, w2, dy = _block_inputs(60, 128, 72, torch.bfloat16, seed=1)
    wide = torch.zeros((60, 320), dtype=torch.bfloat16, device=DEV)
    for view in (x.view(3, 4, 5, 128), x[7], x[::2], x[:0], x.T.contiguous().T, x[4:5].expand(6, 128), wide[:, 64:192].copy_(x), wide[:, 3:131].copy_(x),
                 torch.cat((x.new_zeros(1), x.flatten()))[1:].view(60, 128)):
        lead = view.shape[:-1]
        v = view.detach().requires_grad_(True)
        w13r, w2r = w13.clone().requires_grad_(True), w2.clone().requires_grad_(True)
        y = api.gated_feed_forward(v, w13r, w2r, activation_clamp=2.0)
        assert y.shape == (*lead, 128)
        up = torch.randn(y.shape, generator=_gen(9), device=DEV).to(y.dtype)
        y.backward(up)
        flat, fup = v.detach().reshape(-1, 128), up.reshape(-1, 128)
        ref = R.Block(flat, w13, w2, 2.0, fup)
        R.check("y", y.detach().reshape(-1, 128), ref.y, ref.off["y"])
        assert v.grad.shape == view.shape
        R.check("dx", v.grad.reshape(-1, 128), ref.dx, ref.off["dx"])
        R.check("dw13", w13r.grad, ref.dw13, ref.off["dw13"])
        R.check("dw2", w2r.grad, ref.dw2, ref.off["dw2"])


def test_block_gradient_of_a_sum_and_parts():
    """A gradient that is one value broadcast, a transposed and a misaligned one; each subset of the inputs by itself."""
    api = _api()
    x, w13, w2, dy = _block_inputs(70, 64, 40, torch.bfloat16, seed=2)
    odd = torch.cat((dy.new_zeros(3), dy.flatten()))[3:].view(70, 64)
    for up in (torch.ones((), dtype=dy.dtype, device=DEV).expand(70, 64), dy.T.contiguous().T, odd):
        ref = R.Block(x, w13, w2, None, up)
        for mask in range(1, 8):
            leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w13, w2))]
            y = api.gated_feed_forward(*leaves)
            y.backward(up)
            for i, name in enumerate(("dx", "dw13", "dw2")):
                if mask >> i & 1:
                    R.check(name, leaves[i].grad, getattr(ref, name), ref.off[name])
                else:
                    assert leaves[i].grad is None


def test_block_shared_leaves_accumulate():
    """The same weights and rows in two calls: gradients add up as for any operator."""
    api = _api()
    x, w13, w2, dy = _block_inputs(33, 64, 32, torch.float16, seed=6, grad=True)
    a, b = api.gated_feed_forward(x, w13, w2), api.gated_feed_forward(x, w13, w2, activation_clamp=0.5)
    got = torch.autograd.grad(a + b, (x, w13, w2), dy)
    one = torch.autograd.grad(api.gated_feed_forward(x, w13, w2), (x, w13, w2), dy)
    two = torch.autograd.grad(api.gated_feed_forward(x, w13, w2, activation_clamp=0.5), (x, w13, w2), dy)
    for g, p, q in zip(got, one, two):
        assert torch.equal(g, p + q)


def test_block_of_values_that_are_no_numbers():
    api = _api()
    for m in (1, 40, 300):
        x, w13, w2, dy = _block_inputs(m, 64, 48, torch.bfloat16, seed=m)
        x[m // 2, 3] = math.nan
        y = api.gated_feed_forward(x, w13, w2, activation_clamp=3.0)
        assert torch.isnan(y[m // 2]).all()
        keep = torch.arange(m, device=DEV) != m // 2
        ref = R.Block(x[keep], w13, w2, 3.0)
        R.check("others", y[keep], ref.y, ref.off["y"])
        big = torch.full_like(x, 1e30)                                   # far beyond the clamp: sigmoid and its argument overflow
        y = api.gated_feed_forward(big, w13, w2, activation_clamp=3.0)
        ref = R.Block(big, w13, w2, 3.0)
        R.check("large", y, ref.y, ref.off["y"])


def test_second_derivatives_are_refused_and_changes_noticed():
    api = _api()
    x, w13, w2, dy = _block_inputs(5, 64, 32, torch.bfloat16, seed=3, grad=True)
    y = api.gated_feed_forward(x, w13, w2)
    (dx,) = torch.autograd.grad(y, (x,), dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    y = api.gated_feed_forward(x, w13, w2)
    with torch.no_grad():
        w2.mul_(2)
    with pytest.raises(RuntimeError, match="inplace|in-place"):
        y.backward(dy)


# ---------------------------------------------------------------------------------------------------------------------
# together, and how they are called
# ---------------------------------------------------------------------------------------------------------------------
def _int8_block(api, x, w13, s13, w2, s2, clamp):
    q, s = api.prepare_int8_inputs(x)
    h = api.int8_gated_projection(q, s, w13, s13, activation_clamp=clamp)
    return api.int8_projection(*api.prepare_int8_inputs(h), w2, s2), h


@pytest.mark.parametrize("m", [1, 9, 130, 1000])
def test_the_8_bit_block_is_near_the_16_bit_one(m):
    """Quantiser, gated product, quantiser, second product, as a W8A8 dense layer runs them: each step against its definition, and the
    whole near the 16-bit block with the dequantised weights.  The distance is that of quantisation: a value's rounding is off by s / sqrt(12)
    in the mean, s = max / 127 of its row; with max below 5.5 standard deviations for x and 30 for h (a product of two), 0.0125 and 0.07."""
    api = _api()
    x, w13, w2, _ = _block_inputs(m, 512, 384, torch.bfloat16, seed=m)
    (q13, s13), (q2, s2) = R.quantize(w13), R.quantize(w2)
    y, h = _int8_block(api, x, q13, s13, q2, s2, 10.0)
    qx, sx = R.quantize(x)
    R.check("h", h, *R.gated_projection(qx, sx, q13, s13, 10.0, torch.bfloat16))
    R.check("y", y, *R.projection(*R.quantize(h), q2, s2, None, torch.bfloat16))
    wide = api.gated_feed_forward(x, (q13 * s13[:, None]).bfloat16(), (q2 * s2[:, None]).bfloat16(), activation_clamp=10.0)
    assert float((y.double() - wide.double()).norm() / wide.double().norm()) < 0.1


def test_calls_repeat_bit_for_bit():
    api = _api()
    for m in (1, 48, 333):
        x, w13, w2, dy = _block_inputs(m, 1024, 520, torch.bfloat16, seed=m, grad=True)
        runs = []
        for _ in range(3):
            y = api.gated_feed_forward(x, w13, w2, activation_clamp=1.0)
            runs.append((y.detach(), *torch.autograd.grad(y, (x, w13, w2), dy)))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_two_streams_at_once():
    api = _api()
    args = [_block_inputs(m, 512, 264, torch.bfloat16, seed=m) for m in (1, 300, 64, 700)]
    gen = _gen(4)
    eight = [(*_int8(gen, m, 512), *_int8(gen, 264, 512)) for m in (3, 500, 40, 1)]
    want = [api.gated_feed_forward(*a[:3], activation_clamp=1.5) for a in args]
    want8 = [api.int8_projection(*e) for e in eight]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got, got8 = [], []
    for turn in range(6):
        for i, a in enumerate(args):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, api.gated_feed_forward(*a[:3], activation_clamp=1.5)))
                got8.append((i, api.int8_projection(*eight[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got) and all(torch.equal(y, want8[i]) for i, y in got8)
    api.read_dense_status()


def test_calls_in_graphs():
    """Both blocks captured and replayed on new inputs; two graphs replayed at once on two streams."""
    api = _api()
    graphs = []
    for m in (1, 70, 400):
        x, w13, w2, _ = _block_inputs(m, 256, 136, torch.bfloat16, seed=m)
        w13, w2 = w13[:256].contiguous(), w2[:, :128].contiguous()
        (q13, s13), (q2, s2) = R.quantize(w13), R.quantize(w2)

        def calls(x=x, w13=w13, w2=w2, q13=q13, s13=s13, q2=q2, s2=s2):
            return (api.gated_feed_forward(x, w13, w2, activation_clamp=2.0), *_int8_block(api, x, q13, s13, q2, s2, 2.0))

        calls()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls()
        graphs.append((graph, x, out, calls))
    for seed in (1, 2):
        for graph, x, out, calls in graphs:
            x.copy_(torch.randn(x.shape, generator=_gen(seed), device=DEV))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, x, out, calls in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, calls()))


def test_a_training_step_in_a_graph():
    api = _api()
    x, w13, w2, dy = _block_inputs(50, 128, 64, torch.bfloat16, seed=7, grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        api.gated_feed_forward(x, w13, w2).backward(dy)
        for t in (x, w13, w2):
            t.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = api.gated_feed_forward(x, w13, w2)
        y.backward(dy)
    captured = [t.grad for t in (x, w13, w2)]
    with torch.no_grad():
        x.copy_(torch.randn(x.shape, generator=_gen(3), device=DEV))
        dy.copy_(torch.randn(x.shape, generator=_gen(4), device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    ref = R.Block(x, w13, w2, None, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    for name, got in zip(("dx", "dw13", "dw2"), captured):
        R.check(name, got, getattr(ref, name), ref.off[name])


def test_a_module_made_graphed():
    """A layer around the block through torch.cuda.make_graphed_callables: forward and backward replayed on new inputs."""
    api = _api()

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            _, w13, w2, _ = _block_inputs(1, 128, 72, torch.bfloat16, seed=5)
            self.w13, self.w2 = torch.nn.Parameter(w13), torch.nn.Parameter(w2)

        def forward(self, x):
            return x + api.gated_feed_forward(x, self.w13, self.w2, activation_clamp=1.0)

    layer = Layer()
    w13, w2 = layer.w13.detach().clone(), layer.w2.detach().clone()
    sample = torch.randn(2, 30, 128, device=DEV).bfloat16().requires_grad_(True)
    graphed = torch.cuda.make_graphed_callables(layer, (sample,))
    for seed in (1, 2):
        x = _randn(_gen(seed), 2, 30, 128, dtype=torch.bfloat16).requires_grad_(True)
        dy = _randn(_gen(seed + 9), 2, 30, 128, dtype=torch.bfloat16)
        layer.zero_grad()
        graphed(x).backward(dy)
        ref = R.Block(x.reshape(60, 128), w13, w2, 1.0, dy.reshape(60, 128))
        R.check("dw13", layer.w13.grad, ref.dw13, ref.off["dw13"])
        R.check("dw2", layer.w2.grad, ref.dw2, ref.off["dw2"])
        # the sum with dy is rounded once more
        want = ref.dx + dy.reshape(60, 128).double()
        R.check("dx", x.grad.reshape(60, 128), want, ref.off["dx"] + 2.0 ** -8 * want.abs())


def test_capture_beside_a_graph_made_on_another_stream():
    api = _api()
    x, w13, w2, dy = _block_inputs(50, 128, 64, torch.bfloat16, seed=17, grad=True)
    want = torch.autograd.grad(api.gated_feed_forward(x, w13, w2), (x, w13, w2), dy)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        alive = api.gated_feed_forward(x, w13, w2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.gated_feed_forward(x, w13, w2).backward(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w13, w2), want)) and alive.requires_grad


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    api = _api()
    x, w13, w2, dy = _block_inputs(5, 64, 32, torch.bfloat16, seed=3, grad=True)
    alive = api.gated_feed_forward(x, w13, w2)
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        try:
            api.gated_feed_forward(x, w13, w2)
        except RuntimeError:
            refused = True
        with torch.no_grad():
            y = api.gated_feed_forward(x, w13, w2)           # without gradients there is nothing against it
    assert refused
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive.detach())
    alive.backward(dy)                                         # the eager graph is as it was
    del alive
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        api.gated_feed_forward(x, w13, w2)
    # weights in 32 bits behind the block's, which are no leaves themselves
    master = w13.detach().float().requires_grad_(True)
    alive = api.gated_feed_forward(x.detach(), master.bfloat16(), w2.detach()).sum()
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        weights = master.bfloat16()
        try:
            api.gated_feed_forward(x.detach(), weights, w2.detach())
        except RuntimeError:
            refused = True
    assert refused
    other = w13.detach().float().requires_grad_(True)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        api.gated_feed_forward(x.detach(), other.bfloat16(), w2.detach())        # other leaves
    alive.backward()


def test_beside_the_layer():
    """A shared expert in 16 bits beside the routed ones: the layer's output as its residual, on one stream and in one graph."""
    import helpers as H
    from oracle import mmoe_oracle as O
    api = _api()
    layer = H.make_layer(512, 256, 8, 2, False, seed=0)
    m = 33
    hid = O.make_hidden(m, layer.hidden, 1)
    ids, w = O.make_routing(m, layer.num_experts, layer.num_topk, 2)
    want, buf = H.run_layer(layer, hid, ids, w)
    _, w13, w2, _ = _block_inputs(1, 512, 256, torch.bfloat16, seed=5)
    weights = H.kernel_weights(layer, torch.device(DEV))
    x, ids, w = hid.to(DEV), ids.to(DEV), w.to(DEV)
    y = torch.empty_like(x)

    def step():
        api.stage_inputs_for_mega_moe(buf, x, ids, w)
        shared = api.gated_feed_forward(x, w13, w2, activation_clamp=10.0)
        api.fp8_fp4_mega_moe(y, weights[0], weights[1], buf, activation_clamp=10.0, residual=shared)
        return shared

    shared = step()
    eager = y.clone()
    assert torch.equal(eager, want + shared)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, eager)


@pytest.mark.parametrize("m", [144, 145, 160, 161, 256, 257, 520])
def test_either_side_of_the_line_between_the_kernels(m):
    """Few tokens and many take different kernels: up to 160 in products that read the weights as they are stored, up to 256 in those that read
    them along their rows.  Values, all gradients and the 8-bit products, and rows that do not depend on how many others there are."""
    api = _api()
    x, w13, w2, dy = _block_inputs(m, 392, 200, torch.bfloat16, seed=m, grad=True)
    y = api.gated_feed_forward(x, w13, w2, activation_clamp=1.5)
    grads = torch.autograd.grad(y, (x, w13, w2), dy)
    ref = R.Block(x, w13, w2, 1.5, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        R.check(name, got, getattr(ref, name), ref.off[name])
    gen = _gen(m)
    (q, s), (w, sw) = _int8(gen, m, 336), _int8(gen, 222, 336)
    out = api.int8_projection(q, s, w, sw, out_dtype=torch.float32)
    R.check("y8", out, *R.projection(q, s, w, sw, None, torch.float32))
    assert torch.equal(out[:3], api.int8_projection(q[:3], s[:3], w, sw, out_dtype=torch.float32))     # whole numbers: the same bits


@pytest.mark.parametrize("m", [1, 40, 150, 200, 256])
def test_more_tiles_than_sms(m):
    """Wide weights: few tokens then take half of an SM for each tile, if their sums fit there."""
    api = _api()
    gen = _gen(m)
    (q, s), (w, sw) = _int8(gen, m, 112), _int8(gen, 20003, 112)
    R.check("y8", api.int8_projection(q, s, w, sw), *R.projection(q, s, w, sw, None, torch.bfloat16))
    x, w13, w2, dy = _block_inputs(m, 72, 19456, torch.bfloat16, seed=m, grad=True)
    y = api.gated_feed_forward(x, w13, w2, activation_clamp=1.5)
    dx, = torch.autograd.grad(y, (x,), dy)
    ref = R.Block(x, w13, w2, 1.5, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    R.check("dx", dx, ref.dx, ref.off["dx"])


@pytest.mark.parametrize("mask", range(1, 8))
def test_parts_of_the_gradients_of_many_tokens(mask):
    """Each subset of the gradients by itself, rows of x in a wider tensor: the launches hold one product or two then."""
    api = _api()
    _, w13, w2, dy = _block_inputs(300, 136, 104, torch.float16, seed=mask)
    wide = _randn(_gen(mask), 300, 400, dtype=torch.float16)
    leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((wide[:, 64:200], w13, w2))]
    y = api.gated_feed_forward(*leaves, activation_clamp=1.0)
    ref = R.Block(*leaves, 1.0, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
    names = [n for i, n in enumerate(("dx", "dw13", "dw2")) if mask >> i & 1]
    for name, g in zip(names, got):
        R.check(name, g, getattr(ref, name), ref.off[name])


def test_a_recorded_timeout_is_raised_once():
    """What a kernel that gave up leaves in the status words reaches the caller: at the next read, and at a later call without one."""
    from vllm_plugin_b200.backend import dense as D
    api = _api()
    gen = _gen(1)
    (q, s), (w, sw) = _int8(gen, 4, 64), _int8(gen, 32, 64)
    want = api.int8_projection(q, s, w, sw)
    state = D._on_device(0)
    state.status[:4] = torch.tensor([1, 31, 2, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="kernel 31"):
        api.read_dense_status()
    api.read_dense_status()
    try:
        api.set_kernel_options(status_poll_interval=1)
        for _ in range(3):                                     # whatever an earlier interval had queued is over
            api.int8_projection(q, s, w, sw)
            torch.cuda.synchronize()
        state.status[:4] = torch.tensor([1, 32, 0, 7], dtype=torch.int32)
        with pytest.raises(RuntimeError, match="kernel 32"):
            for _ in range(3):
                api.int8_projection(q, s, w, sw)
                torch.cuda.synchronize()
    finally:
        api.set_kernel_options(status_poll_interval=32)
    assert torch.equal(api.int8_projection(q, s, w, sw), want)
    api.read_dense_status()


def test_backward_twice_and_under_no_grad():
    api = _api()
    x, w13, w2, dy = _block_inputs(40, 64, 48, torch.bfloat16, seed=9, grad=True)
    y = api.gated_feed_forward(x, w13, w2)
    one = torch.autograd.grad(y, (x, w13, w2), dy, retain_graph=True)
    two = torch.autograd.grad(y, (x, w13, w2), dy)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    with torch.no_grad():
        assert not api.gated_feed_forward(x, w13, w2).requires_grad
    with torch.inference_mode():
        assert torch.equal(api.gated_feed_forward(x, w13, w2), y)


def test_a_first_call_from_another_thread():
    """Threads that have not used the GPU yet, at once, each on a stream of its own; gradients too."""
    import threading
    api = _api()
    x, w13, w2, dy = _block_inputs(200, 256, 136, torch.bfloat16, seed=12, grad=True)
    want = [api.gated_feed_forward(x, w13, w2).detach()]
    want += torch.autograd.grad(api.gated_feed_forward(x, w13, w2), (x, w13, w2), dy)
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    y = api.gated_feed_forward(x, w13, w2)
                    got = [y.detach(), *torch.autograd.grad(y, (x, w13, w2), dy)]
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        wrong.append("other bits")
        except Exception as e:  # noqa: BLE001 - reported below, in the test's own thread
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    api = _api()
    x, w13, w2, _ = _block_inputs(4, 64, 32, torch.bfloat16)
    ok = dict(x=x, w13=w13, w2=w2)
    for change, error in ((dict(x=x.float()), AssertionError), (dict(x=x.half()), AssertionError), (dict(x=x[:, :56]), AssertionError),
                          (dict(w13=w13[:62]), AssertionError), (dict(w13=w13[0]), AssertionError), (dict(w2=w2.T), AssertionError),
                          (dict(w13=torch.cat((w13, w13), 1)[:, :64]), AssertionError), (dict(w13=w13.cpu()), AssertionError), (dict(x=x.cpu()), RuntimeError),
                          (dict(x=x[:, :60].contiguous(), w13=w13[:, :60].contiguous(), w2=w2[:60].contiguous()), AssertionError),
                          (dict(w13=torch.cat((w13.new_zeros(1), w13.flatten()))[1:].view(64, 64)), AssertionError),
                          (dict(activation_clamp=0.0), AssertionError), (dict(activation_clamp=-1.0), AssertionError), (dict(activation_clamp=math.nan), AssertionError)):
        with pytest.raises(error):
            api.gated_feed_forward(**{**ok, **change})
    gen = _gen(1)
    (q, s), (w, sw) = _int8(gen, 4, 64), _int8(gen, 32, 64)
    ok = dict(x=q, x_scales=s, w=w, w_scales=sw)
    for change, error in ((dict(x=q.to(torch.uint8)), AssertionError), (dict(x=q[:, :48]), AssertionError), (dict(x_scales=s[:3]), AssertionError),
                          (dict(x_scales=s.double()), AssertionError), (dict(w_scales=sw[:5]), AssertionError), (dict(w=w[:, :40], x=q[:, :40]), AssertionError),
                          (dict(w=w.T), AssertionError), (dict(bias=sw.bfloat16()), AssertionError), (dict(bias=sw[:3]), AssertionError), (dict(x=q.cpu()), RuntimeError),
                          (dict(x_scales=s.cpu()), AssertionError), (dict(out_dtype=torch.float64), AssertionError), (dict(out_dtype=torch.int8), AssertionError),
                          (dict(w=w[:, :40].contiguous(), x=q[:, :40].contiguous()), AssertionError), (dict(w=w[:0]), AssertionError),
                          (dict(w_scales=sw.clone().requires_grad_(True)), NotImplementedError)):
        with pytest.raises(error):
            api.int8_projection(**{**ok, **change})
    with pytest.raises(AssertionError):
        api.int8_gated_projection(q, s, w[:31], sw[:31])
    with pytest.raises(AssertionError):
        api.int8_gated_projection(q, s, w, sw, activation_clamp=0)
    with pytest.raises(ValueError):
        api.prepare_int8_inputs(x.float())
    with pytest.raises(ValueError):
        api.prepare_int8_inputs(x.cpu())
    with pytest.raises(ValueError):
        api.prepare_int8_inputs(x, out=(q[:, :32], s))
    with pytest.raises(NotImplementedError):
        api.prepare_int8_inputs(x.clone().requires_grad_(True))
    api.read_dense_status()
