"""What the experts' products on CTA pairs must not touch or pass on, in the forward pass too: the next expert's values, what is around an output, ends out of
order or changed between replays, strides.  The shapes are those that the pairs take (``grouped_shapes``)."""

import ctypes
import math

import pytest
import torch

import dense_reference as R
import grouped_reference as G
import grouped_shapes as S
from test_gpu_fp8 import _case
from test_gpu_grouped import DEV, _ends, _rand

pytestmark = pytest.mark.gpu


def _api():
    from vllm_plugin_b200 import api
    return api


@pytest.fixture(autouse=True)
def this_device_has_the_shapes_multiprocessors():
    assert torch.cuda.get_device_properties(0).multi_processor_count == S.SMS


def _block(seed, name, dtype=torch.bfloat16):
    rows, experts, hidden, inter = S.BLOCKS[name]
    return (_rand(seed, rows, hidden, dtype=dtype), _rand(seed + 1, experts, 2 * inter, hidden, std=0.03, dtype=dtype),
            _rand(seed + 2, experts, hidden, inter, std=0.03, dtype=dtype))


def _eight(name, gated):
    rows, experts, width, channels = S.EIGHT_BITS[name]
    return _case(rows, experts, channels, width, 1 + gated)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_no_numbers_stay_with_their_expert(bad, dtype):
    """In rows of another expert, in rows of none, in another expert's weights: loads of rows, of weights in order, of gate and up rows by eights, and of
    weights that K or the channels end within a stage or a tile of, give the others nothing."""
    api = _api()
    counts = [33, 40, 0, 70, 65, 12]
    x, w13, w2 = _block(11, "values", dtype)
    rows, ends = x.shape[0], _ends(counts)
    assert rows == sum(counts) + 21
    spoilt = (1, 4)
    good = torch.ones(rows, dtype=torch.bool, device=DEV)
    for e, a, b in G.pieces(ends, rows):
        if e in spoilt:
            good[a:b] = False
    good[sum(counts):] = False
    x2, w13b, w2b = x.clone(), w13.clone(), w2.clone()
    x2[~good] = bad
    for e in (*spoilt, 2):
        w13b[e], w2b[e] = bad, bad
    y = api.grouped_feed_forward(x2, w13b, w2b, ends, activation_clamp=2.0)
    want = G.Block(x, w13, w2, ends, 2.0)
    R.check("y", y[good], want.y[good], want.off["y"][good])
    assert not y[sum(counts):].any()
    y = api.grouped_projection(x2, w13b, ends)
    want = G.Projection(x, w13, ends)
    R.check("projection", y[good], want.y[good], want.off["y"][good])
    assert not y[sum(counts):].any()


@pytest.mark.parametrize("gated", [False, True])
def test_eight_bit_values_that_are_no_numbers_stay_with_their_expert(gated):
    """NaN as values and as scales, of rows and of weights."""
    api = _api()
    counts = [100, 130, 0, 270, 65, 41]
    x, sx, w, sw = _eight("values", gated)
    rows, ends = x.shape[0], _ends(counts)
    assert rows == sum(counts) + 34
    want, off = G.fp8_product(x, sx, w, sw, ends, torch.bfloat16, gated)
    good = torch.ones(rows, dtype=torch.bool, device=DEV)
    for e, a, b in G.pieces(ends, rows):
        if e in (1, 4):
            good[a:b] = False
    good[sum(counts):] = False
    call = api.fp8_gated_projection if gated else api.fp8_projection
    for which in range(4):
        given = [x.clone(), sx.clone(), w.clone(), sw.clone()]
        if which == 0:
            given[0].view(torch.uint8)[~good] = 0x7F
        elif which == 1:
            given[1][~good] = math.nan
        else:
            for e in (1, 2, 4):
                if which == 2:
                    given[2].view(torch.uint8)[e] = 0x7F
                else:
                    given[3][e] = math.nan
        got = call(*given, ends=ends)
        R.check("y", got[good], want[good], off[good])
        assert torch.isnan(got[:sum(counts)][~good[:sum(counts)]]).all() and not got[sum(counts):].any()


@pytest.mark.parametrize("behind", [0, 117])
def test_what_is_around_the_output_is_left(behind):
    """In front of and behind it; rows behind the last expert's are its own, and zero."""
    from vllm_plugin_b200.backend import _native as N, dense as D
    api = _api()
    rows, experts, width, channels = S.PROJECTIONS["room"]
    ends = _ends([350, rows - 350 - behind])
    x, w = _rand(1, rows, width), _rand(2, experts, channels, width, std=0.1)
    api.grouped_projection(x, w, ends)
    lib, status, stream = N.load(), D._on_device(0).status_ptr, torch.cuda.current_stream().cuda_stream
    room = torch.full((rows + 16, channels), 7.0, dtype=x.dtype, device=DEV)
    a = N.MmoeGroupedProduct(0, rows, experts, width, channels, 0, width, x.data_ptr(), w.data_ptr(), ends.data_ptr(), room[8:].data_ptr(), status)
    N.check(lib.mmoe_grouped_projection(ctypes.byref(a), stream))
    want = G.Projection(x, w, ends)
    R.check("y", room[8:-8], want.y, want.off["y"])
    assert (room[:8] == 7).all() and (room[-8:] == 7).all()

    rows, experts, width, channels = S.EIGHT_BITS["room"]
    ends = _ends([350, rows - 350 - behind])
    q, sx, w8, sw = _eight("room", False)
    for code, dtype in ((3, torch.float32), (0, torch.bfloat16)):
        room = torch.full((rows * channels + 512,), 7.0, dtype=dtype, device=DEV)
        b = N.MmoeFp8Product(rows, experts, width, channels, code, math.inf, 0, 0, width, q.data_ptr(), sx.data_ptr(), w8.data_ptr(), sw.data_ptr(), ends.data_ptr(),
                             room[256:].data_ptr(), status)
        N.check(lib.mmoe_fp8_projection(ctypes.byref(b), stream))
        value, off = G.fp8_product(q, sx, w8, sw, ends, dtype)
        R.check("fp8", room[256:-256].view(rows, channels), value, off)
        assert (room[:256] == 7).all() and (room[-256:] == 7).all()


@pytest.mark.parametrize("values", [[200, 120, 390], [-1, 160, 400], [80, 160, 401], [2**31 - 1, 2**31 - 1, 2**31 - 1], [-2**31, 0, 200], [0, -3, 400]])
def test_ends_out_of_order(values):
    """No row is an expert's then: zeros, a report, and nothing that lasts."""
    api = _api()
    bad = torch.tensor(values, dtype=torch.int32, device=DEV)
    x, w13, w2 = _block(4, "bad ends")
    q, sx, w, sw = _eight("bad ends", False)
    _, _, pair, pair_scales = _eight("bad ends", True)
    api.read_dense_status()
    interval = api.get_kernel_options().status_poll_interval
    try:
        api.set_kernel_options(status_poll_interval=0)
        for call in (lambda ends: api.grouped_feed_forward(x, w13, w2, ends), lambda ends: api.grouped_projection(x, w13, ends),
                     lambda ends: api.fp8_projection(q, sx, w, sw, ends=ends), lambda ends: api.fp8_gated_projection(q, sx, pair, pair_scales, ends=ends)):
            assert not call(bad).any()
            with pytest.raises(AssertionError, match="ends"):
                api.read_dense_status()
    finally:
        api.set_kernel_options(status_poll_interval=interval)
    good = _ends([200, 0, 200])
    want = G.Block(x, w13, w2, good, None)
    R.check("y", api.grouped_feed_forward(x, w13, w2, good), want.y, want.off["y"])
    R.check("fp8", api.fp8_projection(q, sx, w, sw, ends=good), *G.fp8_product(q, sx, w, sw, good, torch.bfloat16))
    api.read_dense_status()


def test_a_captured_call_goes_by_the_ends_at_its_replay():
    """Other experts, tiles and parts of tiles at each replay; two graphs at once."""
    api = _api()
    x, w13, w2 = _block(3, "replays")
    q, sx, w8, sw = _eight("replays", True)
    one = sw[:, :3].contiguous()
    ends = _ends([0, 0, 0, 0])

    def calls():
        return (api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=2.0), api.grouped_projection(x, w13, ends),
                api.fp8_gated_projection(q, sx, w8, sw, ends=ends), api.fp8_projection(q, sx, w8, one, ends=ends))

    calls()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for counts in ([600, 0, 0, 0], [1, 2, 3, 4], [0, 0, 0, 0], [150, 151, 149, 150], [0, 300, 0, 299], [33, 257, 1, 255]):
        ends.copy_(_ends(counts))
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        eager = calls()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        want, linear = G.Block(x, w13, w2, ends, 2.0), G.Projection(x, w13, ends)
        R.check("y", eager[0], want.y, want.off["y"])
        R.check("projection", eager[1], linear.y, linear.off["y"])
        R.check("gated", eager[2], *G.fp8_product(q, sx, w8, sw, ends, torch.bfloat16, True))
        R.check("fp8", eager[3], *G.fp8_product(q, sx, w8, one, ends, torch.bfloat16))
    api.read_dense_status()


def test_rows_of_any_stride():
    api = _api()
    x, w13, w2 = _block(1, "strides")
    rows, hidden = x.shape
    ends = _ends([100, 0, 150])

    def inside(at):                             # columns of a wider matrix of its own
        return torch.zeros((rows, hidden + 256), dtype=x.dtype, device=DEV)[:, at:at + hidden].copy_(x)

    block, linear = G.Block(x, w13, w2, ends, 2.0), G.Projection(x, w13, ends)
    for view in (torch.stack((x, x), 1).flatten(0, 1)[::2], x.T.contiguous().T, inside(64), inside(3),
                 torch.cat((x.new_zeros(1), x.flatten()))[1:].view(rows, hidden)):
        R.check("y", api.grouped_feed_forward(view, w13, w2, ends, activation_clamp=2.0), block.y, block.off["y"])
        R.check("projection", api.grouped_projection(view, w13, ends), linear.y, linear.off["y"])
