"""Products in 8-bit floating point with block scales, and their quantiser, against 64-bit plain forms."""

import pytest
import torch

import dense_reference as R
import grouped_reference as G
from test_gpu_grouped import DEV, GROUPS, _ends, _rand

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _eight_bit(seed, *shape):
    return (_rand(seed, *shape, dtype=torch.float32) * 60).clamp(-448, 448).to(E4M3)


def _positive(seed, *shape):
    return _rand(seed, *shape, dtype=torch.float32).exp() * 0.01


def _case(rows, experts, channels, width, parts):
    groups, blocks = -(-width // 128), -(-(channels // parts) // 128) * parts
    return _eight_bit(1, rows, width), _positive(2, rows, groups), _eight_bit(3, experts, channels, width), _positive(4, experts, blocks, groups)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width,channels", [(16, 8), (128, 48), (144, 131), (640, 257), (1040, 520)])
@pytest.mark.parametrize("rows", [1, 2, 17, 33, 127, 256, 300, 777])
def test_projection(rows, width, channels, dtype):
    from vllm_plugin_b200 import api
    x, sx, w, sw = _case(rows, 1, channels, width, 1)
    want, off = G.fp8_product(x, sx, w, sw, None, dtype)
    got = api.fp8_projection(x, sx, w[0], sw[0], out_dtype=dtype)
    assert got.dtype == dtype
    R.check("y", got, want, off)
    api.read_dense_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hidden,inter", [(16, 8), (144, 72), (640, 136), (528, 264)])
@pytest.mark.parametrize("rows", [1, 17, 256, 333])
@pytest.mark.parametrize("clamp", [None, 1.0])
def test_gated(rows, hidden, inter, clamp, dtype):
    from vllm_plugin_b200 import api
    x, sx, w, sw = _case(rows, 1, 2 * inter, hidden, 2)
    want, off = G.fp8_product(x, sx, w, sw, None, dtype, True, clamp)
    got = api.fp8_gated_projection(x, sx, w[0], sw[0], activation_clamp=clamp, out_dtype=dtype)
    assert got.dtype == dtype
    R.check("h", got, want, off)
    api.read_dense_status()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("width,channels", [(16, 16), (400, 272)])
@pytest.mark.parametrize("counts,spare", GROUPS)
def test_grouped(counts, spare, width, channels, gated):
    from vllm_plugin_b200 import api
    rows, ends = sum(counts) + spare, _ends(counts)
    x, sx, w, sw = _case(rows, len(counts), channels, width, 1 + gated)
    for dtype in (torch.bfloat16, torch.float32):
        want, off = G.fp8_product(x, sx, w, sw, ends, dtype, gated, 2.0 if gated else None)
        got = api.fp8_gated_projection(x, sx, w, sw, ends=ends, activation_clamp=2.0, out_dtype=dtype) if gated else api.fp8_projection(
            x, sx, w, sw, ends=ends, out_dtype=dtype)
        R.check("y", got, want, off)
    api.read_dense_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(1, 128), (3, 1), (7, 5120), (5, 130), (65, 264), (130, 1000), (3, 127)])
def test_quantiser(rows, width, dtype):
    from vllm_plugin_b200 import api
    x = _rand(1, rows, width, dtype=torch.float32).exp().mul(_rand(2, rows, width, dtype=torch.float32)).to(dtype)
    q, s = api.prepare_fp8_inputs(x)
    want_q, want_s = G.quantize(x)
    assert q.dtype == E4M3 and torch.equal(s, want_s) and torch.equal(q.double(), want_q)
