"""Products in 8-bit floating point whose tiles are any number of turns and more: the pairs of multiprocessors take whole tiles of 256 columns, and halves of
them where at most half of the pairs would have one of the last."""

import pytest
import torch

import dense_reference as R
import grouped_reference as G
from test_gpu_fp8 import _case
from test_gpu_grouped import _ends

pytestmark = pytest.mark.gpu


def _columns():
    """Tiles of columns, for two tiles of rows each: fewer than half a turn, about half of one, one, more, two and a little."""
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    return [1, pairs // 8, pairs // 4, pairs // 4 + 1, pairs // 2, pairs // 2 + 1, 3 * pairs // 4, 3 * pairs // 4 + 1, pairs, pairs + 1]


def _run(rows, ends, width, channels, gated, dtype):
    from vllm_plugin_b200 import api
    experts = 1 if ends is None else ends.numel()
    x, sx, w, sw = _case(rows, experts, channels * (1 + gated), width, 1 + gated)
    want, off = G.fp8_product(x, sx, w, sw, ends, dtype, gated, 2.0 if gated else None)
    if ends is None:
        w, sw = w[0], sw[0]
    call = (lambda: api.fp8_gated_projection(x, sx, w, sw, ends=ends, activation_clamp=2.0, out_dtype=dtype)) if gated else (
        lambda: api.fp8_projection(x, sx, w, sw, ends=ends, out_dtype=dtype))
    got = call()
    R.check("y", got, want, off)
    assert torch.equal(got, call())
    api.read_dense_status()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("less", [0, 8, 72, 104])
@pytest.mark.parametrize("which", range(10))
def test_two_tiles_of_rows(which, less, gated):
    channels = _columns()[which] * (128 if gated else 256) - less
    _run(300, None, 272, channels, gated, torch.bfloat16)


@pytest.mark.parametrize("less", [1, 65, 130, 193])
@pytest.mark.parametrize("which", range(10))
def test_columns_that_end_anywhere(which, less):
    _run(400, None, 144, _columns()[which] * 256 - less, False, torch.float32)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("which", range(10))
def test_many_groups(which, gated):
    _run(260, None, 1040, _columns()[which] * (128 if gated else 256), gated, torch.float16)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", [[300, 0, 200, 257, 1, 90], [0, 900, 13], [129] * 9 + [300]])
@pytest.mark.parametrize("columns", [1, 2, 5, 7, 12, 20])
def test_experts(columns, counts, gated):
    ends = _ends(counts)
    _run(sum(counts) + 5, ends, 272, columns * (128 if gated else 256) - 16, gated, torch.bfloat16)
