"""Products in 16 bits whose tiles are any number of turns and more: the pairs of multiprocessors take whole tiles, and halves of their columns where at most half
of the pairs would have one of the last."""

import pytest
import torch

import dense_reference as R
import grouped_reference as G
from test_gpu_fp8_turns import _columns
from test_gpu_grouped import _ends, _rand

pytestmark = pytest.mark.gpu

# two tiles of an expert's rows with 256, 224, 160 and 129 or so columns; more experts, tiles of all widths
COUNTS = [[512], [440], [310], [258], [300, 0, 1, 70], [33, 200, 130, 0, 256]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("which", range(10))
def test_projection(which, counts):
    from vllm_plugin_b200 import api
    rows, ends, channels = sum(counts) + 3, _ends(counts), _columns()[which] * 256 - 56
    x, w = _rand(1, rows, 136), _rand(2, len(counts), channels, 136, std=0.1)
    want = G.Projection(x, w, ends)
    y = api.grouped_projection(x, w, ends)
    R.check("y", y, want.y, want.off["y"])
    assert torch.equal(api.grouped_projection(x, w, ends), y)
    api.read_dense_status()


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("which", range(10))
def test_gradients(which, counts):
    from vllm_plugin_b200 import api
    rows, ends, width = sum(counts) + 3, _ends(counts), _columns()[which] * 256 - 40
    x, w, dy = _rand(1, rows, width), _rand(2, len(counts), 72, width, std=0.1), _rand(3, rows, 72)
    x.requires_grad_(True), w.requires_grad_(True)
    want = G.Projection(x, w, ends, dy)
    dx, dw = torch.autograd.grad(api.grouped_projection(x, w, ends), (x, w), dy)
    R.check("dx", dx, want.dx, want.off["dx"])
    R.check("dw", dw, want.dw, want.off["dw"])
    api.read_dense_status()


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("which", range(10))
def test_block(which, counts):
    from vllm_plugin_b200 import api
    rows, ends, inter = sum(counts) + 3, _ends(counts), _columns()[which] * 128 - 8
    x, dy = _rand(1, rows, 136, dtype=torch.float16), _rand(4, rows, 136, dtype=torch.float16)
    w13, w2 = _rand(2, len(counts), 2 * inter, 136, std=0.1, dtype=torch.float16), _rand(3, len(counts), 136, inter, std=0.02, dtype=torch.float16)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    want = G.Block(x, w13, w2, ends, 1.5, dy)
    y = api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=1.5)
    grads = torch.autograd.grad(y, leaves, dy)
    R.check("y", y.detach(), want.y, want.off["y"])
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        R.check(name, got, getattr(want, name), want.off[name])
    api.read_dense_status()
