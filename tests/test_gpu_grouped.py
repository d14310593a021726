"""Products of a layer's experts in 16 bits, with their gradients, against 64-bit plain forms."""

import pytest
import torch

import dense_reference as R
import grouped_reference as G

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rand(seed, *shape, std=1.0, dtype=torch.bfloat16):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _ends(counts):
    return torch.tensor(counts, device=DEV).cumsum(0).to(torch.int32)


# rows of each expert, rows behind the last one's
GROUPS = [([1], 0), ([5], 3), ([0, 7, 0, 0, 33], 0), ([32, 31, 1, 0], 11), ([256], 0), ([257, 255], 1), ([0, 0, 0], 9), ([300, 0, 64, 513, 2], 70),
          ([1] * 40, 0), ([0] * 63 + [17], 0)]
SIZES = [(64, 48), (8, 8), (136, 264), (72, 520), (648, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width,channels", SIZES)
@pytest.mark.parametrize("counts,spare", GROUPS)
def test_projection_and_gradients(counts, spare, width, channels, dtype):
    from vllm_plugin_b200 import api
    rows, ends = sum(counts) + spare, _ends(counts)
    x, w, dy = _rand(1, rows, width, dtype=dtype), _rand(2, len(counts), channels, width, std=0.1, dtype=dtype), _rand(3, rows, channels, dtype=dtype)
    x.requires_grad_(True), w.requires_grad_(True)
    want = G.Projection(x, w, ends, dy)
    y = api.grouped_projection(x, w, ends)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        assert got.dtype == dtype
        R.check(name, got.detach(), getattr(want, name), want.off[name])
    with torch.no_grad():
        assert torch.equal(api.grouped_projection(x, w, ends), y)
    api.read_dense_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden,inter", [(64, 48), (8, 8), (264, 136), (136, 328)])
@pytest.mark.parametrize("counts,spare", GROUPS)
@pytest.mark.parametrize("clamp", [None, 0.5])
def test_block_and_gradients(counts, spare, hidden, inter, clamp, dtype):
    from vllm_plugin_b200 import api
    rows, ends = sum(counts) + spare, _ends(counts)
    x, dy = _rand(1, rows, hidden, dtype=dtype), _rand(4, rows, hidden, dtype=dtype)
    w13, w2 = _rand(2, len(counts), 2 * inter, hidden, std=0.1, dtype=dtype), _rand(3, len(counts), hidden, inter, std=0.1, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    want = G.Block(x, w13, w2, ends, clamp, dy)
    y = api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=clamp)
    grads = torch.autograd.grad(y, leaves, dy)
    for name, got in zip(("y", "dx", "dw13", "dw2"), (y, *grads)):
        assert got.dtype == dtype
        R.check(name, got.detach(), getattr(want, name), want.off[name])
    with torch.no_grad():
        assert torch.equal(api.grouped_feed_forward(x, w13, w2, ends, activation_clamp=clamp), y)
    api.read_dense_status()
