"""Dense products on CTA pairs at every width of tile (``dense_widths.py``), against the plain 64-bit forms."""

import pytest
import torch

import dense_reference as R
import dense_widths as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _pairs_of_a_b200():
    """The tables hold for the number of pairs that they were made for."""
    assert torch.cuda.get_device_properties(0).multi_processor_count // 2 == W.PAIRS


def _randn(seed, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * std).to(dtype)


def _int8(seed, rows, k, most):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randint(-127, 128, (rows, k), generator=gen, device=DEV, dtype=torch.int32).to(torch.int8)
    return q, (torch.rand(rows, generator=gen, device=DEV) + 0.05) * most


def _name(shape):
    return "x".join(map(str, shape))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", W.BLOCKS, ids=_name)
def test_block_and_gradients(shape, dtype):
    """Both products of the block, and the launches of two products of its gradients."""
    from vllm_plugin_b200 import api
    m, hidden, inter = shape
    x, w13 = _randn(1, m, hidden, dtype=dtype), _randn(2, 2 * inter, hidden, dtype=dtype, std=hidden ** -0.5)
    w2, dy = _randn(3, hidden, inter, dtype=dtype, std=inter ** -0.5), _randn(4, m, hidden, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    y = api.gated_feed_forward(*leaves, activation_clamp=1.25)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = R.Block(*leaves, 1.25, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        R.check(name, got, getattr(ref, name), ref.off[name])


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", W.GATED, ids=_name)
def test_gated_product_of_8_bits(shape, out_dtype):
    """g and u of about 0.6: sums of K products with a standard deviation of 73^2, times scales of 0.011 and 0.011 / sqrt(K) in the mean."""
    from vllm_plugin_b200 import api
    m, n, k = shape
    (x, sx), (w, sw) = _int8(m, m, k, 0.02), _int8(n, 2 * n, k, 0.02 * k ** -0.5)
    h = api.int8_gated_projection(x, sx, w, sw, activation_clamp=1.5, out_dtype=out_dtype)
    R.check(f"{out_dtype}", h, *R.gated_projection(x, sx, w, sw, 1.5, out_dtype))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", W.PROJECTIONS, ids=_name)
def test_projection_of_8_bits(shape, out_dtype):
    from vllm_plugin_b200 import api
    m, n, k = shape
    (x, sx), (w, sw) = _int8(m, m, k, 0.02), _int8(n, n, k, 0.02 * k ** -0.5)
    for bias in (None, _randn(5, n)):
        y = api.int8_projection(x, sx, w, sw, bias=bias, out_dtype=out_dtype)
        R.check(f"{out_dtype}", y, *R.projection(x, sx, w, sw, bias, out_dtype))


@pytest.mark.parametrize("shape", [(392, 200), (1032, 264), (520, 1288)], ids=_name)
@pytest.mark.parametrize("m", [160, 161, 176, 191, 192, 193, 208, 224, 256])
def test_gradients_on_either_side_of_the_lines(m, shape):
    """From 161 tokens on the forward products run on pairs, from 193 on those of the gradients that read the weights along their rows."""
    from vllm_plugin_b200 import api
    hidden, inter = shape
    x, w13 = _randn(1, m, hidden, dtype=torch.bfloat16), _randn(2, 2 * inter, hidden, dtype=torch.bfloat16, std=hidden ** -0.5)
    w2, dy = _randn(3, hidden, inter, dtype=torch.bfloat16, std=inter ** -0.5), _randn(4, m, hidden, dtype=torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    y = api.gated_feed_forward(*leaves, activation_clamp=1.25)
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    ref = R.Block(*leaves, 1.25, dy)
    R.check("y", y.detach(), ref.y, ref.off["y"])
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        R.check(name, got, getattr(ref, name), ref.off[name])
    dx, = torch.autograd.grad(y, leaves[:1], dy)
    assert torch.equal(dx, grads[0])
