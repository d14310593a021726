"""How exact the activation is where it is the only thing that is rounded: the gated product of 8-bit integers with an FP32 result."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("clamp", [None, 10.0])
@pytest.mark.parametrize("m", [1, 37, 300])
def test_activation_over_the_whole_range(m, clamp):
    """g from -103 to 103 and u, both exact in FP32.  Bound: the exponential is good to 2^-22 and its correction rounds once (2^-24), the
    reciprocal to 2^-23, the sum and three products round once each: 11 * 2^-24, below 2^-20 of the value.  Where e^g is no normal number, 2 units of
    2^-149 of it, times g and u."""
    from vllm_plugin_b200 import api
    n, k = 255, 48
    steps = torch.arange(-127, 128, device=DEV)
    x = torch.zeros(m, k, dtype=torch.int8, device=DEV)
    x[:, 0], x[:, 17] = 1, 1
    x[m // 2:, 17] = -3
    w = torch.zeros(2 * n, k, dtype=torch.int8, device=DEV)
    w[:n, 0], w[n:, 17] = steps.to(torch.int8), 3
    sw = torch.full((2 * n,), 0.8125, device=DEV)
    sw[n:] = 0.5
    h = api.int8_gated_projection(x, torch.ones(m, device=DEV), w, sw, activation_clamp=clamp, out_dtype=torch.float32).double()
    g = (steps.double() * 0.8125).expand(m, n)
    u = (x[:, 17].double() * 1.5)[:, None]
    if clamp is not None:
        u = u.clamp(-clamp, clamp)
        gc = g.clamp(max=clamp)
    else:
        gc = g
    want = gc / (1 + torch.exp(-gc)) * u
    off = 2.0 ** -20 * want.abs() + 2.0 ** -148 * (gc * u).abs() + 2.0 ** -149
    worst = ((h - want).abs() / off).max(0).values
    assert bool((worst <= 1).all()), [(float(g[0, i]), float(worst[i])) for i in torch.nonzero(worst > 1).flatten().tolist()[:8]]
