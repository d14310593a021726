"""The 8-bit floating point quantiser where a group's values are so far apart that quotients leave the numbers of 32 bits."""

import pytest
import torch

import grouped_reference as G
from test_gpu_fp8 import E4M3

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _groups(exponents):
    """A row for each scale ``2 ** e``: its largest value, and values on a border each beside one far below it (and eight places from one, as those are
    neighbours that are read one by one), either first, either sign."""
    codes = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    borders = (codes[1:] + codes[:-1]) / 2
    rows = []
    for e in exponents:
        row = torch.zeros(128, dtype=torch.float64)
        for i in range(0, 126, 2):
            near, sign = borders[(7 * i + e) % len(borders)] * 2.0 ** e, -1.0 if i % 8 < 4 else 1.0
            far = -sign * 2.0 ** max(-133, min(e - 151 - i % 5, e - 150)) if i % 3 else sign * 2.0 ** -133
            row[i], row[i + 1] = (sign * near, far) if (i // 2 + i // 8) % 2 else (far, sign * near)
        row[126] = 448 * 2.0 ** e
        rows.append(row)
    return torch.stack(rows)


@pytest.mark.parametrize("width", [128, 127, 256])
def test_quotients_far_below_the_smallest_number(width):
    """Zeros with the value's sign, whatever is beside them: 128 and 256 are read eight values at a time, 127 one by one (without the last zero)."""
    from vllm_plugin_b200 import api
    x = _groups(range(17, 119))
    assert torch.equal(x, x.to(torch.bfloat16).double())
    if width == 256:
        x = torch.cat((x, x.flip(1)), 1)
    x = x[:, :width].to(torch.bfloat16).to(DEV)
    for rows in (x, -x):
        q, s = api.prepare_fp8_inputs(rows)
        want_q, want_s = G.quantize(rows)
        assert torch.equal(s, want_s)
        assert torch.equal(q.double(), want_q)
        assert torch.equal(q.view(torch.uint8) >> 7, rows.signbit().to(torch.uint8))
