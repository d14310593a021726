"""The C interface of the 8-bit products and their quantiser refuses numbers that do not stand on their own size.  Nothing is launched."""

import ctypes

import pytest

from test_grouped_refusals import FAKE, _native, _product, _refused


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name", ["x_scales", "w_scales"])
def test_scales_of_products(name, off):
    lib = _native().load()
    for change in (dict(), dict(num_experts=1, ends=None)):
        a = _product(**{name: FAKE + off}, **change)
        _refused(lib.mmoe_fp8_projection(ctypes.byref(a), None))
        _refused(lib.mmoe_fp8_gated_projection(ctypes.byref(a), None))


def test_quantiser():
    lib = _native().load()
    for kind in (0, 1):
        for x, scales in ((FAKE + 1, FAKE), (FAKE + 3, FAKE), (FAKE, FAKE + 1), (FAKE, FAKE + 2), (FAKE, FAKE + 3)):
            _refused(lib.mmoe_quantize_fp8(x, kind, 64, FAKE, scales, 5, 64, None))
