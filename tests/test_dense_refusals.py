"""Dense feed-forward operators without a GPU: every refusal of the C interface comes before anything is launched, and there is no CPU path."""

import ctypes
import math

import pytest
import torch

FAKE = 1 << 20          # an aligned address that nobody follows


def _native():
    from vllm_plugin_b200.backend import _native as N
    return N


def _block(**change):
    a = dict(type=0, hidden=64, intermediate=32, num_tokens=5, clamp=math.inf, timeout_ms=0, x_stride=64, x=FAKE, w13=FAKE, w2=FAKE, h=FAKE, preact=FAKE,
             y=FAKE, status=FAKE)
    return _native().MmoeFeedForward(**{**a, **change})


def _product(**change):
    a = dict(num_tokens=5, width=64, channels=24, out_type=0, clamp=math.inf, timeout_ms=0, x_stride=64, x=FAKE, x_scales=FAKE, w=FAKE, w_scales=FAKE,
             bias=None, out=FAKE, status=FAKE)
    return _native().MmoeInt8Product(**{**a, **change})


def _refused(code):
    N = _native()
    assert code == N.MMOE_ERR_INVALID_ARGUMENT
    with pytest.raises(AssertionError):
        N.check(code)


@pytest.mark.parametrize("change", [dict(type=2), dict(type=3), dict(type=-1), dict(hidden=0), dict(hidden=60), dict(intermediate=4), dict(intermediate=-8),
                                    dict(num_tokens=-1), dict(clamp=0.0), dict(clamp=-3.0), dict(clamp=math.nan), dict(x_stride=56), dict(x_stride=68),
                                    dict(x=None), dict(w13=None), dict(w2=None), dict(status=None), dict(x=FAKE + 2), dict(w13=FAKE + 8), dict(w2=FAKE + 1),
                                    dict(h=FAKE + 4), dict(preact=FAKE + 4), dict(y=FAKE + 8)])
def test_feed_forward_arguments(change):
    lib = _native().load()
    a = _block(**change)
    _refused(lib.mmoe_feed_forward(ctypes.byref(a), None))
    _refused(lib.mmoe_feed_forward_grad(ctypes.byref(a), FAKE, FAKE, FAKE, FAKE, FAKE, None))


def test_sizes_past_32_bit_indexes():
    lib = _native().load()
    for change in (dict(num_tokens=2**30 + 1), dict(hidden=2**29 + 8, x_stride=2**29 + 8), dict(intermediate=2**29 + 8)):
        a = _block(**change)
        _refused(lib.mmoe_feed_forward(ctypes.byref(a), None))
        _refused(lib.mmoe_feed_forward_grad(ctypes.byref(a), FAKE, FAKE, FAKE, FAKE, FAKE, None))
    for change in (dict(num_tokens=2**31 - 1), dict(channels=2**29 + 1)):
        _refused(lib.mmoe_int8_projection(ctypes.byref(_product(**change)), None))
        _refused(lib.mmoe_int8_gated_projection(ctypes.byref(_product(**change)), None))


def test_feed_forward_outputs():
    lib = _native().load()
    for change in (dict(h=None), dict(y=None)):
        a = _block(**change)
        _refused(lib.mmoe_feed_forward(ctypes.byref(a), None))
    _refused(lib.mmoe_feed_forward(None, None))
    _refused(lib.mmoe_feed_forward_grad(None, FAKE, FAKE, FAKE, FAKE, FAKE, None))
    a = _block()
    for args in ((None, FAKE, FAKE, FAKE, FAKE), (FAKE, None, FAKE, None, None), (FAKE, None, None, FAKE, None), (FAKE + 2, FAKE, FAKE, FAKE, FAKE),
                 (FAKE, FAKE + 2, FAKE, FAKE, FAKE), (FAKE, FAKE, FAKE + 4, FAKE, FAKE), (FAKE, FAKE, FAKE, FAKE + 8, FAKE), (FAKE, FAKE, FAKE, FAKE, FAKE + 8)):
        _refused(lib.mmoe_feed_forward_grad(ctypes.byref(a), *args, None))
    a = _block(preact=None)
    _refused(lib.mmoe_feed_forward_grad(ctypes.byref(a), FAKE, FAKE, FAKE, None, None, None))
    a = _block(h=None)
    _refused(lib.mmoe_feed_forward_grad(ctypes.byref(a), FAKE, FAKE, None, None, FAKE, None))
    assert lib.mmoe_feed_forward(ctypes.byref(_block(num_tokens=0, x=None, h=None, y=None)), None) == 0


@pytest.mark.parametrize("change", [dict(num_tokens=-1), dict(width=0), dict(width=40), dict(width=131072), dict(channels=0), dict(out_type=2), dict(out_type=4),
                                    dict(x_stride=48), dict(x_stride=72), dict(x=None), dict(x_scales=None), dict(w=None), dict(w_scales=None),
                                    dict(out=None), dict(status=None), dict(x=FAKE + 8), dict(w=FAKE + 1), dict(out=FAKE + 4)])
def test_int8_arguments(change):
    lib = _native().load()
    a = _product(**change)
    _refused(lib.mmoe_int8_projection(ctypes.byref(a), None))
    _refused(lib.mmoe_int8_gated_projection(ctypes.byref(a), None))


def test_int8_other_arguments():
    lib = _native().load()
    for clamp in (0.0, -1.0, math.nan):
        _refused(lib.mmoe_int8_gated_projection(ctypes.byref(_product(clamp=clamp)), None))
    _refused(lib.mmoe_int8_projection(None, None))
    assert lib.mmoe_int8_projection(ctypes.byref(_product(num_tokens=0, x=None, out=None)), None) == 0
    for args in ((FAKE, 2, 64, FAKE, FAKE, 5, 64), (FAKE, 3, 64, FAKE, FAKE, 5, 64), (FAKE, 0, 63, FAKE, FAKE, 5, 64), (FAKE, 0, 64, FAKE, FAKE, -1, 64),
                 (FAKE, 0, 64, FAKE, FAKE, 5, 0), (None, 0, 64, FAKE, FAKE, 5, 64), (FAKE, 0, 64, None, FAKE, 5, 64), (FAKE, 0, 64, FAKE, None, 5, 64)):
        _refused(lib.mmoe_quantize_int8(*args, None))
    assert lib.mmoe_quantize_int8(None, 0, 64, None, None, 0, 64, None) == 0
    _refused(lib.mmoe_dense_read_status(None, None, None))


def test_there_is_no_cpu_path():
    from vllm_plugin_b200 import api
    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    w13, w2 = torch.zeros((32, 64), dtype=torch.bfloat16), torch.zeros((64, 16), dtype=torch.bfloat16)
    q, s = torch.zeros((3, 64), dtype=torch.int8), torch.ones(3)
    w, sw = torch.zeros((32, 64), dtype=torch.int8), torch.ones(32)
    with pytest.raises(RuntimeError):
        api.gated_feed_forward(x, w13, w2)
    with pytest.raises(ValueError):
        api.prepare_int8_inputs(x)
    with pytest.raises(RuntimeError):
        api.int8_projection(q, s, w, sw)
    with pytest.raises(RuntimeError):
        api.int8_gated_projection(q, s, w, sw)
    if not torch.cuda.is_available():
        with pytest.raises(Exception):
            api.read_dense_status()


def test_quantiser_sizes_past_32_bit_indexes():
    lib = _native().load()
    for tokens, width in ((2**31 - 1, 64), (2**31 - 4095, 8), (5, 2**31 - 1), (5, 2**31 - 4095)):
        _refused(lib.mmoe_quantize_int8(FAKE, 0, max(width, 64), FAKE, FAKE, tokens, width, None))
