"""Products of a layer's experts without a GPU: every refusal of the C interface comes before anything is launched, the operators' own come before
anything is made, and there is no CPU path."""

import ctypes
import math
import os
import types

import pytest
import torch

from helpers import ROOT

FAKE = 1 << 20          # an aligned address that nobody follows
E4M3 = torch.float8_e4m3fn


def _native():
    from vllm_plugin_b200.backend import _native as N
    return N


def _refused(code):
    N = _native()
    assert code == N.MMOE_ERR_INVALID_ARGUMENT
    with pytest.raises(AssertionError):
        N.check(code)


def _projection(**change):
    a = dict(type=0, num_rows=5, num_experts=3, width=64, channels=24, timeout_ms=0, x_stride=64, x=FAKE, w=FAKE, ends=FAKE, out=FAKE, status=FAKE)
    return _native().MmoeGroupedProduct(**{**a, **change})


def _block(**change):
    a = dict(type=1, num_rows=5, num_experts=3, hidden=64, intermediate=32, clamp=math.inf, timeout_ms=0, x_stride=64, x=FAKE, w13=FAKE, w2=FAKE, ends=FAKE,
             h=FAKE, preact=FAKE, y=FAKE, status=FAKE)
    return _native().MmoeGroupedFeedForward(**{**a, **change})


def _product(**change):
    a = dict(num_rows=5, num_experts=3, width=64, channels=24, out_type=0, clamp=math.inf, timeout_ms=0, x_stride=64, x=FAKE, x_scales=FAKE, w=FAKE,
             w_scales=FAKE, ends=FAKE, out=FAKE, status=FAKE)
    return _native().MmoeFp8Product(**{**a, **change})


COMMON = [dict(num_rows=-1), dict(num_rows=2**30 + 1), dict(num_experts=0), dict(num_experts=-1), dict(num_experts=1025), dict(ends=None), dict(ends=FAKE + 2),
          dict(x_stride=48), dict(x_stride=68), dict(x=None), dict(status=None), dict(x=FAKE + 8)]


@pytest.mark.parametrize("change", COMMON + [dict(type=2), dict(type=3), dict(type=4), dict(type=-1), dict(width=0), dict(width=60), dict(width=2**20 + 8, x_stride=2**21),
                                             dict(channels=0), dict(channels=4), dict(channels=-8), dict(channels=2**20 + 8), dict(w=None), dict(w=FAKE + 8)])
def test_projection_arguments(change):
    lib = _native().load()
    a = _projection(**change)
    _refused(lib.mmoe_grouped_projection(ctypes.byref(a), None))
    _refused(lib.mmoe_grouped_projection_grad(ctypes.byref(a), FAKE, FAKE, FAKE, None))


def test_projection_outputs():
    lib = _native().load()
    _refused(lib.mmoe_grouped_projection(None, None))
    _refused(lib.mmoe_grouped_projection_grad(None, FAKE, FAKE, FAKE, None))
    for out in (None, FAKE + 4):
        _refused(lib.mmoe_grouped_projection(ctypes.byref(_projection(out=out)), None))
    a = _projection(out=None)
    for args in ((None, FAKE, FAKE), (FAKE + 8, FAKE, FAKE), (FAKE, FAKE + 8, FAKE), (FAKE, FAKE, FAKE + 4)):
        _refused(lib.mmoe_grouped_projection_grad(ctypes.byref(a), *args, None))
    assert lib.mmoe_grouped_projection(ctypes.byref(_projection(num_rows=0, x=None, out=None, status=None)), None) == 0
    assert lib.mmoe_grouped_projection_grad(ctypes.byref(_projection(num_rows=0, x=None, out=None, status=None)), None, None, None, None) == 0


@pytest.mark.parametrize("change", COMMON + [dict(type=2), dict(type=4), dict(hidden=0), dict(hidden=60), dict(intermediate=4), dict(intermediate=-8),
                                             dict(intermediate=2**20 + 8), dict(clamp=0.0), dict(clamp=-3.0), dict(clamp=math.nan), dict(w13=None), dict(w2=None),
                                             dict(w13=FAKE + 8), dict(w2=FAKE + 1), dict(h=FAKE + 4), dict(preact=FAKE + 4), dict(y=FAKE + 8)])
def test_feed_forward_arguments(change):
    lib = _native().load()
    a = _block(**change)
    _refused(lib.mmoe_grouped_feed_forward(ctypes.byref(a), None))
    _refused(lib.mmoe_grouped_feed_forward_grad(ctypes.byref(a), FAKE, FAKE, FAKE, FAKE, FAKE, None))


def test_feed_forward_outputs():
    lib = _native().load()
    for change in (dict(h=None), dict(y=None)):
        _refused(lib.mmoe_grouped_feed_forward(ctypes.byref(_block(**change)), None))
    _refused(lib.mmoe_grouped_feed_forward(None, None))
    _refused(lib.mmoe_grouped_feed_forward_grad(None, FAKE, FAKE, FAKE, FAKE, FAKE, None))
    a = _block()
    for args in ((None, FAKE, FAKE, FAKE, FAKE), (FAKE, None, FAKE, None, None), (FAKE, None, None, FAKE, None), (FAKE + 2, FAKE, FAKE, FAKE, FAKE),
                 (FAKE, FAKE + 2, FAKE, FAKE, FAKE), (FAKE, FAKE, FAKE + 4, FAKE, FAKE), (FAKE, FAKE, FAKE, FAKE + 8, FAKE), (FAKE, FAKE, FAKE, FAKE, FAKE + 8)):
        _refused(lib.mmoe_grouped_feed_forward_grad(ctypes.byref(a), *args, None))
    _refused(lib.mmoe_grouped_feed_forward_grad(ctypes.byref(_block(preact=None)), FAKE, FAKE, FAKE, None, None, None))
    _refused(lib.mmoe_grouped_feed_forward_grad(ctypes.byref(_block(h=None)), FAKE, FAKE, None, None, FAKE, None))
    assert lib.mmoe_grouped_feed_forward(ctypes.byref(_block(num_rows=0, x=None, h=None, y=None, status=None)), None) == 0


@pytest.mark.parametrize("change", COMMON + [dict(width=0), dict(width=40), dict(width=2**20 + 16, x_stride=2**21), dict(channels=0), dict(channels=2**20 + 1),
                                             dict(out_type=2), dict(out_type=4), dict(out_type=-1), dict(x_scales=None), dict(w=None), dict(w_scales=None), dict(out=None),
                                             dict(w=FAKE + 1), dict(out=FAKE + 4)])
def test_fp8_arguments(change):
    lib = _native().load()
    a = _product(**change)
    _refused(lib.mmoe_fp8_projection(ctypes.byref(a), None))
    _refused(lib.mmoe_fp8_gated_projection(ctypes.byref(a), None))


def test_fp8_other_arguments():
    lib = _native().load()
    for clamp in (0.0, -1.0, math.nan):
        _refused(lib.mmoe_fp8_gated_projection(ctypes.byref(_product(clamp=clamp)), None))
    _refused(lib.mmoe_fp8_gated_projection(ctypes.byref(_product(channels=20)), None))
    _refused(lib.mmoe_fp8_projection(None, None))
    _refused(lib.mmoe_fp8_gated_projection(None, None))
    for rows in (-1, 2**30 + 1):
        _refused(lib.mmoe_fp8_projection(ctypes.byref(_product(num_experts=1, ends=None, num_rows=rows)), None))
    assert lib.mmoe_fp8_projection(ctypes.byref(_product(num_rows=0, x=None, out=None, status=None)), None) == 0
    assert lib.mmoe_fp8_projection(ctypes.byref(_product(num_rows=0, num_experts=1, ends=None, x=None, out=None, status=None)), None) == 0
    for args in ((FAKE, 2, 64, FAKE, FAKE, 5, 64), (FAKE, 3, 64, FAKE, FAKE, 5, 64), (FAKE, 0, 63, FAKE, FAKE, 5, 64), (FAKE, 0, 64, FAKE, FAKE, -1, 64),
                 (FAKE, 0, 64, FAKE, FAKE, 5, 0), (None, 0, 64, FAKE, FAKE, 5, 64), (FAKE, 0, 64, None, FAKE, 5, 64), (FAKE, 0, 64, FAKE, None, 5, 64),
                 (FAKE, 0, 2**31 - 1, FAKE, FAKE, 5, 2**31 - 1), (FAKE, 0, 64, FAKE, FAKE, 2**31 - 1, 64), (FAKE, 0, 2**30, FAKE, FAKE, 2**30, 2**30)):
        _refused(lib.mmoe_quantize_fp8(*args, None))
    assert lib.mmoe_quantize_fp8(None, 0, 64, None, None, 0, 64, None) == 0


def test_the_structures_are_those_of_the_header(tmp_path):
    """Sizes and places of the members, as a C compiler has them."""
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    N = _native()
    names = ("MmoeGroupedProduct", "MmoeGroupedFeedForward", "MmoeFp8Product")
    lines = []
    for n in names:
        lines.append(f'printf("%zu\\n", sizeof({n}));')
        lines += [f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in getattr(N, n)._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "mmoe.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for n in names:
        s = getattr(N, n)
        want += [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_there_is_no_cpu_path():
    from vllm_plugin_b200 import api
    ends = torch.tensor([1, 3], dtype=torch.int32)
    x, w13, w2 = (torch.zeros(s, dtype=torch.bfloat16) for s in ((3, 64), (2, 32, 64), (2, 64, 16)))
    q, s, w, sw = torch.zeros((3, 64), dtype=E4M3), torch.ones((3, 1)), torch.zeros((32, 64), dtype=E4M3), torch.ones((1, 1))
    for call in (lambda: api.grouped_projection(x, w13, ends), lambda: api.grouped_feed_forward(x, w13, w2, ends), lambda: api.fp8_projection(q, s, w, sw),
                 lambda: api.fp8_gated_projection(q, s, w, sw)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError):
        api.prepare_fp8_inputs(x)


@pytest.fixture
def stubbed(monkeypatch):
    """The operators on CPU tensors; the C library writes nothing.  The list of what was called."""
    class Event:
        def record(self, *args):
            pass

        def query(self):
            return True

        def synchronize(self):
            pass

    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t, *a: t)
    from vllm_plugin_b200.backend import dense as D, grouped as G
    calls = []
    lib = types.SimpleNamespace(**{n: (lambda *a, n=n: calls.append(n) or 0) for n in (
        "mmoe_grouped_projection", "mmoe_grouped_projection_grad", "mmoe_grouped_feed_forward", "mmoe_grouped_feed_forward_grad")})
    monkeypatch.setattr(D, "_lib", lib)
    monkeypatch.setattr(D, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(D, "_current_device", lambda: -1)
    monkeypatch.setattr(D, "_capturing", lambda: False)
    monkeypatch.setattr(G, "_check_rows", lambda *a: None)
    monkeypatch.setitem(D._devices, -1, D._Device(torch.device("cpu")))
    return calls


def _inputs(rows=5):
    return (torch.randn(rows, 64).bfloat16(), torch.randn(2, 64, 64).bfloat16(), torch.randn(2, 64, 32).bfloat16(), torch.tensor([2, rows], dtype=torch.int32))


def test_tangents_are_refused(stubbed):
    import torch.autograd.forward_ad as fwd
    from vllm_plugin_b200.backend import grouped as G
    x, w13, w2, ends = _inputs()
    with fwd.dual_level():
        for grad in (False, True):
            for i in range(3):
                a = [t.detach().requires_grad_(grad) for t in (x, w13, w2)]
                a[i] = fwd.make_dual(a[i], torch.ones_like(a[i]))
                with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                    G.grouped_feed_forward(*a, ends)
                if i < 2:
                    with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                        G.grouped_projection(a[0], a[1], ends)
        assert not stubbed
        G.grouped_feed_forward(x, w13, w2, ends)                 # a level by itself is no obstacle
        G.grouped_projection(x, w13, ends)
        leaves = [t.detach().requires_grad_(True) for t in (x, w13, w2)]
        for y, some in ((G.grouped_feed_forward(*leaves, ends), leaves), (G.grouped_projection(*leaves[:2], ends), leaves[:2])):
            torch.autograd.grad(y, some, torch.ones_like(y), retain_graph=True)
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(y, some, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
        scale = fwd.make_dual(torch.ones(5, 1), torch.ones(5, 1))
        with pytest.raises(NotImplementedError, match="forward"):
            G._scales(scale, (5, 1), "x_scales", -1)


def test_traces_are_refused(stubbed):
    from torch.fx.experimental.proxy_tensor import make_fx
    from vllm_plugin_b200.backend import grouped as G
    for rows in (5, 2):
        x, w13, w2, ends = _inputs(rows)
        for run, args in ((G.grouped_feed_forward, (x, w13, w2, ends)), (G.grouped_projection, (x, w13, ends))):
            for grad in (False, True):
                a = tuple(t.clone().requires_grad_(grad) if t.is_floating_point() else t for t in args)
                with pytest.raises((NotImplementedError, TypeError)):
                    torch.jit.trace(lambda *b: run(*b), a, check_trace=False)
                with pytest.raises(NotImplementedError, match="trace"):
                    make_fx(lambda *b: run(*b))(*a)
            y = run(*a)
            with pytest.raises(NotImplementedError, match="trace"):
                make_fx(lambda dy: torch.autograd.grad(y, a[:-1], dy))(torch.ones_like(y))
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(lambda t: G._fp8_product(t, None, None, None, None, torch.bfloat16, 1.0, False))(torch.zeros(5, 64, dtype=E4M3))
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(G.prepare_fp8_inputs)(x, None)


def test_arguments_of_the_operators(stubbed):
    from vllm_plugin_b200.backend import grouped as G
    x, w13, w2, ends = _inputs()
    for bad in (ends.long(), ends[:1], ends[None], [2, 5], ends.float(), torch.tensor([1, 2, 5], dtype=torch.int32)):
        with pytest.raises(AssertionError, match="ends"):
            G.grouped_projection(x, w13, bad)
        with pytest.raises(AssertionError, match="ends"):
            G.grouped_feed_forward(x, w13, w2, bad)
    with pytest.raises(AssertionError):
        G.grouped_projection(x[:, :56], w13, ends)
    with pytest.raises(AssertionError):
        G.grouped_projection(x, w13[0], ends)
    with pytest.raises(AssertionError):
        G.grouped_projection(x, w13.half(), ends)
    with pytest.raises(AssertionError):
        G.grouped_projection(x, w13.transpose(1, 2), ends)
    with pytest.raises(AssertionError, match="multiple of 8"):
        G.grouped_projection(x, torch.zeros(2, 12, 64, dtype=torch.bfloat16), ends)
    with pytest.raises(AssertionError):
        G.grouped_feed_forward(x, w13, w2[:, :, :16].contiguous(), ends)
    with pytest.raises(AssertionError):
        G.grouped_feed_forward(x, w13, w2, ends, activation_clamp=0.0)
    with pytest.raises(AssertionError, match="experts"):
        G.grouped_projection(x, torch.zeros(1025, 8, 64, dtype=torch.bfloat16), torch.zeros(1025, dtype=torch.int32))
    with pytest.raises(AssertionError, match="experts"):
        G.grouped_projection(x, torch.zeros(0, 8, 64, dtype=torch.bfloat16), torch.zeros(0, dtype=torch.int32))
    assert not stubbed
    G.grouped_projection(x, w13, torch.stack((ends, ends), 1)[:, 0])             # any stride
    assert stubbed == ["mmoe_grouped_projection"]


def test_rows_past_32_bit_indexes():
    from vllm_plugin_b200.backend import grouped as G
    row = torch.zeros(1, 64, dtype=torch.bfloat16)
    for rows in (2**32 + 5, 2**31, 2**30 + 1):
        x = types.SimpleNamespace(is_cuda=True, dtype=torch.bfloat16, dim=lambda: 2, shape=(rows, 64))
        with pytest.raises(AssertionError, match="tokens"):
            G._check_rows(x, "grouped_projection")
    G._check_rows(types.SimpleNamespace(is_cuda=True, dtype=torch.bfloat16, dim=lambda: 2, shape=(2**30, 64)), "grouped_projection")
    assert row.shape == (1, 64)


def test_bad_ends_are_named(stubbed):
    """Ends that are not in order are reported as such, once, and not as expert ids of the layer."""
    from vllm_plugin_b200.backend import dense as D
    state = D._Device(torch.device("cpu"))
    state.status[4] = 2
    state.poll.after_call(state, 1)
    with pytest.raises(AssertionError, match="2 launches of earlier grouped operators had ends"):
        state.poll.before_call(state)
    assert not state.status.any()
    state.poll.after_call(state, 1)
    state.poll.before_call(state)


def test_what_the_launch_in_front_writes_is_not_read_as_constant():
    """The launches start beside the ones in front of them, which write their rows, ends and scales: read with ordinary loads, never through the
    read-only path."""
    for name in ("mmoe_grouped.cu", "mmoe_grouped_few.cu", "mmoe_fp8.cu", "mmoe_grouped_device.cuh", "mmoe_grouped.cuh"):
        with open(os.path.join(ROOT, "vllm_plugin_b200", "csrc", name)) as f:
            text = f.read()
        for form in ("__ldg(", "__restrict__", ".nc."):
            assert form not in text, (name, form)
