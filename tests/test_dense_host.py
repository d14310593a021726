"""Host side of the dense feed-forward operators on the CPU, launches and CUDA's own objects stubbed."""

import types

import pytest
import torch


@pytest.fixture
def stubbed(monkeypatch):
    """Events that are always complete, and host memory that needs no pinning."""
    class Event:
        def record(self, *args):
            pass

        def query(self):
            return True

        def synchronize(self):
            pass

    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t, *a: t)


@pytest.mark.parametrize("make_in_inference", [True, False])
def test_status_words_work_in_any_mode(stubbed, make_in_inference):
    """Whatever mode the first call ran in: polls, reports and the words' reset work outside inference mode and inside."""
    from vllm_plugin_b200.backend import dense as D
    with torch.inference_mode(make_in_inference):
        state = D._Device(torch.device("cpu"))
    assert not state.status.is_inference() and not state.poll.host.is_inference()
    for inference in (False, True, False):
        with torch.inference_mode(inference):
            state.poll.before_call(state)
            state.poll.after_call(state, 1)
            state.poll.before_call(state)
            state.status[:4] = torch.tensor([1, 31, 2, 5], dtype=torch.int32)
            state.poll.after_call(state, 1)
            with pytest.raises(RuntimeError, match="kernel 31"):
                state.poll.before_call(state)
            assert not state.status.any()


def test_a_buffer_made_in_inference_mode_can_be_reset_outside(stubbed, monkeypatch):
    """The layer's own words, which its poll resets as well."""
    from vllm_plugin_b200.backend import frontend as F, workspace as W
    empty = torch.empty

    def aligned(size, **kind):                       # on 1024 bytes, as CUDA's memory is
        room = empty(size + 1024, **kind)
        return room[-room.data_ptr() % 1024:][:size]

    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch, "empty", lambda size, **kind: aligned(size, **kind) if isinstance(size, int) else empty(size, **kind))
    with torch.inference_mode():
        buffer = W.SymmBuffer(types.SimpleNamespace(size=lambda: 1, rank=lambda: 0), 8, 64, 2, 512, 256, device=torch.device("cpu"))
        poll = F._StatusPoll(buffer)
    buffer.status[0] = 1
    poll.after_call(buffer, 1)
    with pytest.raises(RuntimeError, match="expired"):
        poll.before_call(buffer)
    assert not buffer.status.any()


def test_a_read_forgets_the_copy_that_was_queued(stubbed, monkeypatch):
    """A failure that a read has reported and cleared is not raised once more by a copy of the words queued in front of the read."""
    import contextlib
    from vllm_plugin_b200.backend import _native, dense as D, frontend as F
    state = D._Device(torch.device("cpu"))
    raised = []

    def read(*args):                                 # the C call: the words as they are, then cleared
        raised.append(int(state.status[0]))
        state.status.zero_()
        return 0

    monkeypatch.setattr(F, "require_sm100", lambda: None)
    monkeypatch.setattr(_native, "load", lambda: types.SimpleNamespace(mmoe_dense_read_status=read, mmoe_read_status=read))
    monkeypatch.setattr(_native, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    monkeypatch.setitem(D._devices, 0, state)
    buffer = types.SimpleNamespace(device=None, geo=_native.MmoeGeometry(), base_ptr=0, status=state.status, _status_poll=state.poll)
    for reader in (lambda: D.read_dense_status("cuda:0"), lambda: F.read_status(buffer)):
        state.status[:4] = torch.tensor([1, 31, 2, 5], dtype=torch.int32)
        state.poll.after_call(state, 1)
        assert state.poll.pending
        reader()
        assert raised.pop() == 1 and not state.status.any()
        state.status[0] = 1                          # what a newer call leaves stays for the next look
        state.poll.before_call(state)
        assert state.status[0] == 1
        state.status.zero_()
    buffer._status_poll = None                       # no call has looked yet
    F.read_status(buffer)


def test_a_timeout_names_the_kind_of_call(stubbed):
    from vllm_plugin_b200.backend import dense as D, frontend as F
    state = D._Device(torch.device("cpu"))
    for poll, name in ((state.poll, "dense operator's call"), (F._StatusPoll(state), "MegaMoE call")):
        state.status[0] = 1
        poll.after_call(state, 1)
        with pytest.raises(RuntimeError, match=f"wait of an earlier {name} expired"):
            poll.before_call(state)


@pytest.fixture
def launches(stubbed, monkeypatch):
    """The operators on CPU tensors; the C library writes nothing.  The list of what was called."""
    from vllm_plugin_b200.backend import dense as D
    calls = []
    lib = types.SimpleNamespace(**{n: (lambda *a, n=n: calls.append(n) or 0) for n in (
        "mmoe_feed_forward", "mmoe_feed_forward_grad", "mmoe_quantize_int8", "mmoe_int8_projection")})
    monkeypatch.setattr(D, "_lib", lib)
    monkeypatch.setattr(D, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(D, "_current_device", lambda: -1)
    monkeypatch.setattr(D, "_capturing", lambda: False)
    monkeypatch.setattr(D, "_check_block", lambda *a: None)
    monkeypatch.setitem(D._devices, -1, D._Device(torch.device("cpu")))
    return calls


def _block():
    return torch.randn(5, 64).bfloat16(), torch.randn(64, 64).bfloat16(), torch.randn(64, 32).bfloat16()


def test_tangents_are_refused(launches):
    """Forward-mode derivatives through any input, and through the gradient of the output, with and without a backward graph."""
    import torch.autograd.forward_ad as fwd
    from vllm_plugin_b200.backend import dense as D
    args = _block()
    with fwd.dual_level():
        for grad in (False, True):
            for i in range(3):
                inputs = [t.detach().requires_grad_(grad) for t in args]
                inputs[i] = fwd.make_dual(inputs[i], torch.ones_like(inputs[i]))
                for run in (D.gated_feed_forward, torch.no_grad()(D.gated_feed_forward)):
                    with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                        run(*inputs)
        assert not launches
        scale = fwd.make_dual(torch.ones(5), torch.ones(5))
        with pytest.raises(NotImplementedError, match="forward"):
            D._float_vector(scale, (5,), "x_scales", -1)
        D.gated_feed_forward(*args)                          # a level by itself is no obstacle
        D._float_vector(torch.ones(5), (5,), "x_scales", -1)
        assert launches == ["mmoe_feed_forward"]
        inputs = [t.detach().requires_grad_(True) for t in args]
        y = D.gated_feed_forward(*inputs)
        torch.autograd.grad(y, inputs, torch.ones_like(y), retain_graph=True)
        with pytest.raises(NotImplementedError, match="forward"):
            torch.autograd.grad(y, inputs, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
        with fwd._set_fwd_grad_enabled(False):               # as inference mode has it: nobody asks for tangents
            D.gated_feed_forward(fwd.make_dual(args[0], args[0]), *args[1:])
    D.gated_feed_forward(*args)


def test_traces_are_refused(launches):
    """torch.jit.trace and make_fx would record the allocation of the output and not what fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    from vllm_plugin_b200.backend import dense as D
    for tokens in (5, 0):
        x, w13, w2 = _block()
        x = x[:tokens]

        def forward(a, b, c):
            return D.gated_feed_forward(a, b, c)

        def gradient(a, b, c):
            return torch.autograd.grad(D.gated_feed_forward(a, b, c), (a, b, c), torch.ones_like(a))

        for grad in (False, True):
            args = tuple(t.clone().requires_grad_(grad) for t in (x, w13, w2))
            with pytest.raises((NotImplementedError, TypeError)):           # TypeError: with gradients PyTorch's own, at the function's number argument
                torch.jit.trace(forward, args, check_trace=False)
            for early in (False, True):
                with pytest.raises(NotImplementedError, match="trace"):
                    make_fx(gradient if grad else forward, pre_dispatch=early)(*args)
        args = tuple(t.clone().requires_grad_(True) for t in (x, w13, w2))
        y = D.gated_feed_forward(*args)
        with pytest.raises(NotImplementedError, match="trace"):                                  # the gradient alone
            make_fx(lambda dy: torch.autograd.grad(y, args, dy))(torch.ones_like(y))

    class Counts(TorchDispatchMode):                     # a mode that runs what it sees is no trace
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    launches.clear()
    with Counts(), torch.device("cpu"):
        D.gated_feed_forward(*_block())
    assert launches == ["mmoe_feed_forward"]
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(lambda t: D._int8_product(t, None, None, None, None, torch.bfloat16, 1.0, False))(torch.zeros(5, 64, dtype=torch.int8))
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(D.prepare_int8_inputs)(_block()[0], None)


def test_what_the_launch_in_front_writes_is_not_read_as_constant():
    """The dense launches start beside the ones in front of them, which write their tokens, scales, weights and bias: behind the wait they
    are read with ordinary loads, never through the read-only path, which is for memory that nobody writes while a kernel runs."""
    import os
    from helpers import ROOT
    for name in ("mmoe_dense.cu", "mmoe_dense.cuh"):
        with open(os.path.join(ROOT, "vllm_plugin_b200", "csrc", name)) as f:
            text = f.read()
        for form in ("__ldg(", "__restrict__", ".nc."):
            assert form not in text, (name, form)


def test_sizes_past_32_bits_are_refused_before_anything_is_made(launches):
    """The C interface takes 32-bit sizes; what does not fit is not cut to its low bits.  Broadcast tensors: nothing of that size exists."""
    from vllm_plugin_b200.backend import dense as D
    x, w13, w2 = _block()
    for tokens in (2**32 + 5, 2**32, 2**31, 2**30 + 1):
        many = x[:1].expand(tokens, 64)
        for rows in (many, many.view(1, tokens, 64)):
            with pytest.raises(AssertionError, match="tokens"):
                D._rows(rows)
        with pytest.raises(AssertionError, match="tokens"):
            D.gated_feed_forward(many, w13, w2)
        rows = types.SimpleNamespace(shape=(tokens, 64))                       # dense rows, of which no copy would be made
        with pytest.raises(AssertionError, match="tokens"):
            D._launch_block(rows, w13, w2, 1.0, False)
    assert not launches
    D.gated_feed_forward(x[:1].expand(7, 64), w13, w2)
    assert launches


def test_first_calls_at_once_find_all_of_the_library(monkeypatch):
    """A thread that finds the library loaded by another one finds the look-up of streams as well, at every line in between."""
    import sys
    from vllm_plugin_b200.backend import _native, dense as D
    monkeypatch.setattr(D, "_lib", None)
    monkeypatch.setattr(D, "_raw_stream", None)
    monkeypatch.setattr(_native, "load", lambda: object())
    half = []

    def watch(frame, event, arg):
        if frame.f_code is D._library.__code__:
            half.append(D._lib is not None and D._raw_stream is None)
            return watch

    sys.settrace(watch)
    try:
        D._library()
    finally:
        sys.settrace(None)
    assert half and not any(half) and D._lib is not None and D._raw_stream is not None


def test_live_graphs_are_listed_while_others_are_made(monkeypatch):
    """Eager calls of other threads come and go while a captured call looks through the live graphs."""
    import sys
    import threading
    from vllm_plugin_b200.backend import dense as D

    class Node:
        next_functions = ()

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    stop, wrong = threading.Event(), []

    def make():
        while not stop.is_set():
            nodes = [Node() for _ in range(50)]
            for n in nodes:
                D._remember(n)

    threads = [threading.Thread(target=make) for _ in range(3)]
    try:
        for t in threads:
            t.start()
        kept = Node()
        D._remember(kept)
        for _ in range(3000):
            if kept not in D._live_graphs():
                wrong.append("lost")
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
    assert not wrong
    del kept, make
    threads.clear()
    import gc
    gc.collect()
    assert not D._live_graphs()


def test_the_combine_does_not_read_its_inputs_as_constant():
    """What it adds is written by launches in front of it, beside which it starts: the routed rows, and a residual that a dense operator left or that is
    the output itself.  No restrict pointers, so that nothing tells the compiler that they stay as they are."""
    import os
    import re
    from helpers import ROOT
    with open(os.path.join(ROOT, "vllm_plugin_b200", "csrc", "mmoe_support.cu")) as f:
        text = f.read()
    for name in ("combine_narrow_kernel", "combine_kernel"):
        (arguments,) = re.findall(rf"__launch_bounds__\(256\) {name}\((.*?)\) {{", text, re.S)
        assert "residual" in arguments and "__restrict__" not in arguments, name
