"""Dense feed-forward operators in fresh processes and in PyTorch's modes."""

import os
import subprocess
import sys

import pytest
import torch
import torch.utils.flop_counter

from helpers import ROOT

pytestmark = pytest.mark.gpu


def _fresh(program):
    """Runs ``program`` in a process that has made no call yet."""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr


def test_a_first_call_in_inference_mode():
    """A serving warm-up, then more calls than lie between two looks at the status words, without a mode and training."""
    _fresh("""
import torch
import torch.utils.flop_counter
from vllm_plugin_b200 import api
x, w13, w2 = (torch.randn(s, device="cuda").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
with torch.inference_mode():
    want = api.gated_feed_forward(x, w13, w2).clone()
for _ in range(80):
    y = api.gated_feed_forward(x, w13, w2)
    torch.cuda.synchronize()
assert torch.equal(y, want)
w13.requires_grad_(True)
for _ in range(80):
    api.gated_feed_forward(x, w13, w2).sum().backward()
    torch.cuda.synchronize()
with torch.inference_mode():
    for _ in range(80):
        api.gated_feed_forward(x, w13, w2)
        torch.cuda.synchronize()
api.read_dense_status()
print("ok")
""")


def test_a_timeout_read_beside_a_queued_copy_is_raised_once():
    from vllm_plugin_b200 import api
    from vllm_plugin_b200.backend import dense as D
    x, w13, w2 = (torch.randn(s, device="cuda:0").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
    want = api.gated_feed_forward(x, w13, w2)
    state = D._on_device(0)
    try:
        api.set_kernel_options(status_poll_interval=1)
        for _ in range(3):
            api.gated_feed_forward(x, w13, w2)
            torch.cuda.synchronize()
        state.status[:4] = torch.tensor([1, 31, 2, 5], dtype=torch.int32)
        torch.cuda.synchronize()
        state.poll.pending = False
        state.poll.after_call(state, 1)                          # the look that a call takes: queued, not yet inspected
        with pytest.raises(RuntimeError, match="kernel 31"):
            api.read_dense_status()
        for _ in range(3):
            assert torch.equal(api.gated_feed_forward(x, w13, w2), want)
            torch.cuda.synchronize()
    finally:
        api.set_kernel_options(status_poll_interval=32)
    api.read_dense_status()


def test_tangents_are_refused():
    """Forward mode, alone and through a backward pass; scales and bias of the 8-bit products and the quantiser's input too."""
    import torch.autograd.forward_ad as fwd
    from vllm_plugin_b200 import api
    x, w13, w2 = (torch.randn(s, device="cuda:0").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
    q, s = api.prepare_int8_inputs(x)
    w, sw = api.prepare_int8_inputs(w13)
    bias = torch.zeros(64, device="cuda:0")
    want = x + api.gated_feed_forward(x, w13, w2)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for args in ((dual(x), w13, w2), (x, dual(w13), w2), (x, w13, dual(w2))):
            with pytest.raises(NotImplementedError):
                api.gated_feed_forward(*args)
        with pytest.raises(NotImplementedError):
            api.prepare_int8_inputs(dual(x))
        for args, b in (((q, dual(s), w, sw), bias), ((q, s, w, dual(sw)), bias), ((q, s, w, sw), dual(bias))):
            with pytest.raises(NotImplementedError):
                api.int8_projection(*args, bias=b)
        with pytest.raises(NotImplementedError):
            api.int8_gated_projection(q, s, w, dual(sw))
        assert torch.equal(x + api.gated_feed_forward(x, w13, w2), want)      # a level by itself is no obstacle
        leaf = x.detach().requires_grad_(True)
        y = api.gated_feed_forward(leaf, w13, w2)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, leaf, dual(torch.ones_like(y)))


def test_traces_are_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    from vllm_plugin_b200 import api
    x, w13, w2 = (torch.randn(s, device="cuda:0").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
    q, s = api.prepare_int8_inputs(x)
    w, sw = api.prepare_int8_inputs(w13)
    for run, args in ((lambda a, b, c: api.gated_feed_forward(a, b, c), (x, w13, w2)), (lambda a: api.prepare_int8_inputs(a), (x,)),
                      (lambda a, b, c, d: api.int8_projection(a, b, c, d), (q, s, w, sw)),
                      (lambda a, b, c, d: api.int8_gated_projection(a, b, c, d), (q, s, w, sw))):
        run(*args)
        with pytest.raises(NotImplementedError):
            make_fx(run)(*args)
        with pytest.raises(NotImplementedError):
            torch.jit.trace(run, args, check_trace=False)
    leaves = [t.clone().requires_grad_(True) for t in (x, w13, w2)]
    y = api.gated_feed_forward(*leaves)
    with pytest.raises(NotImplementedError):                     # the backward pass runs on a thread of its own
        make_fx(lambda dy: torch.autograd.grad(y, leaves, dy, retain_graph=True))(x)
    want = torch.autograd.grad(y, leaves, x)
    with torch.utils.flop_counter.FlopCounterMode(display=False):        # a mode that runs what it sees
        y = api.gated_feed_forward(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, x), want))


def test_the_limit_is_that_of_a_wait_not_of_a_launch():
    """Launches that take longer than the limit of a wait, none of whose waits does: the same results, and nothing recorded."""
    from vllm_plugin_b200 import api
    gen = torch.Generator(device="cuda:0").manual_seed(1)
    m, n, k = 20000, 16384, 16384
    x, w = (torch.randint(-127, 128, (r, k), generator=gen, device="cuda:0", dtype=torch.int32).to(torch.int8) for r in (m, n))
    sx, sw = torch.rand(m, generator=gen, device="cuda:0"), torch.rand(n, generator=gen, device="cuda:0")
    want = api.int8_projection(x, sx, w, sw)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    limit = api.get_kernel_options().timeout_ms
    try:
        api.set_kernel_options(timeout_ms=1)
        start.record()
        got = api.int8_projection(x, sx, w, sw)
        end.record()
        api.read_dense_status()
    finally:
        api.set_kernel_options(timeout_ms=limit)
    assert start.elapsed_time(end) > 2                  # 1.1e13 operations in one launch
    assert torch.equal(got, want)


def test_sizes_past_32_bits_are_refused():
    """Broadcast rows, so that nothing of that size exists: refused before a copy or an output is made."""
    from vllm_plugin_b200 import api
    x, w13, w2 = (torch.randn(s, device="cuda:0").bfloat16() for s in ((1, 64), (64, 64), (64, 32)))
    q, s = api.prepare_int8_inputs(x)
    w, sw = api.prepare_int8_inputs(w13)
    held = torch.cuda.memory_allocated()
    for tokens in (2**32 + 5, 2**32, 2**31):
        with pytest.raises(AssertionError):
            api.gated_feed_forward(x.expand(tokens, 64), w13, w2)
        with pytest.raises(AssertionError):
            api.int8_projection(q.expand(tokens, 64), s.expand(tokens), w, sw)
        with pytest.raises(AssertionError):
            api.int8_gated_projection(q.expand(tokens, 64), s.expand(tokens), w, sw)
        with pytest.raises(ValueError):
            api.prepare_int8_inputs(x.expand(tokens, 64))
        with pytest.raises(ValueError):
            api.prepare_int8_inputs(x[:, :1].expand(1, tokens))
    assert torch.cuda.memory_allocated() == held


def test_a_first_call_of_the_quantiser_in_a_capture():
    """The one operator that needs no preparation."""
    _fresh("""
import torch
from vllm_plugin_b200 import api
x = torch.randn(5, 64, device="cuda").bfloat16()
many = torch.randn(600, 64, device="cuda").half()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s = api.prepare_int8_inputs(x)
    q2, s2 = api.prepare_int8_inputs(many)
graph.replay()
torch.cuda.synchronize()
want, want2 = api.prepare_int8_inputs(x), api.prepare_int8_inputs(many)
assert torch.equal(q, want[0]) and torch.equal(s, want[1]) and torch.equal(q2, want2[0]) and torch.equal(s2, want2[1])
print("ok")
""")


def test_a_first_call_of_the_others_in_a_capture_is_refused():
    _fresh("""
import torch
from vllm_plugin_b200 import api
x, w13, w2 = (torch.randn(s, device="cuda").bfloat16() for s in ((5, 64), (64, 64), (64, 32)))
refused = 0
with torch.cuda.graph(torch.cuda.CUDAGraph()):
    try:
        api.gated_feed_forward(x, w13, w2)
    except RuntimeError:
        refused += 1
y = api.gated_feed_forward(x, w13, w2)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    z = api.gated_feed_forward(x, w13, w2)
graph.replay()
torch.cuda.synchronize()
assert refused == 1 and torch.equal(y, z)
api.read_dense_status()
print("ok")
""")
