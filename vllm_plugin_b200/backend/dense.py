"""Dense feed-forward operators beside the MegaMoE layer: the gated block of a model's dense layers (or of a shared expert
that is not MXFP8) in 16 bits with its gradients, and the same block's products in 8-bit integers, with a scale per token and
one per channel, behind their per-token quantiser.  The reference has no counterpart.

Every function launches on the current stream of its tensors' device and never synchronises (but the first call on a device, which
prepares the kernels and therefore has to come before CUDA-graph capture).  Errors are those of the layer: ``AssertionError`` for
arguments, ``ValueError`` in the quantiser, ``NotImplementedError`` for what is not supported, ``RuntimeError`` for the wrong
device, a first call inside a capture, and waits on the device that expired.
"""

from __future__ import annotations

import ctypes
import math
import sys
import weakref
from typing import Dict, Optional, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _native
from . import frontend as _f

_CODES = {torch.bfloat16: _native.MMOE_BF16, torch.float16: _native.MMOE_FP16, torch.float32: _native.MMOE_FP32}
_FF_TYPES = (torch.bfloat16, torch.float16)


# ---------------------------------------------------------------------------------------------------------------------
# per device: prepared kernels, and the words in which they record that a wait expired
# ---------------------------------------------------------------------------------------------------------------------
class _Device:
    def __init__(self, device: torch.device):
        with torch.inference_mode(False):    # kept for calls in any mode, whatever the first one runs in
            self.status = torch.zeros(8, dtype=torch.int32, device=device)
        self.status_ptr = self.status.data_ptr()
        self.poll = _f._StatusPoll(self, "dense operator's call", "launches of earlier grouped operators had ends that fall or pass the last row: "
                                                                  "no row was taken to be an expert's")
        self.calls = self.due = 0            # launching calls so far, and the one at which to look at the words ...
        self.options = None                  # ... by these options


_devices: Dict[int, _Device] = {}
_byref = ctypes.byref
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)


def _prepare(index: int) -> _Device:
    _f.require_sm100()
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the dense operators must be called once on a device before CUDA-graph capture")
    _native.check(_native.load().mmoe_dense_prepare(_native.raw_stream(index)))
    state = _Device(torch.device("cuda", index))
    torch.cuda.synchronize(index)                   # the words are zero before a call on another stream may look at them
    return _devices.setdefault(index, state)


def _on_device(index: int) -> _Device:
    """State of the current device ``index``, made at the first call."""
    return _devices.get(index) or _prepare(index)


def _library():
    """The C library; what a call looks up is kept from here on."""
    global _lib, _raw_stream
    _raw_stream = torch._C._cuda_getCurrentRawStream    # first: a thread that finds the library takes this to be there
    _lib = _native.load()
    return _lib


_lib = _raw_stream = None


def _launch(function, index: int, arguments, *more) -> None:
    """One call of the C library on the current stream of device ``index``: ``arguments`` is its structure but for the status words."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return _launch(function, index, arguments, *more)
    state = _devices.get(index) or _prepare(index)
    options = _f._kernel_options
    arguments.status = state.status_ptr
    arguments.timeout_ms = options.timeout_ms
    state.calls += 1
    if state.calls >= state.due or options is not state.options:
        _watch(state, options)
    code = function(_byref(arguments), *more, _raw_stream(index))
    if code:
        _native.check(code)


def _watch(state: _Device, options) -> None:
    """Non-blocking look at the status words, as the layer's calls take it: every so many eager calls a copy of the words is queued, and a
    later call that finds it complete raises what it says."""
    interval = options.status_poll_interval
    state.options = options
    state.due = state.calls + 1
    if interval <= 0 or _capturing():
        return
    state.poll.before_call(state)
    if not state.poll.pending:
        if state.calls >= state.poll.calls + interval:
            state.poll.calls = state.calls - 1
            state.poll.after_call(state, 1)
        else:
            state.due = state.poll.calls + interval


def read_dense_status(device=None) -> None:
    """Synchronise and raise ``RuntimeError`` if a device-side wait of a dense or grouped operator expired on ``device`` since the last
    read, ``AssertionError`` if the ``ends`` of a grouped one were not in order; clears the condition."""
    _f.require_sm100()
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    with torch.cuda.device(index):
        state = _on_device(index)
        words = (ctypes.c_int32 * 8)()
        code = _native.load().mmoe_dense_read_status(state.status_ptr, words, _native.raw_stream(index))
        state.poll.forget()
        _native.check(code)


# ---------------------------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------------------------
def _clamp_of(activation_clamp: Optional[float]) -> float:
    if activation_clamp is None:
        return math.inf
    value = float(activation_clamp)
    if not value > 0:
        raise AssertionError("activation_clamp must be positive")
    return value


# the C interface's limits.  Its sizes have 32 bits, of which ctypes would take the low ones
_MOST_TOKENS, _MOST_CHANNELS, _MOST_QUANTIZED = 1 << 30, 1 << 29, 2**31 - 4096


def _too_many(tokens: int) -> AssertionError:
    return AssertionError(f"{tokens} tokens: at most {_MOST_TOKENS}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as ``(rows, width)`` whose rows are dense and start on 16 bytes: a view where there is one, else a copy."""
    if t.is_contiguous():
        r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
        return r if r.data_ptr() % 16 == 0 else r.clone()
    r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    tokens, width = r.shape
    if tokens > _MOST_TOKENS:                    # before a copy of them is made
        raise _too_many(tokens)
    dense = r.stride(1) == 1 or width == 1
    if tokens > 1:
        dense = dense and r.stride(0) >= width and r.stride(0) * r.element_size() % 16 == 0
    return r if dense and r.data_ptr() % 16 == 0 else r.clone(memory_format=torch.contiguous_format)


def _stride(r: torch.Tensor) -> int:
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def _refuse_weight(w: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device) -> None:
    if w.dim() != 2 or w.dtype != dtype:
        raise AssertionError(f"{what} must be 2-D {dtype}, got {tuple(w.shape)} {w.dtype}")
    if w.device != device:
        raise AssertionError(f"{what} must be on {device}, got {w.device}")
    raise AssertionError(f"{what} must be contiguous and 16-byte aligned")


def _check_weight(w: torch.Tensor, what: str, dtype: torch.dtype, x: torch.Tensor) -> None:
    if w.dtype is not dtype or w.dim() != 2 or not w.is_contiguous() or w.data_ptr() % 16 != 0 or w.get_device() != x.get_device():
        _refuse_weight(w, what, dtype, x.device)


def _refuse_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """To be called inside a level of forward-mode differentiation only (``_forward_ad._current_level >= 0``).  Outputs are written where
    PyTorch does not see it: they would come back without a tangent, and what is computed from them with a wrong one."""
    if torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")


# A trace, or a mode of PyTorch that may be one, is on when one of these is not zero.  Asked in place: a call of 11 us is 0.2 us longer for a function's sake.
_tracing, _dispatch_modes, _function_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack


def _refuse_traces(what: str) -> None:
    """A trace records the allocation of an output and not the launch that fills it.  Modes that run what they see are no obstacle."""
    tracer = sys.modules.get("torch.fx.experimental.proxy_tensor")
    if _tracing() or (tracer is not None and tracer.get_proxy_mode() is not None):
        raise NotImplementedError(f"{what} cannot be traced (torch.jit.trace, make_fx)")


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------
def _check_block(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError("gated_feed_forward runs on the GPU only (there is no CPU path).")
    dtype = x.dtype
    if dtype not in _FF_TYPES or x.dim() < 1:
        raise AssertionError(f"x must be BF16 or FP16 (..., H), got {tuple(x.shape)} {dtype}")
    _check_weight(w13, "w13", dtype, x)
    _check_weight(w2, "w2", dtype, x)
    hidden, inter = w2.shape
    if x.shape[-1] != hidden or w13.shape != (2 * inter, hidden):
        raise AssertionError(f"expected x (..., H), w13 (2 I, H) and w2 (H, I), got {tuple(x.shape)}, {tuple(w13.shape)} and {tuple(w2.shape)}")
    if hidden <= 0 or inter <= 0 or hidden % 8 != 0 or inter % 8 != 0:
        raise AssertionError(f"H={hidden} and I={inter} must be positive multiples of 8")


def _launch_block(x2: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, clamp: float, keep: bool):
    """``(y, kept)`` of rows ``x2``: ``kept`` holds h, and behind it (``keep``) g and u for the backward pass, in bytes."""
    tokens, hidden = x2.shape
    inter = w2.shape[1]
    if tokens > _MOST_TOKENS:
        raise _too_many(tokens)
    y = x2.new_empty((tokens, hidden))
    kept = x2.new_empty(tokens * inter * (5 if keep else 1))       # 16-bit elements: 1 for h, 2 x 2 for g and u
    if tokens > 0:
        h = kept.data_ptr()
        _launch((_lib or _library()).mmoe_feed_forward, x2.get_device(),
                _native.MmoeFeedForward(_CODES[x2.dtype], hidden, inter, tokens, clamp, 0, _stride(x2), x2.data_ptr(), w13.data_ptr(),
                                        w2.data_ptr(), h, h + 2 * tokens * inter if keep else None, y.data_ptr()))
    return y, kept


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _launch_block_grad(x2, w13, w2, kept, dy2, clamp: float, wanted):
    tokens, hidden = x2.shape
    inter = w2.shape[1]
    inner = wanted[0] or wanted[1]
    dx = x2.new_empty((tokens, hidden)) if wanted[0] else None
    dw13 = w13.new_empty(w13.shape) if wanted[1] else None
    dw2 = w2.new_empty(w2.shape) if wanted[2] else None
    dpre = x2.new_empty((tokens, 2 * inter)) if inner else None
    h = kept.data_ptr()
    _launch((_lib or _library()).mmoe_feed_forward_grad, x2.get_device(),
            _native.MmoeFeedForward(_CODES[x2.dtype], hidden, inter, tokens, clamp, 0, _stride(x2), x2.data_ptr(), w13.data_ptr(),
                                    w2.data_ptr(), h, h + 2 * tokens * inter if inner else None, None),
            dy2.data_ptr(), _ptr(dpre), _ptr(dx), _ptr(dw13), _ptr(dw2))
    return dx, dw13, dw2


# Nodes of the calls on a default stream whose graphs are alive, by weak references that leave by themselves.  A plain set of them, which is listed and
# changed in one step each: threads may make and drop graphs while another one captures.
_eager_graphs = set()


def _remember(node) -> None:
    _eager_graphs.add(weakref.ref(node, _eager_graphs.discard))


def _live_graphs() -> list:
    return [node for node in [r() for r in list(_eager_graphs)] if node is not None]


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, clamp):
        x2 = _rows(x)
        need = ctx.needs_input_grad
        y, kept = _launch_block(x2, w13, w2, clamp, need[0] or need[1])
        ctx.clamp = clamp
        # x is kept beside a copy of its rows, where there had to be one, so that a change of x is noticed
        if x2.data_ptr() == x.data_ptr():
            ctx.save_for_backward(x, w13, w2, kept)
        else:
            ctx.save_for_backward(x, w13, w2, kept, x2)
        if (_raw_stream or _native.raw_stream)(x.get_device()) == 0:
            _remember(ctx)
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses second derivatives costs some microseconds, and only a graph of the gradients can have them)
        return _Block._once(ctx, dy) if torch.is_grad_enabled() else _Block._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        if _tracing() or _dispatch_modes() or _function_modes():
            _refuse_traces("the gradient of gated_feed_forward")
        if _forward_ad._current_level >= 0:
            _refuse_tangents("the gradient of gated_feed_forward", dy)
        x, w13, w2, kept, *copy = ctx.saved_tensors
        dy2 = dy if dy.dim() == 2 and dy.is_contiguous() else dy.reshape(-1, w2.shape[0]).contiguous()
        if dy2.data_ptr() % 16 != 0:
            dy2 = dy2.clone()
        dx, dw13, dw2 = _launch_block_grad(copy[0] if copy else _rows(x), w13, w2, kept, dy2, ctx.clamp, ctx.needs_input_grad)
        return dx.view(x.shape) if dx is not None and x.dim() != 2 else dx, dw13, dw2, None


_Block._once = staticmethod(once_differentiable(_Block._gradients))


def _refuse_beside_eager_graph(inputs, what: str = "gated_feed_forward") -> None:
    """The node that accumulates a leaf's gradient belongs to the stream on which the first live graph made it.  A captured backward
    pass lets that stream wait for its own, which takes it into the capture; a default stream cannot be captured, and the process would
    end.  Graphs made on other streams, as by a warm-up, are no obstacle."""
    if not _eager_graphs:
        return
    mine = _accumulators([torch.autograd.graph.get_gradient_edge(t).node for t in inputs if t.requires_grad])
    if mine & _accumulators(_live_graphs()):
        raise RuntimeError("a graph of an eager call of gated_feed_forward, grouped_feed_forward or grouped_projection with the same leaves on the "
                           f"default stream is still alive: drop its output before the call of {what} is captured for training")


def _accumulators(nodes) -> set:
    """The nodes behind ``nodes`` that accumulate the gradients of leaves."""
    seen, found = set(nodes), set()
    nodes = list(seen)
    while nodes:
        node = nodes.pop()
        if hasattr(node, "variable"):
            found.add(node)
        for behind, _ in node.next_functions:
            if behind is not None and behind not in seen:
                seen.add(behind)
                nodes.append(behind)
    return found


def gated_feed_forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, *, activation_clamp: Optional[float] = None) -> torch.Tensor:
    """``y = h w2^T`` with ``h = silu(min(x wg^T, c)) * clip(x wu^T, -c, c)`` and ``w13 = [wg; wu]``.  See ``api.gated_feed_forward``."""
    if _tracing() or _dispatch_modes() or _function_modes():
        _refuse_traces("gated_feed_forward")
    _check_block(x, w13, w2)
    clamp = _clamp_of(activation_clamp)
    if _forward_ad._current_level >= 0:
        _refuse_tangents("gated_feed_forward", x, w13, w2)
    if not ((x.requires_grad or w13.requires_grad or w2.requires_grad) and torch.is_grad_enabled()):
        y = _launch_block(_rows(x), w13, w2, clamp, False)[0]
        return y if x.dim() == 2 else y.view(x.shape)
    if _capturing():
        _refuse_beside_eager_graph((x, w13, w2))
    return _Block.apply(x, w13, w2, clamp)


# ---------------------------------------------------------------------------------------------------------------------
# 8-bit integers
# ---------------------------------------------------------------------------------------------------------------------
def _refuse_gradient(what: str) -> None:
    if torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or with tensors that need none")


def prepare_int8_inputs(hidden_states: torch.Tensor, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-token 8-bit quantiser.  See ``api.prepare_int8_inputs``."""
    if _tracing() or _dispatch_modes() or _function_modes():
        _refuse_traces("INT8 staging")
    x = hidden_states
    code = _CODES.get(x.dtype)
    if code is None or code == _native.MMOE_FP32 or not x.is_cuda or x.dim() < 1:
        raise ValueError("INT8 staging requires BF16 or FP16 CUDA hidden states.")
    if x.requires_grad:
        _refuse_gradient("INT8 staging")
    if _forward_ad._current_level >= 0:
        _refuse_tangents("INT8 staging", x)
    shape = x.shape
    width, lead = shape[-1], shape[:-1]
    if width == 0:
        raise ValueError("INT8 staging requires a positive hidden_size.")
    if len(shape) != 2:
        x = x.reshape(-1, width)
    tokens = x.shape[0]
    if tokens > _MOST_QUANTIZED or width > _MOST_QUANTIZED:
        raise ValueError(f"INT8 staging takes at most {_MOST_QUANTIZED} tokens and as many channels, got {tokens} and {width}.")
    if not x.is_contiguous() and (width > 1 and x.stride(1) != 1 or tokens > 1 and x.stride(0) < width):
        x = x.contiguous()
    if out is None:
        q, scales = x.new_empty(shape, dtype=torch.int8), x.new_empty(lead, dtype=torch.float32)
    else:
        q, scales = out
        if (q.shape != shape or scales.shape != lead or q.dtype != torch.int8 or scales.dtype != torch.float32
                or q.device != x.device or scales.device != x.device or not q.is_contiguous() or not scales.is_contiguous()):
            raise ValueError("INT8 staging requires out=(int8 of the shape of hidden_states, float32 of its leading shape), contiguous.")
    if tokens > 0:
        _quantize(x, code, q, scales, tokens, width)
    return q, scales


def _quantize(x, code, q, scales, tokens, width) -> None:
    index = x.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return _quantize(x, code, q, scales, tokens, width)
    code = (_lib or _library()).mmoe_quantize_int8(x.data_ptr(), code, _stride(x), q.data_ptr(), scales.data_ptr(), tokens, width,
                                                   _raw_stream(index))
    if code:
        _native.check(code)


def _float_vector(t: torch.Tensor, shape, what: str, index: int) -> torch.Tensor:
    """A float32 tensor of ``shape`` (or with one more dimension of 1), dense; ``t`` itself where it is that."""
    if t.dtype is not torch.float32 or t.get_device() != index or (t.shape != shape and t.shape != (*shape, 1)):
        raise AssertionError(f"{what} must be float32 {tuple(shape)} on cuda:{index}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.requires_grad:
        _refuse_gradient("a product of 8-bit integers")
    if _forward_ad._current_level >= 0:
        _refuse_tangents("a product of 8-bit integers", t)
    return t if t.is_contiguous() else t.contiguous()


def _int8_product(x, x_scales, w, w_scales, bias, out_dtype, clamp: float, gated: bool) -> torch.Tensor:
    if _tracing() or _dispatch_modes() or _function_modes():
        _refuse_traces("a product of 8-bit integers")
    index = x.get_device()
    if index < 0:
        raise RuntimeError("products of 8-bit integers run on the GPU only (there is no CPU path).")
    shape = x.shape
    if x.dtype is not torch.int8 or len(shape) < 1:
        raise AssertionError(f"x must be int8 (..., K), got {tuple(shape)} {x.dtype}")
    _check_weight(w, "w13" if gated else "w", torch.int8, x)
    rows, width = w.shape
    if shape[-1] != width or width < 16 or width >= 131072 or width % 16 != 0:
        raise AssertionError(f"x (..., K) and the weights (N, K) must agree on K, a multiple of 16 below 131072, got {shape[-1]} and {width}")
    if not 1 <= rows <= 2 * _MOST_CHANNELS or (gated and rows % 2 != 0):
        raise AssertionError(f"the weights have {rows} rows" + (": the gated projection needs as many gate as up rows" if gated else ""))
    code = _CODES.get(out_dtype)
    if code is None:
        raise AssertionError(f"out_dtype must be BF16, FP16 or FP32, got {out_dtype}")
    lead = shape[:-1]
    x2 = _rows(x)
    tokens = x2.shape[0]
    if tokens > _MOST_TOKENS:
        raise _too_many(tokens)
    x_scales = _float_vector(x_scales, lead, "x_scales", index)
    w_scales = _float_vector(w_scales, (rows,), "w_scales", index)
    if bias is not None:
        bias = _float_vector(bias, (rows,), "bias", index)
    channels = rows // 2 if gated else rows
    out = x.new_empty((*lead, channels), dtype=out_dtype)
    if tokens > 0:
        lib = _lib or _library()
        _launch(lib.mmoe_int8_gated_projection if gated else lib.mmoe_int8_projection, index,
                _native.MmoeInt8Product(tokens, width, channels, code, clamp, 0, _stride(x2), x2.data_ptr(), x_scales.data_ptr(), w.data_ptr(),
                                        w_scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr()))
    return out


def int8_projection(x, x_scales, w, w_scales, *, bias=None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _int8_product(x, x_scales, w, w_scales, bias, torch.bfloat16 if out_dtype is None else out_dtype, math.inf, False)


def int8_gated_projection(x, x_scales, w13, w13_scales, *, activation_clamp: Optional[float] = None,
                          out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _int8_product(x, x_scales, w13, w13_scales, None, torch.bfloat16 if out_dtype is None else out_dtype, _clamp_of(activation_clamp), True)
