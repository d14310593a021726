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
from typing import Dict, Optional, Tuple

import torch
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
        self.status = torch.zeros(8, dtype=torch.int32, device=device)
        self.status_ptr = self.status.data_ptr()
        self.poll = None


_devices: Dict[int, _Device] = {}


def _on_device(index: int) -> _Device:
    """State of the current device ``index``, made at the first call."""
    state = _devices.get(index)
    if state is None:
        _f.require_sm100()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the dense operators must be called once on a device before CUDA-graph capture")
        device = torch.device("cuda", index)
        _native.check(_native.load().mmoe_dense_prepare(_native.raw_stream(index)))
        state = _Device(device)
        torch.cuda.synchronize(device)              # the words are zero before a call on another stream may look at them
        _devices[index] = state
    return state


def _watch(state: _Device):
    """Non-blocking look at the status words, as the layer's calls do it: returns what to call behind the launch."""
    interval = _f._kernel_options.status_poll_interval
    if interval <= 0 or torch.cuda.is_current_stream_capturing():
        return None
    if state.poll is None:
        state.poll = _f._StatusPoll(state)
    state.poll.before_call(state)
    return state.poll


def read_dense_status(device=None) -> None:
    """Synchronise and raise ``RuntimeError`` if a device-side wait of a dense operator expired on ``device`` since the last
    read; clears the condition."""
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    with torch.cuda.device(index):
        state = _on_device(index)
        words = (ctypes.c_int32 * 8)()
        _native.check(_native.load().mmoe_dense_read_status(state.status_ptr, words, _native.raw_stream(index)))


# ---------------------------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------------------------
def _need(condition: bool, message: str) -> None:
    if not condition:
        raise AssertionError(message)


def _clamp_of(activation_clamp: Optional[float]) -> float:
    if activation_clamp is None:
        return math.inf
    value = float(activation_clamp)
    _need(value > 0, "activation_clamp must be positive")
    return value


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as ``(rows, width)`` whose rows are dense and start on 16 bytes: a view where there is one, else a copy."""
    width = t.shape[-1]
    r = t if t.dim() == 2 else t.reshape(-1, width)
    unit = 16 // r.element_size()
    if r.shape[0] <= 1:
        dense = r.stride(1) == 1 or width == 1
    else:
        dense = (r.stride(1) == 1 or width == 1) and r.stride(0) >= width and r.stride(0) % unit == 0
    if dense and r.data_ptr() % 16 == 0:
        return r
    return r.contiguous() if not r.is_contiguous() else r.clone(memory_format=torch.contiguous_format)


def _stride(r: torch.Tensor) -> int:
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def _check_weight(w: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device) -> None:
    _need(w.dim() == 2 and w.dtype == dtype, f"{what} must be 2-D {dtype}, got {tuple(w.shape)} {w.dtype}")
    _need(w.device == device, f"{what} must be on {device}")
    _need(w.is_contiguous() and w.data_ptr() % 16 == 0, f"{what} must be contiguous and 16-byte aligned")


def _needs_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU only (there is no CPU path).")


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------
def _check_block(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor) -> Tuple[int, int]:
    _needs_cuda(x, "gated_feed_forward")
    _need(x.dim() >= 1 and x.dtype in _FF_TYPES, f"x must be BF16 or FP16 (..., H), got {tuple(x.shape)} {x.dtype}")
    _check_weight(w13, "w13", x.dtype, x.device)
    _check_weight(w2, "w2", x.dtype, x.device)
    hidden, inter = w2.shape
    _need(x.shape[-1] == hidden and tuple(w13.shape) == (2 * inter, hidden),
          f"expected x (..., H), w13 (2 I, H) and w2 (H, I), got {tuple(x.shape)}, {tuple(w13.shape)} and {tuple(w2.shape)}")
    _need(hidden > 0 and inter > 0 and hidden % 8 == 0 and inter % 8 == 0, f"H={hidden} and I={inter} must be positive multiples of 8")
    return hidden, inter


def _launch_block(x2: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, clamp: float, keep: bool):
    """``(y, h, preact or None)`` of rows ``x2``."""
    tokens, hidden = x2.shape
    inter = w2.shape[1]
    y = torch.empty((tokens, hidden), dtype=x2.dtype, device=x2.device)
    h = torch.empty((tokens, inter), dtype=x2.dtype, device=x2.device)
    preact = torch.empty((tokens, 2 * inter), dtype=torch.float32, device=x2.device) if keep else None
    if tokens > 0:
        index = x2.get_device()
        state = _on_device(index)
        poll = _watch(state)
        a = _native.MmoeFeedForward(_CODES[x2.dtype], hidden, inter, tokens, clamp, _f._kernel_options.timeout_ms, _stride(x2),
                                    x2.data_ptr(), w13.data_ptr(), w2.data_ptr(), h.data_ptr(),
                                    preact.data_ptr() if keep else None, y.data_ptr(), state.status_ptr)
        _native.check(_native.load().mmoe_feed_forward(ctypes.byref(a), _native.raw_stream(index)))
        if poll is not None:
            poll.after_call(state, _f._kernel_options.status_poll_interval)
    return y, h, preact


def _launch_block_grad(x2, w13, w2, h, preact, dy2, clamp: float, wanted):
    tokens, hidden = x2.shape
    inter = w2.shape[1]
    dx, dw13, dw2 = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if w else None for t, w in zip((x2, w13, w2), wanted))
    dpre = torch.empty((tokens, 2 * inter), dtype=x2.dtype, device=x2.device) if wanted[0] or wanted[1] else None
    index = x2.get_device()
    state = _on_device(index)
    poll = _watch(state)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = _native.MmoeFeedForward(_CODES[x2.dtype], hidden, inter, tokens, clamp, _f._kernel_options.timeout_ms, _stride(x2),
                                x2.data_ptr(), w13.data_ptr(), w2.data_ptr(), ptr(h), ptr(preact), None, state.status_ptr)
    _native.check(_native.load().mmoe_feed_forward_grad(ctypes.byref(a), dy2.data_ptr(), ptr(dpre), ptr(dx), ptr(dw13), ptr(dw2),
                                                        _native.raw_stream(index)))
    if poll is not None:
        poll.after_call(state, _f._kernel_options.status_poll_interval)
    return dx, dw13, dw2


_EAGER = "mmoe_eager_graph"


def _accumulators(leaves):
    return [torch.autograd.graph.get_gradient_edge(t).node for t in leaves if t.requires_grad and t.is_leaf]


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, clamp):
        x2 = _rows(x.detach())
        w13d, w2d = w13.detach(), w2.detach()
        need_x, need_13, need_2 = ctx.needs_input_grad[:3]
        with torch.cuda.device(x.device):
            y, h, preact = _launch_block(x2, w13d, w2d, clamp, need_x or need_13)
        ctx.clamp, ctx.x_shape = clamp, x.shape
        # the rows as the products read them (x itself unless its rows had to be copied), so that a change of x is noticed
        own_rows = x2.data_ptr() != x.data_ptr()
        ctx.save_for_backward(x, w13, w2, h if need_2 else None, preact, x2 if own_rows else None)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w13, w2, h, preact, x2 = ctx.saved_tensors
        x2 = _rows(x.detach()) if x2 is None else x2
        with torch.cuda.device(x.device):
            dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
            if dy2.data_ptr() % 16 != 0:
                dy2 = dy2.clone()
            dx, dw13, dw2 = _launch_block_grad(x2, w13, w2, h, preact, dy2, ctx.clamp, ctx.needs_input_grad[:3])
        return None if dx is None else dx.view(ctx.x_shape), dw13, dw2, None


def gated_feed_forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, *, activation_clamp: Optional[float] = None) -> torch.Tensor:
    """``y = h w2^T`` with ``h = silu(min(x wg^T, c)) * clip(x wu^T, -c, c)`` and ``w13 = [wg; wu]``.  See ``api.gated_feed_forward``."""
    _check_block(x, w13, w2)
    clamp = _clamp_of(activation_clamp)
    if not (torch.is_grad_enabled() and (x.requires_grad or w13.requires_grad or w2.requires_grad)):
        with torch.cuda.device(x.device):
            return _launch_block(_rows(x.detach()), w13.detach(), w2.detach(), clamp, False)[0].view(x.shape)
    leaves = (x, w13, w2)
    if torch.cuda.is_current_stream_capturing():
        # The node that accumulates a leaf's gradient belongs to the stream on which the first live graph made it.  A captured
        # backward pass would wait for that stream, which is not being captured, and the process would end.
        if any(_EAGER in node.metadata for node in _accumulators(leaves)):
            raise RuntimeError("a graph of an eager gated_feed_forward call with the same leaves is still alive: drop its output "
                               "before the call is captured for training")
        return _Block.apply(x, w13, w2, clamp)
    y = _Block.apply(x, w13, w2, clamp)
    for node in _accumulators(leaves):
        node.metadata[_EAGER] = True
    return y


# ---------------------------------------------------------------------------------------------------------------------
# 8-bit integers
# ---------------------------------------------------------------------------------------------------------------------
def _no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or with tensors that need none")


def prepare_int8_inputs(hidden_states: torch.Tensor, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-token 8-bit quantiser.  See ``api.prepare_int8_inputs``."""
    if hidden_states.dtype not in _FF_TYPES or not hidden_states.is_cuda or hidden_states.dim() < 1:
        raise ValueError("INT8 staging requires BF16 or FP16 CUDA hidden states.")
    _no_gradient("INT8 staging", hidden_states)
    width = hidden_states.shape[-1]
    if width == 0:
        raise ValueError("INT8 staging requires a positive hidden_size.")
    lead = hidden_states.shape[:-1]
    x = hidden_states.detach() if hidden_states.dim() == 2 else hidden_states.detach().reshape(-1, width)
    if width > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < width:
        x = x.contiguous()
    tokens = x.shape[0]
    if out is None:
        q = torch.empty((*lead, width), dtype=torch.int8, device=x.device)
        scales = torch.empty(lead, dtype=torch.float32, device=x.device)
    else:
        q, scales = out
        if (q.shape != hidden_states.shape or scales.shape != lead or q.dtype != torch.int8 or scales.dtype != torch.float32
                or q.device != x.device or scales.device != x.device or not q.is_contiguous() or not scales.is_contiguous()):
            raise ValueError("INT8 staging requires out=(int8 of the shape of hidden_states, float32 of its leading shape), contiguous.")
    if tokens > 0:
        index = x.get_device()
        with torch.cuda.device(index):
            _native.check(_native.load().mmoe_quantize_int8(x.data_ptr(), _CODES[x.dtype], _stride(x), q.data_ptr(), scales.data_ptr(),
                                                            tokens, width, _native.raw_stream(index)))
    return q, scales


def _int8_product(what: str, x, x_scales, w, w_scales, bias, out_dtype, clamp: float, gated: bool) -> torch.Tensor:
    _needs_cuda(x, what)
    _no_gradient(what, x_scales, w_scales, bias)
    _need(x.dtype == torch.int8 and x.dim() >= 1, f"x must be int8 (..., K), got {tuple(x.shape)} {x.dtype}")
    _check_weight(w, "w13" if gated else "w", torch.int8, x.device)
    rows, width = w.shape
    lead = x.shape[:-1]
    _need(x.shape[-1] == width and 16 <= width < 131072 and width % 16 == 0,
          f"x (..., K) and the weights (N, K) must agree on K, a multiple of 16 below 131072, got {x.shape[-1]} and {width}")
    _need(rows > 0 and (not gated or rows % 2 == 0), "the gated projection needs as many gate as up rows" if gated else "w has no rows")
    _need(out_dtype in _CODES, f"out_dtype must be BF16, FP16 or FP32, got {out_dtype}")
    for t, shape, name in ((x_scales, lead, "x_scales"), (w_scales, (rows,), "w_scales"), (bias, (rows,), "bias")):
        if t is not None:
            _need(t.dtype == torch.float32 and t.device == x.device and tuple(t.shape) in (tuple(shape), (*shape, 1)),
                  f"{name} must be float32 {tuple(shape)} on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    channels = rows // 2 if gated else rows
    out = torch.empty((*lead, channels), dtype=out_dtype, device=x.device)
    index = x.get_device()
    with torch.cuda.device(index):
        x2 = _rows(x)
        if x2.shape[0] > 0:
            x_scales, w_scales = x_scales.detach().contiguous(), w_scales.detach().contiguous()
            bias = bias.detach().contiguous() if bias is not None else None
            state = _on_device(index)
            poll = _watch(state)
            a = _native.MmoeInt8Product(x2.shape[0], width, channels, _CODES[out_dtype], clamp, _f._kernel_options.timeout_ms,
                                        _stride(x2), x2.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
                                        bias.data_ptr() if bias is not None else None, out.data_ptr(), state.status_ptr)
            lib = _native.load()
            run = lib.mmoe_int8_gated_projection if gated else lib.mmoe_int8_projection
            _native.check(run(ctypes.byref(a), _native.raw_stream(index)))
            if poll is not None:
                poll.after_call(state, _f._kernel_options.status_poll_interval)
    return out


def int8_projection(x, x_scales, w, w_scales, *, bias=None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return _int8_product("int8_projection", x, x_scales, w, w_scales, bias, out_dtype, math.inf, False)


def int8_gated_projection(x, x_scales, w13, w13_scales, *, activation_clamp: Optional[float] = None,
                          out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return _int8_product("int8_gated_projection", x, x_scales, w13, w13_scales, None, out_dtype, _clamp_of(activation_clamp), True)
