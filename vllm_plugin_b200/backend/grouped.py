"""Products of a layer's experts beside the MXFP8 x MXFP4 layer: rows that are grouped by expert, in 16 bits with their gradients (experts
that are trained or not quantised), and products in 8-bit floating point with block scales, of such rows or of all rows by one weight,
behind their quantiser.  The reference has no counterpart.

The experts' rows are given by ``ends``, int32 ``(E,)`` on the device: expert e's end before row ``ends[e]`` (``torch.cumsum(counts, 0,
dtype=torch.int32)``).  The kernels read them; nothing comes back to the host, and a captured call goes by what they hold at each replay.

Launches, status words and errors are those of the dense operators (``dense.py``).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _native
from . import dense as _d

_MOST_EXPERTS, _MOST_WIDTH = _native.MOST_EXPERTS, _native.MOST_GROUPED_WIDTH
_BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_tracing, _dispatch_modes, _function_modes = _d._tracing, _d._dispatch_modes, _d._function_modes


# ---------------------------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------------------------
# A call that is right is told by one condition; what is wrong with any other is looked for afterwards.
_INT32 = torch.int32


def _refuse_rows(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU only (there is no CPU path).")
    if x.dtype not in _d._FF_TYPES or x.dim() != 2:
        raise AssertionError(f"x must be BF16 or FP16 (T, width), got {tuple(x.shape)} {x.dtype}")
    if x.shape[0] > _d._MOST_TOKENS:
        raise _d._too_many(x.shape[0])


def _weights_fit(w: torch.Tensor, dtype: torch.dtype, index: int) -> bool:
    return w.dtype is dtype and w.dim() == 3 and w.is_contiguous() and w.data_ptr() % 16 == 0 and w.get_device() == index


def _check_weights(w: torch.Tensor, what: str, dtype: torch.dtype, index: int) -> None:
    if _weights_fit(w, dtype, index):
        return
    if w.dim() != 3 or w.dtype != dtype:
        raise AssertionError(f"{what} must be 3-D {dtype} (experts first), got {tuple(w.shape)} {w.dtype}")
    if w.get_device() != index:
        raise AssertionError(f"{what} must be on cuda:{index}, got {w.device}")
    raise AssertionError(f"{what} must be contiguous and 16-byte aligned")


def _dense_ends(ends: torch.Tensor, experts: int, index: int) -> torch.Tensor:
    if not isinstance(ends, torch.Tensor) or ends.dtype is not _INT32 or ends.get_device() != index or ends.shape != (experts,):
        got = f"{tuple(ends.shape)} {ends.dtype} on {ends.device}" if isinstance(ends, torch.Tensor) else repr(type(ends))
        raise AssertionError(f"ends must be int32 ({experts},) on cuda:{index}, got {got}")
    if not 1 <= experts <= _MOST_EXPERTS:
        raise AssertionError(f"{experts} experts: at least one and at most {_MOST_EXPERTS}")
    return ends if ends.is_contiguous() else ends.contiguous()


def _size_fits(size: int, step: int) -> bool:
    return 0 < size <= _MOST_WIDTH and size % step == 0


def _refuse_size(name: str, size: int, step: int) -> None:
    raise AssertionError(f"{name}={size} must be a positive multiple of {step}, at most {_MOST_WIDTH}")


def _check_sizes(step: int, a: str, first: int, b: str, second: int) -> None:
    if not _size_fits(first, step):
        _refuse_size(a, first, step)
    if not _size_fits(second, step):
        _refuse_size(b, second, step)


def _check_rows(x: torch.Tensor, what: str) -> None:
    if x.dtype not in _d._FF_TYPES or x.dim() != 2 or not x.is_cuda or x.shape[0] > _d._MOST_TOKENS:
        _refuse_rows(x, what)


def _dense_gradient(dy: torch.Tensor) -> torch.Tensor:
    dy = dy.contiguous()
    return dy if dy.data_ptr() % 16 == 0 else dy.clone()


_ptr = _d._ptr


def _keep(ctx, x, x2, *more) -> None:
    """x is kept beside a copy of its rows, where there had to be one, so that a change of x is noticed."""
    if x2.data_ptr() == x.data_ptr():
        ctx.save_for_backward(x, *more)
    else:
        ctx.save_for_backward(x, *more, x2)
    if (_d._raw_stream or _native.raw_stream)(x.get_device()) == 0:
        _d._remember(ctx)


# ---------------------------------------------------------------------------------------------------------------------
# one product
# ---------------------------------------------------------------------------------------------------------------------
def _projection_of(x2, w, ends, out):
    experts, channels, width = w.shape
    rows = x2.shape[0]
    return _native.MmoeGroupedProduct(_d._CODES[x2.dtype], rows, experts, width, channels, 0, x2.stride(0) if rows > 1 else width, x2.data_ptr(), w.data_ptr(),
                                      ends.data_ptr(), out)


def _launch_projection(x2, w, ends):
    rows = x2.shape[0]
    out = x2.new_empty((rows, w.shape[1]))
    if rows > 0:
        _d._launch((_d._lib or _d._library()).mmoe_grouped_projection, x2.get_device(), _projection_of(x2, w, ends, out.data_ptr()))
    return out


class _Projection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ends):
        x2 = _d._rows(x)
        out = _launch_projection(x2, w, ends)
        _keep(ctx, x, x2, w, ends)
        return out

    @staticmethod
    def backward(ctx, dy):
        return _Projection._once(ctx, dy) if torch.is_grad_enabled() else _Projection._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        if _tracing() or _dispatch_modes() or _function_modes():
            _d._refuse_traces("the gradient of grouped_projection")
        if _forward_ad._current_level >= 0:
            _d._refuse_tangents("the gradient of grouped_projection", dy)
        x, w, ends, *copy = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        dy = _dense_gradient(dy)
        x2 = copy[0] if copy else _d._rows(x)
        dx = x2.new_empty(x2.shape) if wanted[0] else None
        dw = torch.empty_like(w) if wanted[1] else None
        _d._launch((_d._lib or _d._library()).mmoe_grouped_projection_grad, x2.get_device(), _projection_of(x2, w, ends, None), dy.data_ptr(), _ptr(dx),
                   _ptr(dw))
        return dx, dw, None


_Projection._once = staticmethod(once_differentiable(_Projection._gradients))


def grouped_projection(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """``y[t] = w[e] x[t]`` for the rows of expert e.  See ``api.grouped_projection``."""
    if _tracing() or _dispatch_modes() or _function_modes():
        _d._refuse_traces("grouped_projection")
    _check_rows(x, "grouped_projection")
    index = x.get_device()
    _check_weights(w, "w", x.dtype, index)
    experts, channels, width = w.shape
    if x.shape[1] != width:
        raise AssertionError(f"expected x (T, K) and w (E, N, K), got {tuple(x.shape)} and {tuple(w.shape)}")
    _check_sizes(8, "K", width, "N", channels)
    ends = _dense_ends(ends, experts, index)
    if _forward_ad._current_level >= 0:
        _d._refuse_tangents("grouped_projection", x, w)
    if not ((x.requires_grad or w.requires_grad) and torch.is_grad_enabled()):
        return _launch_projection(_d._rows(x), w, ends)
    if _d._capturing():
        _d._refuse_beside_eager_graph((x, w), "grouped_projection")
    return _Projection.apply(x, w, ends)


# ---------------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------
def _block_of(x2, w13, w2, ends, clamp, h, preact, y):
    experts, hidden, inter = w2.shape
    return _native.MmoeGroupedFeedForward(_d._CODES[x2.dtype], x2.shape[0], experts, hidden, inter, clamp, 0, 0, _d._stride(x2), x2.data_ptr(),
                                          w13.data_ptr(), w2.data_ptr(), ends.data_ptr(), h, preact, _ptr(y))


def _launch_block(x2, w13, w2, ends, clamp: float, keep: bool):
    """``(y, kept)``: ``kept`` holds h, and behind it (``keep``) g and u for the backward pass, in bytes."""
    rows, hidden = x2.shape
    inter = w2.shape[2]
    y = x2.new_empty((rows, hidden))
    kept = x2.new_empty(rows * inter * (5 if keep else 1))        # 16-bit elements: 1 for h, 2 x 2 for g and u
    if rows > 0:
        h = kept.data_ptr()
        _d._launch((_d._lib or _d._library()).mmoe_grouped_feed_forward, x2.get_device(),
                   _block_of(x2, w13, w2, ends, clamp, h, h + 2 * rows * inter if keep else None, y))
    return y, kept


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, ends, clamp):
        x2 = _d._rows(x)
        need = ctx.needs_input_grad
        y, kept = _launch_block(x2, w13, w2, ends, clamp, need[0] or need[1])
        ctx.clamp = clamp
        _keep(ctx, x, x2, w13, w2, ends, kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _Block._once(ctx, dy) if torch.is_grad_enabled() else _Block._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        if _tracing() or _dispatch_modes() or _function_modes():
            _d._refuse_traces("the gradient of grouped_feed_forward")
        if _forward_ad._current_level >= 0:
            _d._refuse_tangents("the gradient of grouped_feed_forward", dy)
        x, w13, w2, ends, kept, *copy = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        inner = wanted[0] or wanted[1]
        dy = _dense_gradient(dy)
        x2 = copy[0] if copy else _d._rows(x)
        rows, inter = x2.shape[0], w2.shape[2]
        dx = x2.new_empty(x2.shape) if wanted[0] else None
        dw13 = torch.empty_like(w13) if wanted[1] else None
        dw2 = torch.empty_like(w2) if wanted[2] else None
        dpre = x2.new_empty((rows, 2 * inter)) if inner else None
        h = kept.data_ptr()
        _d._launch((_d._lib or _d._library()).mmoe_grouped_feed_forward_grad, x2.get_device(),
                   _block_of(x2, w13, w2, ends, ctx.clamp, h, h + 2 * rows * inter if inner else None, None), dy.data_ptr(), _ptr(dpre), _ptr(dx), _ptr(dw13),
                   _ptr(dw2))
        return dx, dw13, dw2, None, None


_Block._once = staticmethod(once_differentiable(_Block._gradients))


def grouped_feed_forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, ends: torch.Tensor, *,
                         activation_clamp: Optional[float] = None) -> torch.Tensor:
    """The gated feed-forward block with the weights of each row's expert.  See ``api.grouped_feed_forward``."""
    if _tracing() or _dispatch_modes() or _function_modes():
        _d._refuse_traces("grouped_feed_forward")
    _check_rows(x, "grouped_feed_forward")
    index = x.get_device()
    _check_weights(w13, "w13", x.dtype, index)
    _check_weights(w2, "w2", x.dtype, index)
    experts, hidden, inter = w2.shape
    if x.shape[1] != hidden or w13.shape != (experts, 2 * inter, hidden):
        raise AssertionError(f"expected x (T, H), w13 (E, 2 I, H) and w2 (E, H, I), got {tuple(x.shape)}, {tuple(w13.shape)} and {tuple(w2.shape)}")
    _check_sizes(8, "H", hidden, "I", inter)
    ends = _dense_ends(ends, experts, index)
    clamp = _d._clamp_of(activation_clamp)
    if _forward_ad._current_level >= 0:
        _d._refuse_tangents("grouped_feed_forward", x, w13, w2)
    if not ((x.requires_grad or w13.requires_grad or w2.requires_grad) and torch.is_grad_enabled()):
        return _launch_block(_d._rows(x), w13, w2, ends, clamp, False)[0]
    if _d._capturing():
        _d._refuse_beside_eager_graph((x, w13, w2), "grouped_feed_forward")
    return _Block.apply(x, w13, w2, ends, clamp)


# ---------------------------------------------------------------------------------------------------------------------
# 8-bit floating point
# ---------------------------------------------------------------------------------------------------------------------
def prepare_fp8_inputs(hidden_states: torch.Tensor, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Quantiser by groups of 128 values.  See ``api.prepare_fp8_inputs``."""
    if _tracing() or _dispatch_modes() or _function_modes():
        _d._refuse_traces("FP8 staging")
    x = hidden_states
    code = _d._CODES.get(x.dtype)
    if code is None or code == _native.MMOE_FP32 or not x.is_cuda or x.dim() < 1:
        raise ValueError("FP8 staging requires BF16 or FP16 CUDA hidden states.")
    if x.requires_grad and torch.is_grad_enabled():
        _d._refuse_gradient("FP8 staging")
    if _forward_ad._current_level >= 0:
        _d._refuse_tangents("FP8 staging", x)
    shape = x.shape
    width = shape[-1]
    if width == 0:
        raise ValueError("FP8 staging requires a positive hidden_size.")
    groups = -(-width // _BLOCK)
    scale_shape = (*shape[:-1], groups)
    if len(shape) != 2:
        x = x.reshape(-1, width)
    rows = x.shape[0]
    most = _d._MOST_QUANTIZED
    if rows > most or width > most or rows * groups >= 1 << 32:
        raise ValueError(f"FP8 staging takes at most {most} tokens, as many channels and 2^32 - 1 groups of 128, got {rows} and {width}.")
    if not x.is_contiguous() and (width > 1 and x.stride(1) != 1 or rows > 1 and x.stride(0) < width):
        x = x.contiguous()
    if out is None:
        q, scales = x.new_empty(shape, dtype=_E4M3), x.new_empty(scale_shape, dtype=torch.float32)
    else:
        q, scales = out
        if (q.shape != shape or scales.shape != scale_shape or q.dtype != _E4M3 or scales.dtype != torch.float32
                or q.device != x.device or scales.device != x.device or not q.is_contiguous() or not scales.is_contiguous()):
            raise ValueError("FP8 staging requires out=(float8_e4m3fn of the shape of hidden_states, float32 with a scale for each 128 values), contiguous.")
    if rows > 0:
        _quantize(x, code, q, scales, rows, width)
    return q, scales


def _quantize(x, code, q, scales, rows, width) -> None:
    index = x.get_device()
    if _d._current_device() != index:
        with torch.cuda.device(index):
            return _quantize(x, code, q, scales, rows, width)
    code = (_d._lib or _d._library()).mmoe_quantize_fp8(x.data_ptr(), code, _d._stride(x), q.data_ptr(), scales.data_ptr(), rows, width, _d._raw_stream(index))
    if code:
        _native.check(code)


def _scales(t: torch.Tensor, shape, what: str, index: int) -> torch.Tensor:
    """A float32 tensor of ``shape``, dense; ``t`` itself where it is that."""
    if t.dtype is not torch.float32 or t.get_device() != index or t.shape != shape:
        raise AssertionError(f"{what} must be float32 {tuple(shape)} on cuda:{index}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        _d._refuse_gradient("a product in 8-bit floating point")
    if _forward_ad._current_level >= 0:
        _d._refuse_tangents("a product in 8-bit floating point", t)
    return t if t.is_contiguous() else t.contiguous()


def _fp8_product(x, x_scales, w, w_scales, ends, out_dtype, clamp: float, gated: bool) -> torch.Tensor:
    if _tracing() or _dispatch_modes() or _function_modes():
        _d._refuse_traces("a product in 8-bit floating point")
    index = x.get_device()
    if index < 0:
        raise RuntimeError("products in 8-bit floating point run on the GPU only (there is no CPU path).")
    shape = x.shape
    what = "w13" if gated else "w"
    if x.dtype is not _E4M3 or (len(shape) < 1 if ends is None else len(shape) != 2):
        raise AssertionError(f"x must be float8_e4m3fn {'(..., K)' if ends is None else '(T, K)'}, got {tuple(shape)} {x.dtype}")
    if ends is None:
        _d._check_weight(w, what, _E4M3, x)
        experts, (rows, width) = 1, w.shape
    else:
        _check_weights(w, what, _E4M3, index)
        experts, rows, width = w.shape
        ends = _dense_ends(ends, experts, index)
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        _d._refuse_gradient("a product in 8-bit floating point")
    if _forward_ad._current_level >= 0:
        _d._refuse_tangents("a product in 8-bit floating point", x, w)
    if shape[-1] != width:
        raise AssertionError(f"x (..., K) and the weights (..., N, K) must agree on K, got {shape[-1]} and {width}")
    if gated and rows % 2 != 0:
        raise AssertionError(f"the weights have {rows} rows: the gated projection needs as many gate as up rows")
    channels = rows // 2 if gated else rows
    if not _size_fits(width, 16):
        _refuse_size("K", width, 16)
    if not _size_fits(channels, 8 if gated else 1):
        _refuse_size("N", channels, 8 if gated else 1)
    code = _d._CODES.get(out_dtype)
    if code is None:
        raise AssertionError(f"out_dtype must be BF16, FP16 or FP32, got {out_dtype}")
    lead, groups, blocks = shape[:-1], -(-width // _BLOCK), -(-channels // _BLOCK) * (2 if gated else 1)
    x2 = _d._rows(x)
    tokens = x2.shape[0]
    if tokens > _d._MOST_TOKENS:
        raise _d._too_many(tokens)
    x_scales = _scales(x_scales, (*lead, groups), "x_scales", index)
    w_scales = _scales(w_scales, (blocks, groups) if ends is None else (experts, blocks, groups), what + "_scales", index)
    out = x.new_empty((*lead, channels), dtype=out_dtype)
    if tokens > 0:
        lib = _d._lib or _d._library()
        _d._launch(lib.mmoe_fp8_gated_projection if gated else lib.mmoe_fp8_projection, index,
                   _native.MmoeFp8Product(tokens, experts, width, channels, code, clamp, 0, 0, _d._stride(x2), x2.data_ptr(), x_scales.data_ptr(), w.data_ptr(),
                                          w_scales.data_ptr(), None if ends is None else ends.data_ptr(), out.data_ptr()))
    return out


def fp8_projection(x, x_scales, w, w_scales, *, ends: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _fp8_product(x, x_scales, w, w_scales, ends, torch.bfloat16 if out_dtype is None else out_dtype, math.inf, False)


def fp8_gated_projection(x, x_scales, w13, w13_scales, *, ends: Optional[torch.Tensor] = None, activation_clamp: Optional[float] = None,
                         out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return _fp8_product(x, x_scales, w13, w13_scales, ends, torch.bfloat16 if out_dtype is None else out_dtype, _d._clamp_of(activation_clamp), True)
