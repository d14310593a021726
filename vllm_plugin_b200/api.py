"""Public operator surface of the B200 MegaMoE expert backend.

Same names, signatures and semantics as the reference's ``vllm_sm107_megamoe/api.py`` (:39-266, which itself follows
DeepGEMM's MegaMoE API), so that a layer written against that module -- the ``DeepGemmMegaMoEExperts`` subclass reaches
it through ``_import_backend()`` -- can switch backend without other changes.  Every function hands off to
``vllm_plugin_b200.backend`` through function-local imports: importing this module imports neither torch nor CUDA.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple, Union

# implementations of the per-step functions, looked up once (a function-local import costs about a microsecond per call)
_mega_moe = _stage = _route_and_stage = None
_feed_forward = _quantize_int8 = _int8_projection = _int8_gated_projection = None
_grouped_projection = _grouped_feed_forward = _quantize_fp8 = _fp8_projection = _fp8_gated_projection = None


def get_symm_buffer_for_mega_moe(group, num_experts: int, num_max_tokens_per_rank: int, num_topk: int, hidden: int,
                                 intermediate_hidden: int, num_shared_experts: int = 0,
                                 use_fp8_dispatch: Union[bool, None] = None, mma_type: str = "fp8xfp4",
                                 activation: str = "swiglu"):
    """Allocate (collectively) the workspace of the layer; returns a ``SymmBuffer``.  ``num_max_tokens_per_rank`` is
    aligned up to 1920; the aligned value is ``SymmBuffer.num_max_tokens_per_rank``."""
    from .backend.frontend import require_sm100
    from .backend.workspace import get_symm_buffer_for_mega_moe as _impl

    require_sm100()
    return _impl(group, num_experts, num_max_tokens_per_rank, num_topk, hidden, intermediate_hidden,
                 num_shared_experts, use_fp8_dispatch, mma_type, activation)


def transform_weights_for_mega_moe(l1_weights, l2_weights, activation: str = "swiglu"):
    """Rearrange ``(weights, scale factors)`` pairs into the layout the kernels read (pure torch, any device)."""
    from .backend.weights import transform_weights_for_mega_moe as _impl

    return _impl(l1_weights, l2_weights, activation)


def fp8_fp4_mega_moe(y, l1_weights: Tuple[Any, Any], l2_weights: Tuple[Any, Any], sym_buffer,
                     shared_l1_weights: Optional[Tuple[Any, Any]] = None,
                     shared_l2_weights: Optional[Tuple[Any, Any]] = None, cumulative_local_expert_recv_stats=None,
                     recipe: Tuple[int, int, int] = (1, 1, 32), activation: str = "swiglu",
                     activation_clamp: Optional[float] = None, fast_math: bool = True, activation_alpha: float = 1.0,
                     activation_beta: float = 0.0, *, residual=None):
    """Fused MegaMoE for one rank.  The BLOCK_M variant is selected from ``y.size(0)`` of this call.  ``residual``
    (keyword only, an addition to the reference's signature): BF16 ``(M, H)`` added to the output in the combine pass."""
    global _mega_moe
    if _mega_moe is None:
        from .backend.frontend import fp8_fp4_mega_moe as _mega_moe
    return _mega_moe(y, l1_weights, l2_weights, sym_buffer, shared_l1_weights, shared_l2_weights,
                     cumulative_local_expert_recv_stats, recipe, activation, activation_clamp, fast_math, activation_alpha,
                     activation_beta, residual=residual)


def get_block_m_for_mega_moe(num_ranks: int, num_experts: int, num_max_tokens_per_rank: int, num_tokens: int,
                             num_topk: int, mma_type: str = "fp8xfp4") -> int:
    """BLOCK_M used for ``num_tokens`` tokens on the calling rank (a forced value, ``set_kernel_options(block_m=...)``, wins)."""
    from .backend.frontend import get_block_m_for_mega_moe as _impl

    return _impl(num_ranks, num_experts, num_max_tokens_per_rank, num_tokens, num_topk, mma_type)


def get_token_alignment_for_mega_moe() -> int:
    """Alignment (1920 = lcm of the candidate BLOCK_M) applied to ``num_max_tokens_per_rank``."""
    from .backend.heuristics import get_token_alignment_for_mega_moe as _impl

    return _impl()


def get_unsupported_reason_for_mega_moe(num_ranks: int, num_experts: int, num_max_tokens_per_rank: int, num_topk: int,
                                        hidden: int, intermediate_hidden: int, num_shared_experts: int = 0,
                                        mma_type: str = "fp8xfp4", activation: str = "swiglu", *,
                                        fast_math: bool = True, localized_shared_weights: bool = False,
                                        allow_unvalidated: bool = False) -> Optional[str]:
    """``None`` when this backend can serve the geometry, else a short reason.  Total: never raises."""
    from .backend.heuristics import get_mega_moe_unsupported_reason as _impl

    return _impl(num_ranks, num_experts, num_max_tokens_per_rank, num_topk, hidden, intermediate_hidden,
                 num_shared_experts, mma_type, activation, fast_math=fast_math,
                 localized_shared_weights=localized_shared_weights, allow_unvalidated=allow_unvalidated)


def stage_inputs_for_mega_moe(sym_buffer, hidden_states, topk_ids, topk_weights, *, is_padding=None,
                              block_m: Optional[int] = None) -> int:
    """Quantise and stage one call's inputs into ``sym_buffer`` (one CUDA launch); returns the BLOCK_M used."""
    global _stage
    if _stage is None:
        from .backend.staging import stage_inputs as _stage
    return _stage(sym_buffer, hidden_states, topk_ids, topk_weights, is_padding=is_padding, block_m=block_m)


def route_and_stage_inputs_for_mega_moe(sym_buffer, hidden_states, router_logits, *, replica_map=None, is_padding=None,
                                        block_m: Optional[int] = None) -> int:
    """Router (top-k by logit, softmax over the selected, optional logical -> physical replica choice) fused in front of
    the input staging: one CUDA launch; returns the BLOCK_M used.  Not part of the reference's surface: there the
    serving engine routes before it calls the layer."""
    global _route_and_stage
    if _route_and_stage is None:
        from .backend.staging import route_and_stage_inputs as _route_and_stage
    return _route_and_stage(sym_buffer, hidden_states, router_logits, replica_map=replica_map, is_padding=is_padding, block_m=block_m)


def prepare_megamoe_nvfp4_inputs(hidden_states, global_scale: float, out=None):
    """NVFP4 (E2M1 + E4M3 scale per 16 + per-tensor scale) staging of BF16 hidden states; returns ``(packed, scales)``."""
    from .backend.staging import prepare_megamoe_nvfp4_inputs as _impl

    return _impl(hidden_states, global_scale, out)


def gated_feed_forward(x, w13, w2, *, activation_clamp: Optional[float] = None):
    """Gated feed-forward block of a dense layer, or of a shared expert that is not MXFP8, with its gradients (no counterpart in
    the reference): ``y = h w2^T`` with ``h = silu(min(g, c)) * clip(u, -c, c)``, ``g = x wg^T``, ``u = x wu^T``.

    ``x``: BF16 or FP16 ``(..., H)``, any strides (rows that are not dense or do not start on 16 bytes are copied).  ``w13``: ``(2 I, H)``
    in checkpoint order, the gate's rows first; ``w2``: ``(H, I)``; both contiguous, on 16 bytes and of x's type; H and I multiples of 8.
    ``activation_clamp``: ``c``, none by default.  Returns ``(..., H)`` of the same type.

    Sums are FP32; the activation is within ``2^-21 + 2^-24 |g|`` of its value, and 0 for g below -87.  ``h`` is rounded to the type, as the second product's operand, and so are the gradients of g and u in the backward
    pass (in FP16 they overflow past 65504); g and u themselves are kept for it in FP32.  A value on the border of the clamp passes its gradient, one beyond it does not.
    First derivatives only, in backward mode.  Tangents and traces (``torch.jit.trace``, ``make_fx``) are refused by all dense operators,
    ``NotImplementedError``.  A training step can be captured into a CUDA graph behind a first call, but not while the graph of an eager
    call with the same leaves on the default stream is alive (``RuntimeError``); warm up on another stream, as PyTorch asks for anyway
    (graphs of other operators with the same leaves end a capture as they do in PyTorch; they are not looked for)."""
    global _feed_forward
    if _feed_forward is None:
        from .backend.dense import gated_feed_forward as _feed_forward
    return _feed_forward(x, w13, w2, activation_clamp=activation_clamp)


def prepare_int8_inputs(hidden_states, out=None):
    """Per-token 8-bit quantiser of BF16 or FP16 hidden states ``(..., K)``; returns ``(int8 (..., K), float32 scales (...))``.
    ``scale = max|x| / 127`` (1 for a row of zeros), values ``x / scale`` rounded to the nearest, ties to even.  A row that holds an infinity or
    a NaN gets the scale NaN and zeros, so that what is computed from it is NaN.  ``out``: the two tensors, contiguous."""
    global _quantize_int8
    if _quantize_int8 is None:
        from .backend.dense import prepare_int8_inputs as _quantize_int8
    return _quantize_int8(hidden_states, out)


def int8_projection(x, x_scales, w, w_scales, *, bias=None, out_dtype=None):
    """``(x w^T) * x_scales[..., None] * w_scales + bias`` with exact integer sums: ``x`` int8 ``(..., K)`` with float32 scales ``(...)``, ``w`` int8
    ``(N, K)`` with ``(N,)``, optional ``bias`` float32 ``(N,)``; ``w`` contiguous and on 16 bytes, K a multiple of 16 below 131072.  ``out_dtype``: BF16 (default), FP16 or
    FP32.  No gradient."""
    global _int8_projection
    if _int8_projection is None:
        from .backend.dense import int8_projection as _int8_projection
    return _int8_projection(x, x_scales, w, w_scales, bias=bias, out_dtype=out_dtype)


def int8_gated_projection(x, x_scales, w13, w13_scales, *, activation_clamp: Optional[float] = None, out_dtype=None):
    """The first half of a gated feed-forward block in 8-bit integers: both products (``w13`` int8 ``(2 I, K)``, the gate's rows first, scales
    ``(2 I,)``), the activation and their product in one kernel, ``silu(min(g, c)) * clip(u, -c, c)`` in ``(..., I)``.  Quantise it with
    :func:`prepare_int8_inputs` for :func:`int8_projection`.  Otherwise as there.  The activation is within 2^-20 of its value in FP32 (and, for g below
    -87, 2^-148 |g u|); in 16 bits within ``2^-21 + 2^-24 |g|``, far below the rounding, and 0 for g below -87."""
    global _int8_gated_projection
    if _int8_gated_projection is None:
        from .backend.dense import int8_gated_projection as _int8_gated_projection
    return _int8_gated_projection(x, x_scales, w13, w13_scales, activation_clamp=activation_clamp, out_dtype=out_dtype)


def grouped_projection(x, w, ends):
    """Product of rows that are grouped by expert with their expert's weights, with its gradients (no counterpart in the reference):
    ``y[t] = w[e] x[t]``.

    ``x``: BF16 or FP16 ``(T, K)``, any strides (rows that are not dense or do not start on 16 bytes are copied), the rows of expert 0
    first.  ``w``: ``(E, N, K)``, contiguous, on 16 bytes and of x's type; K and N multiples of 8, at most 2^20; at most 1024 experts.
    ``ends``: int32 ``(E,)`` on the device, ``torch.cumsum(counts, 0, dtype=torch.int32)``: expert e's rows end before ``ends[e]`` and begin where those of
    the one before end.  An expert may have no rows.  Rows behind the last expert's get zeros, in the output and in x's gradient, whatever they hold.
    Returns ``(T, N)`` of x's type.

    The kernels read ``ends``; nothing comes back to the host.  A call that is captured into a CUDA graph goes by what they hold at each
    replay.  Where they fall, are negative or pass T, no row is taken to be an expert's (all results are zero), and a later call or :func:`read_dense_status`
    raises ``AssertionError``.

    Sums are FP32, rounded once.  Gradients, captures, tangents and traces as for :func:`gated_feed_forward`; the gradient of an expert without rows is
    zero.  The same bits in every call."""
    global _grouped_projection
    if _grouped_projection is None:
        from .backend.grouped import grouped_projection as _grouped_projection
    return _grouped_projection(x, w, ends)


def grouped_feed_forward(x, w13, w2, ends, *, activation_clamp: Optional[float] = None):
    """:func:`gated_feed_forward` with the weights of each row's expert, with its gradients: ``x`` ``(T, H)``, ``w13`` ``(E, 2 I, H)`` in checkpoint order, the
    gate's rows first, ``w2`` ``(E, H, I)``; rows and ``ends`` as in :func:`grouped_projection`.  Returns ``(T, H)``.  As there, ``h`` and in the backward pass the
    gradients of g and u are rounded to the type, as operands of the next product: in FP16 they overflow past 65504."""
    global _grouped_feed_forward
    if _grouped_feed_forward is None:
        from .backend.grouped import grouped_feed_forward as _grouped_feed_forward
    return _grouped_feed_forward(x, w13, w2, ends, activation_clamp=activation_clamp)


def prepare_fp8_inputs(hidden_states, out=None):
    """Quantiser of BF16 or FP16 hidden states ``(..., K)`` by groups of 128 values; returns ``(float8_e4m3fn (..., K), float32 scales (..., ceil(K / 128)))``.
    ``scale = max|x| / 448`` (1 for a group of zeros), values ``x / scale`` rounded to the nearest, ties to even.  A group that holds an infinity or a
    NaN gets the scale NaN and zeros, so that what is computed from it is NaN.  ``out``: the two tensors, contiguous."""
    global _quantize_fp8
    if _quantize_fp8 is None:
        from .backend.grouped import prepare_fp8_inputs as _quantize_fp8
    return _quantize_fp8(hidden_states, out)


def fp8_projection(x, x_scales, w, w_scales, *, ends=None, out_dtype=None):
    """Product in 8-bit floating point with a scale for each 128 values of a row and each block of 128 x 128 weights: ``y[t, n] = sum_k x[t, k] sx[t, k / 128]
    w[n, k] sw[n / 128, k / 128]``.  ``x``: float8_e4m3fn ``(..., K)`` with float32 scales ``(..., ceil(K / 128))`` (:func:`prepare_fp8_inputs`); ``w``:
    float8_e4m3fn ``(N, K)``, contiguous and on 16 bytes, with ``(ceil(N / 128), ceil(K / 128))``; K a multiple of 16, K and N at most 2^20.  With
    ``ends`` rows are grouped by expert as in :func:`grouped_projection`: ``x`` ``(T, K)``, ``w`` ``(E, N, K)``, ``w_scales`` ``(E, ..., ...)``.  ``out_dtype``:
    BF16 (default), FP16 or FP32.  Scales may be any numbers; each sum over 128 values is multiplied by their product and added in FP32.  No gradient."""
    global _fp8_projection
    if _fp8_projection is None:
        from .backend.grouped import fp8_projection as _fp8_projection
    return _fp8_projection(x, x_scales, w, w_scales, ends=ends, out_dtype=out_dtype)


def fp8_gated_projection(x, x_scales, w13, w13_scales, *, ends=None, activation_clamp: Optional[float] = None, out_dtype=None):
    """The first half of a gated feed-forward block in 8-bit floating point: both products (``w13`` ``(2 I, K)``, the gate's rows first, I a multiple of 8, scales
    ``(2 ceil(I / 128), ceil(K / 128))``, the gate's blocks first and those of the up rows begun anew), the activation and their product in one
    kernel, ``silu(min(g, c)) * clip(u, -c, c)`` in ``(..., I)``.  Quantise it with :func:`prepare_fp8_inputs` for :func:`fp8_projection`.  Otherwise as there; the
    activation as in :func:`int8_gated_projection`."""
    global _fp8_gated_projection
    if _fp8_gated_projection is None:
        from .backend.grouped import fp8_gated_projection as _fp8_gated_projection
    return _fp8_gated_projection(x, x_scales, w13, w13_scales, ends=ends, activation_clamp=activation_clamp, out_dtype=out_dtype)


def read_dense_status(device=None) -> None:
    """:func:`read_status` of the dense and grouped operators' calls on ``device`` (default: the current one): ``RuntimeError`` for a wait that
    expired, ``AssertionError`` for ``ends`` that were not in order."""
    from .backend.dense import read_dense_status as _impl

    return _impl(device)


def precompile_mega_moe_variants(num_ranks: int, num_experts: int, num_max_tokens_per_rank: int, num_topk: int,
                                 hidden: int, intermediate_hidden: int, num_shared_experts: int = 0, *,
                                 activation_clamp: Optional[float] = None, activation_alpha: float = 1.0,
                                 activation_beta: float = 0.0, fast_math: bool = True, per_die: bool = False,
                                 localized_weights: bool = False, localized_shared_weights: bool = False
                                 ) -> Tuple[int, ...]:
    """Prepare every BLOCK_M variant the geometry can select, before CUDA-graph capture; returns the variants."""
    from .backend.frontend import precompile_mega_moe_variants as _impl

    return _impl(num_ranks, num_experts, num_max_tokens_per_rank, num_topk, hidden, intermediate_hidden,
                 num_shared_experts, activation_clamp=activation_clamp, activation_alpha=activation_alpha,
                 activation_beta=activation_beta, fast_math=fast_math, per_die=per_die,
                 localized_weights=localized_weights, localized_shared_weights=localized_shared_weights)


def read_status(sym_buffer) -> None:
    """Synchronise and raise if a device-side wait expired (``RuntimeError``) or an expert id was out of range
    (``AssertionError``) in any call on ``sym_buffer`` since the last read; clears the condition."""
    from .backend.frontend import read_status as _impl

    return _impl(sym_buffer)


def set_kernel_options(**kwargs):
    from .backend.frontend import set_kernel_options as _impl

    return _impl(**kwargs)


def get_kernel_options():
    from .backend.frontend import get_kernel_options as _impl

    return _impl()


def is_localization_available() -> bool:
    from .backend.locality import is_localization_available as _impl

    return _impl()


def get_balanced_sm_locality_domains():
    from .backend.locality import get_balanced_sm_locality_domains as _impl

    return _impl()


def localize(t, dim: int = -2):
    from .backend.locality import localize as _impl

    return _impl(t, dim)


def localize_mega_moe_weights(l1_weights, l2_weights):
    """Two-slice form of the routed weight tensors of ``(weights, sf)`` pairs; scale factors are left as they are."""
    from .backend.locality import localize as _impl

    return (_impl(l1_weights[0]), l1_weights[1]), (_impl(l2_weights[0]), l2_weights[1])


def __getattr__(name: str):
    if name == "SymmBuffer":
        from .backend.workspace import SymmBuffer

        return SymmBuffer
    raise AttributeError(name)


__all__ = [
    "get_symm_buffer_for_mega_moe", "transform_weights_for_mega_moe", "fp8_fp4_mega_moe", "get_block_m_for_mega_moe",
    "get_token_alignment_for_mega_moe", "get_unsupported_reason_for_mega_moe", "stage_inputs_for_mega_moe",
    "route_and_stage_inputs_for_mega_moe", "prepare_megamoe_nvfp4_inputs",
    "precompile_mega_moe_variants", "set_kernel_options", "get_kernel_options", "is_localization_available",
    "get_balanced_sm_locality_domains", "localize", "localize_mega_moe_weights", "read_status", "SymmBuffer",
    "gated_feed_forward", "prepare_int8_inputs", "int8_projection", "int8_gated_projection", "read_dense_status",
    "grouped_projection", "grouped_feed_forward", "prepare_fp8_inputs", "fp8_projection", "fp8_gated_projection",
]
