"""Softmax attention over a sliding window with a few first tokens that stay visible: whole sequences, for prompts, evaluation and training.

    o_t = sum_j softmax_j(scale q_t . k_j) v_j        over the keys j <= p of its sequence with j > p - window or j < sinks

    q               [B, T, H, D]    bf16 (or fp32), last dim contiguous
    k, v            [B, S, HK, D]   HK divides H (query head h reads head h / (H / HK)); query t stands at position p = t + S - T
    window          visible keys up to a query's own, itself among them; None = all
    sinks           first tokens of a sequence that every query of it sees
    cu_seqlens      [N + 1]         int32 with leading 0 (then B must be 1 and T == S)
    returns  o [B, T, H, D] in q.dtype

D is a multiple of 8, at most 256.  Queries that see no key, and tokens that belong to no sequence (padding, tokens in front of and behind the
packed sequences), read as zeros in ``o`` and in the gradients.  A query's output depends on nothing but the keys and values that it sees,
whatever the others hold; a gradient may be spoiled by values of the same sequence or batch row that are not finite, seen or not.

Differentiable in q, k and v; the backward works from the saved inputs, the output and one number per row.  Second derivatives and dual
tensors (forward mode) are refused, and in bf16 gradients with more than 65280 query heads to one of k and v.  The kernels are those of ``csrc/gdn_window_attention*.hip``; there is no fallback.
"""

from __future__ import annotations

import torch

from ._autograd import as_int32, kernel_rows, refuse_tangents
from ._host import host, raw_stream
from .kernels import Kernel, is_kernel_allowed
from .layer_ops import _dtype_code
from .rotary import refused


_MAX_D = 256
_LONG = 1 << 30  # windows from here on hold every key


def check_window(window, sinks) -> tuple[int, int]:
    """As the kernels take them: a window of 0 is none."""
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 (a query sees itself) or None, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return (0 if window is None or window >= _LONG else int(window)), min(int(sinks), _LONG)


def _check_inputs(q, k, v, cu_seqlens, left_padded) -> None:
    if not is_kernel_allowed(Kernel.window_attention):
        raise RuntimeError("Kernel.window_attention is disabled and this package ships no other implementation of it; "
                           "enable it (it is on by default) with lm_engine_amd.kernels.enable_kernels")  # fmt: skip
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [B, T, H, D] tensors")
    B, T, H, D = q.shape
    if v.shape != k.shape:
        raise ValueError(f"v {tuple(v.shape)} must have the shape of k {tuple(k.shape)}")
    if k.size(0) != B or k.size(3) != D:
        raise ValueError(f"k {tuple(k.shape)} must share B and D with q {tuple(q.shape)}")
    HK = k.size(2)
    if H == 0 or HK == 0 or H % HK != 0:
        raise ValueError(f"the heads of q ({H}) must be a multiple of the heads of k and v ({HK})")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    _dtype_code(q.dtype, "q, k, v")
    if D == 0 or D % 8 != 0 or D > _MAX_D:
        raise ValueError(f"head dim D={D} is not supported (a multiple of 8, at most {_MAX_D})")
    if cu_seqlens is not None:
        if cu_seqlens.is_floating_point() or cu_seqlens.dtype == torch.bool:
            raise ValueError(f"cu_seqlens must hold integers, got {cu_seqlens.dtype}")
        if k.size(1) != T:
            raise ValueError(f"with cu_seqlens q and k have the same tokens, got {T} and {k.size(1)}")
        if left_padded and (cu_seqlens.dim() != 1 or cu_seqlens.numel() != B + 1):
            raise ValueError(f"left_padded needs cu_seqlens [B + 1] = [{B + 1}]: the prefix sums of the valid lengths")
        if not left_padded and B != 1:
            raise ValueError(f"with cu_seqlens the batch dim must be 1 (tokens packed along T), got B={B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
            raise ValueError("cu_seqlens must be a 1-D tensor [N + 1]")
    elif left_padded:
        raise ValueError(f"left_padded needs cu_seqlens [B + 1] = [{B + 1}]: the prefix sums of the valid lengths")
    if not q.is_cuda:
        raise ValueError("sliding_window_attention runs on the GPU only; inputs must be device tensors")
    for name, x in (("k", k), ("v", v), ("cu_seqlens", cu_seqlens)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} is on {x.device}, q is on {q.device}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x``, or a copy where its rows cannot be read in 16-byte pieces or lie too far apart for the kernels' 32-bit offsets in a tile."""
    x = x.detach()
    far = x.stride(1) > 1 << 23 or x.stride(2) * x.size(2) > 1 << 28
    return x.clone(memory_format=torch.contiguous_format) if far else kernel_rows(x, 16 // x.element_size())


def _empty_lse(q: torch.Tensor) -> torch.Tensor:
    """Of rows that see no key: one number each, fp32 two."""
    return q.new_full(q.shape[:3], float("inf"), dtype=torch.float32) if q.dtype == torch.bfloat16 else q.new_zeros(*q.shape[:3], 2)


def _forward(q, k, v, window, sinks, scale, cu_seqlens, left_padded, wants_lse):
    """(o, lse or None)"""
    _check_inputs(q, k, v, cu_seqlens, left_padded)
    refuse_tangents("sliding_window_attention", q, k, v)
    if q.numel() == 0 or k.numel() == 0:
        return torch.zeros_like(q, memory_format=torch.contiguous_format), _empty_lse(q) if wants_lse else None
    with torch.cuda.device(q.device), torch.no_grad():
        cu_seqlens = as_int32(cu_seqlens)
        result = host().window_attention(raw_stream(q.get_device()), _rows(q), _rows(k), _rows(v), window, sinks, scale, cu_seqlens, left_padded, wants_lse)
        if result is None:
            raise refused("sliding_window_attention", q)
    return result


def _backward(q, k, v, o, lse, window, sinks, scale, cu_seqlens, left_padded, do):
    """(dq, dk, dv)"""
    _check_inputs(q, k, v, cu_seqlens, left_padded)
    refuse_tangents("the backward of sliding_window_attention", q, k, v, do)
    if q.numel() == 0 or k.numel() == 0:
        return tuple(torch.zeros_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    with torch.cuda.device(q.device), torch.no_grad():
        cu_seqlens = as_int32(cu_seqlens)
        result = host().window_attention_bwd(raw_stream(q.get_device()), _rows(q), _rows(k), _rows(v), _rows(o), lse, window, sinks, scale, cu_seqlens,
                                             left_padded, _rows(do.to(q.dtype)))  # fmt: skip
        if result is None:
            raise refused("the backward of sliding_window_attention", q, k, v)
    return result


def _on_host_path(q, *operands):
    """``(o, lse)``, or None where the operands need a conversion, a gradient or a report."""
    if not q.is_cuda or not is_kernel_allowed(Kernel.window_attention):
        return None
    return host().window_attention(raw_stream(q.get_device()), q, *operands)


class _WindowAttention(torch.autograd.Function):
    """Forward and backward on the HIP kernels; the forward keeps its inputs, its output and one number per row."""

    @staticmethod
    def forward(ctx, window, sinks, scale, left_padded, q, k, v, cu_seqlens):
        operands = (q, k, v, window, sinks, scale, cu_seqlens, left_padded, True)
        result = _on_host_path(*operands)
        o, lse = _forward(*operands) if result is None else result
        ctx.save_for_backward(q, k, v, o, lse, cu_seqlens)
        ctx.options = (window, sinks, scale)
        ctx.left_padded = left_padded
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, cu_seqlens = ctx.saved_tensors
        operands = (q, k, v, o, lse, *ctx.options, cu_seqlens, ctx.left_padded, do)
        grads = None
        if is_kernel_allowed(Kernel.window_attention):
            grads = host().window_attention_bwd(raw_stream(q.get_device()), *operands)
        if grads is None:
            grads = _backward(*operands)
        return (None, None, None, None, *grads, None)


def sliding_window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
    cu_seqlens: torch.Tensor | None = None,
    left_padded: bool = False,
) -> torch.Tensor:
    """Whole sequences: prompts, evaluation, training; with fewer queries than keys the continuation of a sequence whose keys and values are
    at hand.  ``scale=None`` is ``D ** -0.5``.

    bf16 inputs run on the matrix units: scores, weights and sums are fp32, the weights are rounded to bf16 as operands of ``o`` (and with
    their gradients of those of q, k and v).  fp32 inputs are computed in fp32 throughout.

    ``left_padded=True`` keeps a padded batch ``[B, T, ...]`` as it is, as in ``chunk_gated_delta_rule``: ``cu_seqlens`` ``[B + 1]``
    holds the prefix sums of the valid lengths, sequence b is the last ``cu_seqlens[b+1] - cu_seqlens[b]`` tokens of row b."""
    window, sinks = check_window(window, sinks)
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    if torch.compiler.is_compiling():  # a graph is being captured: the kernels go in as opaque operators
        from . import _opaque

        return _opaque.sliding_window_attention(q, k, v, window, sinks, scale, cu_seqlens, left_padded)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(window, sinks, scale, left_padded, q, k, v, cu_seqlens)
    result = _on_host_path(q, k, v, window, sinks, scale, cu_seqlens, left_padded, False)
    return (_forward(q, k, v, window, sinks, scale, cu_seqlens, left_padded, False) if result is None else result)[0]
