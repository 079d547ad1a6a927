"""Layer norm, forward and backward, one HIP kernel each (the sums over rows behind the parameters' gradients one more).

What lm_engine/modeling_utils/normalization.py builds for a ``layernorm`` block: the norm of a hidden size in front of a mixer's
projections, or of a head's size behind it.  There is no torch fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._autograd import refuse_tangents
from ._host import host, raw_stream
from .kernels import Kernel, is_kernel_allowed
from .layer_ops import _dtype_code, column_sums


def _check(x, weight, bias) -> int:
    if not is_kernel_allowed(Kernel.layer_norm):
        raise RuntimeError("Kernel.layer_norm is disabled and this package ships no other implementation of it")
    if not x.is_cuda:
        raise ValueError("x must be a device tensor: layer norm runs on the GPU only")
    if x.dim() < 1:
        raise ValueError("x must be [..., D]")
    D = x.size(-1)
    _dtype_code(x.dtype, "x")
    if D == 0 or D > _lib.GDN_LAYER_NORM_MAX_D:
        raise ValueError(f"rows of D={D} are not supported (1 to {_lib.GDN_LAYER_NORM_MAX_D})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (D,):
            raise ValueError(f"{name} must be [D] = {(D,)}, got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name} is on {p.device}, x is on {x.device}")
        _dtype_code(p.dtype, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must share a dtype, got {weight.dtype} and {bias.dtype}")
    return D


def _as_rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """``(x or a copy, elements between rows, rows)``: the leading dims as one, where they collapse."""
    D = x.size(-1)
    if x.stride(-1) != 1 and D > 1:
        x = x.contiguous()
    rows = x.reshape(-1, D)  # a view whenever the leading dims collapse
    return rows, (rows.stride(0) if rows.size(0) > 1 else D), rows.size(0)


def _forward(x, weight, bias, eps):
    D = _check(x, weight, bias)
    refuse_tangents("layer norm", x, weight, bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    rows, stride, count = _as_rows(x)
    weight, bias = (None if p is None else p.contiguous() for p in (weight, bias))
    args = _lib.GdnLayerNormArgs()
    args.x, args.y = rows.data_ptr(), y.data_ptr()
    args.weight = None if weight is None else weight.data_ptr()
    args.bias = None if bias is None else bias.data_ptr()
    args.x_stride, args.y_stride, args.rows, args.D = stride, D, count, D
    args.dtype = _dtype_code(x.dtype, "x")
    parameter = weight if weight is not None else bias
    args.w_dtype = _lib.GDN_F32 if parameter is None else _dtype_code(parameter.dtype, "weight")
    args.eps = eps
    lib = _lib.load_library()
    with torch.cuda.device(x.device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)
        _lib.check_status(lib.gdn_layer_norm_fwd(ctypes.byref(args), stream), "gdn_layer_norm_fwd")
    return y


def _backward(x, weight, bias_dtype, eps, dy, needs_dw, needs_db):
    """``gdn_layer_norm_bwd``: (dx, dweight or None, dbias or None)."""
    D = _check(x, weight, None)
    refuse_tangents("the backward of layer norm", x, weight, dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return dx, (torch.zeros_like(weight) if needs_dw else None), (torch.zeros(D, dtype=bias_dtype, device=x.device) if needs_db else None)
    rows, stride, count = _as_rows(x)
    dy_rows, dy_stride, _ = _as_rows(dy.to(x.dtype))
    weight = None if weight is None else weight.contiguous()
    lib = _lib.load_library()
    with torch.cuda.device(x.device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)
        code = _dtype_code(x.dtype, "x")
        blocks = lib.gdn_layer_norm_partial_blocks(count, D, code)
        new = lambda: torch.empty(blocks, D, dtype=torch.float32, device=x.device)  # noqa: E731
        dw, db = new() if needs_dw else None, new() if needs_db else None
        args = _lib.GdnLayerNormBwdArgs()
        args.x, args.dy, args.dx = rows.data_ptr(), dy_rows.data_ptr(), dx.data_ptr()
        args.weight = None if weight is None else weight.data_ptr()
        args.dweight_partial = None if dw is None else dw.data_ptr()
        args.dbias_partial = None if db is None else db.data_ptr()
        args.x_stride, args.dy_stride, args.dx_stride, args.rows, args.D = stride, dy_stride, D, count, D
        args.dtype = code
        args.w_dtype = _lib.GDN_F32 if weight is None else _dtype_code(weight.dtype, "weight")
        args.eps, args.partial_blocks = eps, blocks
        _lib.check_status(lib.gdn_layer_norm_bwd(ctypes.byref(args), stream), "gdn_layer_norm_bwd")
        wanted = ([(dw, weight.dtype)] if needs_dw else []) + ([(db, bias_dtype)] if needs_db else [])
        sums = column_sums(lib, stream, *wanted) if wanted else []
    return dx, (sums[0] if needs_dw else None), (sums[-1] if needs_db else None)


def _on_host_path(x, weight, bias, eps):
    """y, or None where the operands need a conversion, a gradient or a report."""
    if not x.is_cuda or not is_kernel_allowed(Kernel.layer_norm):
        return None
    return host().layer_norm(raw_stream(x.get_device()), x, weight, bias, eps)


class _LayerNorm(torch.autograd.Function):
    """Forward and backward on the HIP kernels; the forward keeps nothing but its inputs."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y = _on_host_path(x, weight, bias, eps)
        if y is None:
            y = _forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight)
        ctx.options = (None if bias is None else bias.dtype, eps)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        bias_dtype, eps = ctx.options
        needs_dw, needs_db = ctx.needs_input_grad[1:3]
        grads = None
        if is_kernel_allowed(Kernel.layer_norm):
            grads = host().layer_norm_bwd(raw_stream(x.get_device()), x, weight, eps, dy, needs_dw, needs_db, bias_dtype == torch.bfloat16)
        if grads is None:
            grads = _backward(x, weight, bias_dtype, eps, dy, needs_dw, needs_db)
        return (*grads, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """x ``[..., D]`` (bf16 or fp32, D up to 16384; leading dims that collapse to rows of one stride are read where they lie); weight and
    bias ``[D]`` (bf16 or fp32) or None.  Returns ``(x - mean) / sqrt(var + eps) * weight + bias`` over D, shape and dtype of x, contiguous;
    mean, variance and everything up to the result in fp32.  Differentiable, but neither twice nor in forward mode."""
    eps = float(eps)
    if torch.compiler.is_compiling():  # a graph is being captured: the kernel goes in as an opaque operator
        from . import _opaque

        return _opaque.layer_norm(x, weight, bias, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    y = _on_host_path(x, weight, bias, eps)
    return _forward(x, weight, bias, eps) if y is None else y
