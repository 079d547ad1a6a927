"""RMS norm of every head of the queries and keys and the rotation by position, in one pass: what stands between a mixer's projection and
its attention.  Forward and backward are one HIP kernel each (the sums over rows behind the weights' gradients one more).

Per head x of a token at position p, with the first R dims rotated in pairs (i, i + R / 2):

    n = x / sqrt(mean(x^2) + eps) * weight
    y_i = n_i cos[p, i] - n_{i + R/2} sin[p, i]        y_{i + R/2} = n_{i + R/2} cos[p, i] + n_i sin[p, i]        y_i = n_i for i >= R

There is no torch fallback.
"""

from __future__ import annotations

import torch

from . import _lib
from ._autograd import as_int32, kernel_rows, refuse_tangents
from ._host import host, raw_stream
from .kernels import Kernel, is_kernel_allowed
from .layer_ops import _dtype_code


def rotary_table(
    positions: int, dims: int, base: float = 10000.0, device: torch.device | str | None = "cuda"
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)``, fp32 ``[positions, dims / 2]``: angle ``p base^(-2 i / dims)``, formed in 64 bits (at position 65536 an angle in 32
    bits is off by 2e-3).  Made once, for all layers and steps."""
    if dims <= 0 or dims % 2 != 0:
        raise ValueError(f"dims must be an even number of rotated dims, got {dims}")
    if positions <= 0:
        raise ValueError(f"positions must be positive, got {positions}")
    pair = torch.arange(dims // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * float(base) ** (-2.0 * pair / dims)
    return angle.cos().to(torch.float32), angle.sin().to(torch.float32)


def _check(q, k, q_weight, k_weight, cos, sin, positions) -> None:
    if not is_kernel_allowed(Kernel.qk_norm_rotary):
        raise RuntimeError("Kernel.qk_norm_rotary is disabled and this package ships no other implementation of it")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be [B, T, H, D] tensors")
    if k.shape[:2] != q.shape[:2] or k.size(-1) != q.size(-1):
        raise ValueError(f"k {tuple(k.shape)} must share [B, T, ., D] with q {tuple(q.shape)}")
    B, T, H, D = q.shape
    if H == 0 or k.size(2) == 0:
        raise ValueError("q and k need at least one head")
    if k.dtype != q.dtype:
        raise ValueError(f"q and k must share a dtype, got {q.dtype} and {k.dtype}")
    _dtype_code(q.dtype, "q and k")
    if D == 0 or D % 8 != 0 or D > _lib.GDN_QK_ROTARY_MAX_D:
        raise ValueError(f"head dim D={D} is not supported (a multiple of 8, at most {_lib.GDN_QK_ROTARY_MAX_D})")
    if cos.dim() != 2 or cos.shape != sin.shape or not cos.is_floating_point() or not sin.is_floating_point():
        raise ValueError(f"cos and sin must be floating-point tables [positions, R / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    R = 2 * cos.size(1)
    if R == 0 or R % 8 != 0 or R > D or cos.size(0) == 0:
        raise ValueError(f"the tables rotate R={R} dims; a multiple of 8, at most D={D}, and at least one position are needed")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if tuple(w.shape) != (D,):
                raise ValueError(f"{name} must be [D] = {(D,)}, got {tuple(w.shape)}")
            _dtype_code(w.dtype, name)
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"q_weight and k_weight must share a dtype, got {q_weight.dtype} and {k_weight.dtype}")
    if positions is None:
        if T > cos.size(0):
            raise ValueError(f"{T} tokens, and the tables have {cos.size(0)} positions")
    elif tuple(positions.shape) not in ((B, T), (T,)) or positions.is_floating_point() or positions.dtype == torch.bool:
        raise ValueError(f"positions must be integers [B, T] = {(B, T)} or [T], got {positions.dtype} {tuple(positions.shape)}")
    if not q.is_cuda:
        raise ValueError("qk_norm_rotary runs on the GPU only; q must be a device tensor")
    for name, x in (("k", k), ("q_weight", q_weight), ("k_weight", k_weight), ("cos", cos), ("sin", sin), ("positions", positions)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} is on {x.device}, q is on {q.device}")


def _dense(x, dtype=None):
    """Contiguous, at a multiple of 16 bytes, of ``dtype``."""
    if x is None:
        return None
    x = (x if dtype is None else x.to(dtype)).detach().contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _operands(q, k, q_weight, k_weight, cos, sin, positions):
    """In the form the kernels read: copies where rows or tables do not lie so."""
    rows = lambda x: kernel_rows(x.detach(), 16 // x.element_size())  # noqa: E731
    return rows(q), rows(k), _dense(q_weight), _dense(k_weight), _dense(cos, torch.float32), _dense(sin, torch.float32), as_int32(positions)


def refused(what: str, *outputs: torch.Tensor) -> Exception:
    """For a call that its host path has refused although every operand was checked.  Where memory was short, allocating results of that
    size raises torch's own error here."""
    for x in outputs:
        torch.empty_like(x)
    return ValueError(f"{what}: these operands are not supported (a size past the kernels' 32-bit counts, or a tensor that is no plain one)")


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps):
    _check(q, k, q_weight, k_weight, cos, sin, positions)
    refuse_tangents("qk_norm_rotary", q, k, q_weight, k_weight, cos, sin)
    if q.size(0) * q.size(1) == 0:
        return q.new_empty(q.shape), k.new_empty(k.shape)
    with torch.cuda.device(q.device), torch.no_grad():
        operands = _operands(q, k, q_weight, k_weight, cos, sin, positions)
        result = host().qk_rotary(raw_stream(q.get_device()), *operands, eps)
        if result is None:
            raise refused("qk_norm_rotary", q, k)
    return result


def _backward(q, k, q_weight, k_weight, cos, sin, positions, eps, dq, dk, needs_q, needs_k):
    """(gradients of q, k, q_weight or None, k_weight or None) from those of the results."""
    _check(q, k, q_weight, k_weight, cos, sin, positions)
    refuse_tangents("the backward of qk_norm_rotary", q, k, q_weight, k_weight, dq, dk)
    if q.size(0) * q.size(1) == 0:
        return q.new_empty(q.shape), k.new_empty(k.shape), torch.zeros_like(q_weight) if needs_q else None, torch.zeros_like(k_weight) if needs_k else None
    with torch.cuda.device(q.device), torch.no_grad():
        operands = _operands(q, k, q_weight, k_weight, cos, sin, positions)
        dq, dk = (kernel_rows(d.detach().to(x.dtype), 16 // x.element_size()) for d, x in ((dq, q), (dk, k)))
        result = host().qk_rotary_bwd(raw_stream(q.get_device()), *operands, eps, dq, dk, needs_q, needs_k)
        if result is None:
            raise refused("the backward of qk_norm_rotary", q, k)
    return result


def _on_host_path(*operands):
    """(q', k'), or None where the operands need a conversion, a gradient or a report."""
    q = operands[0]
    if not q.is_cuda or not is_kernel_allowed(Kernel.qk_norm_rotary):
        return None
    return host().qk_rotary(raw_stream(q.get_device()), *operands)


class _QkNormRotary(torch.autograd.Function):
    """Forward and backward on the HIP kernels; the forward keeps nothing but its inputs."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        result = _on_host_path(q, k, q_weight, k_weight, cos, sin, positions, eps)
        if result is None:
            result = _forward(q, k, q_weight, k_weight, cos, sin, positions, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return result

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        saved = ctx.saved_tensors
        needs = ctx.needs_input_grad[2:4]
        grads = None
        if is_kernel_allowed(Kernel.qk_norm_rotary):
            grads = host().qk_rotary_bwd(raw_stream(saved[0].get_device()), *saved, ctx.eps, dq, dk, *needs)
        if grads is None:
            grads = _backward(*saved, ctx.eps, dq, dk, *needs)
        return (*grads, None, None, None, None)


def qk_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """q ``[B, T, H, D]``, k ``[B, T, HK, D]`` (bf16 or fp32, any strides; column blocks of one projection are read where they lie), weights
    ``[D]`` (bf16 or fp32) or None, the tables ``[positions, R / 2]`` fp32 (``rotary_table``), ``positions`` integers ``[B, T]`` or ``[T]`` or
    None (token t stands at position t).  Returns the normed and rotated q and k, contiguous, computed in fp32 and rounded once.

    D and R are multiples of 8, D at most 512.  A position that the tables do not have makes its rows NaN.  Differentiable in q, k and the
    weights, but neither twice nor in forward mode; the tables are constants, and refused where a gradient of theirs is wanted."""
    eps = float(eps)
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):  # (before a Function, inside of which nothing wants one)
        raise ValueError("cos and sin are constants: they get no gradient")
    if torch.compiler.is_compiling():  # a graph is being captured: the kernels go in as opaque operators
        from . import _opaque

        return _opaque.qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
    result = _on_host_path(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps) if result is None else result
