"""Linear attention with a decay for each head: chunked form for prompts and training, recurrent form for single tokens.

The reference's ``linear_attention_torch`` (lm_engine/modeling_utils/sequence_mixer_blocks/linear_attention/op.py:10-44) with a
log-decay per head: per (sequence, head), w = exp(g), state S ``[K, V]`` in fp32,

    S_t = w S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t

    q, k            [B, T, HK, K]   bf16 (or fp32), last dim contiguous; HK divides H (value head h reads head h / (H / HK))
    v               [B, T, H, V]
    g               [H]             log-decay of one token (<= 0); None = no decay.  Differentiable.
    initial_state   [N, H, K, V]    fp32; N = B, or number of packed sequences
    cu_seqlens      [N + 1]         int32 with leading 0 (then B must be 1)
    returns  o [B, T, H, V] in v.dtype, final_state [N, H, K, V] fp32 or None

K and V are multiples of 8, K at most 256.  Tokens that belong to no sequence (padding, tokens behind the last packed sequence)
read as zeros in ``o`` and in the gradients.  A token whose values are not finite spoils the outputs of the 64 tokens around it that
are computed together with it, earlier ones among them.

Both forms are differentiable; the backward works from the saved inputs (``gdn_linear_attn_bwd``).  Second derivatives and dual tensors
(forward mode) are refused.  The kernels
are those of ``csrc/gdn_linear_*.hip``; there is no fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._autograd import kernel_rows, mark_written, refuse_tangents
from ._host import host, raw_stream
from .kernels import Kernel, is_kernel_allowed
from .ops import RECURRENT_MAX_TOKENS, _dtype_code


_MAX_K = 256


def _require_hip_path() -> None:
    if not is_kernel_allowed(Kernel.linear_attention):
        raise RuntimeError("Kernel.linear_attention is disabled and this package ships no other implementation of it; "
                           "enable it (it is on by default) with lm_engine_amd.kernels.enable_kernels")  # fmt: skip


def _check_inputs(q, k, v, g, initial_state, cu_seqlens, left_padded):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [B, T, H, D] tensors")
    B, T, HK, K = q.shape
    H, V = v.size(2), v.size(-1)
    if k.shape != q.shape:
        raise ValueError(f"k {tuple(k.shape)} must have the shape of q {tuple(q.shape)}")
    if v.shape[:2] != q.shape[:2]:
        raise ValueError(f"v {tuple(v.shape)} must share [B, T] with q {tuple(q.shape)}")
    if HK == 0 or H == 0 or H % HK != 0:
        raise ValueError(f"the heads of v ({H}) must be a multiple of the heads of q and k ({HK})")
    if not q.is_cuda:
        raise ValueError("linear attention runs on the GPU only; inputs must be device tensors")
    for name, x in (("k", k), ("v", v), ("g", g), ("initial_state", initial_state), ("cu_seqlens", cu_seqlens)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} is on {x.device}, q is on {q.device}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    _dtype_code(q.dtype, "q, k, v")
    if K == 0 or K % 8 != 0 or K > _MAX_K:
        raise ValueError(f"head dim K={K} is not supported (a multiple of 8, at most {_MAX_K})")
    if V == 0 or V % 8 != 0:
        raise ValueError(f"value head dim V={V} must be a multiple of 8")
    if g is not None and (tuple(g.shape) != (H,) or not g.is_floating_point()):
        raise ValueError(f"g must be a floating-point tensor [H] = {(H,)}, got {g.dtype} {tuple(g.shape)}")
    N = B
    if cu_seqlens is not None and cu_seqlens.is_floating_point():
        raise ValueError(f"cu_seqlens must hold integers, got {cu_seqlens.dtype}")
    if left_padded:
        if cu_seqlens is None or cu_seqlens.dim() != 1 or cu_seqlens.numel() != B + 1:
            raise ValueError(f"left_padded needs cu_seqlens [B + 1] = [{B + 1}]: the prefix sums of the valid lengths")
    elif cu_seqlens is not None:
        if B != 1:
            raise ValueError(f"with cu_seqlens the batch dim must be 1 (tokens packed along T), got B={B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
            raise ValueError("cu_seqlens must be a 1-D tensor [N + 1]")
        N = cu_seqlens.numel() - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (N, H, K, V):
            raise ValueError(f"initial_state must be [N, H, K, V] = {(N, H, K, V)}, got {tuple(initial_state.shape)}")
        if initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be float32, got {initial_state.dtype}")
    return B, T, H, K, V, N


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor at a multiple of 16 bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x``, or a copy where its rows cannot be read in 16-byte pieces or lie too far apart for the kernels' 32-bit offsets in a chunk."""
    return x.clone(memory_format=torch.contiguous_format) if x.stride(1) > 1 << 24 else kernel_rows(x, 16 // x.element_size())


def _set_rows(args, name, x) -> None:
    setattr(args, name, x.data_ptr())
    for i, d in enumerate("bth"):
        setattr(args, f"{name}_stride_{d}", x.stride(i))


def _fill(q, k, v, g, h0, cu_seqlens, scale, left_padded, dims) -> _lib.GdnLinearAttnArgs:
    B, T, H, K, V, N = dims
    a = _lib.GdnLinearAttnArgs()
    for name, x in (("q", q), ("k", k), ("v", v)):
        _set_rows(a, name, x)
    a.g = None if g is None else g.data_ptr()
    a.h0 = None if h0 is None else h0.data_ptr()
    a.cu_seqlens = None if cu_seqlens is None else cu_seqlens.data_ptr()
    a.B, a.T, a.H, a.K, a.V, a.N = B, T, H, K, V, N
    a.qk_heads = 0 if q.size(2) == H else q.size(2)
    a.dtype = _dtype_code(q.dtype, "q, k, v")
    a.flags = _lib.GDN_FLAG_ZERO_PADDING | (_lib.GDN_FLAG_LEFT_PADDED if left_padded else 0)
    a.scale = float(K**-0.5 if scale is None else scale)
    return a


def _operands(q, k, v, g, cu_seqlens):
    q, k, v = _rows(q), _rows(k), _rows(v)
    g = None if g is None else g.to(torch.float32).contiguous()
    cu_seqlens = None if cu_seqlens is None else cu_seqlens.to(torch.int32).contiguous()
    return q, k, v, g, cu_seqlens


def _run(mode, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded):
    _require_hip_path()
    dims = _check_inputs(q, k, v, g, initial_state, cu_seqlens, left_padded)
    B, T, H, K, V, N = dims
    refuse_tangents("linear attention", q, k, v, g, initial_state)
    if inplace_state and (mode != "recurrent" or not output_final_state or initial_state is None or not initial_state.is_contiguous()
                          or initial_state.data_ptr() % 16 != 0):  # fmt: skip
        raise ValueError("inplace_state needs a contiguous initial_state to update and output_final_state=True")
    h0 = None if initial_state is None else _aligned(initial_state)
    o = torch.empty(B, T, H, V, dtype=v.dtype, device=v.device)
    ht = None
    if output_final_state:
        ht = h0 if inplace_state else torch.empty(N, H, K, V, dtype=torch.float32, device=v.device)
    if o.numel() == 0:  # no token: the states stay what they are
        if ht is not None and not inplace_state:
            ht.zero_() if h0 is None else ht.copy_(h0)
        return o, (initial_state if inplace_state else ht)

    q, k, v, g, cu_seqlens = _operands(q, k, v, g, cu_seqlens)
    args = _fill(q, k, v, g, h0, cu_seqlens, scale, left_padded, dims)
    args.ht = None if ht is None else ht.data_ptr()
    _set_rows(args, "o", o)
    lib = _lib.load_library()
    with torch.cuda.device(q.device):
        stream = ctypes.c_void_p(torch.cuda.current_stream(q.device).cuda_stream)
        if mode == "chunk":
            nbytes = int(lib.gdn_linear_attn_workspace_bytes(ctypes.byref(args)))
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            args.workspace, args.workspace_bytes = (None if workspace is None else workspace.data_ptr()), nbytes
            _lib.check_status(lib.gdn_linear_attn_chunk_fwd(ctypes.byref(args), stream), "gdn_linear_attn_chunk_fwd")
        else:
            _lib.check_status(lib.gdn_linear_attn_recurrent_fwd(ctypes.byref(args), stream), "gdn_linear_attn_recurrent_fwd")
    if inplace_state:
        mark_written(initial_state)
    return o, (initial_state if inplace_state else ht)


def _on_host_path(mode, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded):
    """``(o, final_state)``, or None where the operands need a conversion, a gradient or a report."""
    if not q.is_cuda or not is_kernel_allowed(Kernel.linear_attention):
        return None
    return host().linear_attention(raw_stream(q.get_device()), mode == "chunk", q, k, v, g, scale, initial_state, cu_seqlens, left_padded,
                                   output_final_state, inplace_state)  # fmt: skip


def _backward(q, k, v, g, scale, initial_state, cu_seqlens, left_padded, do, dht, needs_dg, needs_dh0):
    """``gdn_linear_attn_bwd``: (dq, dk, dv, dg or None, dh0 or None)."""
    _require_hip_path()
    dims = _check_inputs(q, k, v, g, initial_state, cu_seqlens, left_padded)
    B, T, H, K, V, N = dims
    refuse_tangents("the backward of linear attention", q, k, v, g, initial_state, do, dht)
    HK, dev, dtype = q.size(2), q.device, v.dtype
    new = lambda *shape: torch.empty(*shape, dtype=dtype, device=dev)  # noqa: E731
    dq, dk, dv = new(B, T, HK, K), new(B, T, HK, K), new(B, T, H, V)
    dg = torch.empty(H, dtype=torch.float32, device=dev) if needs_dg else None
    dh0 = torch.empty(N, H, K, V, dtype=torch.float32, device=dev) if needs_dh0 else None
    if v.numel() == 0:
        if dg is not None:
            dg.zero_()
        if dh0 is not None:
            dh0.zero_() if dht is None else dh0.copy_(dht)
        return torch.empty_like(q), torch.empty_like(k), dv, None if dg is None else dg.to(g.dtype), dh0

    g_dtype = None if g is None else g.dtype
    q, k, v, g, cu_seqlens = _operands(q, k, v, g, cu_seqlens)
    do = torch.zeros_like(v, memory_format=torch.contiguous_format) if do is None else _rows(do.to(dtype))
    dht = None if dht is None else _aligned(dht.to(torch.float32))
    h0 = None if initial_state is None else _aligned(initial_state)
    b = _lib.GdnLinearAttnBwdArgs()
    b.fwd = _fill(q, k, v, g, h0, cu_seqlens, scale, left_padded, dims)
    for name, x in (("dout", do), ("dq", dq), ("dk", dk), ("dv", dv)):
        _set_rows(b, name, x)
    b.dht = None if dht is None else dht.data_ptr()
    b.dh0 = None if dh0 is None else dh0.data_ptr()
    b.dg = None if dg is None else dg.data_ptr()
    lib = _lib.load_library()
    with torch.cuda.device(dev):
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        nbytes = int(lib.gdn_linear_attn_bwd_workspace_bytes(ctypes.byref(b)))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        b.workspace, b.workspace_bytes = (None if workspace is None else workspace.data_ptr()), nbytes
        _lib.check_status(lib.gdn_linear_attn_bwd(ctypes.byref(b), stream), "gdn_linear_attn_bwd")
    return dq, dk, dv, (None if dg is None else dg.to(g_dtype)), dh0


class _LinearAttention(torch.autograd.Function):
    """Forward and backward on the HIP kernels; the forward keeps nothing but its inputs."""

    @staticmethod
    def forward(ctx, mode, scale, output_final_state, left_padded, q, k, v, g, initial_state, cu_seqlens):
        operands = (q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, False, left_padded)
        result = _on_host_path(mode, *operands)
        o, ht = _run(mode, *operands) if result is None else result
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, initial_state, cu_seqlens)
        ctx.options = (scale, left_padded)
        return o, ht

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dht):
        q, k, v, g, initial_state, cu_seqlens = ctx.saved_tensors
        scale, left_padded = ctx.options
        if do is None and dht is None:
            return (None,) * 10
        needs_dg, needs_dh0 = ctx.needs_input_grad[7:9]
        grads = None
        if do is not None and is_kernel_allowed(Kernel.linear_attention):
            grads = host().linear_attention_bwd(raw_stream(q.get_device()), q, k, v, g, scale, initial_state, cu_seqlens, left_padded, do, dht,
                                                needs_dg, needs_dh0)  # fmt: skip
        if grads is None:
            grads = _backward(q, k, v, g, scale, initial_state, cu_seqlens, left_padded, do, dht, needs_dg, needs_dh0)
        return None, None, None, None, *grads, None


def _dispatch(mode, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded):
    if torch.compiler.is_compiling():  # a graph is being captured: the kernels go in as opaque operators
        from . import _opaque

        return _opaque.linear_attention(mode, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (g is not None and g.requires_grad)
                                    or (initial_state is not None and initial_state.requires_grad)):  # fmt: skip
        if inplace_state:
            raise ValueError("inplace_state overwrites the initial state the backward needs; it is for inference")
        return _LinearAttention.apply(mode, scale, output_final_state, left_padded, q, k, v, g, initial_state, cu_seqlens)
    operands = (q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded)
    result = _on_host_path(mode, *operands)
    return _run(mode, *operands) if result is None else result


def chunk_linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor | None = None,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.Tensor | None = None,
    head_first: bool = False,
    left_padded: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Whole sequences: prompts, evaluation, training.  ``scale=None`` is ``K ** -0.5``.

    bf16 inputs run in chunks of 64 tokens on the matrix units: the state is kept, and returned, to fp32 accuracy; as an operand of
    ``o`` (and of the gradients) it is rounded to bf16, like the chunk's own weights.  fp32 inputs are computed in fp32, token by token.

    ``left_padded=True`` keeps a padded batch ``[B, T, ...]`` as it is, as in ``chunk_gated_delta_rule``: ``cu_seqlens`` ``[B + 1]``
    holds the prefix sums of the valid lengths, sequence b is the last ``cu_seqlens[b+1] - cu_seqlens[b]`` tokens of row b."""
    if head_first:
        raise ValueError("head_first layouts are not supported; pass [B, T, H, D] tensors")
    return _dispatch("chunk", q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, False, left_padded)


def fused_recurrent_linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor | None = None,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.Tensor | None = None,
    inplace_state: bool = False,
    left_padded: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """One token per sequence, or a few: every state passes through registers once, fp32 throughout.

    With ``inplace_state=True`` (and ``output_final_state=True``) the final state overwrites ``initial_state`` and that same tensor is
    returned, as in ``fused_recurrent_gated_delta_rule``; autograd counts it as written (not where a captured graph is replayed)."""
    return _dispatch("recurrent", q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, inplace_state, left_padded)


def linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(o, final_state)``: the recurrent form up to 64 tokens per row, the chunked form for anything longer, as ``gated_delta_rule``.

    bf16, recurrent | chunked, us, for 1, 16, 32 and 64 tokens a row: 1 sequence of 16 heads of 128 6 | 18, 11 | 18, 18 | 18, 32 | 18; 16 of them
    8 | 20, 18 | 20, 30 | 20, 53 | 21; 256 of them 92 | 190, 169 | 193, 281 | 199, 502 | 222; 16 sequences of 2 heads of 256 x 512 8 | 23, 16 | 23,
    26 | 23, 47 | 23.  So from about 20 tokens on the chunked form is the faster one; the recurrent form, with every product in fp32, is the
    more exact one."""
    fn = fused_recurrent_linear_attention if q.size(1) <= RECURRENT_MAX_TOKENS else chunk_linear_attention
    return fn(q, k, v, g, scale=scale, initial_state=initial_state, output_final_state=True, cu_seqlens=cu_seqlens)
