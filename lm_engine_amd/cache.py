"""A paged cache of keys and values in 8 bits, and attention over it: the serving side of ``sliding_window_attention``.

    cache = new_paged_cache(pages=4096, heads=8, head_dim=128)            # once, for a layer
    write_paged_cache(cache, k, v, block_table, start)                     # new tokens behind the `start` ones that are held
    o = paged_cache_attention(q, cache, block_table, lengths)              # one token per sequence, or a few

A code c (e4m3) of a page and head whose scale is s stands for c 2^(s - 127).  A page's scale is the smallest with which none of its tokens
passes 448; a page that is gone on with keeps its scale or takes a larger one, and the codes that it holds are rounded to it (exact but for
e4m3's smallest exponent, so nothing wears off).  Pages belong to whom ``block_table`` says; pages that several sequences share
are full ones that none of them writes.  The kernels are those of ``csrc/gdn_paged_cache.hip`` and ``csrc/gdn_cache_attention.hip``; there is
no fallback.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._autograd import as_int32, kernel_rows, refuse_tangents
from ._host import host, raw_stream
from .kernels import Kernel, is_kernel_allowed
from .layer_ops import _dtype_code
from .rotary import refused


_LOWEST_SCALE = 27  # an exponent of -100


class PagedCache(NamedTuple):
    """``k`` ``[pages, heads, page_size, D]``, ``v`` ``[pages, heads, page_size / 16, D, 16]`` (16 tokens of a column lie together, as the
    product with the weights reads them), both float8_e4m3fn; their scales ``[pages, heads]`` uint8."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new_paged_cache(pages: int, heads: int, head_dim: int, page_size: int = 64, device: torch.device | str | None = "cuda") -> PagedCache:
    """A cache of zeros.  ``page_size``: tokens of a page, a multiple of 16 up to 256; ``head_dim``: a multiple of 16 up to 256."""
    if pages <= 0 or heads <= 0 or heads > 65535:
        raise ValueError(f"pages and heads must be positive (heads at most 65535), got {pages} and {heads}")
    if page_size <= 0 or page_size % 16 != 0 or page_size > 256:
        raise ValueError(f"page_size={page_size} is not supported (a multiple of 16, at most 256)")
    if head_dim <= 0 or head_dim % 16 != 0 or head_dim > 256:
        raise ValueError(f"head_dim={head_dim} is not supported (a multiple of 16, at most 256)")
    codes = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)  # noqa: E731
    scales = lambda: torch.full((pages, heads), _LOWEST_SCALE, dtype=torch.uint8, device=device)  # noqa: E731
    return PagedCache(codes(pages, heads, page_size, head_dim), codes(pages, heads, page_size // 16, head_dim, 16), scales(), scales())


def _require() -> None:
    if not is_kernel_allowed(Kernel.paged_cache):
        raise RuntimeError("Kernel.paged_cache is disabled and this package ships no other implementation of it")


def _check_cache(cache, block_table, **per_sequence):
    """(HK, P, D, N) of a well-formed cache; ``per_sequence``: integer tensors [N]."""
    _require()
    k, v, k_scale, v_scale = cache
    if k.dim() != 4 or v.dim() != 5:
        raise ValueError("cache.k must be [pages, heads, page_size, D] and cache.v [pages, heads, page_size / 16, D, 16]")
    pages, HK, P, D = k.shape
    if tuple(v.shape) != (pages, HK, P // 16, D, 16) or P % 16 != 0 or P == 0 or P > 256 or D % 16 != 0 or D == 0 or D > 256 or pages == 0 or HK == 0:
        raise ValueError(f"cache.k {tuple(k.shape)} and cache.v {tuple(v.shape)} do not belong together, or their page size or head dim is not "
                         "a multiple of 16 up to 256")  # fmt: skip
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise ValueError(f"cache.k and cache.v must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if tuple(s.shape) != (pages, HK) or s.dtype != torch.uint8:
            raise ValueError(f"cache.{name} must be uint8 [pages, heads] = {(pages, HK)}, got {s.dtype} {tuple(s.shape)}")
    if block_table.dim() != 2 or block_table.is_floating_point() or block_table.dtype == torch.bool:
        raise ValueError(f"block_table must be integers [N, pages of a sequence], got {block_table.dtype} {tuple(block_table.shape)}")
    N = block_table.size(0)
    for name, x in per_sequence.items():
        if tuple(x.shape) != (N,) or x.is_floating_point() or x.dtype == torch.bool:
            raise ValueError(f"{name} must be integers [N] = {(N,)}, got {x.dtype} {tuple(x.shape)}")
    if not k.is_cuda:
        raise ValueError("the paged cache lives on the GPU; its tensors must be device tensors")
    for name, x in (("cache.v", v), ("cache.k_scale", k_scale), ("cache.v_scale", v_scale), ("block_table", block_table), *per_sequence.items()):
        if x.device != k.device:
            raise ValueError(f"{name} is on {x.device}, cache.k is on {k.device}")
    for name, x in zip(PagedCache._fields, cache):
        if not x.is_contiguous() or (x.dim() > 2 and x.data_ptr() % 16 != 0):
            raise ValueError(f"cache.{name} must be contiguous (codes at a multiple of 16 bytes)")
    return HK, P, D, N


def _check_rows(x, name, like, heads, D):
    if x.dim() != 4 or x.size(2) != heads or x.size(3) != D:
        raise ValueError(f"{name} must be [B, T, {heads}, {D}], got {tuple(x.shape)}")
    if x.device != like.device:
        raise ValueError(f"{name} is on {x.device}, cache.k is on {like.device}")


def _write(cache, k, v, block_table, start, cu_seqlens, left_padded):
    HK, P, D, N = _check_cache(cache, block_table, start=start)
    _check_rows(k, "k", cache.k, HK, D)
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError(f"v must have the shape, dtype and device of k, got {v.dtype} {tuple(v.shape)} and {k.dtype} {tuple(k.shape)}")
    _dtype_code(k.dtype, "k and v")
    B, T = k.shape[:2]
    if cu_seqlens is not None:
        if cu_seqlens.is_floating_point() or cu_seqlens.dtype == torch.bool or cu_seqlens.dim() != 1 or cu_seqlens.numel() != N + 1 or cu_seqlens.device != k.device:
            raise ValueError(f"cu_seqlens must be integers [N + 1] = [{N + 1}] on {k.device}")
        if not left_padded and B != 1:
            raise ValueError(f"with cu_seqlens the batch dim must be 1 (tokens packed along T), got B={B}")
    elif left_padded:
        raise ValueError(f"left_padded needs cu_seqlens [B + 1] = [{B + 1}]: the prefix sums of the valid lengths")
    if (cu_seqlens is None or left_padded) and B != N:
        raise ValueError(f"k has {B} rows, block_table has {N}")
    refuse_tangents("write_paged_cache", k, v)
    if B * T == 0 or block_table.size(1) == 0:
        return
    with torch.cuda.device(k.device), torch.no_grad():
        rows = (kernel_rows(x.detach(), 16 // x.element_size()) for x in (k, v))
        done = host().cache_write(raw_stream(k.get_device()), *cache, as_int32(block_table), *rows, as_int32(start), as_int32(cu_seqlens), left_padded)
        if done is None:
            raise refused("write_paged_cache")


def write_paged_cache(
    cache: PagedCache,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table: torch.Tensor,
    start: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    left_padded: bool = False,
) -> PagedCache:
    """Writes k, v ``[B, T, heads, D]`` (bf16 or fp32) behind the ``start`` ``[N]`` tokens that the cache holds of every sequence, and returns
    the cache.  ``block_table`` ``[N, pages]``: the pages of every sequence in order, those of the new tokens among them.  A row of tokens
    per sequence; or packed (B = 1, ``cu_seqlens`` ``[N + 1]``), or ``left_padded``, as in ``sliding_window_attention``.

    What lay behind the new tokens of a page counts as gone: a sequence that is cut back (rejected drafts) is written on from where it
    was cut.  Values that are not finite become NaN and do not count for the scale.  New tokens without a page (a number outside of the
    cache, past the table, in front of position 0) are dropped.  Autograd counts the cache as written; it gets no gradient."""
    if torch.compiler.is_compiling():
        from . import _opaque

        return _opaque.write_paged_cache(cache, k, v, block_table, start, cu_seqlens, left_padded)
    done = None
    if k.is_cuda and is_kernel_allowed(Kernel.paged_cache):
        with torch.no_grad():
            done = host().cache_write(raw_stream(k.get_device()), *cache, block_table, k, v, start, cu_seqlens, left_padded)
    if done is None:
        _write(cache, k, v, block_table, start, cu_seqlens, left_padded)
    return cache


def _read(cache, block_table, lengths, max_tokens, dtype):
    HK, P, D, N = _check_cache(cache, block_table, lengths=lengths)
    code = _dtype_code(dtype, "dtype")
    if max_tokens < 0 or max_tokens > block_table.size(1) * P:
        raise ValueError(f"max_tokens={max_tokens}: block_table has pages for {block_table.size(1) * P} tokens")
    if N * max_tokens == 0:
        empty = cache.k.new_empty((N, max_tokens, HK, D), dtype=dtype)
        return empty, empty.clone()
    with torch.cuda.device(cache.k.device):
        result = host().cache_read(raw_stream(cache.k.get_device()), *cache, as_int32(block_table), as_int32(lengths), max_tokens, code == 0)
        if result is None:
            raise refused("read_paged_cache", *[torch.empty(N, max_tokens, HK, D, dtype=dtype, device=cache.k.device)] * 2)
    return result


def read_paged_cache(
    cache: PagedCache, block_table: torch.Tensor, lengths: torch.Tensor, max_tokens: int | None = None, dtype: torch.dtype = torch.bfloat16
) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds of every sequence's first ``lengths`` ``[N]`` tokens: k, v ``[N, max_tokens, heads, D]`` in ``dtype`` (bf16 holds
    every code exactly), zeros behind a sequence's last token; NaN where its page number is outside of the cache.  ``max_tokens``: what the
    block table has room for, if not given."""
    max_tokens = block_table.size(1) * cache.k.size(2) if max_tokens is None else int(max_tokens)
    if torch.compiler.is_compiling():
        from . import _opaque

        return _opaque.read_paged_cache(cache, block_table, lengths, max_tokens, dtype)
    result = None
    if cache.k.is_cuda and is_kernel_allowed(Kernel.paged_cache) and dtype in (torch.bfloat16, torch.float32):
        result = host().cache_read(raw_stream(cache.k.get_device()), *cache, block_table, lengths, max_tokens, dtype == torch.bfloat16)
    return _read(cache, block_table, lengths, max_tokens, dtype) if result is None else result


def _attend(q, cache, block_table, lengths, window, sinks, scale):
    HK, P, D, N = _check_cache(cache, block_table, lengths=lengths)
    if q.dim() != 4 or q.size(0) != N or q.size(3) != D or q.size(2) == 0 or q.size(2) % HK != 0:
        raise ValueError(f"q must be [N, T, H, D] = [{N}, T, a multiple of {HK}, {D}], got {tuple(q.shape)}")
    if q.device != cache.k.device:
        raise ValueError(f"q is on {q.device}, cache.k is on {cache.k.device}")
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bfloat16, got {q.dtype}")
    refuse_tangents("paged_cache_attention", q)
    if q.numel() == 0 or block_table.size(1) == 0:
        return torch.zeros_like(q, memory_format=torch.contiguous_format)
    with torch.cuda.device(q.device), torch.no_grad():
        result = host().cache_attention(raw_stream(q.get_device()), kernel_rows(q.detach()), *cache, as_int32(block_table), as_int32(lengths), window, sinks, scale)
        if result is None:
            raise refused("paged_cache_attention", q)
    return result


def paged_cache_attention(
    q: torch.Tensor,
    cache: PagedCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of the last T tokens of every sequence, q ``[N, T, H, D]`` bf16, over its ``lengths`` ``[N]`` tokens in the cache, their own
    among them (written before).  Query i stands at position ``lengths - T + i`` and sees the keys up to its own, of them
    the last ``window`` (None: all) and the first ``sinks``.  Rows that see none are zeros.  A page number outside of the cache makes the rows
    that see it NaN.  The scores, weights and sums are fp32; the weights are rounded to bf16 as operands.

    For single tokens and a few (drafts that are verified).  The contexts of few sequences are split over the GPU, so that one long sequence is read
    as fast as many; parts go by the number of sequences, not by their lengths, so a long one among many short ones is read by few workgroups.
    For inference: q gets no gradient."""
    from .attention import check_window

    window, sinks = check_window(window, sinks)
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("paged_cache_attention is for inference: q gets no gradient (call it under torch.no_grad())")
    if torch.compiler.is_compiling():
        from . import _opaque

        return _opaque.paged_cache_attention(q, cache, block_table, lengths, window, sinks, scale)
    result = None
    if q.is_cuda and is_kernel_allowed(Kernel.paged_cache):
        result = host().cache_attention(raw_stream(q.get_device()), q, *cache, block_table, lengths, window, sinks, scale)
    return _attend(q, cache, block_table, lengths, window, sinks, scale) if result is None else result
