"""Windowed softmax attention, the norm and rotation of its queries and keys, and its paged cache, in 64 bits as they are defined: test
infrastructure.  Gradients are those of autograd through the formulas."""

from __future__ import annotations

import torch

from .linear_attention_oracle import sequences_of


LOWEST = -100


def visible_keys(queries, keys, window=None, sinks=0):
    """[queries, keys]: query i stands at position i + keys - queries."""
    i = torch.arange(queries)[:, None] + keys - queries
    j = torch.arange(keys)[None, :]
    near = j > i - window if window is not None else torch.ones(queries, keys, dtype=torch.bool)
    return (j <= i) & (near | (j < sinks))


def attend(q, k, v, mask, scale):
    """q [T, H, D], k and v [S, HK, D], mask [T, S], float64; rows that see nothing are zeros.  What a row does not see does not enter."""
    T, H, D = q.shape
    group = H // k.size(1)
    out = []
    for h in range(H):
        kh, vh = k[:, h // group], v[:, h // group]
        scores = torch.where(mask, scale * (q[:, h] @ torch.where(mask.any(0)[:, None], kh, torch.zeros_like(kh)).T), -torch.inf)
        top = scores.max(dim=1, keepdim=True).values.clamp(min=-1e300).detach() if scores.size(1) else scores.new_zeros(T, 1)
        weights = torch.exp(scores - top)
        total = weights.sum(dim=1, keepdim=True)
        weights = weights / torch.where(total > 0, total, torch.ones_like(total))
        if vh.isfinite().all():
            out.append(weights @ vh)
        else:
            out.append(torch.where(mask[:, :, None], weights[:, :, None] * vh[None], torch.zeros(()).double()).sum(dim=1))
    return torch.stack(out, dim=1)


def window_attention_ref(q, k, v, window=None, sinks=0, scale=None, cu_seqlens=None, left_padded=False):
    """o [B, T, H, D] in float64; ``cu_seqlens`` is a list.  Tokens of no sequence read as zeros.  Differentiable."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, H, D = q.shape
    S = k.size(1)
    scale = D**-0.5 if scale is None else scale
    if cu_seqlens is None:
        return torch.stack([attend(q[b], k[b], v[b], visible_keys(T, S, window, sinks), scale) for b in range(B)])
    pieces, at = [[] for _ in range(B)], [0] * B
    for b, first, length in sequences_of(B, T, cu_seqlens, left_padded):
        pick = slice(first, first + length)
        o = attend(q[b, pick], k[b, pick], v[b, pick], visible_keys(length, length, window, sinks), scale)
        pieces[b] += [q.new_zeros(first - at[b], H, D), o]
        at[b] = first + length
    return torch.stack([torch.cat(p + [q.new_zeros(T - end, H, D)]) for p, end in zip(pieces, at)])


def norm_rotary_ref(x, weight, cos, sin, positions, eps=1e-6):
    """x [B, T, H, D], tables [positions, R / 2], positions [B, T]; float64, differentiable."""
    x = x.double()
    n = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + eps)
    n = n if weight is None else n * weight.double()
    half = cos.size(1)
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    a, b = n[..., :half], n[..., half : 2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, n[..., 2 * half :]], dim=-1)


def _e4m3_values():
    return torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def to_e4m3(x):
    """The nearest value of e4m3's grid, ties to the even code: by looking for it among all of them."""
    grid = _e4m3_values()[:127]  # 0 .. 448, in the codes' order
    y = x.double()
    hi = torch.searchsorted(grid, y.abs().contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y.abs(), y.abs() - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(y.abs() >= 448, torch.full_like(code, 126), code)
    return torch.where(y.isfinite(), torch.copysign(grid[code], y), torch.full_like(y, torch.nan))


def exponent_of(values):
    """The smallest exponent, from -100 on, with which no finite value passes 448."""
    top = values[values.isfinite()].abs().max().item() if values.isfinite().any() else 0.0
    e = LOWEST
    while top > 448.0 * 2.0**e:
        e += 1
    return e


class PagedCacheRef:
    """Values in grid steps [pages, heads, P, D] and exponents [pages, heads] of keys and values, one token after the other."""

    def __init__(self, pages, heads, D, P):
        self.P = P
        self.codes = [torch.zeros(pages, heads, P, D, dtype=torch.float64) for _ in range(2)]
        self.exponents = [torch.full((pages, heads), LOWEST) for _ in range(2)]

    def write(self, k, v, table, start):
        """One sequence's new tokens k, v [T, heads, D]; table: its pages."""
        pages, heads = self.exponents[0].shape
        for which, x in enumerate((k.double(), v.double())):
            codes, exponents = self.codes[which], self.exponents[which]
            for index in range(len(table)):
                first, last = index * self.P - start, (index + 1) * self.P - start  # of the new tokens
                lo, hi = max(first, 0, -start), min(last, x.size(0))
                page = table[index]
                if lo >= hi or not 0 <= page < pages:
                    continue
                offset = start + lo - index * self.P
                for h in range(heads):
                    new = x[lo:hi, h]
                    e = exponent_of(new)
                    if offset > 0:
                        before = int(exponents[page, h])
                        e = max(e, before)
                        if e > before:
                            codes[page, h, :offset] = to_e4m3(codes[page, h, :offset] * 2.0 ** (before - e))
                    codes[page, h, offset : offset + hi - lo] = to_e4m3(new * 2.0**-e)
                    exponents[page, h] = e

    def read(self, table, length):
        """k, v [length, heads, D] of one sequence; NaN where a page is not there."""
        out = []
        for codes, exponents in zip(self.codes, self.exponents):
            x = codes * torch.exp2(exponents.double())[:, :, None, None]
            rows = [x[p] if 0 <= p < x.size(0) else torch.full_like(x[0], torch.nan) for p in table]
            out.append(torch.cat(rows, dim=1).transpose(0, 1)[:length] if rows else x.new_zeros(0, x.size(1), x.size(3)))
        return out
