"""Softmax attention over a window, its 8-bit cache and what stands in front of it, as cases that can be timed and compared.

Paths:

* ``rotate``        ``qk_norm_rotary``: RMS norm of every head of q and k and the rotation by position, one pass
* ``rotate_train``  the same under autograd: both results and the gradients of q, k and the weights
* ``window``        ``sliding_window_attention``: prompts and evaluation; whole, packed or left-padded batches, a few first tokens stay visible
* ``window_train``  the same under autograd: output and the gradients of q, k, v
* ``write``         ``write_paged_cache``: new tokens of every sequence into its pages, 8 bits each, a scale for each page and head
* ``write_read``    the same, and ``read_paged_cache``: what the pages then stand for
* ``decode``        ``paged_cache_attention``: one new token per sequence (or a few) over the 8-bit pages

A query at position p sees the keys j <= p with j > p - window or j < sinks.  A page of the cache holds e4m3 codes c that stand for
c 2^(s - 127); s is the smallest exponent for which none of the page's tokens passes 448.  A page that is gone on with keeps its
exponent or takes a larger one, its older codes rounded to it.

Head shapes are those of the package's benchmark configurations (16 and 32 heads of 128), of the reference's shipped model configurations (2 heads of
256), of its smallest tests (heads of 64), and odd ones between them; keys and values are shared by 1 to 8 heads.
"""

from __future__ import annotations

import math

import torch


own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": BF16, "fp32": F32}
EPS = 1e-6
ROTARY_BASE = 10000.0
LOWEST = -100  # exponent of a page that holds nothing but (nearly) zeros


def _rotate(path, B, T, H, HK, D, R=None, context=4096, dtype="bf16", weights="fp32", name=None):
    """``R``: dims that are rotated; ``context``: positions that the table has; ``weights``: their dtype, or "none"."""
    case = dict(path=path, B=B, T=T, H=H, HK=HK, D=D, R=D if R is None else R, context=context, dtype=dtype, weights=weights)
    return case if name is None else dict(case, name=name)


def _window(path, B, T, H, HK, D, window, sinks, S=None, N=0, padded=False, dtype="bf16", name=None):
    """``T`` queries and ``S`` keys per row (packed: one row that holds ``N`` sequences); ``window`` 0: all keys up to the query's own."""
    case = dict(path=path, B=B, T=T, S=T if S is None else S, H=H, HK=HK, D=D, window=window, sinks=sinks, N=N, padded=padded, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _write(path, B, T, HK, D, page, context, N=0, dtype="bf16", name=None):
    """``T`` new tokens per sequence (packed: of the one row that holds ``N`` sequences) behind up to ``context`` - ``T`` held ones."""
    case = dict(path=path, B=B, T=T, HK=HK, D=D, page=page, context=context, N=N, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _decode(B, T, H, HK, D, page, context, window=0, sinks=0, name=None):
    """``T`` new tokens of each of ``B`` sequences of up to ``context`` tokens."""
    case = dict(path="decode", B=B, T=T, H=H, HK=HK, D=D, page=page, context=context, window=window, sinks=sinks)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # a serving step of 53 chats far into their contexts, one layer: latency
        _rotate("rotate", 53, 1, 16, 2, 128, context=65536, name="rotate_step"),
        # a training step's batch in front of attention
        _rotate("rotate_train", 4, 4096, 16, 2, 128, name="rotate_train"),
        # a prompt of ordinary length at the shipped head shape, length not a multiple of anything
        _window("window", 1, 777, 2, 1, 256, 512, 4, name="window_prompt"),
        # a training-sized batch, forward only (evaluation)
        _window("window", 4, 4096, 16, 2, 128, 1024, 4, name="window_batch"),
        # prefill of documents of very different lengths, packed
        _window("window", 1, 16384, 16, 2, 128, 2048, 16, N=11, name="window_packed"),
        # training step of the operator at the benchmark's batch
        _window("window_train", 4, 4096, 16, 2, 128, 1024, 4, name="window_train"),
        # training on left-padded rows, every key up to the query's own, small heads
        _window("window_train", 6, 1500, 16, 8, 64, 0, 0, padded=True, name="causal_train_padded"),
        # the exact fp32 path (debugging, small checks)
        _window("window_train", 1, 256, 2, 2, 64, 100, 3, dtype="fp32", name="window_train_fp32"),
        # a serving step's new tokens into 256 sequences' pages: latency
        _write("write", 256, 1, 8, 128, 64, 512, name="write_step"),
        # prompts behind a shared beginning into the cache, and the cache handed to another layer's check or a swap to host
        _write("write_read", 8, 4001, 8, 128, 64, 4736, name="write_prompts"),
        # one user's chat with a long context: latency, the context split over the chip
        _decode(1, 1, 16, 2, 128, 64, 32768, name="decode_single"),
        # a serving batch, contexts from a handful of tokens to 4096
        _decode(256, 1, 32, 8, 128, 64, 4096, name="decode_256"),
    ]


_HEAD_DIMS = [64, 64, 128, 128, 128, 256, 96, 80, 24, 200]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _heads(rng, most=32):
    HK = rng.choice([h for h in (1, 2, 3, 4, 8, 16) if h <= most])
    return HK * rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * HK <= most]), HK


def draw(rng):
    """One more case, sizes over the whole range.  Odd lengths, head shapes and page ends among them."""
    path = rng.choice(["rotate", "rotate_train", "window", "window", "window_train", "window_train", "write", "write_read", "decode", "decode"])
    H, HK = _heads(rng)
    D = rng.choice(_HEAD_DIMS)
    if path.startswith("rotate"):
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        tokens = _log_int(rng, 1, max(1, (1 << (25 if path == "rotate" else 24)) // ((H + HK) * D)))
        B = min(rng.choice([1, 2, 5, 8]), tokens)
        T = tokens // B
        R = D if rng.random() < 0.7 else max(8, D // 4 // 8 * 8)
        return _rotate(path, B, T, H, HK, D, R=R, context=T + _log_int(rng, 1, 100000), dtype=dtype,
                       weights=rng.choice(["bf16", "fp32", "none"] if path == "rotate" else ["bf16", "fp32"]))  # fmt: skip
    if path.startswith("window"):
        train, dtype = path == "window_train", "fp32" if rng.random() < 0.2 else "bf16"
        limit = (1 << 26) if dtype == "fp32" else (1 << 29) if train else (1 << 31)
        kind = rng.choice(["batch", "batch", "padded", "packed"] + ([] if train else ["behind"]))
        S = _log_int(rng, 1 if kind == "behind" else 17, 4096 if train else 16384)
        T = _log_int(rng, 1, S) if kind == "behind" else S
        B = 1 if kind == "packed" else rng.choice([1, 2, 3, 4, 8])
        while B * H * T * S > limit and B > 1:
            B -= 1
        while B * H * T * S > limit:
            S, T = S // 2, max(1, T // 2)
        return _window(path, B, T, H, HK, D, 0 if rng.random() < 0.25 else _log_int(rng, 1, 4096), rng.choice([0, 0, 1, 4, 16, 100]), S=S,
                       N=min(rng.choice([2, 5, 11, 24]), max(1, S // 8)) if kind == "packed" else 0, padded=kind == "padded", dtype=dtype)  # fmt: skip
    D = rng.choice([64, 128, 128, 256, 96, 80])
    page = rng.choice([16, 32, 64, 64, 128])
    if path == "decode":
        T = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        context = _log_int(rng, max(page, T), 65536)
        B = _log_int(rng, 1, max(1, min(512, (1 << 29) // (context * HK * D))))
        return _decode(B, T, H, HK, D, page, context, window=0 if rng.random() < 0.6 else _log_int(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 64]))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    tokens = _log_int(rng, 1, (1 << 24) // (HK * D))
    if rng.random() < 0.3 and tokens > 60:
        N = rng.choice([2, 5, 11])
        return _write(path, 1, tokens, HK, D, page, tokens + _log_int(rng, 1, 1000), N=N, dtype=dtype)
    B = min(tokens, _log_int(rng, 1, 64))
    T = tokens // B
    return _write(path, B, T, HK, D, page, T + _log_int(rng, 1, 600), dtype=dtype)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens of every sequence.  They go by the case alone, so that its work is the same for every seed."""
    gen = torch.Generator().manual_seed(1000 * case.get("T", 1) + case.get("B", 1) + case.get("context", 0))
    if case.get("N"):
        if case["N"] == 1:
            return [case["T"]]
        # cuts of the row at random places: lengths from a handful of tokens to a large part of the row
        cuts = (torch.randperm(case["T"] - 1, generator=gen)[: case["N"] - 1] + 1).sort().values.tolist()
        return [b - a for a, b in zip([0] + cuts, cuts + [case["T"]])]
    if case.get("padded"):
        lens = torch.randint(max(1, case["T"] // 4), case["T"] + 1, (case["B"],), generator=gen).tolist()
        lens[-1] = case["T"]
        return lens
    if case["path"] == "decode":  # contexts, the new tokens among them
        lens = torch.randint(case["T"], case["context"] + 1, (case["B"],), generator=gen).tolist()
        lens[-1] = max(case["T"], case["context"] - 5)
        return lens
    return [case["T"]] * case["B"]


def _held(case, lens):
    """Tokens that the cache holds of every sequence before the call; some pages are begun, some are not."""
    gen = torch.Generator().manual_seed(case["context"] + len(lens))
    return [int(torch.randint(0, case["context"] - n + 1, (1,), generator=gen)) for n in lens]


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _pages(case, counts, gen):
    """``(block_table [N, most], number of pages)``: pages in an order of their own, -1 behind a sequence's last."""
    most, total = -(-case["context"] // case["page"]), sum(counts) + 3
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(counts), most), -1, dtype=torch.int32, device="cuda")
    begin = 0
    for n, count in enumerate(counts):
        table[n, :count] = order[begin : begin + count]
        begin += count
    return table, total


def _rows(randn, tokens, HK, D):
    """Keys and values as a cache meets them: a few strong channels in the keys, tokens of different size."""
    k = randn(tokens, HK, D) * (1.0 + 5.0 * (randn(1, HK, D) > 2.0)) * torch.exp(0.3 * randn(tokens, 1, 1))
    return k, randn(tokens, HK, D) * torch.exp(0.3 * randn(tokens, 1, 1))


def _full_pages(x):
    """Pages [n, P, HK, D] of values -> (codes [n, HK, P, D], exponents [n, HK])."""
    e = _exponent(x.abs().amax(dim=(1, 3)))
    codes = torch.ldexp(x, -e[:, None, :, None]).to(E4M3)
    return codes.permute(0, 2, 1, 3).contiguous(), (e + 127).to(torch.uint8)


def _interleave(codes):
    """[n, HK, P, D] -> [n, HK, P / 16, D, 16], how the cache holds values."""
    n, HK, P, D = codes.shape
    return codes.view(n, HK, P // 16, 16, D).transpose(3, 4).contiguous()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(case)
    if case["path"].startswith("rotate"):
        _prepare_rotate(s, case, gen, randn)
    elif case["path"].startswith("window"):
        _prepare_window(s, case, randn)
    else:
        _prepare_cache(s, case, gen, randn)
    return s


def _prepare_rotate(s, case, gen, randn):
    B, T, H, HK, D, R = (case[n] for n in ("B", "T", "H", "HK", "D", "R"))
    train = case["path"] == "rotate_train"
    # what a layer hands over: q, k, v are the column blocks of one projection's output
    qkv = (randn(B, T, (H + 2 * HK) * D) * 1.7).to(DTYPES[case["dtype"]])
    q, k, _ = qkv.split((H * D, HK * D, HK * D), dim=-1)
    s["q"], s["k"] = q.view(B, T, H, D), k.view(B, T, HK, D)
    s["wq"] = s["wk"] = None
    if case["weights"] != "none":
        s["wq"], s["wk"] = ((1.0 + 0.2 * randn(D)).to(DTYPES[case["weights"]]) for _ in range(2))
    angle = torch.arange(case["context"], device="cuda", dtype=F64)[:, None] * ROTARY_BASE ** (-torch.arange(R // 2, device="cuda", dtype=F64) / (R // 2))
    s["cos"], s["sin"] = angle.cos().to(F32), angle.sin().to(F32)
    if train:
        s["positions"] = None  # rows from their first token on
        s["leaves"] = [n for n in ("q", "k", "wq", "wk") if s[n] is not None]
        for n in s["leaves"]:
            s[n] = s[n].detach().requires_grad_()
        s["dq"], s["dk"] = randn(B, T, H, D).to(q.dtype), randn(B, T, HK, D).to(q.dtype)
    else:
        first = torch.randint(0, case["context"] - T + 1, (B, 1), device="cuda", generator=gen)
        s["positions"] = (first + torch.arange(T, device="cuda")).to(torch.int32)


def _prepare_window(s, case, randn):
    B, T, S, H, HK, D = (case[n] for n in ("B", "T", "S", "H", "HK", "D"))
    dtype = DTYPES[case["dtype"]]
    # heads from broad to sharp; the first keys draw all queries, as they do in trained models
    towards = randn(H, D) * 0.3
    q = (randn(B, T, H, D) + towards) * (0.5 + 2.0 * torch.arange(1, H + 1, device="cuda")[:, None] / H)
    k = randn(B, S, HK, D)
    k[:, :4] += 2.0 * towards[:: H // HK]
    s["q"], s["k"], s["v"] = q.to(dtype), k.to(dtype), randn(B, S, HK, D).to(dtype)
    s["lens"], s["cu"] = _lengths(case), None
    if case["N"] or case["padded"]:
        s["cu"] = _cu(s["lens"])
    if case["path"] == "window_train":
        for n in ("q", "k", "v"):
            s[n] = s[n].requires_grad_()
        s["do"] = randn(B, T, H, D).to(dtype)


def _prepare_cache(s, case, gen, randn):
    HK, D, P = case["HK"], case["D"], case["page"]
    s["lens"] = lens = _lengths(case)
    s["held"] = held = [0] * len(lens) if case["path"] == "decode" else _held(case, lens)
    s["table"], total = _pages(case, [-(-(h + n) // P) for h, n in zip(held, lens)], gen)
    k, v = _rows(randn, total * P, HK, D)
    s["k_cache"], s["k_scale"] = _full_pages(k.view(total, P, HK, D))
    codes, s["v_scale"] = _full_pages(v.view(total, P, HK, D))
    s["v_cache"] = _interleave(codes)
    if case["path"] == "decode":
        s["q"] = (1.5 * randn(case["B"], case["T"], case["H"], D)).to(BF16)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return
    k, v = _rows(randn, case["B"] * case["T"], HK, D)
    s["k"], s["v"] = (x.view(case["B"], case["T"], HK, D).to(DTYPES[case["dtype"]]) for x in (k, v))
    s["start"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    s["cu"] = _cu(lens) if case["N"] else None
    s["counts"] = torch.tensor(lens, device="cuda")
    s["after"] = torch.tensor([h + n for h, n in zip(held, lens)], dtype=torch.int32, device="cuda")
    s["most"] = max(h + n for h, n in zip(held, lens))


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    path = s["path"]
    if path.startswith("rotate"):
        q, k = _call_rotate(s) if own else _plain_rotate(s)
        if path == "rotate":
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), [s[n] for n in s["leaves"]], (s["dq"], s["dk"])))
    if path.startswith("window"):
        o = _call_window(s) if own else _plain_window(s)
        if path == "window":
            return o
        return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
    if path == "decode":
        return _call_decode(s) if own else _plain_decode(s)
    held = (s["k_scale"], s["v_scale"])
    if path == "write":
        (_call_write if own else _plain_write)(s)
        return (s["k_cache"], s["v_cache"], *held)
    if own:
        _call_write(s)
        return (*_call_read(s), *held)
    _plain_write(s)
    return (*_plain_read(s), *held)


def _cache(s):
    from lm_engine_amd import PagedCache

    return PagedCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])


def _call_rotate(s):
    from lm_engine_amd import qk_norm_rotary

    return qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], positions=s["positions"], eps=EPS)


def _call_window(s):
    from lm_engine_amd import sliding_window_attention

    return sliding_window_attention(s["q"], s["k"], s["v"], window=s["window"] or None, sinks=s["sinks"], cu_seqlens=s["cu"], left_padded=s["padded"])


def _call_write(s):
    from lm_engine_amd import write_paged_cache

    write_paged_cache(_cache(s), s["k"], s["v"], s["table"], s["start"], cu_seqlens=s["cu"])


def _call_read(s):
    from lm_engine_amd import read_paged_cache

    return read_paged_cache(_cache(s), s["table"], s["after"], s["most"], dtype=s["k"].dtype)


def _call_decode(s):
    from lm_engine_amd import paged_cache_attention

    return paged_cache_attention(s["q"], _cache(s), s["table"], s["lengths"], window=s["window"] or None, sinks=s["sinks"])


# ---------------------------------------------------------------------------------------------------------------------
# the plain form, in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _plain_rotate_one(x, weight, cos, sin, half):
    n = x.float()
    n = n * torch.rsqrt((n * n).mean(dim=-1, keepdim=True) + EPS)
    if weight is not None:
        n = n * weight.float()
    a, b, rest = n[..., :half], n[..., half : 2 * half], n[..., 2 * half :]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1).to(x.dtype)


def _plain_rotate(s):
    half = s["R"] // 2
    if s["positions"] is None:
        cos, sin = s["cos"][None, : s["T"], None], s["sin"][None, : s["T"], None]
    else:
        at = s["positions"].long()
        cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    return _plain_rotate_one(s["q"], s["wq"], cos, sin, half), _plain_rotate_one(s["k"], s["wk"], cos, sin, half)


def _take(codes, pages):
    return codes.view(torch.uint8)[pages].view(E4M3)


def _visible(query, key, window, sinks):
    """Positions [.., T], [.., S] -> which keys a query sees [.., T, S].  Negative positions are of no sequence."""
    query, key = query[..., :, None], key[..., None, :]
    near = key > query - window if window else torch.ones_like(key > query)
    return (query >= 0) & (key >= 0) & (key <= query) & (near | (key < sinks))


def _plain_softmax(q, k, v, mask, scale):
    """q [B, HK, G, T, D], k and v [B, HK, S, D], mask broadcast over [B, HK, G, T, S] -> [B, HK, G, T, D].  No visible key: zeros."""
    B, HK, G, T, D = q.shape
    scores = torch.matmul(q.reshape(B, HK, G * T, D), k.transpose(-1, -2)).view(B, HK, G, T, -1) * scale
    scores = scores.masked_fill(~mask, float("-inf"))
    top = scores.detach().amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(p.view(B, HK, G * T, -1), v).view(B, HK, G, T, D)


def _window_mask(s):
    """[B, T, S]"""
    T, S = s["T"], s["S"]
    t = torch.arange(S, device="cuda")
    if s["cu"] is None:
        return _visible(t[S - T :] if T < S else t, t, s["window"], s["sinks"])[None]
    if s["padded"]:
        at = t[None] - (T - (s["cu"][1:] - s["cu"][:-1]).long())[:, None]
        return _visible(at, at, s["window"], s["sinks"])
    sequence = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    at = t - s["cu"].long()[sequence]
    return (_visible(at, at, s["window"], s["sinks"]) & (sequence[:, None] == sequence[None, :]))[None]


def _plain_window(s):
    B, T, H, HK, D = (s[n] for n in ("B", "T", "H", "HK", "D"))
    q = s["q"].float().view(B, T, HK, H // HK, D).permute(0, 2, 3, 1, 4)
    k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    o = _plain_softmax(q, k, v, _window_mask(s)[:, None, None], D**-0.5)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(s["q"].dtype)


def _exponent(top):
    """The smallest e with top <= 448 2^e, from LOWEST on; exact: a float is m 2^x with m in [0.5, 1), and 448 is 0.875 2^9."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 9 + (m > 0.875).to(x.dtype), torch.full_like(x, LOWEST)).clamp(min=LOWEST)


def _plain_write_one(new, codes, scales, pages, begun, fresh, source):
    """``new`` [tokens, HK, D]; ``codes`` [pages, HK, P, D] and ``scales`` [pages, HK] are returned as they become.  ``pages`` [m]:
    the touched ones; ``begun``, ``fresh`` [m, P]: places held before, places written; ``source`` [m, P]: tokens."""
    x = new[source].float() * fresh[:, :, None, None]  # [m, P, HK, D]
    e = _exponent(x.abs().amax(dim=(1, 3)))  # [m, HK]
    before = scales[pages].to(torch.int32) - 127
    e = torch.where(begun.any(dim=1)[:, None], torch.maximum(e, before), e)
    old = _take(codes, pages)  # [m, HK, P, D]
    again = torch.ldexp(old.float(), (before - e)[:, :, None, None]).to(E4M3)
    value = torch.ldexp(x, -e[:, None, :, None]).to(E4M3).permute(0, 2, 1, 3)
    bits = torch.where(fresh[:, None, :, None], value.view(torch.uint8), torch.where(begun[:, None, :, None], again.view(torch.uint8), old.view(torch.uint8)))
    codes.view(torch.uint8)[pages] = bits
    scales[pages] = (e + 127).to(torch.uint8)


def _plain_write(s):
    P, N = s["page"], len(s["lens"])
    start, counts = s["start"].long(), s["counts"]
    slots = (max(s["lens"]) + P - 2) // P + 1  # pages that a sequence's new tokens can lie in
    nth = start[:, None] // P + torch.arange(slots, device="cuda")  # [N, slots]
    used = (nth * P < (start + counts)[:, None]) & (counts > 0)[:, None]
    row = torch.arange(N, device="cuda")[:, None].expand(N, slots)[used]
    nth = nth[used]
    pages = s["table"].long()[row, nth]
    at = nth[:, None] * P + torch.arange(P, device="cuda")  # positions [m, P]
    begun, fresh = at < start[row][:, None], (at >= start[row][:, None]) & (at < (start + counts)[row][:, None])
    first = row * s["T"] if s["cu"] is None else s["cu"].long()[row]
    source = (first[:, None] + at - start[row][:, None]).clamp(0, s["B"] * s["T"] - 1)
    HK, D = s["HK"], s["D"]
    _plain_write_one(s["k"].reshape(-1, HK, D), s["k_cache"], s["k_scale"], pages, begun, fresh, source)
    straight = s["v_cache"].view(torch.uint8).transpose(3, 4).reshape(-1, HK, P, D).view(E4M3)
    _plain_write_one(s["v"].reshape(-1, HK, D), straight, s["v_scale"], pages, begun, fresh, source)
    s["v_cache"].view(torch.uint8).copy_(straight.view(torch.uint8).view(-1, HK, P // 16, 16, D).transpose(3, 4))


def _plain_values(codes, scales, table):
    """[N, HK, tokens, D] in fp32 of the pages of ``table``."""
    pages = table.long().clamp(min=0)
    x = torch.ldexp(_take(codes, pages).float(), (scales[pages].to(torch.int32) - 127)[..., None, None])  # [N, most, HK, P, D]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_cache(s, table):
    k = _plain_values(s["k_cache"], s["k_scale"], table)
    return k, _plain_values(s["v_cache"].view(torch.uint8).transpose(3, 4).flatten(2, 3).view(E4M3), s["v_scale"], table)


def _plain_read(s):
    most = s["most"]
    there = torch.arange(most, device="cuda")[None] < s["after"][:, None]
    k, v = _plain_cache(s, s["table"][:, : -(-most // s["page"])])
    return tuple((x[:, :, :most].transpose(1, 2) * there[:, :, None, None]).to(s["k"].dtype) for x in (k, v))


def _plain_decode(s):
    B, T, H, HK, D = (s[n] for n in ("B", "T", "H", "HK", "D"))
    k, v = _plain_cache(s, s["table"])
    t = torch.arange(k.size(2), device="cuda")
    lengths = s["lengths"].long()[:, None]
    query = lengths - T + torch.arange(T, device="cuda")
    mask = _visible(query, t[None].expand(B, -1), s["window"], s["sinks"])
    q = s["q"].float().view(B, T, HK, H // HK, D).permute(0, 2, 3, 1, 4)
    return _plain_softmax(q, k, v, mask[:, None, None], D**-0.5).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(BF16)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _pairs(queries, length, window, sinks):
    """Visible (query, key) pairs of a sequence whose last ``queries`` tokens ask."""
    total = 0
    for p in range(length - queries, length):
        total += p + 1 if not window or p < window else window + min(sinks, p - window + 1)
    return total


def _seen(queries, length, window, sinks):
    """Keys that one of them sees."""
    near = min(length, window + queries - 1) if window else length
    return near + min(sinks, length - near)


def work(case):
    size = {"bf16": 2, "fp32": 4}
    path = case["path"]
    if path.startswith("rotate"):
        cells, rows = case["B"] * case["T"] * (case["H"] + case["HK"]) * case["D"], case["B"] * case["T"]
        table = (rows if path == "rotate" else case["T"]) * case["R"] * 4
        e = size[case["dtype"]]
        if path == "rotate":
            return dict(bytes=2 * cells * e + table, flops=8 * cells)
        return dict(bytes=5 * cells * e + table, flops=24 * cells)  # forward: x, y; backward: x, dy, dx
    HK, D = case["HK"], case["D"]
    if path == "decode":
        seen = sum(_seen(case["T"], n, case["window"], case["sinks"]) for n in _lengths(case))
        pairs = sum(_pairs(case["T"], n, case["window"], case["sinks"]) for n in _lengths(case))
        return dict(bytes=2 * seen * HK * D + 4 * case["B"] * case["T"] * case["H"] * D, flops=4 * pairs * case["H"] * D)
    if path.startswith("window"):
        e, H, lens = size[case["dtype"]], case["H"], _lengths(case)
        if case["N"] or case["padded"]:
            pairs, queries, keys = sum(_pairs(n, n, case["window"], case["sinks"]) for n in lens), sum(lens), sum(lens)
        else:
            pairs = case["B"] * _pairs(case["T"], case["S"], case["window"], case["sinks"])
            queries, keys = case["B"] * case["T"], case["B"] * case["S"]
        rows, shared = queries * H * D * e, keys * HK * D * e
        if path == "window":
            return dict(bytes=2 * rows + 2 * shared, flops=4 * pairs * H * D)
        # forward; then q, k, v, o, do read and dq, dk, dv written; five products where the forward has two
        return dict(bytes=6 * rows + 6 * shared, flops=14 * pairs * H * D)
    lens = _lengths(case)
    held = _held(case, lens)
    new = sum(lens) * HK * D
    if path == "write":
        return dict(bytes=2 * new * (size[case["dtype"]] + 1), flops=4 * new)
    back = sum(h + n for h, n in zip(held, lens)) * HK * D
    out = len(lens) * max(h + n for h, n in zip(held, lens)) * HK * D
    return dict(bytes=2 * new * (size[case["dtype"]] + 1) + 2 * back + 2 * out * size[case["dtype"]], flops=4 * new + 2 * back)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_rotate(s):
    R, T = s["R"], s["T"]
    at = torch.arange(T, device="cuda")[None].expand(s["B"], T) if s["positions"] is None else s["positions"].long()
    turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[at][:, :, None]  # [B, T, 1, R / 2]
    results, grads, weights = [], [], []
    for x, w, dy in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
        x = x.detach().to(F64)
        r = 1.0 / torch.sqrt(x.square().sum(-1, keepdim=True) / x.size(-1) + EPS)
        unit = x * r
        gain = torch.ones(x.size(-1), device="cuda", dtype=F64) if w is None else w.detach().to(F64)
        turned = lambda z, by: torch.cat([(c := torch.complex(z[..., : R // 2], z[..., R // 2 : R]) * by).real, c.imag, z[..., R:]], dim=-1)  # noqa: E731
        results.append(turned(unit * gain, turn))
        if dy is None:
            continue
        dn = turned(dy.to(F64), turn.conj())
        weights.append((dn * unit).sum(dim=(0, 1, 2)))
        du = dn * gain
        grads.append(r * (du - unit * (du * unit).mean(-1, keepdim=True)))
    return (*results, *grads, *(weights if s["wq"] is not None else []))


def _exact_attention(q, k, v, mask, scale, do=None):
    """One head's queries [T, D], its keys and values [S, D], all in 64 bits."""
    scores = (q @ k.T) * scale
    scores[~mask] = -math.inf
    empty = ~mask.any(dim=1)
    scores[empty] = 0.0
    p = torch.softmax(scores, dim=1)
    p[empty] = 0.0
    o = p @ v
    if do is None:
        return o
    ds = p * (do @ v.T - (do * o).sum(dim=1, keepdim=True)) * scale
    return o, ds @ k, ds.T @ q, p.T @ do


def _exact_window(s):
    B, T, S, H, HK = (s[n] for n in ("B", "T", "S", "H", "HK"))
    q, k, v = (s[n].detach().to(F64) for n in ("q", "k", "v"))
    train = s["path"] == "window_train"
    do = s["do"].to(F64) if train else None
    outs = [torch.zeros_like(q)] + ([torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)] if train else [])
    if s["cu"] is None:
        parts = [(b, 0, T, 0, S) for b in range(B)]
    elif s["padded"]:
        parts = [(b, T - n, T, T - n, T) for b, n in enumerate(s["lens"])]
    else:
        ends = torch.tensor(s["lens"]).cumsum(0).tolist()
        parts = [(0, end - n, end, end - n, end) for n, end in zip(s["lens"], ends)]
    for b, q0, q1, k0, k1 in parts:
        i = torch.arange(q1 - q0, device="cuda")[:, None] + (k1 - k0) - (q1 - q0)
        j = torch.arange(k1 - k0, device="cuda")[None, :]
        gap = i - j
        mask = gap >= 0
        if s["window"]:
            mask = mask & ((gap < s["window"]) | (j < s["sinks"]).expand_as(gap))
        for h in range(H):
            g = h * HK // H
            got = _exact_attention(q[b, q0:q1, h], k[b, k0:k1, g], v[b, k0:k1, g], mask, q.size(-1) ** -0.5, do[b, q0:q1, h] if train else None)
            if not train:
                outs[0][b, q0:q1, h] = got
                continue
            outs[0][b, q0:q1, h], outs[1][b, q0:q1, h] = got[:2]
            outs[2][b, k0:k1, g] += got[2]
            outs[3][b, k0:k1, g] += got[3]
    return tuple(outs) if train else outs[0]


def _exact_decode(s):
    T, H, HK, P = (s[n] for n in ("T", "H", "HK", "page"))
    out = torch.zeros(s["q"].shape, device="cuda", dtype=F64)
    v_codes = s["v_cache"].to(F32).permute(0, 1, 2, 4, 3).reshape(s["k_cache"].shape).to(E4M3)
    for b, n in enumerate(s["lens"]):
        pages = s["table"][b, : -(-n // P)].long()
        k, v = ((_take(codes, pages).to(F64) * torch.exp2(scales[pages].to(F64) - 127.0)[:, :, None, None]).transpose(0, 1).reshape(HK, -1, s["D"])[:, :n]
                for codes, scales in ((s["k_cache"], s["k_scale"]), (v_codes, s["v_scale"])))  # fmt: skip
        gap = (n - T + torch.arange(T, device="cuda"))[:, None] - torch.arange(n, device="cuda")[None, :]
        mask = gap >= 0
        if s["window"]:
            mask &= (gap < s["window"]) | (torch.arange(n, device="cuda") < s["sinks"])[None]
        for h in range(H):
            out[b, :, h] = _exact_attention(s["q"][b, :, h].to(F64), k[h * HK // H], v[h * HK // H], mask, s["D"] ** -0.5)
    return out


def _nearest(x, e):
    """x 2^-e in e4m3, x in 64 bits: the grid's step at y is 2^(floor(log2 |y|) - 3), at least 2^-9; ties go to even."""
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.frexp(y)[1].to(F64) - 4.0).clamp(min=2.0**-9)
    return torch.round(y / step) * step


def _exact_write(s):
    HK, D, P = s["HK"], s["D"], s["page"]
    results, scales = {}, {}
    v_codes = s["v_cache"].to(F64).permute(0, 1, 2, 4, 3).reshape(s["k_cache"].shape)
    for name, codes, at, new in (("k", s["k_cache"].to(F64), s["k_scale"], s["k"]), ("v", v_codes, s["v_scale"], s["v"])):
        codes, exponents, new, first = codes.clone(), at.to(torch.int64) - 127, new.reshape(-1, HK, D).to(F64), 0
        for n, count in enumerate(s["lens"]):
            begin, done = s["held"][n], 0
            while done < count:
                page, offset = int(s["table"][n, (begin + done) // P]), (begin + done) % P
                take = min(P - offset, count - done)
                x = new[first + done : first + done + take].transpose(0, 1)  # [HK, take, D]
                top = x.abs().amax(dim=(1, 2))
                e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)), torch.full_like(top, LOWEST))
                e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
                e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=LOWEST)
                if offset:
                    e = torch.maximum(e, exponents[page].to(F64))
                    codes[page, :, :offset] = _nearest(codes[page, :, :offset], (e - exponents[page])[:, None, None])
                codes[page, :, offset : offset + take] = _nearest(x, e[:, None, None])
                exponents[page] = e.to(torch.int64)
                done += take
            first += count
        results[name], scales[name] = codes, exponents
    exact_scales = [(scales[n] + 127).to(torch.uint8) for n in ("k", "v")]
    if s["path"] == "write":
        v = results["v"]
        return (results["k"], v.view(v.size(0), HK, P // 16, 16, D).transpose(3, 4), *exact_scales)
    back = []
    for n in ("k", "v"):
        out = torch.zeros(len(s["lens"]), s["most"], HK, D, device="cuda", dtype=F64)
        for b, count in enumerate(s["lens"]):
            total = s["held"][b] + count
            pages = s["table"][b, : -(-total // P)].long()
            x = results[n][pages] * torch.exp2(scales[n][pages].to(F64))[:, :, None, None]
            out[b, :total] = x.transpose(1, 2).reshape(-1, HK, D)[:total]
        back.append(out)
    return (*back, *exact_scales)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["path"].startswith("rotate"):
            return _exact_rotate(s)
        if case["path"].startswith("window"):
            return _exact_window(s)
        if case["path"] == "decode":
            return _exact_decode(s)
        # (a page at a time: too long for the largest)
        return _exact_write(s) if sum(-(-n // case["page"]) + 1 for n in s["lens"]) <= 8000 else None
