"""Linear attention with a decay for each head, and layer norm, as cases that can be timed and compared.

Paths:

* ``decode``      ``fused_recurrent_linear_attention``: a few new tokens per sequence (mostly one), the state updated in place
* ``forward``     ``chunk_linear_attention``: prompts and evaluation; whole, packed or left-padded batches
* ``train``       ``chunk_linear_attention`` under autograd: output, final state and the gradients of its inputs
* ``norm``        ``layer_norm``: rows of a hidden size in front of the mixer, rows of a head's size behind it
* ``norm_train``  ``layer_norm`` under autograd: output, gradients of rows, weight and bias

Per (sequence, head), with S [K, V] and w = exp(g):  S_t = w S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t.

Head shapes are those of the package's benchmark configurations (K = V = 128; K = 128, V = 256), of the reference's shipped
model configurations (K = 256, V = 512, 2 heads), of its smallest tests (K = V = 64), and odd ones between them.
"""

from __future__ import annotations

import math

import torch


own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp32": F32}
NORM_EPS = 1e-5


def _mix(path, B, T, H, K, V, HK=None, N=0, padded=False, dtype="bf16", decay=True, learned=False, state=True, name=None):
    """``T``: tokens per row (packed: of the one row that holds ``N`` sequences of drawn lengths); ``HK`` heads of q and k;
    ``decay``: with one (else every token weighs the same); ``learned``: the decay's gradient is wanted; ``state``: carried states."""
    case = dict(path=path, B=B, T=T, H=H, HK=H if HK is None else HK, K=K, V=V, N=N, padded=padded, dtype=dtype, decay=decay,
                learned=learned, state=state)  # fmt: skip
    return case if name is None else dict(case, name=name)


def _norm(path, rows, D, dtype="bf16", weights="bf16", bias=True, gap=0, name=None):
    """``rows`` rows of ``D``; ``weights``: dtype of weight and bias, or "none"; ``gap``: elements between the rows (a slice)."""
    case = dict(path=path, rows=rows, D=D, dtype=dtype, weights=weights, bias=bias, gap=gap)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one user's chat, one layer: latency and launches
        _mix("decode", 1, 1, 16, 128, 128, name="decode_single"),
        # a serving batch: 256 sequences x 32 heads, 512 MiB of state through HBM
        _mix("decode", 256, 1, 32, 128, 128, name="decode_256"),
        # a prompt of ordinary length at the shipped head shape, length not a multiple of anything
        _mix("forward", 1, 777, 2, 256, 512, state=False, name="forward_prompt"),
        # a training-sized batch, forward only (evaluation)
        _mix("forward", 4, 4096, 16, 128, 128, state=False, name="forward_batch"),
        # packed documents of very different lengths with carried states
        _mix("forward", 1, 32768, 16, 128, 128, N=11, name="forward_packed"),
        # one very long context, expanded values
        _mix("forward", 1, 65536, 32, 128, 256, name="forward_long"),
        # training step of the operator at the benchmark's batch
        _mix("train", 4, 4096, 16, 128, 128, state=False, name="train_batch"),
        # training on left-padded rows, q and k shared by two value heads, small heads, a learned decay
        _mix("train", 6, 1500, 16, 64, 64, HK=8, padded=True, learned=True, name="train_padded"),
        # the exact fp32 path (debugging, small checks)
        _mix("train", 1, 256, 2, 64, 64, dtype="fp32", name="train_fp32"),
        # the norm of each head's output of a serving batch: few short rows, latency
        _norm("norm", 53 * 16, 128, bias=False, name="norm_heads"),
        # the norm in front of the mixer, 4 x 4096 tokens of 16 x 128 channels
        _norm("norm", 16384, 2048, name="norm_rows"),
        # its training step, parameters kept in fp32
        _norm("norm_train", 16384, 2048, weights="fp32", name="norm_train_rows"),
    ]


_HEADS = [(64, 64), (128, 128), (128, 256), (256, 512), (256, 256), (96, 80), (48, 160), (24, 200)]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case, sizes over the whole range.  Odd lengths and head shapes among them."""
    path = rng.choice(["decode", "forward", "forward", "train", "train", "norm", "norm_train"])
    if path.startswith("norm"):
        D = _log_int(rng, 32, 16384)
        if rng.random() < 0.7:
            D = max(8, D // 8 * 8)
        rows = _log_int(rng, 1, min(1 << 17, (1 << 26) // D))
        return _norm(path, rows, D, dtype=rng.choice(["bf16", "bf16", "fp32"]), weights=rng.choice(["bf16", "fp32", "none"] if path == "norm" else ["bf16", "fp32"]),
                     bias=rng.random() < 0.7, gap=rng.choice([0, 0, 8, 40]))  # fmt: skip
    K, V = rng.choice(_HEADS)
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])
    HK = rng.choice([H, H, H // 2 if H % 2 == 0 else H])
    options = dict(HK=HK, decay=rng.random() < 0.9)
    if path == "decode":
        B = _log_int(rng, 1, 512)
        T = 1 if rng.random() < 0.7 else rng.randint(2, 64)
        while B * H * K * V > 256 * 32 * 128 * 128 // (1 if T == 1 else 4):
            B = max(1, B // 2)
        return _mix(path, B, T, H, K, V, dtype=rng.choice(["bf16", "bf16", "fp32"]), **options)
    dtype = "fp32" if rng.random() < 0.15 else "bf16"
    tokens = _log_int(rng, 65, 2048 if dtype == "fp32" else 65536)
    kind = rng.choice(["batch", "batch", "padded", "packed"])
    B = 1 if kind == "packed" else min(rng.choice([1, 2, 3, 4, 8]), max(1, tokens // 65))
    T, N = max(65, tokens // B), 0
    if kind == "packed":
        N = min(rng.choice([2, 5, 11, 24, 70]), max(2, T // 16))
    limit = (1 << 26) if path == "train" else (1 << 28)
    while B * T * H * (K + V) > limit and T > 130:
        T //= 2
    while B * T * H * (K + V) > limit and H % 2 == 0:
        H, options["HK"] = H // 2, max(1, options["HK"] // 2)
    while N * H * K * V > 1 << 26 and N > 2:
        N //= 2
    return _mix(path, B, T, H, K, V, N=N, padded=kind == "padded", dtype=dtype, state=rng.random() < 0.5,
                learned=path == "train" and options["decay"] and rng.random() < 0.3, **options)  # fmt: skip


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Tokens of every sequence."""
    if case["N"]:
        # cuts of the row at random places: lengths from a handful of tokens to a large part of the row
        gen = torch.Generator().manual_seed(seed + 77)
        cuts = (torch.randperm(case["T"] - 1, generator=gen)[: case["N"] - 1] + 1).sort().values.tolist()
        return [b - a for a, b in zip([0] + cuts, cuts + [case["T"]])]
    if case["padded"]:
        gen = torch.Generator().manual_seed(seed + 78)
        lens = torch.randint(max(1, case["T"] // 4), case["T"] + 1, (case["B"],), generator=gen).tolist()
        lens[seed % len(lens)] = case["T"]
        return lens
    return [case["T"]] * case["B"]


def _decays(H, gen):
    """The usual slopes, one for each head from fast to slow, with a little of the seed in them."""
    slopes = -(2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=F32) / H))
    return slopes * (1.0 + 0.05 * torch.rand(H, device="cuda", generator=gen))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    train = case["path"] in ("train", "norm_train")
    s = dict(case)
    if case["path"].startswith("norm"):
        rows, D = case["rows"], case["D"]
        x = (randn(rows, D + case["gap"]) + randn(rows, 1)).to(dtype)  # a residual stream: every row has a mean of its own
        s["x"] = x[:, :D].requires_grad_() if train else x[:, :D]
        s["weight"] = s["bias"] = None
        if case["weights"] != "none":
            s["weight"] = (1.0 + 0.1 * randn(D)).to(DTYPES[case["weights"]]).requires_grad_(train)
            if case["bias"]:
                s["bias"] = (0.1 * randn(D)).to(DTYPES[case["weights"]]).requires_grad_(train)
        if train:
            s["dy"] = randn(rows, D).to(dtype)
        return s
    B, T, H, HK, K, V = (case[n] for n in ("B", "T", "H", "HK", "K", "V"))
    lens = _lengths(case, seed)
    # what a layer hands over: q, k, v are the column blocks of one projection's output
    qkv = randn(B, T, 2 * HK * K + H * V).to(dtype)
    q, k, v = qkv.split((HK * K, HK * K, H * V), dim=-1)
    s["q"], s["k"], s["v"] = q.view(B, T, HK, K), k.view(B, T, HK, K), v.view(B, T, H, V)
    s["g"] = _decays(H, gen) if case["decay"] else None
    s["h0"] = 0.5 * randn(len(lens), H, K, V) if case["state"] else None
    s["lens"], s["cu"] = lens, None
    if case["N"] or case["padded"]:
        s["cu"] = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    if train:
        s["leaves"] = ["q", "k", "v"] + (["g"] if case["learned"] else []) + (["h0"] if case["state"] else [])
        for name in s["leaves"]:
            s[name] = s[name].detach().requires_grad_()
        s["do"] = randn(B, T, H, V).to(dtype)
        s["dht"] = 0.1 * randn(len(lens), H, K, V)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if s["path"] == "norm":
        return _call_norm(s) if own else _plain_norm(s["x"], s["weight"], s["bias"])
    if s["path"] == "norm_train":
        y = _call_norm(s) if own else _plain_norm(s["x"], s["weight"], s["bias"])
        leaves = [x for x in (s["x"], s["weight"], s["bias"]) if x is not None]
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if s["path"] == "decode":
        if own:
            from lm_engine_amd import fused_recurrent_linear_attention

            return fused_recurrent_linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["h0"], output_final_state=True, inplace_state=True)
        o, ht = _plain_attention(s)
        s["h0"].copy_(ht)
        return o, s["h0"]
    if s["path"] == "forward":
        return _call_attention(s) if own else _plain_attention(s)
    o, ht = _call_attention(s) if own else _plain_attention(s)
    return (o.detach(), ht.detach(), *torch.autograd.grad((o, ht), [s[n] for n in s["leaves"]], (s["do"], s["dht"])))


def _call_norm(s):
    from lm_engine_amd import layer_norm

    return layer_norm(s["x"], s["weight"], s["bias"], NORM_EPS)


def _call_attention(s):
    from lm_engine_amd import chunk_linear_attention

    return chunk_linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["h0"], output_final_state=True, cu_seqlens=s["cu"], left_padded=s["padded"])


# ---------------------------------------------------------------------------------------------------------------------
# the plain form, in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(x, weight, bias):
    x32 = x.float()
    centred = x32 - x32.mean(dim=-1, keepdim=True)
    y = centred * torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + NORM_EPS)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def _plain_chunks(q, k, v, g, state, C):
    """Chunks of C tokens: q, k, v [B, H, n, C, .], g [H], state [B, H, K, V] -> (o [B, H, n, C, V], state)."""
    i = torch.arange(C, device=q.device, dtype=F32)
    distance = i[:, None] - i[None, :]
    weights = torch.exp(g[:, None, None] * distance.clamp(min=0)) * (distance >= 0)  # [H, C, C]
    inside = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * weights[None, :, None], v)
    to_end = torch.exp(g[:, None] * (C - 1 - i))  # [H, C]
    local = torch.matmul((k * to_end[None, :, None, :, None]).transpose(-1, -2), v)
    whole = torch.exp(g * C)[None, :, None, None]
    states = []
    for c in range(q.size(2)):
        states.append(state)
        state = whole * state + local[:, :, c]
    from_start = torch.exp(g[:, None] * (i + 1))
    carried = torch.matmul(q, torch.stack(states, dim=2)) * from_start[None, :, None, :, None]
    return inside + carried, state


def _plain_rows(q, k, v, g, state, scale):
    """Whole sequences: q, k [B, T, H, K], v [B, T, H, V] in fp32 -> (o, state)."""
    B, T, H, _ = q.shape
    q, k, v = ((q * scale).transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
    if state is None:
        state = torch.zeros(B, H, q.size(-1), v.size(-1), device=q.device, dtype=F32)
    out, C = [], 64
    whole = T // C * C
    for begin, end, size in ((0, whole, C), (whole, T, T - whole)):
        if end > begin:
            part = [x[:, :, begin:end].reshape(B, H, -1, size, x.size(-1)) for x in (q, k, v)]
            o, state = _plain_chunks(*part, g, state, size)
            out.append(o.flatten(2, 3))
    return torch.cat(out, dim=2).transpose(1, 2), state


def _plain_attention(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, T, H, HK = s["B"], s["T"], s["H"], s["HK"]
    if HK < H:
        q, k = q.repeat_interleave(H // HK, dim=2), k.repeat_interleave(H // HK, dim=2)
    g = torch.zeros(H, device=q.device, dtype=F32) if s["g"] is None else s["g"]
    scale = s["K"] ** -0.5
    if s["cu"] is None:
        o, ht = _plain_rows(q, k, v, g, s["h0"], scale)
        return o.to(s["v"].dtype), ht
    outs, states, begin = [], [], 0
    for n, length in enumerate(s["lens"]):
        row, first = (n, T - length) if s["padded"] else (0, begin)
        pick = slice(first, first + length)
        o, ht = _plain_rows(*(x[row : row + 1, pick] for x in (q, k, v)), g, None if s["h0"] is None else s["h0"][n : n + 1], scale)
        outs.append(torch.cat([o.new_zeros(1, first, H, s["V"]), o], dim=1) if s["padded"] else o)
        states.append(ht)
        begin += length
    return torch.cat(outs, dim=0 if s["padded"] else 1).to(s["v"].dtype), torch.cat(states, dim=0)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp32": 4}
    e = size[case["dtype"]]
    if case["path"].startswith("norm"):
        cells = case["rows"] * case["D"]
        parameters = 0 if case["weights"] == "none" else case["D"] * size[case["weights"]] * (2 if case["bias"] else 1)
        if case["path"] == "norm":
            return dict(bytes=2 * cells * e + parameters, flops=8 * cells)
        # forward: x, y; backward: x, dy, dx
        return dict(bytes=5 * cells * e + 3 * parameters, flops=24 * cells)
    B, T, H, HK, K, V = (case[n] for n in ("B", "T", "H", "HK", "K", "V"))
    tokens, sequences = B * T, case["N"] or B
    if case["padded"]:
        tokens = tokens * 5 // 8  # lengths are even between a quarter of the row and the whole row
    qk, vo, state = 2 * tokens * HK * K * e, tokens * H * V * e, sequences * H * K * V * 4
    states = state * (2 if case["state"] else 1)
    per_state = 2 * tokens * H * K * V
    if case["path"] != "train":
        return dict(bytes=qk + 2 * vo + states, flops=2 * per_state)
    # forward, then q, k, v, do read again and dq, dk, dv written; the states' gradients
    moved = (qk + 2 * vo + states) + (2 * qk + 3 * vo + state + states)
    return dict(bytes=moved, flops=7 * per_state)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_norm(s):
    with torch.no_grad():
        x = s["x"].detach().to(F64)
        mean = x.sum(-1, keepdim=True) / x.size(-1)
        var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.size(-1)
        r = 1.0 / torch.sqrt(var + NORM_EPS)
        unit = (x - mean) * r
        w = 1.0 if s["weight"] is None else s["weight"].detach().to(F64)
        y = unit * w
        if s["bias"] is not None:
            y = y + s["bias"].detach().to(F64)
        if s["path"] == "norm":
            return y
        dy = s["dy"].to(F64)
        du = dy * w
        dx = r * (du - du.mean(-1, keepdim=True) - unit * (du * unit).mean(-1, keepdim=True))
        grads = [dx]
        if s["weight"] is not None:
            grads.append((dy * unit).sum(0))
        if s["bias"] is not None:
            grads.append(dy.sum(0))
        return (y, *grads)


_BLOCK = 96


def _exact_sequence(q, k, v, w, scale, h0, do=None, dht=None, tangent=False):
    """One batch of whole sequences [B, T, H, .], block by block along T: state and output forward in time, the state's gradient
    and those of k and v backward.  ``w`` [H]: the factor of one token.  Returns (o, state[, dq, dk, dv, dh0, dg])."""
    B, T, H, K = q.shape
    V = v.size(-1)
    heads = lambda x: x.permute(0, 2, 1, 3).to(F64)  # noqa: E731
    power = lambda e: torch.pow(w[:, None], e[None, :])  # noqa: E731
    state = torch.zeros(B, H, K, V, device=q.device, dtype=F64) if h0 is None else h0.to(F64)
    u = torch.zeros_like(state)  # derivative of the state by the log-decay
    o, saved, dg = torch.empty(B, T, H, V, device=q.device, dtype=F64), [], torch.zeros(H, device=q.device, dtype=F64)
    dq = torch.empty(B, T, H, K, device=q.device, dtype=F64) if do is not None else None
    for a in range(0, T, _BLOCK):
        b = min(T, a + _BLOCK)
        qb, kb, vb = heads(q[:, a:b]) * scale, heads(k[:, a:b]), heads(v[:, a:b])
        n = torch.arange(b - a, device=q.device, dtype=F64)
        gap = n[:, None] - n[None, :]
        lower = torch.where(gap >= 0, torch.pow(w[:, None, None], gap.clamp(min=0)), torch.zeros_like(gap))
        first, last = power(n + 1)[None, :, :, None], power(b - a - 1 - n)[None, :, :, None]
        scores = qb @ kb.transpose(-1, -2)
        ob = first * (qb @ state) + (scores * lower) @ vb
        o[:, a:b] = ob.permute(0, 2, 1, 3)
        if do is not None:
            dob = heads(do[:, a:b])
            dqb = scale * (first * (dob @ state.transpose(-1, -2)) + ((dob @ vb.transpose(-1, -2)) * lower) @ kb)
            dq[:, a:b] = dqb.permute(0, 2, 1, 3)
            if tangent:
                by_g = first * ((n + 1)[None, None, :, None] * (qb @ state) + qb @ u) + (scores * lower * gap) @ vb
                dg += (by_g * dob).sum(dim=(0, 2, 3))
                u = (w ** (b - a))[None, :, None, None] * (u + (b - a) * state) + (kb * last * (b - a - 1 - n)[None, None, :, None]).transpose(-1, -2) @ vb
        state = (w ** (b - a))[None, :, None, None] * state + (kb * last).transpose(-1, -2) @ vb
    if do is None:
        return o, state
    back = torch.zeros_like(state) if dht is None else dht.to(F64)  # gradient of the state behind the block
    if tangent and dht is not None:
        dg += (u * back).sum(dim=(0, 2, 3))
    dk, dv = torch.empty_like(dq), torch.empty_like(o)
    for a in reversed(range(0, T, _BLOCK)):
        b = min(T, a + _BLOCK)
        qb, kb, vb, dob = heads(q[:, a:b]) * scale, heads(k[:, a:b]), heads(v[:, a:b]), heads(do[:, a:b])
        n = torch.arange(b - a, device=q.device, dtype=F64)
        gap = n[None, :] - n[:, None]  # from the row's token to a later one
        upper = torch.where(gap >= 0, torch.pow(w[:, None, None], gap.clamp(min=0)), torch.zeros_like(gap))
        last, first = power(b - a - 1 - n)[None, :, :, None], power(n + 1)[None, :, :, None]
        dkb = last * (vb @ back.transpose(-1, -2)) + ((vb @ dob.transpose(-1, -2)) * upper) @ qb
        dvb = last * (kb @ back) + ((kb @ qb.transpose(-1, -2)) * upper) @ dob
        dk[:, a:b], dv[:, a:b] = dkb.permute(0, 2, 1, 3), dvb.permute(0, 2, 1, 3)
        back = (w ** (b - a))[None, :, None, None] * back + (qb * first).transpose(-1, -2) @ dob
    return o, state, dq, dk, dv, back, dg


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"].startswith("norm"):
        return _exact_norm(s)
    with torch.no_grad():
        B, T, H, HK, K, V = (case[n] for n in ("B", "T", "H", "HK", "K", "V"))
        q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
        q, k = (x.repeat_interleave(H // HK, dim=2) if HK < H else x for x in (q, k))
        w = torch.ones(H, device="cuda", dtype=F64) if s["g"] is None else torch.exp(s["g"].detach().to(F64))
        h0 = None if s["h0"] is None else s["h0"].detach()
        train = case["path"] == "train"
        if s["cu"] is None:
            parts = [(slice(0, B), slice(0, T), slice(0, B))]
        elif case["padded"]:
            parts = [(slice(n, n + 1), slice(T - length, T), slice(n, n + 1)) for n, length in enumerate(s["lens"])]
        else:
            ends = [sum(s["lens"][: n + 1]) for n in range(len(s["lens"]))]
            parts = [(slice(0, 1), slice(end - length, end), slice(n, n + 1)) for n, (end, length) in enumerate(zip(ends, s["lens"]))]
        zeros = lambda *shape: torch.zeros(*shape, device="cuda", dtype=F64)  # noqa: E731
        o, ht = zeros(B, T, H, V), zeros(len(s["lens"]), H, K, V)
        if train:
            dq, dk, dv, dh0, dg = zeros(B, T, H, K), zeros(B, T, H, K), zeros(B, T, H, V), torch.zeros_like(ht), zeros(H)
        for rows, tokens, state in parts:
            operands = (q[rows, tokens], k[rows, tokens], v[rows, tokens], w, K**-0.5, None if h0 is None else h0[state])
            if not train:
                o[rows, tokens], ht[state] = _exact_sequence(*operands)
                continue
            o[rows, tokens], ht[state], dq[rows, tokens], dk[rows, tokens], dv[rows, tokens], dh0[state], dg_part = _exact_sequence(
                *operands, s["do"][rows, tokens], s["dht"][state], case["learned"])  # fmt: skip
            dg += dg_part
        if not train:
            return o, ht
        if HK < H:
            dq, dk = (x.view(B, T, HK, H // HK, K).sum(dim=3) for x in (dq, dk))
        return (o, ht, dq, dk, dv, *([dg] if case["learned"] else []), *([dh0] if case["state"] else []))
