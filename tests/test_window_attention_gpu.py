"""Softmax attention over a window on the GPU, through its public entry point, against the formula in 64 bits.

Tolerances, relative-L2 per tensor.  bf16 inputs are exact as they are.  The output's own rounding is off by at most 2^-8 (half a step of bf16)
relative to the value, and each weight, as an operand, by at most 2^-8 of itself: with uniformly spread roundings (rms 1 / sqrt(3) of the
maximum) independent of each other sqrt(2) 2^-8 / sqrt(3) = 3.2e-3; a weighted sum of values of both signs is smaller than the root of the sum of
its terms' squares at worst by what the sum cancels, and 5e-3 is asked.  dv: the same two.  dq, dk: ds = w (dw - delta) is rounded once more as an
operand, and delta comes from the rounded output, 2^-8 / sqrt(3) of each term of delta: three roundings, sqrt(3) 2^-8 / sqrt(3) = 3.9e-3 of terms of
which a row's add up to zero (sum of ds is none), so that what is left is smaller than the terms: 1e-2.  fp32 inputs: sums of up to 1e3
terms and exponents up to 2^5 with an error of 2^-24 relative: 1e-5."""

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import sliding_window_attention
from oracle.attention_oracle import visible_keys, window_attention_ref
from tests.helpers import rel_l2


pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
OUT = {BF16: 5e-3, F32: 1e-5}
GRAD = {BF16: 1e-2, F32: 1e-5}


def inputs(B, T, H, HK, D, S=None, dtype=BF16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    S = T if S is None else S
    return (1.5 * randn(B, T, H, D)).to(dtype), randn(B, S, HK, D).to(dtype), randn(B, S, HK, D).to(dtype)


def check(name, got, want, tolerance):
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} {tuple(want.shape)}"
    error = rel_l2(got, want)
    print(f"{name} {error:.2e}", flush=True)
    assert torch.isfinite(got.float()).all() and error <= tolerance, f"{name}: relative-L2 {error:.3e} above {tolerance:.1e}"


def cu_of(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist()


def check_call(q, k, v, dtype, cu=None, backward=True, **options):
    leaves = [x.cuda().requires_grad_(backward) for x in (q, k, v)]
    cu_gpu = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    o = sliding_window_attention(*leaves, cu_seqlens=cu_gpu, **options)
    ref = [x.double().requires_grad_(backward) for x in (q, k, v)]
    want = window_attention_ref(*ref, cu_seqlens=cu, **options)
    check("o", o, want.detach(), OUT[dtype])
    assert o.dtype == dtype and o.is_contiguous()
    if not backward:
        return
    do = torch.randn(o.shape, generator=torch.Generator().manual_seed(99)).to(dtype)
    got, expected = torch.autograd.grad(o, leaves, do.cuda()), torch.autograd.grad(want, ref, do.double())
    for name, x, y in zip(("dq", "dk", "dv"), got, expected):
        if y.norm() < 1e-9:  # (one visible key each: a weight of one whatever the scores are)
            assert x.float().norm() <= GRAD[dtype] * do.double().norm()
        else:
            check(name, x, y, GRAD[dtype])


# (B, T, H, HK, D, window, sinks)
WHOLE = [
    (1, 1, 1, 1, 64, None, 0),
    (2, 63, 2, 1, 64, None, 0),
    (1, 64, 4, 4, 128, 16, 0),
    (2, 65, 2, 2, 128, 64, 1),
    (1, 130, 8, 1, 128, 33, 5),
    (1, 300, 6, 2, 128, 100, 70),
    (2, 257, 2, 1, 256, 128, 4),
    (1, 200, 3, 3, 96, 50, 2),
    (1, 150, 4, 2, 80, None, 0),
    (1, 140, 2, 1, 24, 7, 3),
    (1, 140, 2, 2, 200, 64, 64),
    (1, 500, 5, 1, 64, 1, 0),
    (1, 500, 2, 1, 64, 1, 1),
    (1, 333, 16, 2, 64, 300, 130),
    (3, 700, 4, 2, 64, 200, 4),
    (1, 90, 2, 1, 64, 5000, 10),
    (1, 700, 2, 1, 8, 90, 300),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B, T, H, HK, D, window, sinks", WHOLE, ids=str)
def test_whole_sequences(B, T, H, HK, D, window, sinks, dtype):
    check_call(*inputs(B, T, H, HK, D, dtype=dtype), dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens, H, HK, D, window, sinks", [
    ([70, 1, 0, 129, 300], 4, 2, 64, 50, 3), ([200], 2, 1, 128, None, 0), ([5, 3, 2, 1, 1, 4, 7, 60, 64, 65], 2, 2, 64, 20, 2),
    ([150, 400], 8, 1, 128, 100, 40), ([1] * 100, 2, 1, 64, 8, 1),
], ids=str)  # fmt: skip
def test_packed_sequences(lens, H, HK, D, window, sinks, dtype):
    check_call(*inputs(1, sum(lens), H, HK, D, dtype=dtype), dtype, cu=cu_of(lens), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T, lens, window, sinks", [(200, [200, 0, 77, 1], 64, 4), (130, [3, 130], None, 0), (400, [399, 100], 30, 150)], ids=str)
def test_left_padded_rows(T, lens, window, sinks, dtype):
    check_call(*inputs(len(lens), T, 4, 2, 64, dtype=dtype), dtype, cu=cu_of(lens), left_padded=True, window=window, sinks=sinks)


# (T queries, S keys): continuations, single tokens over many keys (cut into parts), queries in front of the first key
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T, S, window, sinks", [(1, 700, None, 0), (1, 3000, None, 0), (1, 5000, 2000, 100), (7, 2049, None, 0), (100, 230, 60, 4),
                                                 (50, 20, None, 0), (130, 1, 4, 1), (64, 1500, 700, 64)], ids=str)  # fmt: skip
def test_other_keys_than_queries(T, S, window, sinks, dtype):
    for H, HK, D in ((4, 1, 64), (2, 2, 128)):
        check_call(*inputs(2, T, H, HK, D, S=S, dtype=dtype), dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(scale):
    for dtype in (BF16, F32):
        check_call(*inputs(1, 150, 2, 1, 64, dtype=dtype), dtype, window=100, sinks=3, scale=scale)


@pytest.mark.parametrize("T, H, HK, D, window", [(1200, 4, 2, 64, None), (900, 4, 2, 128, 500), (600, 2, 1, 256, 400), (300, 4, 2, 64, 8)])
def test_gradients_where_keys_and_values_have_a_mean(T, H, HK, D, window):
    """The sum of a row's ds is zero, and what is left of it comes back times the mean key: 1e-2 of dq's norm and more here, if delta were formed
    from the rounded output.  Exact sums leave ds's rounding (rms 2^-8 / sqrt(3) at most of terms that are up to sqrt(2) of dq's size, since a key is
    its mean and a difference of the same size: 3.2e-3) and the result's own (2.3e-3): 4e-3, and half as much again for the few rows whose
    weights are nearly all on one key."""
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, T, h, D, generator=gen) + torch.randn(D, generator=gen) for h in (H, HK, HK))
    q, k, v = (x.to(BF16) for x in (q, k, v))
    do = torch.randn(1, T, H, D, generator=gen).to(BF16)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(sliding_window_attention(*leaves, window=window), leaves, do.cuda())
    ref = [x.double().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(window_attention_ref(*ref, window=window), ref, do.double())
    for name, x, y in zip(("dq", "dk", "dv"), got, want):
        check(name, x, y, 6e-3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_window_of_one_has_no_gradients_of_scores(dtype):
    """Each query sees itself alone: o = v, and dq, dk are zero but for fp32 sums of D terms (1e-6 each of |do . v|, times |k| scale).  In fp32 o is
    v w (1 / w) with w = 2^(c s - m), where m is c s rounded and c s is not: w is next to 1 but not 1, and the two products and the quotient are
    rounded, 3 times 2^-24 of the value."""
    q, k, v = inputs(1, 300, 4, 2, 64, dtype=dtype)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    o = sliding_window_attention(*leaves, window=1)
    dq, dk, dv = torch.autograd.grad(o, leaves, torch.ones_like(o))
    values = leaves[2].repeat_interleave(2, dim=2)
    assert ((o - values).abs() <= (0 if dtype == BF16 else 4 * 2**-24) * values.abs()).all() and (dv - 2).abs().max() <= 2**-6
    assert dq.abs().max() <= 1e-4 and dk.abs().max() <= 1e-4


@pytest.mark.parametrize("sinks", [4, 11, 100, 1 << 20])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_sequences_that_are_first_keys_for_the_most_part(sinks, D):
    """Their gradients need no more memory than there are tokens."""
    lens = [1, 30, 2, 17, 64, 5, 5, 90, 12, 3, 40, 7, 0, 33, 1, 26]
    torch.cuda.reset_peak_memory_stats()
    q, k, v = inputs(1, sum(lens), 4, 2, D)
    check_call(q, k, v, BF16, cu_of(lens), window=6, sinks=sinks)
    assert torch.cuda.max_memory_allocated() < 1 << 30


@pytest.mark.parametrize("weight", [0.3, 0.6, 0.9, 0.98, 0.9999])
@pytest.mark.parametrize("T, H, HK, D, window, sinks", [(1200, 2, 1, 64, 400, 4), (1100, 2, 2, 64, None, 0), (1200, 2, 1, 128, 400, 4), (900, 2, 1, 128, None, 0), (700, 2, 1, 256, 300, 1), (200, 2, 1, 128, 90, 1)])
def test_queries_gradients_where_a_first_key_draws_the_weight(T, H, HK, D, window, sinks, weight):
    """A first key eight times as long as the others, which have no mean, with `weight` of every row's sum.  An error r of delta comes back as r times
    the row's weighted mean of keys, here `weight` times the first one.

    Whole: the coefficients of the keys add up to zero, rounded as they are, so that the first key's is off by what the others' are: 2^-8 / sqrt(3) rms
    at most of the first one's, and that again from the result's own rounding: 3.2e-3, and 4e-3 is asked (below a weight of 1, where ds is no rest).

    Row by row, in norm, with u = 2^-8 (bf16, half a step): delta from the output is off by rho, u sum |do| |o| from its rounding and u sum_j w_j
    sum |do| |v_j| from its weights'.  A key's ds with that, and its weight, are rounded: u (|ds_j| + w_j rho) + u w_j rho; what is taken off again is
    a sum over those, times w_j: w_j u (sum |ds| + 2 rho).  The result: u of itself.  fp32: scores and products of D terms, D 2^-24 of their
    terms' sizes, sums of S terms, S 2^-24."""
    gen = torch.Generator().manual_seed(T + D)
    scale, u, eps = D**-0.5, 2.0**-8, 2.0**-24
    towards = torch.randn(D, generator=gen)
    towards = towards / towards.norm()
    q, k, v = (torch.randn(1, T, h, D, generator=gen) for h in (H, HK, HK))
    seen = visible_keys(T, T, window, sinks)
    q -= (q @ towards)[..., None] * towards
    k[:, 0] = 8 * D**0.5 * towards
    for h in range(H):
        scores = torch.where(seen, q[0, :, h] @ k[0, :, h * HK // H].T * scale, -torch.inf)
        scores[:, 0] = -torch.inf
        rest = scores.logsumexp(dim=1)
        logit = torch.where(rest > -torch.inf, rest + torch.tensor(weight / (1 - weight)).log(), torch.zeros(()))
        q[0, :, h] += (logit / (scale * 8 * D**0.5))[:, None] * towards
    q, k, v, do = (x.to(BF16) for x in (q, k, v, torch.randn(1, T, H, D, generator=gen)))
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    dq, = torch.autograd.grad(sliding_window_attention(*leaves, window=window, sinks=sinks), leaves[:1], do.cuda())
    dq = dq.double().cpu()[0]
    errors, norms, worst = [], [], 0.0
    for h in range(H):
        Q, K, V, G = (x.double() for x in (q[0, :, h], k[0, :, h * HK // H], v[0, :, h * HK // H], do[0, :, h]))
        scores = torch.where(seen, Q @ K.T * scale, -torch.inf)
        w = scores.softmax(dim=1)
        o = w @ V
        dov, delta = G @ V.T, (G * o).sum(dim=1, keepdim=True)
        ds = w * (dov - delta)
        want = ds @ K * scale
        longs, parts = K.norm(dim=1), G.abs() @ V.abs().T
        rho = u * ((G.abs() * o.abs()).sum(1, keepdim=True) + (w * parts).sum(1, keepdim=True)) * (1 + u)
        total = ds.abs().sum(1, keepdim=True)
        bf16 = u * ds.abs() + 2 * u * w * rho + w * u * (total + 2 * rho)
        exponent = eps * ((D + 2) * scale * (Q.abs() @ K.abs().T) + 8 * (scores.nan_to_num(neginf=0.0).abs() + scores.logsumexp(1, keepdim=True).abs() + 1))
        products = (w * exponent * ((dov - delta).abs() + rho)) + w * eps * D * (parts + (G.abs() * o.abs()).sum(1, keepdim=True))
        fp32 = products + w * products.sum(1, keepdim=True) + eps * T * (ds.abs() + w * (total + 3 * rho))
        bound = (1 + u) * scale * ((bf16 + fp32) @ longs) + u * want.norm(dim=1)
        error = (dq[:, h] - want).norm(dim=1)
        worst = max(worst, (error / bound.clamp(min=1e-30)).max().item())
        errors.append(error), norms.append(want.norm(dim=1))
    whole = (torch.cat(errors).norm() / torch.cat(norms).norm()).item()
    print(f"dq {whole:.2e}, rows at {worst:.2f} of their bound", flush=True)
    assert worst <= 1, f"a row's error is {worst:.2f} of its bound"
    assert whole <= 4e-3 or weight > 0.99, f"relative-L2 {whole:.2e}"


@pytest.mark.parametrize("D", [64, 128, 256])
def test_blocks_of_keys_that_no_query_sees(D):
    """Behind a window, and in front of and behind the packed sequences: their gradients are zeros, next to blocks that have some."""
    check_call(*inputs(2, 10, 4, 2, D, S=500), BF16, window=20)
    check_call(*inputs(2, 10, 4, 2, D, S=500), BF16, window=20, sinks=3)
    q, k, v = inputs(1, 600, 2, 1, D)
    check_call(q, k, v, BF16, cu=[200, 210, 390], window=50, sinks=2)
