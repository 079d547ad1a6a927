"""How exact linear attention is, to limits that its arithmetic has to be right for.

fp32, decays near one.  A factor w = e^{n g} held as one fp32 number is off by up to 2^-25 relative, the same way every time it is applied: a
state that remembers m applications is off by m 2^-25, and m is in the thousands here.  Held as 1 and w - 1 it is exact; what is left
are the roundings of the sums, independent of each other: with r of them remembered, each of at most 2^-24 relative (rms 2^-24 / sqrt 3),
sqrt(r / 3) 2^-24.

bf16.  A state that is a result takes the decayed rows in three bf16 parts, all 24 bits of an fp32 product, in 12 additions a chunk of
64 tokens, and is multiplied once a chunk: 13 roundings, 33 chunks at most here, sqrt(13 * 33 / 3) 2^-24 = 7.1e-7 if nothing were forgotten;
1e-6 is asked.  (Two parts leave 2^-17 of a term, 2.4e-6 rms.)  Outputs and gradients: rounding normally distributed values to bf16 changes
them by 1.66e-3 relative-L2; the state as an operand is rounded like that and makes one part of a sum, the weights of the tokens inside the
chunk make the other part, so the sum is off by 1.66e-3 of its own before its own rounding: sqrt(2) 1.66e-3 = 2.35e-3, and 2.6e-3 is asked.
Gradients of heads that share one of q and k are added up in fp32 and rounded once: no more than that.  (A second rounding would make
sqrt(3) 1.66e-3 = 2.9e-3.)"""

import pytest
import torch

from lm_engine_amd import chunk_linear_attention, fused_recurrent_linear_attention
from oracle.linear_attention_oracle import linear_attention_ref
from tests.helpers import rel_l2
from tests.test_linear_attention_gpu import BF16, _check, _cu, _cuda, _gradients, _inputs


pytestmark = pytest.mark.gpu

F32, F64 = torch.float32, torch.float64


def _normal(*shape, seed, mean=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen) + mean


def test_gradient_of_a_slow_decay_in_fp32():
    """As many sequences as it takes to walk each as one segment.  Factors whose fp32 numbers are off by 2.5e-8 to 3e-8, so 256 to 2048
    remembered tokens would make 1e-5 and more.  Two roundings a token in the state's derivative and two in the state, all 2048 tokens
    remembered: sqrt(4 * 2048 / 3) 2^-24 = 3.1e-6 for a single cell; dg sums 256 sequences x 64 cells of them, and its own sums of up to 2048
    terms in order add sqrt(2048 / 3) 2^-24 = 1.6e-6 for a single thread's of 2048.  2e-6 is far above what is left of either."""
    B, T, H, D = 256, 2048, 4, 8
    g = torch.tensor([-0.004792203661054373, -0.004349226597696543, -0.0014639175496995449, -0.0013917526230216026], device="cuda")
    q, k, v, do = (_normal(B, T, H, D, seed=s) for s in range(4))
    learned = g.clone().requires_grad_()
    o, _ = chunk_linear_attention(q, k, v, learned)
    got, = torch.autograd.grad(o, learned, do)
    w = torch.exp(g.to(F64))[:, None, None]
    S = torch.zeros(B, H, D, D, device="cuda", dtype=F64)
    U, want = S.clone(), torch.zeros(H, device="cuda", dtype=F64)
    for t in range(T):
        U = w * (U + S)  # the derivative of the state by g
        S = w * S + k[:, t].to(F64)[..., :, None] * v[:, t].to(F64)[..., None, :]
        want += ((q[:, t].to(F64)[..., :, None] * U).sum(-2) * do[:, t].to(F64)).sum((0, 2))
    want *= D**-0.5
    error = ((got.to(F64) - want) / want).abs()
    print(error.tolist(), flush=True)
    assert (error <= 2e-6).all(), error.tolist()


@pytest.mark.parametrize("g", [-1.5360825273091905e-05, -1.6082474758150056e-05, -1.226804124598857e-05, -1.041237101162551e-05,
                               -1.4845360965409782e-05, -1.1752576938306447e-05])  # fmt: skip
def test_states_of_many_segments_in_fp32(g):
    """1024 segments of 64 tokens of one head, joined by factors e^{64 g} that fp32 numbers are 2.7e-8 off from or more: some 1e-5 in all.
    Two roundings a join and two a token of a segment: sqrt(2 (1024 + 64) / 3) 2^-24 = 1.6e-6 at most, 3e-6 is asked."""
    T, D = 65536, 8
    q, k, v, do = (_normal(1, T, 1, D, seed=s) for s in range(4))
    decay = torch.tensor([g], device="cuda")
    state = torch.zeros(1, 1, D, D, device="cuda", requires_grad=True)
    o, final = chunk_linear_attention(q, k, v, decay, initial_state=state, output_final_state=True)
    dh0, = torch.autograd.grad(o, state, do)
    n = torch.arange(T, device="cuda", dtype=F64)
    flat = lambda x: x[0, :, 0].to(F64)  # noqa: E731
    w = decay.to(F64)
    want = (flat(k) * torch.exp(w * (T - 1 - n))[:, None]).t().contiguous() @ flat(v)
    want_dh0 = D**-0.5 * (flat(q) * torch.exp(w * (n + 1))[:, None]).t().contiguous() @ flat(do)
    errors = rel_l2(final[0, 0], want), rel_l2(dh0[0, 0], want_dh0)
    print(errors, flush=True)
    assert max(errors) <= 3e-6, errors


@pytest.mark.parametrize("g", [-1.5360825273091905e-05, -1.226804124598857e-05, -1.1752576938306447e-05])
def test_gradient_of_a_slow_decay_over_many_segments_in_fp32(g):
    """As above, of the state's derivative, which remembers twice as long: twice the limit."""
    T, D = 65536, 8
    q, k, v, do = (_normal(1, T, 1, D, seed=s) for s in range(4))
    decay = torch.tensor([g], device="cuda", requires_grad=True)
    o, _ = chunk_linear_attention(q, k, v, decay)
    got, = torch.autograd.grad(o, decay, do)
    # sum_t do_t . sum_{j < t} (t - j) w^{t - j} (q_t . k_j) v_j, 1024 tokens of each at a time
    flat = lambda x: x[0, :, 0].to(F64)  # noqa: E731
    qf, kf, vf, df, w, C = flat(q), flat(k), flat(v), flat(do), decay.detach().to(F64), 1024
    S = torch.zeros(D, D, device="cuda", dtype=F64)
    U, want, n = S.clone(), 0.0, torch.arange(C, device="cuda", dtype=F64)
    first, last = torch.exp(w * (n + 1))[:, None], torch.exp(w * (C - 1 - n))[:, None]
    gap = (n[:, None] - n[None, :]).clamp(min=0)
    inside = gap * torch.exp(w * gap) * (gap > 0)
    for a in range(0, T, C):
        qb, kb, vb, db = (x[a : a + C] for x in (qf, kf, vf, df))
        by_g = first * ((n + 1)[:, None] * (qb @ S) + qb @ U) + ((qb @ kb.t().contiguous()) * inside) @ vb
        want += (by_g * db).sum()
        U = torch.exp(w * C) * (U + C * S) + (kb * last * (C - 1 - n)[:, None]).t().contiguous() @ vb
        S = torch.exp(w * C) * S + (kb * last).t().contiguous() @ vb
    want = D**-0.5 * want
    error = abs((got.item() - want) / want).item()
    print(error, flush=True)
    assert error <= 6e-6


STATE, OUT = 1e-6, 2.6e-3

# (B, T, H, K, V, lengths of packed sequences, options): one segment on the walk (K above 128) and on whole sequences, several, shared heads,
# more columns than a backward walk has keys
SHAPES = [
    (1, 64, 3, 128, 128, None, {}),
    (2, 65, 2, 128, 128, None, {}),
    (1, 129, 1, 256, 512, None, {}),
    (2, 130, 2, 96, 80, None, {}),
    (1, 1100, 2, 128, 128, None, {}),
    (1, 2101, 2, 128, 128, None, {}),
    (1, 1790, 1, 256, 64, None, {}),
    (1, 400, 2, 64, 64, None, dict(decay="slow")),
    (1, 700, 4, 64, 64, None, dict(HK=2)),
    (2, 140, 6, 128, 128, None, dict(HK=2)),
    (1, 900, 4, 72, 264, None, dict(HK=1)),
    (1, 2000, 4, 64, 128, [1200, 3, 0, 400, 397], dict(HK=2)),
]


@pytest.mark.parametrize("B, T, H, K, V, lens, options", SHAPES, ids=str)
def test_forward_in_bf16(B, T, H, K, V, lens, options):
    inputs = _inputs(B, T, H, K, V, N=None if lens is None else len(lens), **options)
    cu = None if lens is None else _cu(lens)
    cu_gpu = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    want, want_state = linear_attention_ref(**inputs, cu_seqlens=cu)
    for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
        o, state = fn(**_cuda(inputs), output_final_state=True, cu_seqlens=cu_gpu)
        _check("o", o, want, OUT)
        _check("state", state, want_state, STATE)


@pytest.mark.parametrize("learned", [False, True], ids=["", "decay"])
@pytest.mark.parametrize("B, T, H, K, V, lens, options", SHAPES, ids=str)
def test_gradients_in_bf16(B, T, H, K, V, lens, options, learned):
    """The decay's: sums of fp32 terms and products of bf16 numbers in three parts, 1e-5 (of its own size, which a sum over tokens and
    columns may leave smaller than its terms)."""
    inputs = _inputs(B, T, H, K, V, N=None if lens is None else len(lens), **options)
    got, want = _gradients(inputs, BF16, learned=learned, cu=None if lens is None else _cu(lens))
    for name, x in got.items():
        _check("d" + name, x, want[name], {"initial_state": STATE, "g": 1e-5}.get(name, OUT))
