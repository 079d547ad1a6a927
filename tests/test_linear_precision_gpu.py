"""How exact linear attention is, to limits that its arithmetic has to be right for.

fp32, decays near one.  A factor w = e^{n g} held as one fp32 number is off by up to 2^-25 relative, the same way every time it is applied: a
state that remembers m applications is off by m 2^-25, and m is in the thousands here.  Held as 1 and w - 1 it is exact; what is left
are the roundings of the sums, independent of each other: with r of them remembered, each of at most 2^-24 relative (rms 2^-24 / sqrt 3),
sqrt(r / 3) 2^-24."""

import pytest
import torch

from lm_engine_amd import chunk_linear_attention


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
