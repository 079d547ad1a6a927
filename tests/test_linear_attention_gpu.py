"""Linear attention with a decay for each head on the GPU, through its public entry points, against the token loop in 64 bits.

Tolerances, relative-L2 per tensor.  bf16 inputs are exact as they are; the output's own rounding is off by at most 2^-9 of the value on
average half of that, and what is summed carries independent roundings of the state and of the chunk's weights as operands, each of at
most 2^-8 / 2 relative to the term (bf16: eps / 2 = 2^-8): a sum of terms with independent relative errors of at most e has a relative-L2
error of at most e, three of them together sqrt(3) 2^-8 = 6.8e-3 at the very most; 5e-3 is asked (rms of a rounding is 1 / sqrt(3) of its
maximum: 3.9e-3).  States (and their gradients): the rows that go in are split in two bf16 parts, 2^-17 of a term at most, and fp32 sums
of n terms: 2e-5.  fp32 inputs: sums of up to 1e3 terms in fp32, 1e-5.  A gradient of heads that share one of q and k is a sum of
gradients rounded to bf16 and rounded again: another 2^-8, 7e-3."""

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import chunk_linear_attention, fused_recurrent_linear_attention, linear_attention
from oracle.linear_attention_oracle import linear_attention_ref, sequences_of
from tests.helpers import rel_l2


pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
OUT = {BF16: 5e-3, F32: 1e-5}
STATE = {BF16: 2e-5, F32: 1e-5}


def _inputs(B, T, H, K, V, HK=None, N=None, dtype=BF16, decay="slopes", state=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    HK, N = HK or H, N or B
    g = {"slopes": -(2.0 ** (-8.0 * torch.arange(1, H + 1) / H)), "none": None, "fast": torch.full((H,), -30.0),
         "at once": torch.full((H,), -float("inf")), "slow": torch.full((H,), -1e-4)}[decay]  # fmt: skip
    return dict(q=randn(B, T, HK, K).to(dtype), k=randn(B, T, HK, K).to(dtype), v=randn(B, T, H, V).to(dtype), g=g,
                initial_state=0.5 * randn(N, H, K, V) if state else None)  # fmt: skip


def _cuda(inputs, **more):
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in {**inputs, **more}.items()}


def _check(name, got, want, tolerance):
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} {tuple(want.shape)}"
    error = rel_l2(got, want)
    print(f"{name} {error:.2e}", flush=True)
    assert torch.isfinite(got.float()).all() and error <= tolerance, f"{name}: relative-L2 {error:.3e} above {tolerance:.1e}"


def _cu(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist()


# (B, T, H, K, V, options)
SHAPES = [
    (1, 1, 2, 64, 64, {}),
    (2, 63, 2, 64, 64, {}),
    (1, 64, 3, 128, 128, {}),
    (2, 65, 2, 128, 128, {}),
    (1, 200, 2, 128, 256, {}),
    (1, 129, 1, 256, 512, {}),
    (2, 130, 2, 96, 80, {}),
    (1, 300, 2, 24, 200, {}),
    (1, 70, 2, 8, 8, {}),
    (1, 190, 2, 48, 160, {}),
    (1, 257, 2, 256, 64, {}),
    (1, 700, 4, 64, 64, dict(HK=2)),
    (2, 140, 6, 128, 128, dict(HK=2)),
    (1, 1, 2, 128, 128, dict(state=False)),
    (2, 100, 2, 128, 128, dict(state=False)),
    (1, 150, 2, 64, 128, dict(decay="none")),
    (1, 150, 2, 128, 64, dict(decay="fast")),
    (1, 150, 2, 128, 64, dict(decay="at once")),
    (1, 400, 2, 64, 64, dict(decay="slow")),
]
LAYOUTS = [  # (lengths, left-padded, tokens of a row or of the packed row)
    ([130, 1, 64, 65, 7], False, 267),
    ([5, 0, 200, 0], False, 205),
    ([100, 50], False, 180),  # 30 tokens behind the last sequence
    ([0, 0], False, 40),
    ([130, 70, 0, 1], True, 130),
    ([10, 64, 140], True, 200),
    ([1] * 70 + [40], False, 110),
]
_ID = lambda x: str(x) if not isinstance(x, torch.dtype) else str(x).split(".")[-1]  # noqa: E731


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("form", ["chunk", "recurrent"])
@pytest.mark.parametrize("B, T, H, K, V, options", SHAPES, ids=_ID)
def test_forward(B, T, H, K, V, options, form, dtype):
    inputs = _inputs(B, T, H, K, V, dtype=dtype, **options)
    want, want_state = linear_attention_ref(**inputs)
    fn = chunk_linear_attention if form == "chunk" else fused_recurrent_linear_attention
    o, state = fn(**_cuda(inputs), output_final_state=True)
    assert o.dtype == dtype and state.dtype == F32
    _check("o", o, want, OUT[dtype])
    _check("state", state, want_state, STATE[dtype])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("form", ["chunk", "recurrent"])
@pytest.mark.parametrize("lens, padded, T", LAYOUTS, ids=_ID)
def test_forward_of_packed_and_padded_batches(lens, padded, T, form, dtype):
    B, H, K, V = (len(lens), 3, 64, 96) if padded else (1, 3, 64, 96)
    inputs = _inputs(B, T, H, K, V, N=len(lens), dtype=dtype)
    cu = _cu(lens)
    want, want_state = linear_attention_ref(**inputs, cu_seqlens=cu, left_padded=padded)
    fn = chunk_linear_attention if form == "chunk" else fused_recurrent_linear_attention
    torch.full((1 << 22,), float("nan"), device="cuda")  # what a fresh output's memory may hold
    o, state = fn(**_cuda(inputs, cu_seqlens=torch.tensor(cu, dtype=torch.int32)), output_final_state=True, left_padded=padded)
    outside = torch.ones(B, T, dtype=torch.bool)
    for b, first, length in sequences_of(B, T, cu, padded):
        outside[b, first : first + length] = False
    assert (o.cpu()[outside] == 0).all()
    _check("o", o, want, OUT[dtype])
    _check("state", state, want_state, STATE[dtype])


def _gradients(inputs, dtype, form="chunk", learned=False, cu=None, padded=False, seed=100, **kwargs):
    """(results and gradients of the kernels, the same of autograd through the loop in 64 bits)."""
    gen = torch.Generator().manual_seed(seed)
    names = [n for n in ("q", "k", "v", "initial_state") if inputs[n] is not None] + (["g"] if learned else [])
    ref = {n: x.double().requires_grad_(n in names) if isinstance(x, torch.Tensor) else x for n, x in inputs.items()}
    o, state = linear_attention_ref(**ref, cu_seqlens=cu, left_padded=padded, **kwargs)
    do, dht = torch.randn(o.shape, generator=gen).to(dtype), 0.1 * torch.randn(state.shape, generator=gen)
    o = o + 0 * sum(ref[n].sum() for n in names)  # (sequences without a token leave nothing to differentiate)
    want = torch.autograd.grad((o, state), [ref[n] for n in names], (do.double(), dht.double()))
    own = _cuda(inputs)
    for n in names:
        own[n].requires_grad_()
    fn = chunk_linear_attention if form == "chunk" else fused_recurrent_linear_attention
    cu_gpu = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    o_own, state_own = fn(**own, output_final_state=True, cu_seqlens=cu_gpu, left_padded=padded, **kwargs)
    got = torch.autograd.grad((o_own, state_own), [own[n] for n in names], (do.cuda(), dht.cuda()))
    return dict(zip(names, got)), dict(zip(names, want))


def _check_gradients(got, want, dtype, shared=False):
    for n, x in got.items():
        limit = {"initial_state": STATE[dtype], "g": 1e-4}.get(n, OUT[dtype])
        if shared and dtype == BF16 and n in ("q", "k"):
            limit = 7e-3
        _check("d" + n, x, want[n], limit)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("B, T, H, K, V, options", SHAPES, ids=_ID)
def test_backward(B, T, H, K, V, options, dtype):
    got, want = _gradients(_inputs(B, T, H, K, V, dtype=dtype, **options), dtype)
    _check_gradients(got, want, dtype, shared="HK" in options)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("lens, padded, T", LAYOUTS, ids=_ID)
def test_backward_of_packed_and_padded_batches(lens, padded, T, dtype):
    B = len(lens) if padded else 1
    got, want = _gradients(_inputs(B, T, 3, 64, 96, N=len(lens), dtype=dtype), dtype, cu=_cu(lens), padded=padded)
    outside = torch.ones(B, T, dtype=torch.bool)
    for b, first, length in sequences_of(B, T, _cu(lens), padded):
        outside[b, first : first + length] = False
    for n in ("q", "k", "v"):
        assert (got[n].cpu()[outside] == 0).all(), n
    _check_gradients(got, want, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("B, T, H, K, V, options", [s for s in SHAPES if s[5].get("decay") not in ("none", "at once")], ids=_ID)
def test_gradient_of_the_decay(B, T, H, K, V, options, dtype):
    got, want = _gradients(_inputs(B, T, H, K, V, dtype=dtype, **options), dtype, learned=True)
    _check_gradients(got, want, dtype, shared="HK" in options)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("lens, padded, T", LAYOUTS, ids=_ID)
def test_gradient_of_the_decay_of_packed_and_padded_batches(lens, padded, T, dtype):
    B = len(lens) if padded else 1
    got, want = _gradients(_inputs(B, T, 3, 64, 96, N=len(lens), dtype=dtype), dtype, learned=True, cu=_cu(lens), padded=padded)
    _check_gradients(got, want, dtype)
