"""Layer norm on the GPU, forward and backward, against its definition in 64 bits.

Tolerances.  y: relative to the largest value of the row, half a step of the output's type (bf16 2^-8, fp32 2^-24) for its own rounding,
and fp32 arithmetic: the mean and the centred values carry errors of some 2^-24 of the largest |x|, and are divided by the row's
deviation, |x|_max / deviation times as much (rows here: up to 30); times a few operations: 2^-16.  Gradients, relative-L2: dx as y; dweight and dbias are fp32
sums of n <= 5000 terms, off by sqrt(n) 2^-24 of the terms' norm and rounded to the parameter's type."""

import pytest
import torch

from lm_engine_amd import layer_norm
from oracle.linear_attention_oracle import layer_norm_ref
from tests.helpers import rel_l2


pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0**-8, F32: 2.0**-24}
_ID = lambda x: str(x).split(".")[-1]  # noqa: E731

# every number of threads to a row, whole and cut rows, sizes that are no multiple of anything
SIZES = [(1, 1), (3, 2), (5, 8), (70, 33), (17, 64), (9, 100), (300, 128), (33, 200), (8, 256), (7, 257), (5000, 512), (4, 777), (130, 1024), (6, 1500),
         (600, 2048), (3, 2049), (9, 4096), (2, 5000), (5, 8192), (2, 9001), (3, 16384)]  # fmt: skip


def _rows(n, D, dtype, seed=0, mean=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, D, generator=gen) + mean * torch.randn(n, 1, generator=gen)).to(dtype)


def _check_rows(got, want, dtype):
    assert got.shape == want.shape and got.dtype == dtype
    scale = want.abs().amax(dim=-1, keepdim=True).clamp(min=1e-30)
    error = ((got.double().cpu() - want).abs() / scale).max().item()
    print(f"error {error:.2e}", flush=True)
    assert error <= HALF[dtype] + 2.0**-16, error


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("n, D", SIZES)
def test_forward(n, D, dtype):
    x = _rows(n, D, dtype)
    gen = torch.Generator().manual_seed(1)
    w, b = 1 + 0.1 * torch.randn(D, generator=gen), 0.1 * torch.randn(D, generator=gen)
    for weight, bias in [(None, None), (w, None), (w.to(BF16), b.to(BF16)), (w, b), (None, b)]:
        got = layer_norm(x.cuda(), *(None if p is None else p.cuda() for p in (weight, bias)), 1e-5)
        _check_rows(got, layer_norm_ref(x, weight, bias), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
@pytest.mark.parametrize("n, D", SIZES)
def test_backward(n, D, dtype):
    gen = torch.Generator().manual_seed(2)
    for w_dtype, with_bias in [(F32, True), (BF16, True), (BF16, False), (None, False)]:
        x = _rows(n, D, dtype, seed=3)
        dy = torch.randn(n, D, generator=gen).to(dtype)
        leaves = [x]
        if w_dtype is not None:
            leaves += [(1 + 0.1 * torch.randn(D, generator=gen)).to(w_dtype)] + ([(0.1 * torch.randn(D, generator=gen)).to(w_dtype)] if with_bias else [])
        ref = [t.double().requires_grad_() for t in leaves]
        want = torch.autograd.grad(layer_norm_ref(*ref), ref, dy.double())
        own = [t.cuda().requires_grad_() for t in leaves]
        got = torch.autograd.grad(layer_norm(*own), own, dy.cuda())
        if D > 2:  # (a row of one or two values has no gradient but through eps: both sides are noise around zero)
            error = rel_l2(got[0], want[0])
            assert got[0].dtype == dtype and error <= HALF[dtype] + 2.0**-16, error
        for g, r, t in zip(got[1:], want[1:], leaves[1:]):
            assert g.dtype == t.dtype
            error = ((g.double().cpu() - r).norm() / r.norm().clamp(min=1e-6)).item()
            assert D == 1 or error <= HALF[t.dtype] + 2.0**-16, error


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_ID)
def test_rows_as_they_lie(dtype):
    """Slices, odd offsets, rows of one tensor repeated, a leading shape; the result is contiguous."""
    base = _rows(40, 300, dtype).cuda()
    for x in (base[:, 8:264], base[:, 3:130], base[::2, :256], base[:1].expand(12, 300), base[:, ::2], base.view(4, 10, 300)[:, :, 16:272],
              base.view(4, 10, 300)[:, 2:7], base.t(), base.reshape(-1)[1 : 1 + 39 * 300].view(39, 300), base[7]):  # fmt: skip
        got = layer_norm(x)
        assert got.is_contiguous() and got.shape == x.shape
        _check_rows(got.reshape(-1, x.size(-1)), layer_norm_ref(x.cpu()).reshape(-1, x.size(-1)), dtype)
    leaf = base.detach().requires_grad_()
    part = leaf.view(4, 10, 300)[:, 1:9, 5:205]
    dy = torch.randn(4, 200, 8, device="cuda").to(dtype).transpose(1, 2)
    got = torch.autograd.grad(layer_norm(part), leaf, dy)[0]
    ref = base.cpu().double().requires_grad_()
    want = torch.autograd.grad(layer_norm_ref(ref.view(4, 10, 300)[:, 1:9, 5:205]), ref, dy.cpu().double())[0]
    assert rel_l2(got, want) <= HALF[dtype] + 2.0**-16


def test_rows_far_from_zero_and_constant_rows():
    """The squares are of what is left of the mean: a row at 1000 with a deviation of 1 keeps fp32's digits of x."""
    gen = torch.Generator().manual_seed(5)
    x = 1000 + torch.randn(20, 512, generator=gen)
    got = layer_norm(x.cuda())
    assert (got.cpu().double() - layer_norm_ref(x)).abs().max() <= 4 * 1000 * 2.0**-24 * 4  # fp32 steps of 1000, of x - mean and of the mean
    x = torch.full((3, 96), 7.0)
    assert torch.equal(layer_norm(x.cuda()).cpu(), torch.zeros_like(x))
    x[1, 5] = float("nan")
    y = layer_norm(x.cuda()).cpu()
    assert y[1].isnan().all() and (y[[0, 2]] == 0).all()


def test_no_rows():
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, w.detach().clone().requires_grad_())
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 64) and (dw == 0).all()
