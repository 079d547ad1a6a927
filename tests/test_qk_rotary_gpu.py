"""The norm of every head and the rotation by position on the GPU, against the formulas in 64 bits.

Tolerances, relative-L2.  A bf16 result carries its own rounding, at most 2^-8 (half a step) of the value, rms 2^-8 / sqrt(3) = 2.3e-3 where
roundings are spread evenly; everything in front of it is fp32: 3e-3.  fp32: the sum of up to 512 squares, the root, the quotient and four
products and sums, each 2^-24 relative to its terms, whose sum may be smaller than they are: 2e-6.  The weights' gradients are fp32 sums over
rows of values of both signs (1e-5 of the root of the sum of squares), rounded to the weights' dtype."""

import pytest
import torch

from lm_engine_amd import qk_norm_rotary, rotary_table
from oracle.attention_oracle import norm_rotary_ref
from tests.helpers import rel_l2


pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TOLERANCE = {BF16: 3e-3, F32: 2e-6}
WEIGHT = {BF16: 3e-3, F32: 1e-5}


def check(name, got, want, tolerance):
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} {tuple(want.shape)}"
    error = rel_l2(got, want)
    print(f"{name} {error:.2e}", flush=True)
    assert torch.isfinite(got.float()).all() and error <= tolerance, f"{name}: relative-L2 {error:.3e} above {tolerance:.1e}"


# (B, T, H, HK, D, R, dtype, dtype of the weights or None)
CASES = [
    (1, 1, 1, 1, 64, 64, BF16, F32), (2, 7, 4, 2, 128, 128, BF16, F32), (3, 50, 16, 2, 128, 128, BF16, BF16), (1, 33, 2, 2, 256, 64, BF16, F32),
    (2, 9, 3, 1, 24, 24, BF16, F32), (2, 9, 3, 1, 24, 8, BF16, None), (1, 20, 5, 5, 80, 80, BF16, BF16), (1, 20, 2, 1, 200, 48, BF16, F32),
    (1, 5, 1, 1, 8, 8, BF16, F32), (1, 4, 2, 1, 512, 512, BF16, F32), (1, 4, 2, 1, 504, 504, BF16, F32), (2, 31, 4, 1, 96, 32, F32, F32),
    (1, 3, 2, 2, 512, 128, F32, BF16), (1, 700, 16, 2, 128, 128, F32, F32), (2, 2000, 32, 4, 128, 64, BF16, F32), (1, 3, 1, 1, 8, 8, F32, None),
]  # fmt: skip


@pytest.mark.parametrize("B, T, H, HK, D, R, dtype, w_dtype", CASES, ids=str)
def test_forward_and_gradients(B, T, H, HK, D, R, dtype, w_dtype):
    gen = torch.Generator().manual_seed(T + D)
    randn = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    q, k = (2 * randn(B, T, H, D)).to(dtype), (0.3 * randn(B, T, HK, D)).to(dtype)
    weights = [None if w_dtype is None else (1 + 0.3 * randn(D)).to(w_dtype) for _ in range(2)]
    cos, sin = rotary_table(T + 100, R, device="cpu")
    positions = torch.randint(0, T + 100, (B, T), generator=gen)
    leaves = [None if x is None else x.cuda().requires_grad_() for x in (q, k, *weights)]
    ref = [None if x is None else x.double().requires_grad_() for x in (q, k, *weights)]
    for given in (positions, None):
        at = torch.arange(T).expand(B, T) if given is None else given
        y = qk_norm_rotary(*leaves, cos.cuda(), sin.cuda(), positions=None if given is None else given.to(torch.int32).cuda())
        want = [norm_rotary_ref(x, w, cos, sin, at) for x, w in zip(ref[:2], ref[2:])]
        for name, a, b in zip(("q", "k"), y, want):
            check(name, a, b.detach(), TOLERANCE[dtype])
            assert a.dtype == dtype and a.is_contiguous()
        dy = [randn(*x.shape).to(dtype) for x in (q, k)]
        wanted = [i for i, x in enumerate(leaves) if x is not None]
        got = torch.autograd.grad(y, [leaves[i] for i in wanted], [d.cuda() for d in dy])
        expected = torch.autograd.grad(want, [ref[i] for i in wanted], [d.double() for d in dy])
        for i, a, b in zip(wanted, got, expected):
            check("d" + ("q", "k", "q_weight", "k_weight")[i], a, b, TOLERANCE[dtype] if i < 2 else WEIGHT[w_dtype])


def test_tables():
    cos, sin = rotary_table(70000, 128, base=500000.0)
    assert cos.shape == sin.shape == (70000, 64) and cos.dtype == F32
    p, i = 69999, 1
    angle = torch.tensor(p, dtype=torch.float64) * 500000.0 ** (-2 * i / 128)
    assert abs(cos[p, i].item() - angle.cos().item()) <= 2**-24 and abs(sin[p, i].item() - angle.sin().item()) <= 2**-24
    for bad in ((0, 64), (10, 0), (10, 7)):
        with pytest.raises(ValueError):
            rotary_table(*bad)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_as_they_lie(dtype):
    """Column blocks of a projection, heads in front of tokens, odd offsets, a broadcast head, far positions: the results of dense copies to the bit."""
    B, T, H, HK, D = 2, 40, 4, 2, 64
    base = torch.randn(B, T, (H + 2 * HK) * D + 8, device="cuda").to(dtype)
    cos, sin = rotary_table(5000, D)
    w = torch.rand(D, device="cuda") + 0.5
    positions = torch.randint(0, 5000, (B, 2 * T), device="cuda")[:, ::2]  # int64, every other one
    for first in (0, 8, 3):
        q, k, _ = base[..., first : first + (H + 2 * HK) * D].split([H * D, HK * D, HK * D], dim=-1)
        q, k = q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D))
        got = qk_norm_rotary(q, k, w, w, cos, sin, positions)
        want = qk_norm_rotary(q.contiguous(), k.contiguous(), w, w, cos, sin, positions.int().contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = k[:, :, :1].expand(B, T, HK, D)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    got, want = qk_norm_rotary(heads_first, one, w, None, cos, sin), qk_norm_rotary(q.contiguous(), one.contiguous(), w, None, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    line = torch.arange(T, device="cuda", dtype=torch.int32)  # [T], the same for all rows
    assert torch.equal(qk_norm_rotary(q, k, w, w, cos, sin, line)[0], qk_norm_rotary(q, k, w, w, cos, sin)[0])
    leaf = base.clone().requires_grad_()
    q, k, _ = leaf[..., : (H + 2 * HK) * D].split([H * D, HK * D, HK * D], dim=-1)
    y = qk_norm_rotary(q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D)), w, w, cos, sin)
    spread = torch.ones(1, 1, 1, 1, device="cuda", dtype=dtype)
    grad, = torch.autograd.grad(y, leaf, [spread.expand_as(x) for x in y])
    again, = torch.autograd.grad(qk_norm_rotary(q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D)), w, w, cos, sin), leaf, [torch.ones_like(x) for x in y])
    assert torch.equal(grad, again) and (grad[..., (H + HK) * D :] == 0).all()


def test_positions_and_rows_that_are_not_there():
    q = torch.randn(1, 6, 2, 64, device="cuda").to(BF16)
    k = torch.randn(1, 6, 1, 64, device="cuda").to(BF16)
    cos, sin = rotary_table(10, 32)
    positions = torch.tensor([[0, 9, 10, -1, 2**31 - 1, 5]], device="cuda", dtype=torch.int32)
    for y in qk_norm_rotary(q, k, None, None, cos, sin, positions):
        assert y[:, [0, 1, 5]].isfinite().all() and y[:, [2, 3, 4]].isnan().all()
    q[0, 1, 1, 3] = float("nan")  # a row's own affair
    y, _ = qk_norm_rotary(q, k, None, None, cos, sin)
    assert y[0, 1, 1].isnan().all() and y[0, 1, 0].isfinite().all() and y[0, [0, 2, 3, 4, 5]].isfinite().all()
    zeros = torch.zeros(1, 2, 1, 64, device="cuda", dtype=BF16, requires_grad=True)
    y, z = qk_norm_rotary(zeros, zeros, None, None, cos, sin)
    assert (y == 0).all() and torch.autograd.grad((y, z), zeros, (torch.ones_like(y), torch.ones_like(z)))[0].isfinite().all()
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        y, z = qk_norm_rotary(q, q, w, w, cos, sin)
        assert y.shape == z.shape == q.shape
        dq, dw = torch.autograd.grad((y, z), (q, w), (y, z))
        assert dq.shape == q.shape and (dw == 0).all()


def test_gradients_against_differences():
    """Central differences of the formula in 64 bits, 1e-5 wide (their own error is 1e-10 of the third derivatives), against the kernel's in fp32:
    1e-5 of the terms' size."""
    gen = torch.Generator().manual_seed(4)
    q, k, wq, wk = (torch.randn(*s, generator=gen) for s in ((1, 5, 2, 16), (1, 5, 1, 16), (16,), (16,)))
    dy = [torch.randn(x.shape, generator=gen) for x in (q, k)]
    cos, sin = rotary_table(5, 8, device="cpu")
    leaves = [x.cuda().requires_grad_() for x in (q, k, wq, wk)]
    got = torch.autograd.grad(qk_norm_rotary(*leaves, cos.cuda(), sin.cuda()), leaves, [d.cuda() for d in dy])
    at = torch.arange(5)[None]

    def loss(values):
        return sum((norm_rotary_ref(x, w, cos, sin, at) * d.double()).sum() for x, w, d in zip(values[:2], values[2:], dy))

    for i, x in enumerate((q, k, wq, wk)):
        d = torch.randn(x.shape, generator=gen).double()
        step = lambda e: loss([t.double() + (e * d if j == i else 0) for j, t in enumerate((q, k, wq, wk))])  # noqa: E731, B023
        want = ((step(1e-5) - step(-1e-5)) / 2e-5).item()
        own = got[i].double().cpu() * d
        assert abs(own.sum().item() - want) <= 1e-5 * own.abs().sum().item(), i
