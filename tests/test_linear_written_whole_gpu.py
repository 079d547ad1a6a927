"""Linear attention through its C entries (include/gdn_linear_hip.h) with results and workspaces full of NaN: what a call returns does not
depend on what its memory held, tokens of no sequence read as zeros where that is asked for, and are left alone where it is not."""

import ctypes

import pytest
import torch

from lm_engine_amd import _lib
from lm_engine_amd import linear as la
from oracle.linear_attention_oracle import sequences_of
from tests.test_linear_attention_gpu import BF16, F32, LAYOUTS, _cu, _cuda, _inputs


pytestmark = pytest.mark.gpu

NAN = float("nan")

# (lengths, left-padded, tokens of a row or of the packed row, H, HK, K, V): besides the small ones, sequences cut into segments, shared
# heads, more columns than a backward walk has keys
CASES = [(lens, padded, T, 3, 3, 64, 96) for lens, padded, T in LAYOUTS] + [
    ([40, 0, 333], False, 400, 4, 2, 64, 72),
    ([900, 1, 1500], False, 2500, 2, 2, 128, 128),
    ([700, 1300], True, 1300, 4, 2, 64, 264),
    ([300, 77], True, 300, 2, 1, 256, 64),
]


def _full(*shape, dtype):
    return torch.full(shape, NAN, dtype=dtype, device="cuda")


def _workspace(nbytes):
    # 4-byte pieces, which make NaN as fp32 and as bf16
    return torch.full((nbytes // 4,), -1, dtype=torch.int32, device="cuda") if nbytes else None


def _call(name, args):
    _lib.check_status(getattr(_lib.load_library(), name)(ctypes.byref(args), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), name)


def _outside(B, T, cu, padded):
    mask = torch.ones(B, T, dtype=torch.bool)
    for b, first, length in sequences_of(B, T, cu, padded):
        mask[b, first : first + length] = False
    return mask.cuda()


def _problem(case, dtype):
    lens, padded, T, H, HK, K, V = case
    B = len(lens) if padded else 1
    x = _cuda(_inputs(B, T, H, K, V, HK=HK, N=len(lens), dtype=dtype))
    return x, torch.tensor(_cu(lens), dtype=torch.int32).cuda(), (B, T, H, K, V, len(lens)), _outside(B, T, _cu(lens), padded)


def _forward(case, dtype, entry, flags):
    x, cu, dims, outside = _problem(case, dtype)
    B, T, H, K, V, N = dims
    a = la._fill(x["q"], x["k"], x["v"], x["g"], x["initial_state"], cu, None, case[1], dims)
    a.flags = (a.flags & ~_lib.GDN_FLAG_ZERO_PADDING) | flags
    o, ht = _full(B, T, H, V, dtype=dtype), _full(N, H, K, V, dtype=F32)
    la._set_rows(a, "o", o)
    a.ht = ht.data_ptr()
    a.workspace_bytes = _lib.load_library().gdn_linear_attn_workspace_bytes(ctypes.byref(a))
    workspace = _workspace(a.workspace_bytes)
    a.workspace = None if workspace is None else workspace.data_ptr()
    _call(entry, a)
    fn = la.chunk_linear_attention if entry == "gdn_linear_attn_chunk_fwd" else la.fused_recurrent_linear_attention
    want, want_state = fn(**x, output_final_state=True, cu_seqlens=cu, left_padded=case[1])
    return o, ht, want, want_state, outside


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("entry", ["gdn_linear_attn_chunk_fwd", "gdn_linear_attn_recurrent_fwd"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(case, entry, dtype):
    o, ht, want, want_state, outside = _forward(case, dtype, entry, _lib.GDN_FLAG_ZERO_PADDING)
    assert (o[outside] == 0).all() and torch.equal(o, want)
    assert ht.isfinite().all() and torch.equal(ht, want_state)
    o, ht, want, want_state, outside = _forward(case, dtype, entry, 0)
    assert o[outside].isnan().all() and torch.equal(o[~outside], want[~outside]) and torch.equal(ht, want_state)


@pytest.mark.parametrize("learned", [False, True], ids=["", "decay"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward(case, dtype, learned):
    x, cu, dims, outside = _problem(case, dtype)
    B, T, H, K, V, N = dims
    HK = case[4]
    gen = torch.Generator().manual_seed(5)
    do, dht = torch.randn(B, T, H, V, generator=gen).to(dtype).cuda(), torch.randn(N, H, K, V, generator=gen).cuda()
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "initial_state")]
    g = x["g"].detach().requires_grad_(learned)
    o, state = la.chunk_linear_attention(*leaves[:3], g, initial_state=leaves[3], output_final_state=True, cu_seqlens=cu, left_padded=case[1])
    want = torch.autograd.grad((o, state), leaves + [g] * learned, (do, dht))
    for zeros in (True, False):
        b = _lib.GdnLinearAttnBwdArgs()
        b.fwd = la._fill(x["q"], x["k"], x["v"], x["g"], x["initial_state"], cu, None, case[1], dims)
        if not zeros:
            b.fwd.flags &= ~_lib.GDN_FLAG_ZERO_PADDING
        dq, dk, dv = _full(B, T, HK, K, dtype=dtype), _full(B, T, HK, K, dtype=dtype), _full(B, T, H, V, dtype=dtype)
        dh0, dg = _full(N, H, K, V, dtype=F32), _full(H, dtype=F32)
        for name, t in (("dout", do), ("dq", dq), ("dk", dk), ("dv", dv)):
            la._set_rows(b, name, t)
        b.dht, b.dh0, b.dg = dht.data_ptr(), dh0.data_ptr(), dg.data_ptr() if learned else None
        b.workspace_bytes = _lib.load_library().gdn_linear_attn_bwd_workspace_bytes(ctypes.byref(b))
        workspace = _workspace(b.workspace_bytes)
        b.workspace = None if workspace is None else workspace.data_ptr()
        _call("gdn_linear_attn_bwd", b)
        for name, got, ref in zip(("dq", "dk", "dv"), (dq, dk, dv), want):
            assert torch.equal(got[~outside], ref[~outside]), name
            # (where heads are shared dq and dk are sums over all tokens: zeros either way)
            assert (got[outside] == 0).all() if zeros or (HK < H and name != "dv") else got[outside].isnan().all(), name
        assert dh0.isfinite().all() and torch.equal(dh0, want[3])
        assert torch.equal(dg, want[4]) if learned else dg.isnan().all()
