"""The second part of the C ABI (include/gdn_linear_hip.h) and its Python side without a GPU: every declared symbol is there, the ctypes
mirrors have the header's layout, and bad arguments are refused before anything is launched."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import _lib
from lm_engine_amd.kernels import Kernel


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gdn_linear_hip.h")
FAKE = 0x10000  # an address that is never read: what is refused is refused by the host


def _code(text):
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def test_library_exports_every_declared_symbol():
    text = _code(open(HEADER).read())
    declared = set(re.findall(r"\b(gdn_\w+)\(", text))
    assert declared == set(_lib.LINEAR_SYMBOLS)
    lib = _lib.load_library()
    assert all(hasattr(lib, name) for name in declared)
    version = int(re.search(r"#define GDN_LINEAR_ABI_VERSION (\d+)", text).group(1))
    assert lib.gdn_linear_abi_version() == version == _lib.GDN_LINEAR_ABI_VERSION


STRUCTS = {"gdn_linear_attn_args": _lib.GdnLinearAttnArgs, "gdn_linear_attn_bwd_args": _lib.GdnLinearAttnBwdArgs,
           "gdn_layer_norm_args": _lib.GdnLayerNormArgs, "gdn_layer_norm_bwd_args": _lib.GdnLayerNormBwdArgs}  # fmt: skip


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    source = tmp_path / "layout.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"gdn_linear_hip.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", f"-I{ROOT}/include", str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for mirror in STRUCTS.values():
        want += [ctypes.sizeof(mirror)] + [getattr(mirror, field).offset for field, _ in mirror._fields_]
    assert got == want


def _attention(**over):
    a = _lib.GdnLinearAttnArgs()
    a.q = a.k = a.v = a.o = FAKE
    a.B, a.T, a.H, a.K, a.V, a.N = 2, 40, 4, 64, 96, 2
    a.dtype, a.scale = _lib.GDN_BF16, 0.125
    for n in "qkvo":
        width = a.V if n in "vo" else a.K
        setattr(a, f"{n}_stride_h", width), setattr(a, f"{n}_stride_t", 4 * width), setattr(a, f"{n}_stride_b", 160 * width)
    for name, value in over.items():
        setattr(a, name, value)
    return a


BAD = [
    (dict(q=None), -1), (dict(v=None), -1), (dict(T=0), -2), (dict(B=-1), -2), (dict(N=3), -2), (dict(qk_heads=3), -2), (dict(qk_heads=-1), -2),
    (dict(K=60), -3), (dict(K=264), -3), (dict(V=20), -3), (dict(dtype=7), -3), (dict(flags=1 << 20), -3), (dict(H=65536, qk_heads=0), -3),
    (dict(T=(1 << 30) + 1), -3), (dict(q_stride_t=(1 << 24) + 8), -3), (dict(v_stride_t=-(1 << 24) - 8), -3), (dict(k_stride_t=-8), -3),
    (dict(k=FAKE + 8), -4), (dict(q_stride_h=68), -4), (dict(v_stride_b=4), -4), (dict(h0=FAKE + 4), -4), (dict(g=FAKE + 2), -4),
    (dict(cu_seqlens=FAKE), -6), (dict(flags=_lib.GDN_FLAG_LEFT_PADDED), -1), (dict(flags=_lib.GDN_FLAG_LEFT_PADDED, cu_seqlens=FAKE, N=3), -2),
]  # fmt: skip


@pytest.mark.parametrize("over, status", BAD, ids=str)
def test_attention_rejects_bad_arguments_before_any_launch(over, status):
    lib = _lib.load_library()
    a = _attention(**over)
    assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(a), None) == status
    assert lib.gdn_linear_attn_recurrent_fwd(ctypes.byref(a), None) == status
    b = _lib.GdnLinearAttnBwdArgs()
    b.fwd = a
    assert lib.gdn_linear_attn_bwd(ctypes.byref(b), None) == status
    if status in (-2, -3) and not any("stride" in n for n in over):
        assert lib.gdn_linear_attn_workspace_bytes(ctypes.byref(a)) == lib.gdn_linear_attn_bwd_workspace_bytes(ctypes.byref(b)) == 0


def test_outputs_and_workspaces_are_checked_before_any_launch():
    lib = _lib.load_library()
    assert lib.gdn_linear_attn_chunk_fwd(None, None) == lib.gdn_linear_attn_recurrent_fwd(None, None) == lib.gdn_linear_attn_bwd(None, None) == -1
    for over, status in ((dict(o=None), -1), (dict(o=FAKE + 8), -4), (dict(o_stride_t=4), -4), (dict(o_stride_t=(1 << 24) + 8), -3), (dict(ht=FAKE + 4), -4)):
        assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(_attention(**over)), None) == status, over
        assert lib.gdn_linear_attn_recurrent_fwd(ctypes.byref(_attention(**over)), None) == status, over
    # whole sequences start from a state that the call must not overwrite; a few tokens update it in place
    assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(_attention(h0=FAKE, ht=FAKE)), None) == -3
    long = dict(B=1, N=1, T=30000)
    need = lib.gdn_linear_attn_workspace_bytes(ctypes.byref(_attention(**long)))
    assert need > 0
    assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(_attention(**long)), None) == -5
    assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(_attention(**long, workspace=FAKE, workspace_bytes=need - 1)), None) == -5
    assert lib.gdn_linear_attn_chunk_fwd(ctypes.byref(_attention(**long, workspace=FAKE + 8, workspace_bytes=need)), None) == -4

    def backward(**over):
        b = _lib.GdnLinearAttnBwdArgs()
        b.fwd = _attention(**long)
        b.dout = b.dq = b.dk = b.dv = FAKE
        b.dq_stride_h = b.dk_stride_h = 64
        b.dv_stride_h = b.dout_stride_h = 96
        b.dq_stride_t = b.dk_stride_t = 256
        b.dv_stride_t = b.dout_stride_t = 384
        for name, value in over.items():
            setattr(b, name, value)
        return lib.gdn_linear_attn_bwd(ctypes.byref(b), None)

    for over, status in ((dict(dout=None), -1), (dict(dk=None), -1), (dict(dq=FAKE + 2), -4), (dict(dv_stride_t=12), -4), (dict(dh0=FAKE + 4), -4),
                         (dict(dg=FAKE), -1), (dict(), -5), (dict(dv_stride_t=1 << 25), -3)):  # fmt: skip
        assert backward(**over) == status, over


def test_layer_norm_rejects_bad_arguments_before_any_launch():
    lib = _lib.load_library()

    def forward(**over):
        a = _lib.GdnLayerNormArgs()
        a.x = a.y = FAKE
        a.rows, a.D, a.x_stride, a.y_stride, a.dtype, a.w_dtype, a.eps = 8, 64, 64, 64, _lib.GDN_BF16, _lib.GDN_F32, 1e-5
        for name, value in over.items():
            setattr(a, name, value)
        return lib.gdn_layer_norm_fwd(ctypes.byref(a), None)

    for over, status in ((dict(x=None), -1), (dict(y=None), -1), (dict(rows=0), -2), (dict(D=0), -2), (dict(D=_lib.GDN_LAYER_NORM_MAX_D + 1), -3),
                         (dict(dtype=9), -3), (dict(w_dtype=9), -3), (dict(x=FAKE + 1), -4), (dict(weight=FAKE + 2), -4), (dict(bias=FAKE + 2), -4),
                         (dict(x_stride=-64), -2), (dict(y_stride=63), -2)):  # fmt: skip
        assert forward(**over) == status, over
    assert lib.gdn_layer_norm_fwd(None, None) == lib.gdn_layer_norm_bwd(None, None) == -1

    def backward(**over):
        a = _lib.GdnLayerNormBwdArgs()
        a.x = a.dy = a.dx = FAKE
        a.rows, a.D, a.x_stride, a.dy_stride, a.dx_stride, a.dtype, a.w_dtype, a.eps = 8, 64, 64, 64, 64, _lib.GDN_BF16, _lib.GDN_F32, 1e-5
        for name, value in over.items():
            setattr(a, name, value)
        return lib.gdn_layer_norm_bwd(ctypes.byref(a), None)

    for over, status in ((dict(dy=None), -1), (dict(dx=None), -1), (dict(dx=FAKE + 1), -4), (dict(dx_stride=32), -2), (dict(weight=FAKE + 2), -4),
                         (dict(dweight_partial=FAKE, partial_blocks=100000), -5), (dict(dbias_partial=FAKE + 2, partial_blocks=1), -4)):  # fmt: skip
        assert backward(**over) == status, over
    assert lib.gdn_layer_norm_partial_blocks(0, 64, _lib.GDN_BF16) == lib.gdn_layer_norm_partial_blocks(8, 64, 9) == 0
    assert lib.gdn_layer_norm_partial_blocks(8, 1 << 20, _lib.GDN_BF16) == 0


def test_python_entry_points_validate_and_never_fall_back():
    q = torch.randn(1, 8, 2, 64)
    with pytest.raises(ValueError, match="GPU only"):
        lm_engine_amd.chunk_linear_attention(q, q, q)
    with pytest.raises(ValueError, match="GPU only"):
        lm_engine_amd.fused_recurrent_linear_attention(q, q, q)
    with pytest.raises(ValueError, match="GPU only"):
        lm_engine_amd.linear_attention(q, q, q)
    with pytest.raises(ValueError, match="shape of q"):
        lm_engine_amd.chunk_linear_attention(q, q[..., :32], q)
    with pytest.raises(ValueError, match="share .B, T."):
        lm_engine_amd.chunk_linear_attention(q, q, q[:, :4])
    with pytest.raises(ValueError, match="multiple of the heads"):
        lm_engine_amd.chunk_linear_attention(q, q, q[:, :, :1])
    with pytest.raises(ValueError, match="head_first"):
        lm_engine_amd.chunk_linear_attention(q, q, q, head_first=True)
    with pytest.raises(ValueError, match="device tensor"):
        lm_engine_amd.layer_norm(q)


def test_kernel_flags_switch_the_operators_off():
    q = torch.randn(1, 8, 2, 64)
    with lm_engine_amd.kernels.enable_kernels([Kernel.gated_delta_rule], reset=True):
        with pytest.raises(RuntimeError, match="Kernel.linear_attention is disabled"):
            lm_engine_amd.chunk_linear_attention(q, q, q)
        with pytest.raises(RuntimeError, match="Kernel.layer_norm is disabled"):
            lm_engine_amd.layer_norm(q)


def test_opaque_operators_have_shape_only_implementations():
    meta = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    import lm_engine_amd._opaque  # noqa: F401

    ops = torch.ops.lm_engine_amd
    q, v, g = meta(2, 9, 2, 64), meta(2, 9, 4, 32), meta(4, dtype=torch.float32)
    o, state = ops.linear_attention_forward(q, q, v, g, None, None, "chunk", None, True, False)
    assert o.shape == v.shape and tuple(state.shape) == (2, 4, 64, 32) and state.dtype == torch.float32
    packed = ops.linear_attention_forward(q[:1], q[:1], v[:1], g, None, meta(4, dtype=torch.int32), "chunk", None, True, False)
    assert tuple(packed[1].shape) == (3, 4, 64, 32)
    grads = ops.linear_attention_backward(q, q, v, g, None, None, v, None, None, False, True)
    assert [x.shape for x in grads[:4]] == [q.shape, q.shape, v.shape, g.shape]
    x, w = meta(5, 7, 96), meta(96)
    assert ops.layer_norm_forward(x, w, w, 1e-5).shape == x.shape
    assert [t.shape for t in ops.layer_norm_backward(x, w, w, 1e-5, x)] == [x.shape, w.shape, w.shape]
