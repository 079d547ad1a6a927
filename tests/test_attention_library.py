"""The third part of the C ABI (include/gdn_attention_hip.h) and its Python side without a GPU: every declared symbol is there, the ctypes
mirrors have the header's layout, and bad arguments are refused before anything is launched."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import _lib
from lm_engine_amd.cache import PagedCache
from lm_engine_amd.kernels import Kernel
from oracle.attention_oracle import PagedCacheRef, exponent_of, norm_rotary_ref, to_e4m3, visible_keys, window_attention_ref


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gdn_attention_hip.h")
FAKE = 0x10000  # an address that is never read: what is refused is refused by the host


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(gdn_\w+)\(", text))
    assert declared == set(_lib.ATTENTION_SYMBOLS)
    lib = _lib.load_library()
    assert all(hasattr(lib, name) for name in declared)
    version = int(re.search(r"#define GDN_ATTENTION_ABI_VERSION (\d+)", text).group(1))
    assert lib.gdn_attention_abi_version() == version == _lib.GDN_ATTENTION_ABI_VERSION
    assert int(re.search(r"#define GDN_QK_ROTARY_MAX_D (\d+)", text).group(1)) == _lib.GDN_QK_ROTARY_MAX_D


STRUCTS = {"gdn_qk_rotary_args": _lib.GdnQkRotaryArgs, "gdn_qk_rotary_bwd_args": _lib.GdnQkRotaryBwdArgs, "gdn_window_attn_args": _lib.GdnWindowAttnArgs,
           "gdn_window_attn_bwd_args": _lib.GdnWindowAttnBwdArgs, "gdn_paged_cache": _lib.GdnPagedCache, "gdn_cache_write_args": _lib.GdnCacheWriteArgs,
           "gdn_cache_read_args": _lib.GdnCacheReadArgs, "gdn_cache_attn_args": _lib.GdnCacheAttnArgs}  # fmt: skip


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    source = tmp_path / "layout.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"gdn_attention_hip.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", f"-I{ROOT}/include", str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for mirror in STRUCTS.values():
        want += [ctypes.sizeof(mirror)] + [getattr(mirror, field).offset for field, _ in mirror._fields_]
    assert got == want


def _set(struct, over):
    for name, value in over.items():
        part, _, rest = name.partition("__")
        if rest.isdigit():
            getattr(struct, part)[int(rest)] = value
        elif rest:
            setattr(getattr(struct, part), rest, value)
        else:
            setattr(struct, name, value)
    return struct


def _window(**over):
    a = _lib.GdnWindowAttnArgs()
    a.q = a.k = a.v = a.o = a.lse = FAKE
    a.B, a.T, a.S, a.H, a.HK, a.D, a.N = 2, 40, 40, 4, 2, 64, 2
    a.window, a.sinks, a.dtype, a.scale = 16, 2, _lib.GDN_BF16, 0.125
    for n in "qkvo":
        heads = 4 if n in "qo" else 2
        setattr(a, f"{n}_stride_h", 64), setattr(a, f"{n}_stride_t", 64 * heads), setattr(a, f"{n}_stride_b", 40 * 64 * heads)
    return _set(a, over)


PADDED = _lib.GDN_FLAG_LEFT_PADDED
BAD_WINDOW = [
    (dict(q=None), -1), (dict(v=None), -1), (dict(o=None), -1), (dict(T=0), -2), (dict(S=0), -2), (dict(B=-1), -2), (dict(N=3), -2), (dict(HK=3), -2),
    (dict(HK=0), -2), (dict(window=-1), -2), (dict(sinks=-1), -2), (dict(D=60), -3), (dict(D=264), -3), (dict(dtype=7), -3), (dict(flags=1), -3),
    (dict(S=1 << 29), -3), (dict(T=1 << 29), -3), (dict(B=1 << 24, N=1 << 24, HK=4, T=2000), -3), (dict(q_stride_t=(1 << 23) + 8), -3), (dict(k_stride_t=-64), -3),
    (dict(v_stride_h=1 << 28), -3), (dict(q_stride_h=-64), -3), (dict(k=FAKE + 8), -4), (dict(q_stride_h=68), -4), (dict(v_stride_b=4), -4), (dict(o_stride_t=4), -4),
    (dict(lse=FAKE + 2), -4), (dict(cu_seqlens=FAKE), -6), (dict(cu_seqlens=FAKE, S=41, B=1), -2), (dict(flags=PADDED), -1), (dict(flags=PADDED, cu_seqlens=FAKE, N=3), -2),
    (dict(flags=PADDED, cu_seqlens=FAKE + 2), -4),
]  # fmt: skip


@pytest.mark.parametrize("over, status", BAD_WINDOW, ids=str)
def test_window_attention_rejects_bad_arguments_before_any_launch(over, status):
    lib = _lib.load_library()
    a = _window(**over)
    assert lib.gdn_window_attn_fwd(ctypes.byref(a), None) == status
    b = _lib.GdnWindowAttnBwdArgs()
    b.fwd = a
    assert lib.gdn_window_attn_bwd(ctypes.byref(b), None) == status
    if status in (-2, -3) and not any("stride" in n for n in over):
        assert lib.gdn_window_attn_workspace_bytes(ctypes.byref(a)) == lib.gdn_window_attn_bwd_workspace_bytes(ctypes.byref(b)) == 0


def test_window_attention_checks_workspaces_and_gradients():
    lib = _lib.load_library()
    assert lib.gdn_window_attn_fwd(None, None) == lib.gdn_window_attn_bwd(None, None) == -1
    assert lib.gdn_window_attn_workspace_bytes(None) == lib.gdn_window_attn_bwd_workspace_bytes(None) == 0
    few = dict(T=1, S=5000, window=0)  # one token over many keys: cut into parts
    need = lib.gdn_window_attn_workspace_bytes(ctypes.byref(_window(**few)))
    assert need > 0
    for over, status in ((dict(), -5), (dict(workspace=FAKE, workspace_bytes=need - 1), -5), (dict(workspace=FAKE + 8, workspace_bytes=need), -4)):
        assert lib.gdn_window_attn_fwd(ctypes.byref(_window(**few, **over)), None) == status

    def backward(**over):
        b = _lib.GdnWindowAttnBwdArgs()
        b.fwd = _window()
        b.dout = b.dq = b.dk = b.dv = b.workspace = FAKE
        for n in ("dout", "dq", "dk", "dv"):
            heads = 4 if n in ("dout", "dq") else 2
            setattr(b, f"{n}_stride_h", 64), setattr(b, f"{n}_stride_t", 64 * heads), setattr(b, f"{n}_stride_b", 40 * 64 * heads)
        b.workspace_bytes = lib.gdn_window_attn_bwd_workspace_bytes(ctypes.byref(b))
        assert b.workspace_bytes >= 2 * 40 * 4 * 4
        return lib.gdn_window_attn_bwd(ctypes.byref(_set(b, over)), None)

    for over, status in ((dict(fwd__lse=None), -1), (dict(dout=None), -1), (dict(dk=None), -1), (dict(dq=FAKE + 2), -4), (dict(dv_stride_t=12), -4),
                         (dict(dk_stride_h=1 << 28), -3), (dict(workspace=None), -5), (dict(workspace_bytes=64), -5), (dict(workspace=FAKE + 8), -4)):  # fmt: skip
        assert backward(**over) == status, over


def test_window_attention_backward_refuses_more_heads_to_one_than_it_takes_apart():
    lib = _lib.load_library()
    b = _lib.GdnWindowAttnBwdArgs()
    for heads, dtype, some in ((65280, _lib.GDN_BF16, True), (65281, _lib.GDN_BF16, False), (65281, _lib.GDN_F32, True)):
        b.fwd = _window(H=heads, HK=1, dtype=dtype)
        assert (lib.gdn_window_attn_bwd_workspace_bytes(ctypes.byref(b)) > 0) == some
        assert lib.gdn_window_attn_bwd(ctypes.byref(b), None) == (-1 if some else -3)  # (no gradients to write to, or refused before)


def test_qk_norm_rotary_rejects_bad_arguments_before_any_launch():
    lib = _lib.load_library()

    def args(**over):
        a = _lib.GdnQkRotaryArgs()
        for i, heads in enumerate((4, 2)):
            a.x[i] = a.y[i] = FAKE
            a.heads[i] = heads
            a.x_stride_h[i], a.x_stride_t[i], a.x_stride_b[i] = 64, 64 * heads, 640 * heads
        a.cos = a.sin = FAKE
        a.B, a.T, a.D, a.R, a.table_rows, a.dtype, a.w_dtype, a.eps = 2, 10, 64, 64, 100, _lib.GDN_BF16, _lib.GDN_F32, 1e-6
        return _set(a, over)

    def backward(a, **over):
        b = _lib.GdnQkRotaryBwdArgs()
        b.fwd = a
        for i in range(2):
            b.dy[i] = b.dx[i] = FAKE
            b.dy_stride_h[i], b.dy_stride_t[i], b.dy_stride_b[i] = 64, 64 * (4, 2)[i], 640 * (4, 2)[i]
        return lib.gdn_qk_norm_rotary_bwd(ctypes.byref(_set(b, over)), None)

    for over, status in ((dict(x__0=None), -1), (dict(cos=None), -1), (dict(T=0), -2), (dict(heads__1=0), -2), (dict(table_rows=0), -2), (dict(R=0), -2),
                         (dict(D=60), -3), (dict(D=520), -3), (dict(R=12), -3), (dict(R=72), -3), (dict(dtype=5), -3), (dict(w_dtype=5), -3),
                         (dict(B=1 << 20, T=1 << 20), -3), (dict(x__1=FAKE + 8), -4), (dict(x_stride_h__0=68), -4), (dict(weight__0=FAKE + 2), -4),
                         (dict(cos=FAKE + 4), -4), (dict(pos=FAKE + 2), -4)):  # fmt: skip
        a = args(**over)
        assert lib.gdn_qk_norm_rotary_fwd(ctypes.byref(a), None) == backward(a) == status, over
        if status in (-2, -3):
            assert lib.gdn_qk_rotary_partial_blocks(ctypes.byref(a)) == 0
    assert lib.gdn_qk_norm_rotary_fwd(None, None) == lib.gdn_qk_norm_rotary_bwd(None, None) == -1 and lib.gdn_qk_rotary_partial_blocks(None) == 0
    assert lib.gdn_qk_norm_rotary_fwd(ctypes.byref(args(y__1=None)), None) == -1 and lib.gdn_qk_norm_rotary_fwd(ctypes.byref(args(y__0=FAKE + 8)), None) == -4
    for over, status in ((dict(dy__0=None), -1), (dict(dx__1=None), -1), (dict(dx__0=FAKE + 4), -4), (dict(dy_stride_t__1=4), -4),
                         (dict(dweight_partial__0=FAKE + 2), -4), (dict(dweight_partial__0=FAKE, partial_blocks=10000), -5)):  # fmt: skip
        assert backward(args(), **over) == status, over


def _cache(**over):
    c = _lib.GdnPagedCache()
    c.k_codes = c.v_codes = c.k_scales = c.v_scales = c.table = FAKE
    c.pages, c.P, c.HK, c.D, c.N, c.table_pages, c.table_stride = 10, 64, 2, 64, 3, 4, 4
    return _set(c, over)


BAD_CACHE = [
    (dict(k_codes=None), -1), (dict(v_scales=None), -1), (dict(table=None), -1), (dict(pages=0), -2), (dict(N=0), -2), (dict(table_pages=0), -2), (dict(HK=0), -2),
    (dict(table_stride=-4), -2), (dict(P=24), -3), (dict(P=272), -3), (dict(D=24), -3), (dict(D=272), -3), (dict(HK=65536), -3), (dict(table_pages=1 << 26), -3),
    (dict(k_codes=FAKE + 8), -4), (dict(table=FAKE + 2), -4),
]  # fmt: skip


@pytest.mark.parametrize("over, status", BAD_CACHE, ids=str)
def test_every_cache_entry_checks_the_cache(over, status):
    lib = _lib.load_library()
    for args, entry in ((_lib.GdnCacheWriteArgs(), lib.gdn_cache_write), (_lib.GdnCacheReadArgs(), lib.gdn_cache_read), (_lib.GdnCacheAttnArgs(), lib.gdn_cache_attn)):
        args.cache = _cache(**over)
        if hasattr(args, "B"):
            args.B, args.T = 3, 5
        elif hasattr(args, "H"):
            args.H, args.T = max(args.cache.HK, 1) * 2, 1
        else:
            args.T = 5
        assert entry(ctypes.byref(args), None) == status
    if status in (-2, -3):
        assert lib.gdn_cache_attn_workspace_bytes(ctypes.byref(args)) == 0


def test_cache_entries_reject_bad_arguments_before_any_launch():
    lib = _lib.load_library()
    assert lib.gdn_cache_write(None, None) == lib.gdn_cache_read(None, None) == lib.gdn_cache_attn(None, None) == -1
    assert lib.gdn_cache_attn_workspace_bytes(None) == 0

    def write(**over):
        a = _lib.GdnCacheWriteArgs()
        a.cache = _cache()
        a.k = a.v = a.start = FAKE
        a.B, a.T, a.dtype = 3, 5, _lib.GDN_BF16
        for n in "kv":
            setattr(a, f"{n}_stride_h", 64), setattr(a, f"{n}_stride_t", 128), setattr(a, f"{n}_stride_b", 640)
        return lib.gdn_cache_write(ctypes.byref(_set(a, over)), None)

    for over, status in ((dict(B=0), -2), (dict(T=0), -2), (dict(B=2), -2), (dict(cu_seqlens=FAKE), -6), (dict(flags=PADDED), -1), (dict(flags=4096), -3),
                         (dict(dtype=9), -3), (dict(T=(1 << 30) + 1), -3), (dict(k=None), -1), (dict(v=FAKE + 8), -4), (dict(k_stride_t=4), -4), (dict(start=None), -1),
                         (dict(start=FAKE + 2), -4), (dict(cu_seqlens=FAKE + 2, flags=PADDED), -4)):  # fmt: skip
        assert write(**over) == status, over

    def read(**over):
        a = _lib.GdnCacheReadArgs()
        a.cache = _cache()
        a.k = a.v = a.lengths = FAKE
        a.T, a.dtype = 256, _lib.GDN_BF16
        return lib.gdn_cache_read(ctypes.byref(_set(a, over)), None)

    for over, status in ((dict(T=0), -2), (dict(T=257), -3), (dict(dtype=9), -3), (dict(k=None), -1), (dict(v=FAKE + 8), -4), (dict(lengths=None), -1),
                         (dict(lengths=FAKE + 2), -4)):  # fmt: skip
        assert read(**over) == status, over

    def attend(**over):
        a = _lib.GdnCacheAttnArgs()
        a.cache = _cache(N=1, table_pages=200)
        a.q = a.o = a.lengths = FAKE
        a.T, a.H, a.scale = 1, 4, 0.125
        for n in "qo":
            setattr(a, f"{n}_stride_h", 64), setattr(a, f"{n}_stride_t", 256), setattr(a, f"{n}_stride_b", 256)
        _set(a, over)
        need = lib.gdn_cache_attn_workspace_bytes(ctypes.byref(a))
        if "workspace" not in over:
            a.workspace, a.workspace_bytes = FAKE, need - 1 if need else 0
        return lib.gdn_cache_attn(ctypes.byref(a), None)

    for over, status in ((dict(T=0), -2), (dict(H=3), -2), (dict(window=-1), -2), (dict(sinks=-1), -2), (dict(T=1 << 30), -3), (dict(q=None), -1), (dict(o=FAKE + 8), -4),
                         (dict(q_stride_h=4), -4), (dict(lengths=None), -1), (dict(lengths=FAKE + 2), -4), (dict(), -5),
                         (dict(workspace=FAKE + 8, workspace_bytes=1 << 30), -4)):  # fmt: skip
        assert attend(**over) == status, over


def test_python_entry_points_validate_and_never_fall_back():
    q, k = torch.randn(2, 8, 4, 64), torch.randn(2, 8, 2, 64)
    swa = lm_engine_amd.sliding_window_attention
    for args, options, match in [
        ((q, k, k), {}, "GPU only"), ((q, k, k[:, :4]), {}, "shape of k"), ((q, k[:1], k[:1]), {}, "share B and D"), ((q, k[..., :32], k[..., :32]), {}, "share B and D"),
        ((q[:, :, :3], k, k), {}, "multiple of the heads"), ((q, k.bfloat16(), k.bfloat16()), {}, "share a dtype"), ((q.half(), k.half(), k.half()), {}, "bfloat16 or float32"),
        ((q[..., :60], k[..., :60], k[..., :60]), {}, "head dim"), ((q, k, k), dict(window=0), "window"), ((q, k, k), dict(sinks=-1), "sinks"),
        ((q, k, k), dict(left_padded=True), "prefix sums"), ((q, k, k), dict(cu_seqlens=torch.tensor([0, 16])), "batch dim"),
        ((q, k, k), dict(cu_seqlens=torch.zeros(3)), "integers"), ((q[:, :4], k, k), dict(cu_seqlens=torch.tensor([0, 4, 8]), left_padded=True), "same tokens"), ((q[0], k, k), {}, "tensors"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            swa(*args, **options)
    cos, sin = lm_engine_amd.rotary_table(20, 64, device="cpu")
    rotary = lm_engine_amd.qk_norm_rotary
    w = torch.ones(64)
    for args, match in [
        ((q, k, w, w, cos, sin), "GPU only"), ((q, k[:, :4], w, w, cos, sin), "share"), ((q, k, w[:32], w, cos, sin), "q_weight"), ((q, k, w, w.bfloat16(), cos, sin), "share a dtype"),
        ((q, k, w, w, cos, sin[:5]), "tables"), ((q, k, w, w, cos[:, :3], sin[:, :3]), "rotates?"), ((q, k, w, w, cos[:5], sin[:5]), "8 tokens"),
        ((q, k, w, w, cos, sin, torch.zeros(2, 8)), "positions"), ((q, k, w, w, cos, sin, torch.zeros(3, 8, dtype=torch.int32)), "positions"),
        ((q[..., :60], k[..., :60], None, None, cos, sin), "head dim"), ((q, k, w, w, cos.clone().requires_grad_(), sin), "constants"), ((q.half(), k.half(), w, w, cos, sin), "bfloat16 or float32"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            rotary(*args)
    cache = lm_engine_amd.new_paged_cache(6, 2, 64, device="cpu")
    assert [tuple(x.shape) for x in cache] == [(6, 2, 64, 64), (6, 2, 4, 64, 16), (6, 2), (6, 2)] and (cache.k_scale == 27).all() and (cache.v.float() == 0).all()
    table, start = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    write, read, attend = lm_engine_amd.write_paged_cache, lm_engine_amd.read_paged_cache, lm_engine_amd.paged_cache_attention
    for call, match in [
        (lambda: write(cache, k, k, table, start), "on the GPU"), (lambda: read(cache, table, start), "on the GPU"), (lambda: attend(q.bfloat16(), cache, table, start), "on the GPU"),
        (lambda: write(cache, k, k, table[0], start), "block_table"), (lambda: write(cache, k, k, table.float(), start), "block_table"), (lambda: write(cache, k, k, table, start[:1]), "start"),
        (lambda: read(cache, table, start.float()), "lengths"), (lambda: read(PagedCache(cache.k.float(), *cache[1:]), table, start), "float8"),
        (lambda: read(PagedCache(cache.k, cache.v[:, :1], *cache[2:]), table, start), "belong together"), (lambda: read(PagedCache(*cache[:3], cache.v_scale[:1]), table, start), "v_scale"),
        (lambda: attend(q, cache, table, start, window=0), "window"), (lambda: attend(q.requires_grad_(), cache, table, start), "inference"),
        (lambda: lm_engine_amd.new_paged_cache(0, 2, 64), "pages"), (lambda: lm_engine_amd.new_paged_cache(4, 2, 60), "head_dim"), (lambda: lm_engine_amd.new_paged_cache(4, 2, 64, 20), "page_size"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            call()


def test_kernel_flags_switch_the_operators_off():
    q = torch.randn(1, 8, 2, 64)
    cos, sin = lm_engine_amd.rotary_table(20, 64, device="cpu")
    cache, one = lm_engine_amd.new_paged_cache(1, 2, 64, device="cpu"), torch.zeros(1, dtype=torch.int32)
    with lm_engine_amd.kernels.enable_kernels([Kernel.gated_delta_rule], reset=True):
        for name, call in (("window_attention", lambda: lm_engine_amd.sliding_window_attention(q, q, q)), ("qk_norm_rotary", lambda: lm_engine_amd.qk_norm_rotary(q, q, None, None, cos, sin)),
                           ("paged_cache", lambda: lm_engine_amd.write_paged_cache(cache, q, q, one[None], one)), ("paged_cache", lambda: lm_engine_amd.read_paged_cache(cache, one[None], one)),
                           ("paged_cache", lambda: lm_engine_amd.paged_cache_attention(q.bfloat16(), cache, one[None], one))):  # fmt: skip
            with pytest.raises(RuntimeError, match=f"Kernel.{name} is disabled"):
                call()


def test_opaque_operators_have_shape_only_implementations():
    import lm_engine_amd._opaque  # noqa: F401

    meta = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    ops = torch.ops.lm_engine_amd
    q, k, w = meta(2, 9, 4, 64), meta(2, 9, 2, 64), meta(64)
    o, lse = ops.window_attention_forward(q, k, k, None, 5, 1, 0.125, False)
    assert o.shape == q.shape and lse.shape == q.shape[:3] and lse.dtype == torch.float32
    assert ops.window_attention_forward(q.float(), k.float(), k.float(), None, 5, 1, 0.125, False)[1].shape == (2, 9, 4, 2)
    assert [x.shape for x in ops.window_attention_backward(q, k, k, o, lse, None, o, 5, 1, 0.125, False)] == [q.shape, k.shape, k.shape]
    table = meta(20, 32, dtype=torch.float32)
    assert [x.shape for x in ops.qk_norm_rotary_forward(q, k, w, None, table, table, None, 1e-6)] == [q.shape, k.shape]
    assert [x.shape for x in ops.qk_norm_rotary_backward(q, k, w, None, table, table, None, 1e-6, q, k)] == [q.shape, k.shape, w.shape, (0,)]
    cache = [meta(6, 2, 64, 64, dtype=torch.float8_e4m3fn), meta(6, 2, 4, 64, 16, dtype=torch.float8_e4m3fn), meta(6, 2, dtype=torch.uint8), meta(6, 2, dtype=torch.uint8)]
    pages, lengths = meta(2, 3, dtype=torch.int32), meta(2, dtype=torch.int32)
    assert [x.shape for x in ops.paged_cache_read(*cache, pages, lengths, 70, torch.float32)] == [(2, 70, 2, 64)] * 2
    assert ops.paged_cache_attend(q, *cache, pages, lengths, 0, 0, 0.1).shape == q.shape
    assert ops.paged_cache_write_(*cache, k, k, pages, lengths, None, False) is None


def test_integers_that_32_bits_do_not_hold_stay_out_of_range():
    from lm_engine_amd._autograd import as_int32

    top, low = 2**31 - 1, -(2**31)
    x = torch.tensor([0, 5, -5, 2**31, 2**32 + 5, -(2**32) + 5, 2**63 - 1, -(2**63)])
    assert as_int32(x).tolist() == [0, 5, -5, top, top, low, top, low] and as_int32(x).dtype == torch.int32
    for dtype, values, want in ((torch.uint8, [0, 255], [0, 255]), (torch.int16, [-(2**15), 7], [-(2**15), 7]), (torch.uint16, [65535], [65535]),
                                (torch.uint32, [2**32 - 1, 3], [top, 3]), (torch.uint64, [2**64 - 1, 2**32, 3], [top, top, 3])):  # fmt: skip
        assert as_int32(torch.tensor(values, dtype=dtype)).tolist() == want
    every_other = torch.arange(10, dtype=torch.int32)[::2]
    assert as_int32(every_other).is_contiguous() and as_int32(every_other).tolist() == [0, 2, 4, 6, 8] and as_int32(None) is None


# ---- the oracle itself
def test_oracle_of_the_window():
    mask = visible_keys(3, 6, window=2, sinks=1)  # positions 3, 4, 5
    assert mask.int().tolist() == [[1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert visible_keys(3, 1).int().tolist() == [[0], [0], [1]]
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 7, h, 8, generator=gen, dtype=torch.float64) for h in (4, 2, 2))
    o = window_attention_ref(q, k, v)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True, enable_gqa=True).transpose(1, 2)
    assert torch.allclose(o, want, atol=1e-12)
    assert (window_attention_ref(q, k[:, :3], v[:, :3])[:, :4] == 0).all()  # in front of the first key
    v[:, 5] = float("nan")
    assert window_attention_ref(q, k, v, window=2)[:, :5].isfinite().all()


def test_oracle_of_the_rotation_keeps_norms_and_distances():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(1, 1, 1, 16, generator=gen, dtype=torch.float64)
    cos, sin = lm_engine_amd.rotary_table(50, 16, device="cpu")
    at = [norm_rotary_ref(x, None, cos.double(), sin.double(), torch.tensor([[p]])).flatten() for p in (3, 10, 23, 30)]
    assert torch.allclose(at[0].square().sum(), torch.tensor(16.0).double(), rtol=1e-5)
    assert torch.allclose(at[0] @ at[1], at[2] @ at[3], rtol=1e-5)


def test_oracle_of_the_codes():
    x = torch.tensor([0.0, -0.0, 448.0, 1e9, 2**-9, 2**-10, 2**-10 * 1.01, 3 * 2**-10, 17.0, 18.0, 19.0, -1.0625, float("inf"), float("nan")])
    want = [0, 0, 448, 448, 2**-9, 0, 2**-9, 2**-8, 16, 18, 20, -1.0, float("nan"), float("nan")]
    assert torch.equal(to_e4m3(x).nan_to_num(7), torch.tensor(want, dtype=torch.float64).nan_to_num(7))
    y = torch.randn(5000) * torch.exp(4 * torch.randn(5000))
    y = y.clamp(-448, 448)
    assert torch.equal(to_e4m3(y), y.to(torch.float8_e4m3fn).double())
    assert exponent_of(torch.tensor([448.0])) == 0 and exponent_of(torch.tensor([448.1])) == 1 and exponent_of(torch.tensor([0.0, float("inf")])) == -100
    ref = PagedCacheRef(1, 1, 1, 16)
    ref.write(torch.tensor([1.0]).view(1, 1, 1), torch.tensor([1.0]).view(1, 1, 1), [0], 0)
    ref.write(torch.tensor([400.0]).view(1, 1, 1), torch.tensor([2.0]).view(1, 1, 1), [0], 1)
    k, v = ref.read([0], 2)
    # (steps of 32 from 256 on: 400 lies between 384 = 12 * 32 and 416 = 13 * 32, and the even one is taken)
    assert k.flatten().tolist() == [1.0, 384.0] and v.flatten().tolist() == [1.0, 2.0]
