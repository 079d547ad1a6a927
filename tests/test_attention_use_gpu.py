"""Windowed attention, the norm and rotation in front of it and its paged cache as a user has them: rows as they lie, values that are not finite
in masked places, other streams, captured graphs, one graph of a compiler, the cache in place, and a run of them together.  Tolerances:
tests/test_window_attention_gpu.py, tests/test_paged_cache_gpu.py."""

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import (
    new_paged_cache,
    paged_cache_attention,
    qk_norm_rotary,
    read_paged_cache,
    rotary_table,
    sliding_window_attention,
    write_paged_cache,
)
from oracle.attention_oracle import attend, norm_rotary_ref, visible_keys, window_attention_ref
from tests.helpers import rel_l2
from tests.test_paged_cache_gpu import filled
from tests.test_window_attention_gpu import BF16, F32, GRAD, OUT, check, cu_of, inputs


pytestmark = pytest.mark.gpu


def cuda(*tensors):
    return [x.cuda() for x in tensors]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_as_they_lie(dtype):
    """Column blocks of one tensor, heads in front of tokens, odd offsets, broadcast heads, tokens far apart: the results of dense copies, to the
    bit, and gradients in the views' places."""
    B, T, H, HK, D = 2, 150, 4, 2, 64
    base = torch.randn(B, T, (H + 2 * HK) * D + 8, device="cuda").to(dtype)
    do = torch.randn(B, H, T, D, device="cuda").to(dtype).transpose(1, 2)
    options = dict(window=40, sinks=3)

    def views(x, first):
        q, k, v = x[..., first : first + (H + 2 * HK) * D].split([H * D, HK * D, HK * D], dim=-1)
        return q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D)), v.unflatten(-1, (HK, D))

    for first in (0, 8, 3):
        leaf = base.clone().requires_grad_()
        got = sliding_window_attention(*views(leaf, first), **options)
        dense = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for x in views(base, first)]
        want = sliding_window_attention(*dense, **options)
        assert torch.equal(got, want)
        own, = torch.autograd.grad(got, leaf, do)
        for x, y in zip(views(own, first), torch.autograd.grad(want, dense, do.contiguous())):
            assert torch.equal(x, y)
    q, k, v = (x.detach() for x in views(base, 0))
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(sliding_window_attention(*heads_first, **options), sliding_window_attention(q, k, v, **options))
    one = k[:1, :, :1].expand(B, T, HK, D)
    assert torch.equal(sliding_window_attention(q, one, one, **options), sliding_window_attention(q, one.contiguous(), one.contiguous(), **options))
    apart = torch.zeros(1, 3, (1 << 23) + 8, dtype=dtype, device="cuda")[..., : 2 * 64].view(1, 3, 2, 64)  # tokens beyond 32-bit offsets
    apart.copy_(torch.randn(1, 3, 2, 64))
    assert torch.equal(sliding_window_attention(apart, apart, apart), sliding_window_attention(*[apart.contiguous()] * 3))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_padding_holds_does_not_matter(dtype):
    q, k, v = inputs(3, 200, 4, 2, 64, dtype=dtype)
    packed = [x[:1] for x in inputs(1, 300, 4, 2, 64, dtype=dtype)]
    for tensors, cu, padded in (((q, k, v), cu_of([200, 0, 77]), True), (packed, [20, 60, 60, 281], False)):
        cu = torch.tensor(cu, dtype=torch.int32).cuda()
        results = []
        for dirty in (False, True):
            leaves, do = cuda(*tensors), torch.ones_like(tensors[0]).cuda()
            if dirty:
                for x in (*leaves, do):
                    if padded:
                        x[1], x[2, :123] = float("nan"), float("inf")
                    else:
                        x[:, :20], x[:, 281:] = float("nan"), float("-inf")
            leaves = [x.requires_grad_() for x in leaves]
            o = sliding_window_attention(*leaves, window=50, sinks=4, cu_seqlens=cu, left_padded=padded)
            results.append((o.detach(), *torch.autograd.grad(o, leaves, do)))
        for a, b in zip(*results):
            assert a.isfinite().all() and torch.equal(a, b)
            outside = torch.cat([a[1].flatten(), a[2, :123].flatten()]) if padded else torch.cat([a[:, :20].flatten(), a[:, 281:].flatten()])
            assert (outside == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T, S, window, sinks", [(300, 300, 60, 4), (300, 300, None, 0), (2, 2000, 500, 3), (700, 700, 64, 0)])
def test_values_that_are_not_finite_reach_those_who_see_them(dtype, T, S, window, sinks):
    """Element by element: what sees a NaN or an infinity has it, what does not is as without."""
    q, k, v = inputs(1, T, 4, 2, 64, S=S, dtype=dtype)
    clean = window_attention_ref(q, k, v, window=window, sinks=sinks)
    for at in (1, S // 2, S - 1):
        for value, head, d in ((float("nan"), 0, 5), (float("inf"), 1, 63), (-float("inf"), 0, 0)):
            dirty = v.clone()
            dirty[0, at, head, d] = value
            want = window_attention_ref(q, k, dirty, window=window, sinks=sinks)
            got = sliding_window_attention(*cuda(q, k, dirty), window=window, sinks=sinks).cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
            fine = want.isfinite()
            assert rel_l2(got[fine], clean[fine]) <= OUT[dtype]
        keys = k.clone()
        keys[0, at, 1] = float("nan")
        got = sliding_window_attention(*cuda(q, keys, v), window=window, sinks=sinks).cpu()
        sees = visible_keys(T, S, window, sinks)[:, at]
        assert got[0, sees][:, 2:].isnan().all() and got[0, ~sees].isfinite().all() and got[:, :, :2].isfinite().all()


def test_a_cache_page_that_held_something_else():
    """Codes behind a sequence's last token, NaN among them, and keys outside of the window; and NaN where it is seen."""
    lens = [100, 3, 64]
    cache, table, lengths, (k, v) = filled(lens, 2, 64, 32)
    q = torch.randn(3, 2, 4, 64).to(BF16).cuda()
    want = {w: paged_cache_attention(q, cache, table, lengths, window=w, sinks=s) for w, s in ((None, 0), (20, 5))}
    dirty = [x.clone() for x in cache]
    bytes_k, bytes_v = (dirty[i].view(torch.uint8) for i in range(2))
    for n, length in enumerate(lens):
        page, place = table[n, length // 32] if length % 32 else -1, length % 32
        if page >= 0:
            bytes_k[page, :, place:] = 0x7F
            for p in range(place, 32):
                bytes_v[page, :, p // 16, :, p % 16] = 0xFF
    for (w, s) in ((None, 0), (20, 5)):
        assert torch.equal(paged_cache_attention(q, type(cache)(*dirty), table, lengths, window=w, sinks=s), want[w])
    bytes_v[table[0, 1], 1, 0, 7, 3] = 0x7F  # token 35 of sequence 0, head 1, column 7
    o = paged_cache_attention(q, type(cache)(*dirty), table, lengths, window=20, sinks=5)
    assert torch.equal(o, want[20])
    o = paged_cache_attention(q, type(cache)(*dirty), table, lengths)
    assert o[0, :, 2:, 7].isnan().all() and o.isnan().sum() == 4
    bytes_v[table[0, 3], 0, 0, 9, 3] = 0x7F  # token 99, which the last query alone sees
    o = paged_cache_attention(q, type(cache)(*dirty), table, lengths, window=20, sinks=5)
    assert o[0, 1, :2, 9].isnan().all() and o.isnan().sum() == 2


def test_calls_give_the_same_bits_twice():
    q, k, v = cuda(*inputs(2, 900, 8, 2, 128))
    do = torch.randn_like(q)
    w = torch.rand(128, device="cuda")
    cos, sin = rotary_table(900, 128)
    results = []
    for _ in range(2):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, w)]
        a, b = qk_norm_rotary(leaves[0], leaves[1], leaves[3], leaves[3], cos, sin)
        results.append(torch.autograd.grad(sliding_window_attention(a, b, leaves[2], window=200, sinks=40), leaves, do))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_prefix_sums_out_of_range_are_clamped():
    """[0, 150, 150, 260] over 200 tokens: the last sequence ends where the tokens do.  What is not a prefix sum gives wrong results, not wild reads."""
    q, k, v = inputs(1, 200, 2, 2, 64)
    got = sliding_window_attention(*cuda(q, k, v), window=30, sinks=2, cu_seqlens=torch.tensor([0, 150, 150, 260], dtype=torch.int32).cuda())
    check("o", got, window_attention_ref(q, k, v, window=30, sinks=2, cu_seqlens=[0, 150, 150, 200]), OUT[BF16])
    for bad in ([0, 150, 120, 260], [500, 400, -7, 3], [-100, -50], [2**31 - 1, -(2**31), 100], [0, 0, 0]):
        leaves = [x.requires_grad_() for x in cuda(q, k, v)]
        o = sliding_window_attention(*leaves, window=30, sinks=2, cu_seqlens=torch.tensor(bad, dtype=torch.int32).cuda())
        grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
        assert o.isfinite().all() and all(g.shape == x.shape for g, x in zip(grads, leaves))
    lens = torch.tensor([0, 250, 200], dtype=torch.int32).cuda()  # lengths 250 (of 200) and -50
    two = [torch.cat([x, x]).cuda() for x in (q, k, v)]
    o = sliding_window_attention(*two, cu_seqlens=lens, left_padded=True)
    check("o", o[:1], window_attention_ref(q, k, v), OUT[BF16])
    assert (o[1] == 0).all()


def test_no_tokens():
    for shape_q, shape_k in (((0, 5, 2, 64), (0, 5, 2, 64)), ((2, 0, 2, 64), (2, 0, 2, 64)), ((2, 3, 2, 64), (2, 0, 2, 64)), ((2, 0, 2, 64), (2, 7, 1, 64))):
        for dtype in (BF16, F32):
            q = torch.ones(shape_q, device="cuda", dtype=dtype, requires_grad=True)
            k = torch.ones(shape_k, device="cuda", dtype=dtype, requires_grad=True)
            o = sliding_window_attention(q, k, k, window=3)
            dq, dk = torch.autograd.grad(o, (q, k), torch.ones_like(o))
            assert o.shape == q.shape and (o == 0).all() and (dq == 0).all() and (dk == 0).all() and dk.shape == k.shape
    cache = new_paged_cache(2, 1, 64)
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    empty = torch.zeros(0, 4, 1, 64, device="cuda")
    assert write_paged_cache(cache, empty, empty, none, none[:, 0]) is cache
    assert read_paged_cache(cache, none, none[:, 0])[0].shape == (0, 192, 1, 64)
    assert paged_cache_attention(empty.to(BF16), cache, none, none[:, 0]).shape == empty.shape
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    assert write_paged_cache(cache, empty.view(1, 0, 1, 64), empty.view(1, 0, 1, 64), one, one[0]) is cache
    assert read_paged_cache(cache, one, one[0], 0)[1].shape == (1, 0, 1, 64)
    assert (paged_cache_attention(torch.ones(1, 1, 2, 64, device="cuda", dtype=BF16), cache, one[:, :0], one[0]) == 0).all()


def test_refused_operands():
    q, k, v = cuda(*inputs(2, 10, 4, 2, 64))
    cos, sin = rotary_table(10, 64)
    cache, table, lengths, _ = filled([10, 20], 2, 64, 16)
    new = torch.zeros(2, 1, 2, 64, device="cuda", dtype=BF16)
    for call, match in [
        (lambda: sliding_window_attention(q, k, v.cpu()), "v is on"), (lambda: sliding_window_attention(q, k, v, cu_seqlens=torch.zeros(3, dtype=torch.int32), left_padded=True), "cu_seqlens is on"),
        (lambda: qk_norm_rotary(q, k, None, None, cos.cpu(), sin.cpu()), "cos is on"), (lambda: qk_norm_rotary(q, k, None, None, cos, sin, torch.zeros(2, 10, dtype=torch.int32)), "positions is on"),
        (lambda: write_paged_cache(cache, new, new.float(), table, lengths), "dtype"), (lambda: write_paged_cache(cache, new[:, :, :1], new[:, :, :1], table, lengths), "must be"),
        (lambda: write_paged_cache(cache, new, new, table[:1], lengths[:1]), "rows"), (lambda: write_paged_cache(cache, new, new, table.cpu(), lengths), "block_table is on"),
        (lambda: write_paged_cache(cache, new, new, table, lengths, cu_seqlens=lengths), "cu_seqlens"), (lambda: write_paged_cache(cache, new, new, table, lengths, left_padded=True), "prefix sums"),
        (lambda: write_paged_cache(cache._replace(k=cache.k.transpose(0, 1).contiguous().transpose(0, 1)), new, new, table, lengths), "contiguous"),
        (lambda: read_paged_cache(cache, table, lengths, 1000), "max_tokens"), (lambda: read_paged_cache(cache, table, lengths, dtype=torch.float16), "bfloat16 or float32"),
        (lambda: paged_cache_attention(q.float(), cache, table, lengths), "bfloat16"), (lambda: paged_cache_attention(q[:, :, :3], cache, table, lengths), "must be"),
        (lambda: paged_cache_attention(q[:1], cache, table, lengths), "must be"), (lambda: paged_cache_attention(q.cpu(), cache, table, lengths), "q is on"),
    ]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            call()
    leaf = q.clone().requires_grad_()
    for o in (sliding_window_attention(leaf, k, v), qk_norm_rotary(leaf, k, None, None, cos, sin)[0]):
        dq, = torch.autograd.grad(o.float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):  # a gradient is not itself differentiated
            torch.autograd.grad(dq.float().sum(), leaf)
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: sliding_window_attention(dual, k, v), lambda: qk_norm_rotary(dual, k, None, None, cos, sin), lambda: paged_cache_attention(dual[:, :1], cache, table, lengths)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()
    o = sliding_window_attention(leaf, k, v)
    with lm_engine_amd.kernels.enable_kernels([], reset=True), pytest.raises(RuntimeError, match="disabled"):
        torch.autograd.grad(o, leaf, torch.ones_like(o))


def test_gradients_against_differences():
    """Central differences of the formula in 64 bits, 1e-5 wide, against the kernels' gradients in fp32: 1e-5 of the terms' size and the differences'
    own 1e-9."""
    q, k, v = inputs(1, 40, 4, 2, 16, dtype=F32)
    gen = torch.Generator().manual_seed(8)
    do = torch.randn(q.shape, generator=gen)
    options = dict(window=9, sinks=2)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(sliding_window_attention(*leaves, **options), leaves, do.cuda())
    for i, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, generator=gen).double()
        step = lambda e: (window_attention_ref(*[t.double() + (e * d if j == i else 0) for j, t in enumerate((q, k, v))], **options) * do.double()).sum()  # noqa: E731, B023
        want = ((step(1e-5) - step(-1e-5)) / 2e-5).item()
        own = got[i].double().cpu() * d
        assert abs(own.sum().item() - want) <= 1e-5 * own.abs().sum().item(), i


def test_only_the_gradients_that_are_asked_for():
    tensors = cuda(*inputs(1, 200, 4, 2, 64))
    do = torch.randn_like(tensors[0])
    leaves = [x.clone().requires_grad_() for x in tensors]
    want = torch.autograd.grad(sliding_window_attention(*leaves, window=50), leaves, do)
    for i in range(3):
        part = [x.clone().requires_grad_(i == j) for j, x in enumerate(tensors)]
        got, = torch.autograd.grad(sliding_window_attention(*part, window=50), part[i], do)
        assert torch.equal(got, want[i])
    spread = torch.autograd.grad(sliding_window_attention(*leaves), leaves, torch.ones(1, 1, 1, 1, device="cuda", dtype=BF16).expand_as(do))
    assert all(torch.equal(a, b) for a, b in zip(spread, torch.autograd.grad(sliding_window_attention(*leaves), leaves, torch.ones_like(do))))
    shared = tensors[1].clone().requires_grad_()  # one tensor as keys and values
    both, = torch.autograd.grad(sliding_window_attention(tensors[0], shared, shared, window=50), shared, do)
    apart = [tensors[1].clone().requires_grad_() for _ in range(2)]
    dk, dv = torch.autograd.grad(sliding_window_attention(tensors[0], *apart, window=50), apart, do)
    assert torch.equal(both, dk + dv)


def test_another_stream_and_two_calls_at_once():
    sets = [cuda(*inputs(1, 1200, 8, 2, 128, seed=s)) for s in range(2)]
    cos, sin = rotary_table(1200, 128)
    caches = [filled([900, 30], 2, 128, 64, seed=s)[:3] for s in range(2)]
    few = [x[:, :2, :4].expand(2, 2, 4, 128).contiguous() for x, _, _ in sets]

    def call(i, q, k, v, few):
        a, b = qk_norm_rotary(q, k, None, None, cos, sin)
        cache, table, lengths = caches[i]
        return a, b, sliding_window_attention(a, b, v, window=300, sinks=4), sliding_window_attention(a[:, :1], b, v), paged_cache_attention(few, cache, table, lengths)

    want = [call(i, *s, f) for i, (s, f) in enumerate(zip(sets, few))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                busy = torch.randn(2048, 2048, device="cuda") @ torch.randn(2048, 2048, device="cuda")  # noqa: F841
                got.append(call(i, *[x + 0 for x in sets[i]], few[i] + 0))  # made on this stream, behind the product
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def _capture(fn):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_serving_steps_replay():
    """One decode step - norm and rotation, the token into the cache, attention over it, lengths that move on - and a prompt's attention in parts."""
    H, HK, D, N = 4, 2, 64, 3
    cos, sin = rotary_table(600, D)
    cache, table, lengths, _ = filled([500, 70, 1], HK, D, 32)
    room = torch.cat([table, table.new_full((N, 3), -1)], dim=1)
    room[0, 16], room[1, 3], room[2, 1] = 0, 0, 0  # (behind what these steps reach)
    qkv = torch.randn(N, 1, (H + 2 * HK) * D, device="cuda").to(BF16)
    long = cuda(*inputs(1, 2, H, HK, D, S=1500))

    def run():
        q, k, v = qkv.split([H * D, HK * D, HK * D], dim=-1)
        q, k = qk_norm_rotary(q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D)), None, None, cos, sin, lengths[:, None])
        write_paged_cache(cache, k, v.unflatten(-1, (HK, D)), room, lengths)
        o = paged_cache_attention(q, cache, room, lengths + 1, window=300, sinks=4)
        lengths.add_(1)
        return o, sliding_window_attention(*long)

    first = [x.clone() for x in (*cache, lengths)]

    def restore():
        for x, y in zip((*cache, lengths), first):
            x.view(torch.uint8).copy_(y.view(torch.uint8)) if x.dtype != torch.int32 else x.copy_(y)

    graph, out = _capture(run)
    other, out2 = _capture(lambda: sliding_window_attention(*long))  # a second graph of the same call
    for replay in range(4):
        qkv.normal_()
        long[0].normal_()
        restore()
        graph.replay()
        torch.cuda.synchronize()
        got, after = [x.clone() for x in out], [x.clone() for x in (*cache, lengths)]
        restore()
        other.replay()
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(out2, want[1]), replay
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(after, (*cache, lengths))), replay


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_training_step_replays(dtype):
    tensors = cuda(*inputs(1, 500, 4, 2, 64, dtype=dtype))
    do, w = torch.randn_like(tensors[0]), torch.rand(64, device="cuda")
    cos, sin = rotary_table(500, 64)

    def run():
        q, k, v, wq = [x.detach().requires_grad_() for x in (*tensors, w)]
        a, b = qk_norm_rotary(q, k, wq, wq, cos, sin)
        return torch.autograd.grad(sliding_window_attention(a, b, v, window=100, sinks=4), (q, k, v, wq), do)

    graph, out = _capture(run)
    for replay in range(4):
        for x in tensors:
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for i, (a, b) in enumerate(zip(got, run())):
            assert torch.equal(a, b), (replay, i)


def test_one_graph_of_the_compiler():
    tensors = cuda(*inputs(2, 130, 4, 2, 64))
    w = torch.rand(64, device="cuda")
    cos, sin = rotary_table(130, 64)

    def loss(q, k, v, weight):
        a, b = qk_norm_rotary(q, k, weight, None, cos, sin)
        return sliding_window_attention(a, b, v, window=40, sinks=2).float().square().sum()

    eager, compiled = ([x.detach().clone().requires_grad_() for x in (*tensors, w)] for _ in range(2))
    loss(*eager).backward()
    torch.compile(loss, backend="aot_eager", fullgraph=True)(*compiled).backward()
    for a, b in zip(eager, compiled):
        assert b.grad is not None and torch.equal(a.grad, b.grad)

    def step(q, k, v, cache, table, lengths):
        write_paged_cache(cache, k, v, table, lengths)
        return paged_cache_attention(q, cache, table, lengths + 1, window=30), *read_paged_cache(cache, table, lengths + 1, 20)

    q, k, v = (x[:, :1] for x in tensors)
    results = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        cache, table, lengths, _ = filled([40, 9], 2, 64, 64)
        with torch.no_grad():
            results.append((*fn(q, k, v, cache, table, lengths), *cache))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*results))


def test_a_written_cache_counts_as_written():
    cache, table, lengths, _ = filled([10], 1, 64, 16)
    before = [x._version for x in cache]
    k = torch.zeros(1, 1, 1, 64, device="cuda", dtype=BF16)
    write_paged_cache(cache, k, k, table, lengths)
    assert all(x._version > b for x, b in zip(cache, before))
    with torch.inference_mode():  # (tensors without a version)
        held = new_paged_cache(1, 1, 64, page_size=16)
        write_paged_cache(held, k, k, table * 0, lengths)


def test_a_run_of_them_together():
    """A mixer's middle: norm and rotation of a projection's columns, attention over a prompt and its keys and values into the cache; then
    single tokens over the cache.  Against the same in 64 bits: queries and keys carry a rounding each (2^-8 / sqrt(3) rms), the attention its 5e-3,
    and the cache's codes 2^-4 / sqrt(3) of each key and value (e4m3: half a step is 2^-4) where it is read: scores of keys of norm sqrt(D) change by
    2^-4 / sqrt(3) |q . k| / D^(1/2) spread over D terms, a few hundredths, and values average over the keys seen: 4e-2 of the output's norm.
    With the gradients through both: 3 roundings more, 2e-2."""
    B, T, H, HK, D, window, sinks = 2, 333, 4, 2, 64, 100, 4
    gen = torch.Generator().manual_seed(21)
    qkv = torch.randn(B, T, (H + 2 * HK) * D, generator=gen).to(BF16)
    wq, wk = 1 + 0.1 * torch.randn(D, generator=gen), 1 + 0.1 * torch.randn(D, generator=gen)
    do = torch.randn(B, T, H, D, generator=gen).to(BF16)
    cos, sin = rotary_table(T, D)

    def split(x):
        q, k, v = x.split([H * D, HK * D, HK * D], dim=-1)
        return q.unflatten(-1, (H, D)), k.unflatten(-1, (HK, D)), v.unflatten(-1, (HK, D))

    ref = [x.double().requires_grad_() for x in (qkv, wq, wk)]
    q, k, v = split(ref[0])
    at = torch.arange(T).expand(B, T)
    want = window_attention_ref(norm_rotary_ref(q, ref[1], cos.cpu(), sin.cpu(), at), norm_rotary_ref(k, ref[2], cos.cpu(), sin.cpu(), at), v, window=window, sinks=sinks)
    leaves = [x.cuda().requires_grad_() for x in (qkv, wq, wk)]
    q, k, v = split(leaves[0])
    a, b = qk_norm_rotary(q, k, leaves[1], leaves[2], cos, sin)
    got = sliding_window_attention(a, b, v, window=window, sinks=sinks)
    check("o", got, want.detach(), 1.2e-2)
    for name, x, y in zip(("qkv", "wq", "wk"), torch.autograd.grad(got, leaves, do.cuda()), torch.autograd.grad(want, ref, do.double())):
        check("d" + name, x, y, 2e-2)

    prompt = 300
    with torch.no_grad():
        cache = new_paged_cache(B * 6 + 1, HK, D)
        table = torch.arange(B * 6, dtype=torch.int32, device="cuda").view(B, 6).flip(0).contiguous()
        lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        write_paged_cache(cache, b[:, :prompt], v[:, :prompt], table, lengths)
        lengths += prompt
        outs = []
        for t in range(prompt, T):
            q1, k1, v1 = split(leaves[0][:, t : t + 1])
            q1, k1 = qk_norm_rotary(q1, k1, leaves[1], leaves[2], cos, sin, lengths[:, None])
            write_paged_cache(cache, k1, v1, table, lengths)
            lengths += 1
            outs.append(paged_cache_attention(q1, cache, table, lengths, window=window, sinks=sinks))
        out = torch.cat(outs, dim=1)
        check("single tokens", out, want.detach()[:, prompt:], 4e-2)
        # what the codes stand for, read back: the attention itself is as exact as over bf16
        held_k, held_v = read_paged_cache(cache, table, lengths, T)
        exact = torch.stack([attend(a[n, prompt:].double().cpu(), held_k[n].double().cpu(), held_v[n].double().cpu(), visible_keys(T - prompt, T, window, sinks), D**-0.5) for n in range(B)])
        check("single tokens, on the codes' values", out, exact, 1e-2)
        drafts = paged_cache_attention(a[:, prompt:].contiguous(), cache, table, lengths, window=window, sinks=sinks)  # the same tokens at once
        check("drafts", drafts, exact, OUT[BF16])


def test_lengths_out_of_range():
    """Below zero: no key is seen.  Past the table: what the table has."""
    cache, table, lengths, _ = filled([70, 70, 70, 70], 2, 64, 16)
    q = torch.randn(4, 3, 4, 64).to(BF16).cuda()
    odd = torch.tensor([-(2**31), -1, 2**31 - 1, 70], dtype=torch.int32).cuda()
    for window, sinks in ((None, 0), (20, 4)):
        o = paged_cache_attention(q, cache, table, odd, window=window, sinks=sinks)
        assert (o[:2] == 0).all() and o.isfinite().all()
        at_end = torch.tensor([0, 0, table.size(1) * 16, 70], dtype=torch.int32).cuda()
        assert torch.equal(o, paged_cache_attention(q, cache, table, at_end, window=window, sinks=sinks))
    k, _ = read_paged_cache(cache, table, odd, 70)
    assert (k[:2] == 0).all() and torch.equal(k[2:], read_paged_cache(cache, table, lengths, 70)[0][2:])


def test_a_cache_past_32_bits():
    """Pages of 512 KB, the last ones beyond 4 GB of codes: as in a small cache."""
    HK, P, D, pages = 8, 256, 256, 8300
    gen = torch.Generator("cuda").manual_seed(4)
    k, v = (torch.randn(1, 700, HK, D, device="cuda", generator=gen).to(BF16) for _ in range(2))
    q = torch.randn(1, 2, 16, D, device="cuda", generator=gen).to(BF16)
    results = []
    for total, table in ((4, [[1, 3, 0]]), (pages, [[8298, 8299, 8200]])):
        cache = new_paged_cache(total, HK, D, page_size=P)
        table = torch.tensor(table, dtype=torch.int32).cuda()
        start = torch.zeros(1, dtype=torch.int32, device="cuda")
        write_paged_cache(cache, k[:, :699], v[:, :699], table, start)
        write_paged_cache(cache, k[:, 699:], v[:, 699:], table, start + 699)
        results.append((paged_cache_attention(q, cache, table, start + 700), *read_paged_cache(cache, table, start + 700, 700)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_rows_past_32_bits():
    """Tensors of more than 2^31 elements: the last tokens as in a call that has only them and what they see."""
    T, H, HK, D, window = 140000, 64, 8, 256, 64
    q, k, v, do = (torch.empty(1, T, h, D, dtype=BF16, device="cuda").normal_() for h in (H, HK, HK, H))
    assert q.numel() > 2**31
    few = 256
    tail = [x[:, T - few :].clone().requires_grad_() for x in (q, k, v)]
    want = sliding_window_attention(*tail, window=window)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = sliding_window_attention(*leaves, window=window)
    assert rel_l2(o[:, T - few + window :].detach().cpu(), want[:, window:].detach().cpu()) <= 2 * OUT[BF16]
    do[:, : T - few + window] = 0  # (so that both have the same gradients of the last keys and queries)
    got = torch.autograd.grad(o, leaves, do)
    expected = torch.autograd.grad(want, tail, do[:, T - few :].clone())
    for name, a, b in zip(("dq", "dk", "dv"), got, expected):
        check(name, a[:, T - few :].cpu(), b.cpu(), 2 * 1e-2)
        assert (a[:, : T - few] == 0).all()
    with torch.no_grad():
        cos, sin = rotary_table(T, D)
        a, b = qk_norm_rotary(q, k, None, None, cos, sin)
        at = torch.arange(T - 100, T, dtype=torch.int32, device="cuda")
        c, d = qk_norm_rotary(q[:, T - 100 :], k[:, T - 100 :], None, None, cos, sin, at)
        assert torch.equal(a[:, T - 100 :], c) and torch.equal(b[:, T - 100 :], d)


@pytest.mark.parametrize("dtype, T, S, H, HK, window", [
    (BF16, 1, 50, 4, 2, None), (BF16, 1, 700, 2, 2, None), (BF16, 1, 700, 4, 2, 333), (BF16, 129, 129, 2, 2, None), (BF16, 257, 257, 1, 1, 70), (BF16, 33, 33, 128, 1, None),
    (F32, 1, 50, 4, 2, None), (F32, 1, 700, 2, 2, None), (F32, 40, 40, 16, 1, None), (F32, 40, 40, 16, 1, 21), (F32, 17, 17, 2, 2, None),
], ids=str)  # fmt: skip
def test_values_that_are_not_finite_in_the_last_keys_of_rows_at_one_position(dtype, T, S, H, HK, window):
    """Blocks whose rows all stand at the last key's position: their last tile of keys ends with what they see, and is not whole."""
    q, k, v = inputs(1, T, H, HK, 64, S=S, dtype=dtype)
    for at in {S - 1, S - 2, (S - 1) // 16 * 16, (S - 1) // 64 * 64, S // 2}:
        for value, d in ((float("nan"), 3), (float("inf"), 63), (-float("inf"), 0)):
            dirty = v.clone()
            dirty[0, at, HK - 1, d] = value
            want = window_attention_ref(q, k, dirty, window=window)
            got = sliding_window_attention(*cuda(q, k, dirty), window=window).cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()), (at, value)
            fine = want.isfinite()
            assert rel_l2(got[fine], want[fine]) <= OUT[dtype], (at, value)


# (T, H, HK, D, elements between tokens, between heads): each within what is read as it lies
@pytest.mark.parametrize("T, H, HK, D, apart, heads_apart", [
    (384, 1, 1, 128, 1 << 23, 128), (511, 1, 1, 72, (1 << 22) + (1 << 17), 128), (384, 2, 1, 128, 1 << 23, (1 << 27) - 1024), (300, 1, 1, 64, 1 << 23, 64),
    (384, 2, 1, 64, 1 << 23, (1 << 27) - 1024), (300, 2, 1, 256, 1 << 23, (1 << 27) - 1024), (300, 3, 1, 128, 1 << 23, 89478480),
])  # fmt: skip
def test_gradients_of_first_keys_from_tokens_that_lie_far_apart(T, H, HK, D, apart, heads_apart):
    """Queries and their gradients 2^23 elements apart, of more rows than one tile has: the results of dense copies, to the bit."""
    buffer = torch.empty(T * apart + H * heads_apart + 1024, dtype=BF16, device="cuda")
    q, k, v = cuda(*inputs(1, T, H, HK, D))
    do = torch.randn(1, T, H, D, device="cuda").to(BF16)
    far_q, far_do = (buffer[first:].as_strided((1, T, H, D), (T * apart, apart, heads_apart, 1)) for first in (0, 512))
    far_q.copy_(q), far_do.copy_(do)
    grads = []
    for x, d in ((far_q, far_do), (q, do)):
        leaves = [y.detach().requires_grad_() for y in (x, k, v)]
        grads.append(torch.autograd.grad(sliding_window_attention(*leaves, window=8, sinks=4), leaves, d))
    for name, a, b in zip(("dq", "dk", "dv"), *grads):
        assert torch.equal(a, b), name


def test_as_many_heads_to_one_as_a_division_by_multiplication_holds():
    """Rows are taken apart into tokens and heads by a product with 2^32 / H rounded up, which from 65537 heads on gives a token's last ones the next token."""
    T, H, D = 3, 65280, 8
    more = torch.zeros(1, 2, 65537, D, device="cuda", dtype=BF16, requires_grad=True)
    o = sliding_window_attention(more, *cuda(*inputs(1, 2, 1, 1, D))[1:])
    with pytest.raises(ValueError, match="not supported"):
        torch.autograd.grad(o, more, torch.ones_like(o))
    q, k, v = cuda(*inputs(1, T, H, 1, D))
    do = torch.zeros(1, T, H, D, device="cuda", dtype=BF16)
    do[:, :, -1] = 1
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(sliding_window_attention(*leaves), leaves, do)
    ref = [x.detach().double().requires_grad_() for x in leaves]
    scores = (ref[0][0].transpose(0, 1) @ ref[1][0, :, 0].T) * D**-0.5
    weights = scores.masked_fill(torch.ones(T, T, device="cuda").triu(1) > 0, -torch.inf).softmax(-1)
    want = torch.autograd.grad((weights @ ref[2][0, :, 0]).transpose(0, 1)[None], ref, do.double())
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        check(name, a.cpu(), b.cpu(), GRAD[BF16])


def test_tables_that_want_a_gradient_are_refused():
    q, k = cuda(*inputs(1, 6, 2, 1, 64))[:2]
    cos, sin = rotary_table(6, 64)
    for tables in ((cos.clone().requires_grad_(), sin), (cos, sin.clone().requires_grad_())):
        for leaf in (q, q.clone().requires_grad_()):
            with pytest.raises(ValueError, match="constants"):
                qk_norm_rotary(leaf, k, None, None, *tables)
            with pytest.raises(Exception, match="constants"):
                torch.compile(qk_norm_rotary, backend="aot_eager", fullgraph=True)(leaf, k, None, None, *tables)
        with torch.no_grad():  # none is asked for
            for a, b in zip(qk_norm_rotary(q, k, None, None, *tables), qk_norm_rotary(q, k, None, None, cos, sin)):
                assert torch.equal(a, b)
            odd = [t.T.contiguous().T for t in tables]  # (not as the kernel reads them)
            assert torch.equal(qk_norm_rotary(q, k, None, None, *odd)[0], qk_norm_rotary(q, k, None, None, cos, sin)[0])


@pytest.mark.parametrize("sign", [1, -1])
def test_wide_integers_past_32_bits_are_no_small_ones(sign):
    """Positions, pages, starts, lengths and prefix sums in 64 bits whose lower 32 are those of a valid one."""
    far = sign * 2**32
    q, k, v = cuda(*inputs(1, 4, 4, 2, 64))
    cos, sin = rotary_table(10, 64)
    positions = torch.tensor([[0, far + 1, 2, far]], device="cuda")
    for y in qk_norm_rotary(q, k, None, None, cos, sin, positions):
        assert y[:, [0, 2]].isfinite().all() and y[:, [1, 3]].isnan().all()
    cache, table, lengths, _ = filled([30, 40], 2, 64, 16)
    before = [x.clone() for x in cache]
    bits = lambda x: x.view(torch.uint8)  # noqa: E731
    new = torch.randn(2, 3, 2, 64, device="cuda").to(BF16)
    write_paged_cache(cache, new, new, table, lengths.long() + far)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(cache, before))
    write_paged_cache(cache, new, new, table.long() + far, lengths)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(cache, before))
    wide = table.long()
    wide[0, 1] += far
    held, _ = read_paged_cache(cache, wide, lengths, 40)
    assert held[0, 16:30].isnan().all() and held[0, :16].isfinite().all() and held[1].isfinite().all()
    few = torch.randn(2, 1, 4, 64, device="cuda").to(BF16)
    assert paged_cache_attention(few, cache, wide, lengths)[0].isnan().all()
    ends = torch.full_like(lengths, table.size(1) * 16 if sign > 0 else 0)  # what such a length is clamped to
    got, want = paged_cache_attention(few, cache, table, lengths.long() + far), paged_cache_attention(few, cache, table, ends)
    assert torch.equal(bits(got), bits(want))  # (NaN where the table has no page)
    o = sliding_window_attention(q, k, v, cu_seqlens=torch.tensor([0, far + 2], device="cuda"))
    assert torch.equal(o, sliding_window_attention(q, k, v, cu_seqlens=torch.tensor([0, 4 if sign > 0 else 0], dtype=torch.int32, device="cuda")))


def test_prefix_sums_of_truth_values_are_refused():
    cache, table, lengths, _ = filled([10, 20], 2, 64, 16)
    new = torch.zeros(1, 2, 2, 64, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="cu_seqlens must be integers"):
        write_paged_cache(cache, new, new, table, lengths, cu_seqlens=torch.ones(3, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="cu_seqlens must hold integers"):
        sliding_window_attention(new, new, new, cu_seqlens=torch.ones(3, dtype=torch.bool, device="cuda"))
