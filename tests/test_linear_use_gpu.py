"""Linear attention and layer norm as a user has them: long sequences in several launches, rows as they lie, other streams, captured
graphs, one graph of a compiler, the state in place, and a run of them together.  Tolerances: tests/test_linear_attention_gpu.py."""

import pytest
import torch

import lm_engine_amd
from lm_engine_amd import chunk_linear_attention, fused_recurrent_linear_attention, layer_norm, linear_attention
from oracle.linear_attention_oracle import layer_norm_ref, linear_attention_ref
from tests.helpers import rel_l2
from tests.test_linear_attention_gpu import BF16, F32, OUT, STATE, _check, _check_gradients, _cu, _cuda, _gradients, _inputs


pytestmark = pytest.mark.gpu


# sequences that are cut into segments, on both sides of the rule for whole ones (up to 128 keys, few chunks); 264 and 520 columns are more
# than the 256 keys that a backward walk has at once
@pytest.mark.parametrize(
    "B, T, H, K, V, lens",
    [(1, 1100, 2, 128, 128, None), (1, 2101, 2, 128, 128, None), (2, 1601, 2, 64, 64, None), (1, 1790, 1, 256, 64, None),
     (1, 900, 1, 72, 264, None), (1, 700, 2, 40, 520, None), (1, 3400, 2, 64, 128, [2100, 3, 0, 900, 397])],
)  # fmt: skip
def test_long_sequences(B, T, H, K, V, lens):
    inputs = _inputs(B, T, H, K, V, N=None if lens is None else len(lens))
    cu = None if lens is None else _cu(lens)
    cu_gpu = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    want, want_state = linear_attention_ref(**inputs, cu_seqlens=cu)
    o, state = chunk_linear_attention(**_cuda(inputs), output_final_state=True, cu_seqlens=cu_gpu)
    _check("o", o, want, OUT[BF16])
    _check("state", state, want_state, STATE[BF16])
    _check("o alone", chunk_linear_attention(**_cuda(inputs), cu_seqlens=cu_gpu)[0], want, OUT[BF16])
    for learned in (False, True):
        got, expected = _gradients(inputs, BF16, cu=cu, learned=learned)
        _check_gradients(got, expected, BF16)


def test_two_parts_are_the_whole():
    inputs = _cuda(_inputs(2, 500, 3, 64, 96))
    whole, state = chunk_linear_attention(**inputs, output_final_state=True)
    part = lambda a, b: {n: x[:, a:b] if n in ("q", "k", "v") else x for n, x in inputs.items()}  # noqa: E731
    o1, s1 = chunk_linear_attention(**part(0, 299), output_final_state=True)
    o2, s2 = chunk_linear_attention(**{**part(299, 496), "initial_state": s1}, output_final_state=True)
    outs = [o1, o2]
    for t in range(496, 500):
        o, s2 = fused_recurrent_linear_attention(**{**part(t, t + 1), "initial_state": s2}, output_final_state=True, inplace_state=True)
        outs.append(o)
    _check("o", torch.cat(outs, 1), whole.double(), 2 * OUT[BF16])
    _check("state", s2, state.double(), 2 * STATE[BF16])


def test_short_rows_take_the_recurrent_form():
    for T in (1, 64, 65):
        inputs = _inputs(2, T, 2, 64, 64)
        o, state = linear_attention(**_cuda(inputs))
        want, want_state = linear_attention_ref(**inputs)
        _check("o", o, want, OUT[BF16])
        _check("state", state, want_state, STATE[BF16])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_as_they_lie(dtype):
    """Column blocks of one tensor, heads in front of tokens, odd offsets, shared and broadcast rows: the results of dense copies, to the
    bit, and gradients in the views' places."""
    gen = torch.Generator().manual_seed(3)
    B, T, H, K, V = 2, 150, 3, 64, 48
    base = torch.randn(B, T, H * (2 * K + V) + 8, generator=gen).to(dtype).cuda()
    g = torch.randn(2 * H, generator=gen, dtype=torch.float64).cuda()[::2].abs().neg() * 0.1
    do = torch.randn(B, H, T, V, generator=gen).to(dtype).cuda().transpose(1, 2)

    def views(x, first):
        q, k, v, _ = x[..., first : first + H * (2 * K + V)].split([H * K, H * K, H * V, 0], dim=-1)
        return q.view(B, T, H, K), k.view(B, T, H, K), v.view(B, T, H, V)

    for first in (0, 8, 3):
        leaf = base.clone().requires_grad_()
        got, _ = chunk_linear_attention(*views(leaf, first), g)
        dense = [x.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for x in views(base, first)]
        want, _ = chunk_linear_attention(*dense, g.float())
        assert torch.equal(got, want)
        own, = torch.autograd.grad(got, leaf, do)
        for x, y in zip(views(own, first), torch.autograd.grad(want, dense, do.contiguous())):
            assert torch.equal(x, y)
    q, k, v = (x.detach() for x in views(base, 0))
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
        assert torch.equal(fn(*heads_first, g)[0], fn(q, k, v, g)[0])
        one = k[:1, :, :1].expand(B, T, H, K)  # a broadcast key
        assert torch.equal(fn(q, one, v, g)[0], fn(q, one.contiguous(), v, g)[0])
        state = torch.randn(H, B, K, V, generator=gen).cuda().transpose(0, 1)
        assert torch.equal(fn(q, k, v, g, initial_state=state)[0], fn(q, k, v, g, initial_state=state.contiguous())[0])
    apart = torch.zeros(1, 3, (1 << 24) + 8, dtype=dtype, device="cuda")[..., : 2 * 64].view(1, 3, 2, 64)  # tokens beyond 32-bit offsets
    apart.copy_(torch.randn(1, 3, 2, 64, generator=gen))
    assert torch.equal(chunk_linear_attention(apart, apart, apart)[0], chunk_linear_attention(*[apart.contiguous()] * 3)[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_padding_holds_does_not_matter(dtype):
    inputs = _inputs(3, 200, 2, 64, 64, dtype=dtype)
    cu = torch.tensor(_cu([200, 0, 77]), dtype=torch.int32).cuda()
    clean, dirty = _cuda(inputs), _cuda(inputs)
    for n in ("q", "k", "v"):
        dirty[n][1], dirty[n][2, :123] = float("nan"), float("inf")
    results = []
    for x in (clean, dirty):
        leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "initial_state")]
        o, state = chunk_linear_attention(*leaves[:4], initial_state=leaves[4], output_final_state=True, cu_seqlens=cu, left_padded=True)
        do = torch.ones_like(o)
        do[1], do[2, :123] = float("nan"), float("nan")
        results.append((o.detach(), state.detach(), *torch.autograd.grad((o, state), leaves, (do, torch.ones_like(state)))))
    for a, b in zip(*results):
        assert a.isfinite().all() and torch.equal(a, b)


def test_calls_give_the_same_bits_twice():
    inputs = _inputs(2, 700, 4, 64, 64, HK=2)
    first, _ = _gradients(inputs, BF16, learned=True)
    again, _ = _gradients(inputs, BF16, learned=True)
    for n in first:
        assert torch.equal(first[n], again[n]), n
    x = torch.randn(3000, 512, device="cuda").to(BF16)
    w = torch.randn(512, device="cuda", requires_grad=True)
    grads = [torch.autograd.grad(layer_norm(x, w), w, x)[0] for _ in range(2)]
    assert torch.equal(*grads)


def test_prefix_sums_out_of_range_are_clamped():
    """[0, 150, 120, 260] over 200 tokens: sequences 0 - 149, none (it would end in front of its start), 120 - 199."""
    inputs = _inputs(1, 200, 2, 64, 64, N=3)
    cu = torch.tensor([0, 150, 120, 260], dtype=torch.int32).cuda()
    for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
        _, state = fn(**_cuda(inputs), output_final_state=True, cu_seqlens=cu)
        for n, (first, last) in enumerate(((0, 150), (150, 150), (120, 200))):
            part = {name: x[:, first:last] if name in ("q", "k", "v") else x for name, x in inputs.items()}
            part["initial_state"] = inputs["initial_state"][n : n + 1]
            want = linear_attention_ref(**part)[1] if last > first else part["initial_state"]
            _check("state", state[n : n + 1], want.double(), STATE[BF16])


def test_state_in_place():
    inputs = _cuda(_inputs(4, 1, 2, 128, 128))
    want, want_state = fused_recurrent_linear_attention(**inputs, output_final_state=True)
    state = inputs["initial_state"].clone()
    o, out = fused_recurrent_linear_attention(**{**inputs, "initial_state": state}, output_final_state=True, inplace_state=True)
    assert out is state and torch.equal(state, want_state) and torch.equal(o, want) and not torch.equal(want_state, inputs["initial_state"])
    refuse = lambda **over: pytest.raises(ValueError, match="inplace_state")  # noqa: E731
    with refuse():
        fused_recurrent_linear_attention(**inputs, inplace_state=True)
    with refuse():
        fused_recurrent_linear_attention(**{**inputs, "initial_state": None}, output_final_state=True, inplace_state=True)
    with refuse():
        apart = state.transpose(0, 1).contiguous().transpose(0, 1)
        fused_recurrent_linear_attention(**{**inputs, "initial_state": apart}, output_final_state=True, inplace_state=True)
    with refuse():
        odd = torch.zeros(state.numel() + 1, device="cuda")[1:].view_as(state)
        fused_recurrent_linear_attention(**{**inputs, "initial_state": odd}, output_final_state=True, inplace_state=True)
    with refuse():
        fused_recurrent_linear_attention(**{**inputs, "q": inputs["q"].clone().requires_grad_()}, output_final_state=True, inplace_state=True)


def test_refused_operands():
    x = _cuda(_inputs(2, 10, 4, 64, 64))
    for over, match in [
        (dict(q=x["q"].half(), k=x["k"].half(), v=x["v"].half()), "."), (dict(v=x["v"].float()), "share a dtype"), (dict(g=x["g"][:3]), "g must be"),
        (dict(g=torch.zeros(4, dtype=torch.int32, device="cuda")), "g must be"), (dict(g=x["g"].cpu()), "g is on"),
        (dict(initial_state=x["initial_state"][:1]), "initial_state must be"), (dict(initial_state=x["initial_state"].to(BF16)), "float32"),
        (dict(cu_seqlens=torch.tensor([0, 20], dtype=torch.int32).cuda()), "batch dim must be 1"), (dict(left_padded=True), "prefix sums"),
        (dict(cu_seqlens=torch.zeros(3, device="cuda"), left_padded=True), "integers"), (dict(q=x["q"][..., :60], k=x["k"][..., :60]), "head dim K"),
        (dict(v=x["v"][..., :60]), "value head dim"),
    ]:  # fmt: skip
        for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
            with pytest.raises((ValueError, TypeError), match=match):
                fn(**{**x, **over})
    q = x["q"].clone().requires_grad_()
    o, _ = chunk_linear_attention(**{**x, "q": q})
    dq, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):  # a gradient is not itself differentiated
        torch.autograd.grad(dq.float().sum(), q)
    rows = torch.randn(4, 64, device="cuda")
    for args, match in [((rows, rows[0, :32]), "weight must be"), ((rows, None, rows[0, :32]), "bias must be"), ((rows, rows[0].cpu()), "weight is on"),
                        ((rows, rows[0], rows[0].to(BF16)), "share a dtype"), ((rows.double(),), "."), ((torch.zeros(2, 16385, device="cuda"),), "not supported")]:  # fmt: skip
        with pytest.raises((ValueError, TypeError), match=match):
            layer_norm(*args)


def test_no_tokens():
    for B, T in ((0, 5), (2, 0)):
        q = torch.zeros(B, T, 2, 64, device="cuda", dtype=BF16, requires_grad=True)
        state = torch.randn(B, 2, 64, 64, device="cuda", requires_grad=True)
        for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
            o, out = fn(q, q, q, torch.zeros(2, device="cuda"), initial_state=state, output_final_state=True)
            assert o.shape == q.shape and torch.equal(out, state)
            dq, ds = torch.autograd.grad((o, out), (q, state), (torch.zeros_like(o), torch.ones_like(out)))
            assert dq.shape == q.shape and (ds == 1).all()


def test_gradients_against_differences():
    """The result is linear in q, k, v and the state each, so a central difference of any width is the directional derivative; the two sides
    are sums of fp32 terms, held to 1e-4 of their size.  The decay's is taken of the loop in 64 bits, 1e-4 wide: 40 tokens make the
    rest of the series (40 * 1e-4)^2 / 6 = 3e-6."""
    inputs = _inputs(1, 40, 2, 16, 24, dtype=F32)
    gen = torch.Generator().manual_seed(8)
    do, dht = torch.randn(1, 40, 2, 24, generator=gen), torch.randn(1, 2, 16, 24, generator=gen)

    def loss(x):
        o, state = chunk_linear_attention(**_cuda(x), output_final_state=True)
        return ((o.double().cpu() * do).sum() + (state.double().cpu() * dht).sum()).item()

    def exact(x):
        o, state = linear_attention_ref(**x)
        return ((o * do).sum() + (state * dht).sum()).item()

    leaves = {n: x.cuda().requires_grad_() for n, x in inputs.items()}
    o, state = chunk_linear_attention(**leaves, output_final_state=True)
    grads = dict(zip(leaves, torch.autograd.grad((o, state), list(leaves.values()), (do.cuda(), dht.cuda()))))
    for n, x in inputs.items():
        d = torch.randn(x.shape, generator=gen)
        if n == "g":
            wide = {**inputs, "g": x.double()}
            step = lambda e: exact({**wide, "g": x.double() + e * d.double()})  # noqa: E731
            want, size = (step(1e-4) - step(-1e-4)) / 2e-4, abs(exact(wide))
        else:
            up, down = loss({**inputs, n: x + d}), loss({**inputs, n: x - d})
            want, size = (up - down) / 2, abs(up) + abs(down)
        got = (grads[n].double().cpu() * d.double()).sum().item()
        size += (grads[n].double().cpu() * d.double()).abs().sum().item()
        print(n, got, want, flush=True)
        assert abs(got - want) <= 1e-4 * size, n
    x, dy = torch.randn(6, 40, generator=gen).cuda(), torch.randn(6, 40, generator=gen).cuda()
    w, b = torch.randn(40, generator=gen).cuda(), torch.randn(40, generator=gen).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for i, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=gen).double()
        at = lambda e: (layer_norm_ref(*[(s.cpu().double() + (e * d if j == i else 0)) for j, s in enumerate((x, w, b))]) * dy.cpu().double()).sum()  # noqa: E731, B023
        want = ((at(1e-5) - at(-1e-5)) / 2e-5).item()
        own = got[i].double().cpu() * d
        assert abs(own.sum().item() - want) <= 1e-5 * own.abs().sum().item()


def test_another_stream_and_two_calls_at_once():
    inputs = [_cuda(_inputs(1, 1500, 4, 128, 128, seed=s)) for s in range(2)]
    x = torch.randn(4000, 1024, device="cuda").to(BF16)
    want = [chunk_linear_attention(**i, output_final_state=True) for i in inputs]
    rows = layer_norm(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                busy = torch.randn(2048, 2048, device="cuda") @ torch.randn(2048, 2048, device="cuda")  # noqa: F841
                moved = {n: t + 0 for n, t in i.items()}  # made on this stream, behind the product
                got.append((*chunk_linear_attention(**moved, output_final_state=True), layer_norm(x + 0)))
        torch.cuda.synchronize()
        for (o, state, y), (o_want, state_want) in zip(got, want):
            assert torch.equal(o, o_want) and torch.equal(state, state_want) and torch.equal(y, rows)


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


def test_captured_forward_calls_replay():
    inputs = _cuda(_inputs(1, 2200, 2, 128, 128))  # several segments and a workspace
    x = torch.randn(500, 256, device="cuda").to(BF16)
    w = torch.randn(256, device="cuda")
    step = _cuda(_inputs(3, 1, 2, 128, 128, seed=9))
    start = step["initial_state"].clone()

    def run():
        o, state = chunk_linear_attention(**inputs, output_final_state=True)
        d, _ = fused_recurrent_linear_attention(**step, output_final_state=True, inplace_state=True)
        return o, state, d, layer_norm(x, w, w)

    graph, out = _capture(run)
    other, out2 = _capture(lambda: chunk_linear_attention(**inputs, output_final_state=True))  # a second graph of the same calls
    for replay in range(4):
        for n in ("q", "k", "v"):
            inputs[n].normal_()
        x.normal_()
        step["initial_state"].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        got, after = [t.clone() for t in out], step["initial_state"].clone()
        step["initial_state"].copy_(start)
        other.replay()
        want = run()
        for a, b in zip(got, want):
            assert torch.equal(a, b), replay
        assert torch.equal(after, step["initial_state"]) and torch.equal(out2[0], want[0]) and torch.equal(out2[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_training_step_replays(dtype):
    T = 1700 if dtype == BF16 else 300
    inputs = _cuda(_inputs(1, T, 4, 64, 64, HK=2, dtype=dtype))
    do = torch.randn(1, T, 4, 64, device="cuda").to(dtype)
    w = torch.randn(64, device="cuda")

    def run():
        leaves = [inputs[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "initial_state")] + [w.detach().requires_grad_()]
        o, _ = chunk_linear_attention(*leaves[:4], initial_state=leaves[4])
        return torch.autograd.grad(layer_norm(o, leaves[5]), leaves, do)

    graph, out = _capture(run)
    for replay in range(4):
        for n in ("q", "k", "v"):
            inputs[n].normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for i, (a, b) in enumerate(zip(got, run())):
            assert torch.equal(a, b), (replay, i)


def test_one_graph_of_the_compiler():
    inputs = _inputs(2, 200, 4, 64, 64, HK=2)
    w = torch.randn(64, device="cuda")

    def loss(q, k, v, g, initial_state, weight):
        o, state = chunk_linear_attention(q, k, v, g, initial_state=initial_state, output_final_state=True)
        return layer_norm(o, weight).float().square().sum() + state.sum()

    def leaves():
        return [x.detach().clone().requires_grad_() for x in (*_cuda(inputs).values(), w)]

    eager, compiled = leaves(), leaves()
    loss(*eager).backward()
    torch.compile(loss, backend="aot_eager", fullgraph=True)(*compiled).backward()
    for a, b in zip(eager, compiled):
        assert b.grad is not None and torch.equal(a.grad, b.grad)

    step = _cuda(_inputs(3, 1, 2, 128, 128))
    decode = lambda s: fused_recurrent_linear_attention(**{**step, "initial_state": s}, output_final_state=True, inplace_state=True)  # noqa: E731
    s1, s2 = step["initial_state"].clone(), step["initial_state"].clone()
    o1, _ = decode(s1)
    o2, _ = torch.compile(decode, backend="aot_eager", fullgraph=True)(s2)
    assert torch.equal(o1, o2) and torch.equal(s1, s2)


def test_only_the_gradients_that_are_asked_for():
    inputs = _cuda(_inputs(2, 150, 2, 64, 64))
    full = {n: x.clone().requires_grad_() for n, x in inputs.items()}
    o, state = chunk_linear_attention(**full, output_final_state=True)
    do, dht = torch.randn_like(o), torch.randn_like(state)
    want = dict(zip(full, torch.autograd.grad((o, state), list(full.values()), (do, dht), retain_graph=True)))
    for n in full:
        part = {m: x.clone().requires_grad_(m == n) for m, x in inputs.items()}
        o1, s1 = chunk_linear_attention(**part, output_final_state=True)
        got, = torch.autograd.grad((o1, s1), part[n], (do, dht))
        # (with the decay's the states between the segments come from its own launch)
        assert rel_l2(got, want[n]) <= 2 * STATE[BF16] if n == "initial_state" else rel_l2(got, want[n]) <= OUT[BF16], n
    only_state = torch.autograd.grad(state, full["v"], dht, retain_graph=True)[0]
    both = torch.autograd.grad((o, state), full["v"], (torch.zeros_like(o), dht), retain_graph=True)[0]
    assert torch.equal(only_state, both)
    spread = torch.autograd.grad(o, full["q"], torch.ones(1, 1, 1, 1, device="cuda", dtype=BF16).expand_as(o), retain_graph=True)[0]
    assert torch.equal(spread, torch.autograd.grad(o, full["q"], torch.ones_like(o))[0])


def test_a_run_of_them_together():
    """A mixer's middle: the norm of a hidden size, its columns as q, k and v, the attention over a prompt, the norm of every head; then
    single tokens on the state.  Against the same in 64 bits: q, k and v carry a rounding each (2^-8 / sqrt(3) rms), the attention its
    5e-3, the last norm one more rounding; independent they are 7.2e-3 rms, of rows that the sum may leave smaller than its
    terms: 1.5e-2.  The gradient goes through all of it twice: 3e-2."""
    gen = torch.Generator().manual_seed(21)
    B, T, H, D = 2, 333, 4, 64
    x = torch.randn(B, T, 3 * H * D, generator=gen).to(BF16)
    w, b = 1 + 0.1 * torch.randn(3 * H * D, generator=gen), 0.1 * torch.randn(3 * H * D, generator=gen)
    wh = 1 + 0.1 * torch.randn(D, generator=gen)
    g = -(2.0 ** (-8.0 * torch.arange(1, H + 1) / H))
    dy = torch.randn(B, T, H, D, generator=gen).to(BF16)

    def mixer(norm, attention, x, w, b, wh, g, state=None):
        q, k, v = (t.unflatten(-1, (H, D)) for t in norm(x, w, b).chunk(3, dim=-1))
        o, state = attention(q, k, v, g, initial_state=state)
        return norm(o, wh), state

    def own_attention(q, k, v, g, initial_state):
        return linear_attention(q, k, v, g, initial_state=initial_state)

    ref = [t.double().requires_grad_() for t in (x, w, b, wh, g)]
    want, _ = mixer(layer_norm_ref, lambda q, k, v, g, initial_state: linear_attention_ref(q, k, v, g, initial_state=initial_state), *ref)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, wh, g)]
    got, _ = mixer(layer_norm, own_attention, *leaves)
    _check("y", got, want.detach(), 1.5e-2)
    for name, a, r in zip(("x", "w", "b", "wh", "g"), torch.autograd.grad(got, leaves, dy.cuda()), torch.autograd.grad(want, ref, dy.double())):
        _check("d" + name, a, r, 3e-2)
    with torch.no_grad():
        parts = [leaves[0][:, :330], *(leaves[0][:, t : t + 1] for t in range(330, 333))]
        state, outs = None, []
        for part in parts:
            y, state = mixer(layer_norm, own_attention, part, *leaves[1:], state=state)
            outs.append(y)
        _check("y of a prompt and three tokens", torch.cat(outs, 1), want.detach(), 1.5e-2)


def test_a_switched_off_kernel_is_refused_in_the_backward_too():
    q = torch.randn(1, 8, 1, 64, device="cuda").to(BF16).requires_grad_()
    o, y = chunk_linear_attention(q, q, q)[0], layer_norm(q)
    with lm_engine_amd.kernels.enable_kernels([], reset=True):
        for out in (o, y):
            with pytest.raises(RuntimeError, match="disabled"):
                torch.autograd.grad(out, q, torch.ones_like(out), retain_graph=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shared_heads_of_a_packed_batch_leave_zeros_outside(dtype):
    """The fold of shared heads reads every token: those in front of and behind the sequences are zeros, whatever the workspace held."""
    lens, T = [40, 0, 333], 400
    inputs = _inputs(1, T, 4, 64, 72, HK=2, N=3, dtype=dtype)
    torch.full((1 << 24,), float("nan"), device="cuda")
    got, want = _gradients(inputs, dtype, cu=_cu(lens))
    for n in ("q", "k", "v"):
        assert (got[n][:, 373:] == 0).all(), n
    _check_gradients(got, want, dtype, shared=True)
    shifted = torch.tensor([20, 60, 60, 393], dtype=torch.int32).cuda()
    leaves = {n: x.cuda().requires_grad_() for n, x in inputs.items()}
    o, _ = chunk_linear_attention(**leaves, cu_seqlens=shifted)
    for n, x in zip(("q", "k", "v"), torch.autograd.grad(o, [leaves[n] for n in ("q", "k", "v")], torch.ones_like(o))):
        assert x.isfinite().all() and (x[:, :20] == 0).all() and (x[:, 393:] == 0).all() and (x[:, 20:393] != 0).any(), n


def test_a_decay_at_either_end():
    """No memory at all (-inf: 0 to the power 0 is 1), none of it lost (0), and in between the products of 64 tokens below fp32's range."""
    inputs = _inputs(1, 200, 4, 64, 64)
    inputs["g"] = torch.tensor([-float("inf"), 0.0, -87.0, -1e-30])
    want, want_state = linear_attention_ref(**inputs)
    for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
        o, state = fn(**_cuda(inputs), output_final_state=True)
        _check("o", o, want, OUT[BF16])
        _check("state", state, want_state, STATE[BF16])
