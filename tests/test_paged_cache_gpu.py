"""The paged cache in 8 bits on the GPU, against its definition token by token, and attention over it against the formula in 64 bits.

Codes and scales are exact: what is written has to be what the definition says, to the bit.  The attention's output against the formula on
the values that the codes stand for: its own rounding and that of each weight as an operand, as in tests/test_window_attention_gpu.py: 5e-3."""

import pytest
import torch

from lm_engine_amd import new_paged_cache, paged_cache_attention, read_paged_cache, write_paged_cache
from oracle.attention_oracle import PagedCacheRef, attend, to_e4m3, visible_keys
from tests.helpers import rel_l2


pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
OUT = 5e-3


def tables(counts, pages, most, seed=0):
    """Pages in an order of their own, -1 behind a sequence's last."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    rows = []
    for count in counts:
        rows.append(order[:count] + [-1] * (most - count))
        order = order[count:]
    return rows


def same(cache, ref):
    """The cache's codes and scales against the definition's."""
    pages, heads, P, D = cache.k.shape
    v = cache.v.float().permute(0, 1, 2, 4, 3).reshape(pages, heads, P, D)
    for codes, want, scale, exponents in zip((cache.k.float(), v), ref.codes, (cache.k_scale, cache.v_scale), ref.exponents):
        assert torch.equal(scale.cpu().long() - 127, exponents.long())
        codes = codes.double().cpu()
        assert torch.equal(codes.nan_to_num(1e3), want.nan_to_num(1e3))


def rows(gen, T, heads, D, dtype):
    x = torch.randn(T, heads, D, generator=gen) * torch.exp(torch.randn(T, 1, 1, generator=gen))
    return x.to(dtype)


def test_every_code():
    """All of bf16, one value a page's head beside the one that sets the scale: every rounding, ties among them, and values that vanish."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    x = x[x.isfinite() & (x.float().abs() <= 448)]
    x = torch.cat([x, x.new_zeros(-x.numel() % 15)]).view(-1, 15)
    x = torch.cat([torch.full((x.size(0), 1), 448.0, dtype=BF16), x], dim=1)[:, None, None]  # [pages, 1, 1, 16]
    pages = x.size(0)
    cache = new_paged_cache(pages, 1, 16, page_size=16)
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[:, None]
    write_paged_cache(cache, x.cuda(), x.cuda(), table, torch.zeros(pages, dtype=torch.int32, device="cuda"))
    assert (cache.k_scale == 127).all() and (cache.v_scale == 127).all()
    want = to_e4m3(x[:, 0, 0])
    assert torch.equal(cache.k[:, 0, 0].double().cpu(), want) and torch.equal(cache.v[:, 0, 0, :, 0].double().cpu(), want)
    k, v = read_paged_cache(cache, table, torch.ones(pages, dtype=torch.int32, device="cuda"), 1)
    assert torch.equal(k[:, 0, 0].double().cpu(), want) and torch.equal(v, k)


# (page size, heads, D, dtype, tokens of each call's sequences)
WRITES = [
    (16, 1, 16, BF16, [[1, 5]] * 6), (64, 2, 128, BF16, [[70, 3], [1, 1], [1, 1], [130, 62], [1, 1]]), (32, 3, 80, F32, [[33, 0, 31], [2, 90, 1]]),
    (128, 1, 256, BF16, [[300], [1]]), (256, 1, 256, F32, [[257, 10], [300, 300]]), (48, 2, 96, BF16, [[47, 48, 49], [1, 1, 1], [100, 1, 2]]),
]  # fmt: skip


@pytest.mark.parametrize("layout", ["packed", "left padded", "rows"])
@pytest.mark.parametrize("P, heads, D, dtype, calls", WRITES, ids=str)
def test_write_and_read(P, heads, D, dtype, calls, layout):
    gen = torch.Generator().manual_seed(P + D)
    N, totals = len(calls[0]), [sum(x) for x in zip(*calls)]
    if layout == "rows":
        calls = [[max(c)] * N for c in calls]
        totals = [sum(x) for x in zip(*calls)]
    counts = [-(-t // P) for t in totals]
    most, pages = max(counts) + 1, sum(counts) + 2
    table = tables(counts, pages, most)
    cache, ref = new_paged_cache(pages, heads, D, page_size=P), PagedCacheRef(pages, heads, D, P)
    gpu_table = torch.tensor(table, dtype=torch.int32).cuda()
    start = [0] * N
    for lens in calls:
        T = max(lens)
        new = [(rows(gen, n, heads, D, dtype), rows(gen, n, heads, D, dtype)) for n in lens]
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
        if layout == "packed":
            k, v = (torch.cat([x[i] for x in new])[None] for i in range(2))
            options = dict(cu_seqlens=cu)
        else:
            pad = lambda x: torch.cat([torch.full((T - x.size(0), heads, D), float("nan"), dtype=dtype), x])  # noqa: E731, B023
            k, v = (torch.stack([pad(x[i]) for x in new]) for i in range(2))
            options = dict(cu_seqlens=cu, left_padded=True) if layout == "left padded" else {}
        out = write_paged_cache(cache, k.cuda(), v.cuda(), gpu_table, torch.tensor(start, dtype=torch.int32).cuda(), **options)
        assert out is cache
        for n in range(N):
            ref.write(*new[n], table[n], start[n])
            start[n] += lens[n]
        same(cache, ref)
    for read in (BF16, F32):
        k, v = read_paged_cache(cache, gpu_table, torch.tensor(start, dtype=torch.int32).cuda(), max(start) + 3, dtype=read)
        for n in range(N):
            want = ref.read(table[n], start[n])
            for got, w in zip((k[n], v[n]), want):
                assert got.dtype == read and torch.equal(got[: start[n]].double().cpu(), w) and (got[start[n] :] == 0).all()


def test_a_sequence_that_is_cut_back_is_written_on():
    gen = torch.Generator().manual_seed(3)
    cache, ref = new_paged_cache(4, 2, 32, page_size=32), PagedCacheRef(4, 2, 32, 32)
    table = torch.tensor([[2, 0]], dtype=torch.int32).cuda()
    for start, T, size in ((0, 20, 1.0), (20, 8, 50.0), (22, 4, 1.0), (26, 10, 300.0), (0, 5, 1e-3)):
        k, v = size * torch.randn(T, 2, 32, generator=gen), size * torch.randn(T, 2, 32, generator=gen)
        write_paged_cache(cache, k[None].cuda(), v[None].cuda(), table, torch.tensor([start], dtype=torch.int32).cuda())
        ref.write(k, v, [2, 0], start)
        got = read_paged_cache(cache, table, torch.tensor([start + T], dtype=torch.int32).cuda(), start + T, dtype=F32)
        for a, b in zip(got, ref.read([2, 0], start + T)):
            assert torch.equal(a[0].double().cpu(), b)


def test_values_at_the_edges():
    """Nothing but zeros, the smallest and largest numbers, and what is not finite: NaN, and nothing to the scale."""
    gen = torch.Generator().manual_seed(5)
    for dtype in (BF16, F32):
        for size in (0.0, 1e-38, 2.0**-100, 3e38):
            x = (size * torch.rand(20, 1, 16, generator=gen)).to(dtype)
            x[3, 0, 2], x[17, 0, 1], x[18, 0, 5] = float("inf"), float("nan"), -float("inf")
            cache, ref = new_paged_cache(2, 1, 16, page_size=16), PagedCacheRef(2, 1, 16, 16)
            write_paged_cache(cache, x[None].cuda(), x[None].cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda())
            ref.write(x, x, [1, 0], 0)
            same(cache, ref)


def test_pages_that_are_not_there():
    gen = torch.Generator().manual_seed(6)
    cache = new_paged_cache(3, 1, 32, page_size=16)
    before = [x.clone() for x in cache]
    k = torch.randn(1, 100, 1, 32, generator=gen).to(BF16).cuda()
    table = torch.tensor([[1, -1, 3, 2**31 - 1, -(2**31)]], dtype=torch.int32).cuda()
    write_paged_cache(cache, k, k, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    for now, old in zip(cache, before):
        assert torch.equal(now.view(torch.uint8)[[0, 2]], old.view(torch.uint8)[[0, 2]])
    got, _ = read_paged_cache(cache, table, torch.tensor([100], dtype=torch.int32).cuda())
    assert got.shape == (1, 80, 1, 32) and got[0, :16].isfinite().all() and got[0, 16:].isnan().all()
    # in front of position 0 and past the table: dropped, the rest where it belongs
    for start in (-30, 70, 80, 1000, -1000, 2**31 - 1, -(2**31)):
        write_paged_cache(cache, k, k, table, torch.tensor([start], dtype=torch.int32).cuda())
    cache2 = new_paged_cache(3, 1, 32, page_size=16)
    write_paged_cache(cache2, k, k, table, torch.tensor([-30], dtype=torch.int32).cuda())
    ref = PagedCacheRef(3, 1, 32, 16)
    ref.write(k[0, 30:].cpu(), k[0, 30:].cpu(), table[0].tolist(), 0)
    same(cache2, ref)
    q = torch.randn(1, 20, 2, 32, generator=gen).to(BF16).cuda()
    o = paged_cache_attention(q, cache2, table, torch.tensor([20], dtype=torch.int32).cuda())
    assert o[0, :16].isfinite().all() and o[0, 16:].isnan().all()
    o = paged_cache_attention(q, cache2, table, torch.tensor([16], dtype=torch.int32).cuda())  # queries in front of position 0
    assert (o[0, :4] == 0).all() and o.isfinite().all()


# (N, T, H, HK, D, page size, lengths, window, sinks)
ATTENTION = [
    (1, 1, 1, 1, 16, 16, [1], None, 0), (3, 1, 4, 2, 64, 64, [1, 64, 200], None, 0), (2, 1, 16, 2, 128, 64, [1000, 63], None, 0),
    (2, 3, 8, 1, 128, 32, [500, 2], None, 0), (2, 1, 8, 8, 256, 128, [300, 129], None, 0), (1, 1, 2, 1, 96, 48, [700], None, 0),
    (2, 5, 12, 3, 80, 16, [333, 5], 100, 7), (2, 1, 4, 1, 64, 64, [2000, 40], 200, 4), (1, 8, 40, 4, 128, 64, [1500], 64, 130),
    (1, 1, 16, 2, 128, 64, [30000], None, 0), (1, 1, 4, 2, 128, 256, [9000], 5000, 70), (4, 2, 2, 2, 64, 16, [0, 1, 2, 3], 2, 1), (1, 100, 3, 1, 64, 64, [180], 20, 3),
    (40, 1, 32, 8, 64, 16, list(range(1, 200, 5)), None, 0),
]  # fmt: skip


def filled(lens, heads, D, P, seed=0):
    """(cache, table, its pages as lists, k and v of every sequence as the codes have them, float64)"""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // P) for n in lens]
    most = max(1, *counts)
    table, cache = tables(counts, sum(counts) + 1, most, seed), new_paged_cache(sum(counts) + 1, heads, D, page_size=P)
    gpu = torch.tensor(table, dtype=torch.int32).cuda()
    k, v = (torch.randn(1, max(1, sum(lens)), heads, D, generator=gen).to(BF16).cuda() for _ in range(2))
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    write_paged_cache(cache, k, v, gpu, torch.zeros(len(lens), dtype=torch.int32, device="cuda"), cu_seqlens=cu)
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    return cache, gpu, lengths, [x.double().cpu() for x in read_paged_cache(cache, gpu, lengths, most * P, dtype=F32)]


@pytest.mark.parametrize("N, T, H, HK, D, P, lens, window, sinks", ATTENTION, ids=str)
def test_attention(N, T, H, HK, D, P, lens, window, sinks):
    cache, table, lengths, (k, v) = filled(lens, HK, D, P)
    q = (1.5 * torch.randn(N, T, H, D, generator=torch.Generator().manual_seed(1))).to(BF16)
    for scale in (None, -0.1):
        o = paged_cache_attention(q.cuda(), cache, table, lengths, window=window, sinks=sinks, scale=scale)
        by = D**-0.5 if scale is None else scale
        want = torch.stack([attend(q[n].double(), k[n, : lens[n]], v[n, : lens[n]], visible_keys(T, lens[n], window, sinks), by) for n in range(N)])
        error = rel_l2(o, want)
        print(f"o {error:.2e}", flush=True)
        assert o.shape == q.shape and o.dtype == BF16 and o.isfinite().all() and error <= OUT, error
