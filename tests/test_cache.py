"""GPU tests of cache_write and cache_read against plain indexing and quantisation in 64 bits."""

import math

import pytest
import torch

from paged_testlib import LEVELS, Sequences, rows, stored, values
from sol_attn_amd import PagedCache, PagedPlan, cache_read, cache_write
from sol_testlib import HAS_GPU

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not HAS_GPU, reason="AMD ROCm GPU required")]

FORMATS = ("bf16", "int8", "fp8")


def bits(x):
    return x.view(torch.int8) if x.dtype == torch.float8_e4m3fn else x


def assert_same_cache(a, b):
    assert torch.equal(bits(a.k), bits(b.k)) and torch.equal(bits(a.v), bits(b.v))
    if a.k_scales is not None:
        for x, y in ((a.k_scales, b.k_scales), (a.v_scales, b.v_scales)):
            assert torch.equal(x.nan_to_num(-1.0), y.nan_to_num(-1.0))


def written(seqs, k, v):
    """The batch's cache with its new rows written by the operator, from a cache that holds the older ones."""
    new_k, new_v = seqs.k, seqs.v
    seqs.cache = PagedCache.create(seqs.pages, seqs.page_size, k.shape[1], k.shape[2], format=seqs.fmt)
    seqs.k = [x[:len(x) - n] for x, n in zip(new_k, seqs.new)]
    seqs.v = [x[:len(x) - n] for x, n in zip(new_v, seqs.new)]
    seqs.store()
    cache_write(k, v, seqs.cache, seqs.plan)
    seqs.k, seqs.v = new_k, new_v
    return seqs.cache


def new_rows(seqs, of):
    return torch.cat([x[len(x) - n:] for x, n in zip(of, seqs.new)]).cuda()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (128, 64, 2), (128, 16, 1), (64, 256, 8)])
@pytest.mark.parametrize("lengths,new", [
    ([1, 1, 1], [1, 1, 1]), ([17, 0, 64, 65, 1], [17, 0, 3, 1, 0]), ([300, 129], [300, 1]),
    (list(range(1, 80)), [1] * 79), ([40] * 5, [0] * 5),
])
def test_write_equals_plain_indexing(fmt, dim, page, heads, lengths, new):
    seqs = Sequences(lengths, new, heads=heads, dim=dim, fmt=fmt, page_size=page, seed=3)
    whole = seqs.cache
    got = written(seqs, new_rows(seqs, seqs.k), new_rows(seqs, seqs.v))
    assert_same_cache(got, whole)


@pytest.mark.parametrize("lengths,new,heads,dim", [
    ([1511], [1503], 24, 128), ([900, 0, 1400, 5], [897, 0, 1301, 1], 40, 64), ([5600], [5589], 24, 128),
])
def test_write_of_a_frame(lengths, new, heads, dim):
    # From one round of waves up, and past four.
    seqs = Sequences(lengths, new, heads=heads, dim=dim, page_size=64, seed=51)
    whole = seqs.cache
    assert_same_cache(written(seqs, new_rows(seqs, seqs.k), new_rows(seqs, seqs.v)), whole)


@pytest.mark.parametrize("lengths,new,heads,dim", [
    ([2250], [2243], 24, 128), ([1500, 0, 2400, 5], [1497, 0, 2301, 1], 40, 64), ([2100], [2070], 24, 128),
])
def test_write_of_a_frame_in_one_round(lengths, new, heads, dim):
    # From one and a half rounds of waves up to four, which take four groups of rows each, and just below.
    seqs = Sequences(lengths, new, heads=heads, dim=dim, page_size=64, seed=52)
    whole = seqs.cache
    assert_same_cache(written(seqs, new_rows(seqs, seqs.k), new_rows(seqs, seqs.v)), whole)


def test_write_takes_many_sequences():
    # More sequences than one workgroup keeps offsets of.
    lengths = [1 + i % 3 for i in range(1500)]
    new = [i % 2 for i in range(1500)]
    seqs = Sequences(lengths, new, heads=1, dim=64, fmt="int8", page_size=16, seed=4)
    whole = seqs.cache
    assert_same_cache(written(seqs, new_rows(seqs, seqs.k), new_rows(seqs, seqs.v)), whole)


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_takes_strided_and_misaligned_rows(fmt):
    seqs = Sequences([50, 20], [37, 5], heads=3, dim=64, fmt=fmt, page_size=16, seed=5)
    whole = seqs.cache
    k, v = new_rows(seqs, seqs.k), new_rows(seqs, seqs.v)
    fused = torch.zeros((42, 2, 6, 64), dtype=torch.bfloat16, device="cuda")
    fused[:, 0, ::2], fused[:, 1, 1::2] = k, v
    assert_same_cache(written(seqs, fused[:, 0, ::2], fused[:, 1, 1::2]), whole)
    odd = torch.zeros(42 * 3 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(42, 3, 64)
    odd.copy_(k)
    assert_same_cache(written(seqs, odd, v), whole)


@pytest.mark.parametrize("fmt", ("int8", "fp8"))
def test_codes_are_the_rounded_quotients_everywhere(fmt):
    # Every magnitude as the row's largest beside every finite BF16 value that does not exceed it: exact ties, the
    # smallest and the largest exponents among them.
    everything = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    finite = everything[torch.isfinite(everything.float())]
    g = torch.Generator().manual_seed(6)
    picks = torch.cat([torch.tensor([0, 1, 2, 127, 128, 129, len(finite) - 2, len(finite) - 1]),
                       torch.randint(1, len(finite), (1016,), generator=g)])
    x = torch.zeros((len(picks), 64), dtype=torch.bfloat16)
    for i, at in enumerate(picks.tolist()):
        most = finite[at]
        low = max(0, at - 128 * 12)  # twelve powers of two below it
        x[i] = finite[torch.randint(low, at + 1, (64,), generator=g)]
        x[i, 7] = most
    x[:, ::3] = -x[:, ::3]
    n = len(picks)
    plan = PagedPlan.create([list(range(n // 64))], [n], [n], pages=n // 64, page_size=64).to("cuda")
    cache = PagedCache.create(n // 64, 64, 1, 64, format=fmt)
    cache_write(x[:, None].cuda(), x[:, None].cuda(), cache, plan)
    codes, scale = stored(x, fmt)
    for store, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        assert torch.equal(store.float().double().view(n, 64).cpu(), codes)
        assert torch.equal(scales.view(n).cpu(), scale)


@pytest.mark.parametrize("fmt", ("int8", "fp8"))
def test_rows_of_zeros_infinities_and_nan(fmt):
    x = rows(6, 2, 64, seed=7)
    x[1, 0] = 0
    x[2, 1, 5] = math.inf
    x[3, 0, 63] = -math.inf
    x[4, 1, 0] = math.nan
    plan = PagedPlan.create([[0]], [6], [6], pages=1, page_size=16).to("cuda")
    cache = PagedCache.create(1, 16, 2, 64, format=fmt)
    cache_write(x.cuda(), x.cuda(), cache, plan)
    k, v = cache_read(cache, plan, 6)
    assert torch.equal(k.isnan(), v.isnan())
    bad = k[0].isnan().cpu()
    expected = torch.zeros_like(bad)
    expected[2, 1] = expected[3, 0] = expected[4, 1] = True
    assert torch.equal(bad, expected)
    assert not k[0, 1, 0].any() and float(cache.k_scales[0, 0, 1]) == 0.0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (128, 64, 2), (128, 128, 5)])
@pytest.mark.parametrize("lengths,start,tokens", [([1], 0, 1), ([17, 0, 64, 200], 0, 200), ([130, 70], 33, 60),
                                                  ([5, 300], 290, 20), ([16], 500, 3)])
def test_read_equals_the_stored_values(fmt, dim, page, heads, lengths, start, tokens):
    seqs = Sequences(lengths, [0] * len(lengths), heads=heads, dim=dim, fmt=fmt, page_size=page, seed=8, fill=math.nan)
    k, v = cache_read(seqs.cache, seqs.plan, tokens, start=start)
    for got, of in ((k, seqs.k), (v, seqs.v)):
        assert got.shape == (len(lengths), tokens, heads, dim) and got.is_contiguous()
        for s, x in enumerate(of):
            codes, scale = stored(x[start:start + tokens], fmt)
            want = codes if scale is None else codes.float() * scale[..., None]
            assert torch.equal(got[s, :len(want)].cpu(), want.to(torch.bfloat16))
            assert not got[s, len(want):].any()


def test_zero_tokens_and_zero_sequences():
    seqs = Sequences([20], [0], heads=2, dim=64, seed=9)
    k, v = cache_read(seqs.cache, seqs.plan, 0)
    assert k.shape == v.shape == (1, 0, 2, 64)
    none = PagedPlan.create([], [], [], pages=4, page_size=16).to("cuda")
    k, v = cache_read(seqs.cache, none, 5)
    assert k.shape == (0, 5, 2, 64)
    before = seqs.cache.k.clone()
    cache_write(rows(0, 2, 64, device="cuda"), rows(0, 2, 64, device="cuda"), seqs.cache, seqs.plan)
    cache_write(rows(3, 2, 64, device="cuda"), rows(3, 2, 64, device="cuda"), seqs.cache, none)
    assert torch.equal(seqs.cache.k, before)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_the_plan_does_not_name_stays(fmt):
    # Rows behind the last sequence, pages outside the cache, offsets and lengths outside their ranges.
    cache = PagedCache.create(4, 16, 2, 64, format=fmt)
    fill = rows(64, 2, 64, seed=10, device="cuda")
    full = PagedPlan.create([[0, 1, 2, 3]], [64], [64], pages=4, page_size=16).to("cuda")
    cache_write(fill, fill, cache, full)
    before = [bits(x).clone() for x in (cache.k, cache.v)]
    new = rows(40, 2, 64, seed=11, device="cuda")

    def plan(table, lengths, offsets):
        i32 = dict(dtype=torch.int32, device="cuda")
        return PagedPlan(torch.tensor(table, **i32), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32))

    nothing = [plan([[-1, 4]], [20], [0, 20]), plan([[2 ** 31 - 1, -2 ** 31]], [32], [0, 32]),
               plan([[0, 1]], [-5], [0, 10]), plan([[0, 1]], [0], [0, 10]), plan([[0, 1]], [20], [7, 7]),
               plan([[0, 1]], [20], [30, -3]), plan([[0, 1]], [20], [60, 90])]
    for p in nothing:
        cache_write(new, new, cache, p)
        torch.cuda.synchronize()
        assert torch.equal(bits(cache.k), before[0]) and torch.equal(bits(cache.v), before[1])
    # More new rows than keys: the first ones have no position.  A length past the table is the table's.
    cache_write(new, new, cache, plan([[0, 1]], [3], [0, 20]))
    k, _ = cache_read(cache, full, 64)
    codes, scale = stored(new[17:20], fmt)
    want = (codes if scale is None else codes.float() * scale[..., None]).to(torch.bfloat16)
    assert torch.equal(k[0, :3].cpu(), want)
    cache_write(fill, fill, cache, plan([[0, 1, 2, 3]], [2 ** 31 - 1], [0, 2 ** 31 - 1]))
    assert torch.equal(bits(cache.k), before[0]) and torch.equal(bits(cache.v), before[1])
    k, v = cache_read(cache, plan([[-1, 2]], [2 ** 31 - 1], [0, 0]), 40)
    assert not k[0, :16].any() and not k[0, 32:].any() and torch.equal(k[0, 16:32], cache_read(cache, full, 64)[0][0, 32:48])


def test_rows_behind_the_last_sequence_are_not_written():
    cache = PagedCache.create(2, 16, 2, 64)
    x = rows(9, 2, 64, seed=12, device="cuda")
    plan = PagedPlan.create([[0], [1]], [2, 3], [2, 3], pages=2, page_size=16).to("cuda")
    cache_write(x, x, cache, plan)
    assert torch.equal(cache.k[0, :, :2], x[:2].transpose(0, 1)) and torch.equal(cache.v[1, :, :3], x[2:5].transpose(0, 1))
    assert not cache.k[0, :, 2:].any() and not cache.k[1, :, 3:].any()


@pytest.mark.parametrize("fmt", ("bf16", "int8"))
def test_offsets_past_32_bits(fmt):
    # 2^31 elements and 2^32 bytes into a cache: pages at its far end.
    pages, heads, dim = (1 << 19) + 40, 1, 128
    cache = PagedCache.create(pages, 64, heads, dim, format=fmt)
    far = [pages - 1, 3, pages - 7]
    plan = PagedPlan.create([far], [150], [150], pages=pages, page_size=64).to("cuda")
    x, y = rows(150, heads, dim, seed=13, device="cuda"), rows(150, heads, dim, seed=14, device="cuda")
    cache_write(x, y, cache, plan)
    k, v = cache_read(cache, plan, 150)
    for got, want in ((k, x), (v, y)):
        codes, scale = stored(want, fmt)
        want = (codes if scale is None else codes.float() * scale[..., None]).to(torch.bfloat16)
        assert torch.equal(got[0].cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_capture_follows_the_plan(fmt):
    # One captured step, replayed as the sequences grow: lengths and pages are changed in place between replays.
    heads, dim, page, steps = 2, 64, 16, 5
    cache = PagedCache.create(6, page, heads, dim, format=fmt)
    plan = PagedPlan.create([[0, 1, 2], [3, 4, 5]], [15, 31], [1, 1], pages=6, page_size=page).to("cuda")
    k, v = rows(2, heads, dim, seed=15, device="cuda"), rows(2, heads, dim, seed=16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_write(k, v, cache, plan)
        cache_read(cache, plan, 40)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_write(k, v, cache, plan)
        out = cache_read(cache, plan, 40)
    for step in range(steps):
        k.copy_(rows(2, heads, dim, seed=20 + step))
        v.copy_(rows(2, heads, dim, seed=40 + step))
        graph.replay()
        torch.cuda.synchronize()
        again = cache_read(cache, plan, 40)
        torch.cuda.synchronize()
        for got, eager, new in zip(out, again, (k, v)):
            assert torch.equal(got, eager)
            for s, first in enumerate((15, 31)):
                codes, scale = stored(new[s], fmt)
                want = (codes if scale is None else codes.float() * scale[..., None]).to(torch.bfloat16)
                assert torch.equal(got[s, first - 1 + step].cpu(), want)
        plan.context_lengths.add_(1)


def test_values_stand_for_the_rows():
    # The stored values are within half a step of the rows: 1/254 of the row's largest (INT8), 2^-4 of themselves or, below
    # e4m3's normal range, 2^-10 of its unit (FP8).  The scale's own rounding to FP32 moves a value by 2^-24 of itself:
    # at most 254 * 2^-24 < 2^-16 of such a half step.
    x = rows(40, 2, 128, seed=17)
    for fmt, tol in (("int8", 0.5 / 127), ("fp8", None)):
        off = (values(x, fmt) - x.double()).abs()
        most = x.double().abs().amax(-1, keepdim=True)
        limit = tol * most if tol else 2 ** -4 * x.double().abs() + 2 ** -10 / LEVELS["fp8"] * most
        assert (off <= limit * (1 + 2 ** -16)).all()


def test_a_page_copied_to_another():
    # Rows read from the cache's own pages: a shared page that two sequences go on to write differently.
    seqs = Sequences([30], [30], heads=2, dim=64, page_size=16, seed=50)
    src, dst = seqs.table[0][0], next(p for p in range(seqs.pages) if p not in seqs.table[0])
    k, v = (x[src].transpose(0, 1) for x in (seqs.cache.k, seqs.cache.v))
    copy = PagedPlan.create([[dst]], [16], [16], pages=seqs.pages, page_size=16).to("cuda")
    before = [x.clone() for x in (seqs.cache.k, seqs.cache.v)]
    cache_write(k, v, seqs.cache, copy)
    for x, b in zip((seqs.cache.k, seqs.cache.v), before):
        b[dst] = b[src]
        assert torch.equal(x, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths", [[33, 20], [35, 40], [64, 2 ** 31 - 1]])
def test_a_length_past_the_table_leaves_stored_rows_alone(fmt, lengths):
    # Two sequences of two pages: a step whose lengths have outgrown the table (a captured one replayed too often) drops
    # the tokens past it, and those before keep their places.
    cache = PagedCache.create(4, 16, 2, 64, format=fmt)
    full = PagedPlan.create([[0, 1], [2, 3]], [32, 32], [32, 32], pages=4, page_size=16).to("cuda")
    fill, new = rows(64, 2, 64, seed=60, device="cuda"), rows(6, 2, 64, seed=61, device="cuda")
    cache_write(fill, fill, cache, full)
    want = cache_read(cache, full, 32)[0]
    full.context_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    full.query_offsets.copy_(torch.tensor([0, 2, 6], dtype=torch.int32))
    cache_write(new, new, cache, full)
    codes, scale = stored(new, fmt)
    now = (codes if scale is None else codes.float() * scale[..., None]).to(torch.bfloat16).cuda()
    for s, (length, first, n) in enumerate(zip(lengths, (0, 2), (2, 4))):
        for i in range(n):
            if length - n + i < 32:
                want[s, length - n + i] = now[first + i]
    full.context_lengths.fill_(32)
    for got in cache_read(cache, full, 32):
        assert torch.equal(got, want)
