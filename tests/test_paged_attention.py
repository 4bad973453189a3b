"""GPU tests of paged_attention and window_attention against their 64-bit forms."""

import math

import pytest
import torch

from paged_testlib import Sequences, assert_within, attend, rows
from sol_attn_amd import (PagedCache, PagedPlan, cache_read, cache_write, dense_attention, paged_attention,
                          sol_attention, window_attention)
from sol_testlib import HAS_GPU

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not HAS_GPU, reason="AMD ROCm GPU required")]

FORMATS = ("bf16", "int8", "fp8")


def check(seqs, q, **how):
    named = dict(how)
    if "sinks" in named:
        named["sink_tokens"] = named.pop("sinks")
    out = paged_attention(q, seqs.cache, seqs.plan, **named)
    assert_within(out, *seqs.expected(q, **how))
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (64, 256), (128, 32)])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 8), (3, 3), (2, 12)])
def test_single_tokens(fmt, dim, page, heads, group):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 128, 300, 511, 1025]
    seqs = Sequences(lengths, [1] * len(lengths), heads=heads, dim=dim, fmt=fmt, page_size=page, seed=1, fill=math.nan)
    check(seqs, rows(len(lengths), heads * group, dim, seed=2, device="cuda"))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page,heads,group", [(64, 16, 2, 1), (128, 64, 1, 4), (128, 16, 2, 3)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 3), (64, 64), (100, 1), (65, 200), (1000, 0)])
def test_chunks_under_a_window(fmt, dim, page, heads, group, causal, window, sinks):
    lengths, new = [70, 1, 0, 200, 64, 333, 130], [70, 1, 0, 33, 64, 5, 129]
    seqs = Sequences(lengths, new, heads=heads, dim=dim, fmt=fmt, page_size=page, seed=3, fill=math.nan)
    check(seqs, rows(sum(new), heads * group, dim, seed=4, device="cuda"), causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("causal", [True, False])
def test_a_long_chunk(fmt, causal):
    seqs = Sequences([700, 450], [389, 450], heads=1, dim=128, fmt=fmt, page_size=64, seed=5)
    check(seqs, rows(839, 2, 128, seed=6, device="cuda"), causal=causal)
    check(seqs, rows(839, 2, 128, seed=7, device="cuda"), causal=causal, window=150, sinks=70)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_long_cache_with_few_rows(fmt, dim):
    # The keys are split over many workgroups.
    seqs = Sequences([9001, 3, 700], [1, 1, 1], heads=1, dim=dim, fmt=fmt, page_size=64, seed=8)
    q = rows(3, 5, dim, seed=9, device="cuda")
    check(seqs, q)
    check(seqs, q, window=4000, sinks=130)
    seqs = Sequences([6000], [40], heads=1, dim=dim, fmt=fmt, page_size=16, seed=10)
    check(seqs, rows(40, 3, dim, seed=11, device="cuda"))


def test_one_step_among_long_prompts():
    # Single tokens and chunks of several sequences in one call.
    lengths, new = [900, 500, 64, 1, 777, 300], [1, 400, 64, 1, 1, 2]
    seqs = Sequences(lengths, new, heads=2, dim=128, page_size=32, seed=12)
    check(seqs, rows(sum(new), 4, 128, seed=13, device="cuda"))
    lengths, new = [40 + i for i in range(60)] + [300], [1] * 60 + [260]
    seqs = Sequences(lengths, new, heads=1, dim=64, page_size=16, seed=14)
    check(seqs, rows(sum(new), 1, 64, seed=15, device="cuda"))


def test_many_sequences():
    lengths = [1 + (7 * i) % 90 for i in range(1300)]
    new = [i % 3 if lengths[i] > 2 else 1 for i in range(1300)]
    seqs = Sequences(lengths, new, heads=1, dim=64, page_size=16, seed=16)
    check(seqs, rows(sum(new), 1, 64, seed=17, device="cuda"))


def check_sampled(out, q, ks, vs, new, picks, **how):
    """Some rows of each sequence against the 64-bit form: row i of a causal sequence is the last of its first keys."""
    at = 0
    for k, v, n in zip(ks, vs, new):
        for i in sorted({min(x, n - 1) for x in picks} if n else ()):
            end = len(k) - n + i + 1
            assert_within(out[at + i:at + i + 1], *attend(q[at + i:at + i + 1], k[:end], v[:end], **how))
        at += n


@pytest.mark.parametrize("fmt", FORMATS)
def test_chunks_split_by_lengths_that_differ(fmt):
    # Enough keys that parts of one size even the sequences out: one, two or no parts a row tile.
    lengths, new = [2600, 700, 0, 1900, 300, 2300, 1200], [300, 250, 0, 310, 300, 1, 299]
    seqs = Sequences(lengths, new, heads=16, dim=64, fmt=fmt, page_size=16, seed=84)
    q = rows(sum(new), 32, 64, seed=85, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan)
    from paged_testlib import values
    check_sampled(out, q, [values(x, fmt) for x in seqs.k], [values(x, fmt) for x in seqs.v], new, (0, 63, 64, 200, 309))


@pytest.mark.parametrize("dim", [64, 128])
def test_one_chunk_split_into_many_parts(dim):
    # Several row tiles, up to 32 parts each; the last tile is not full.
    seqs = Sequences([9000], [300], heads=2, dim=dim, page_size=64, seed=86)
    q = rows(300, 2, dim, seed=87, device="cuda")
    check_sampled(paged_attention(q, seqs.cache, seqs.plan), q, seqs.k, seqs.v, [300], (0, 127, 128, 256, 299))
    out = paged_attention(q, seqs.cache, seqs.plan, causal=False)
    for i in (0, 128, 299):  # without a mask a row's place does not matter
        assert_within(out[i:i + 1], *attend(q[i:i + 1], seqs.k[0], seqs.v[0], causal=False))


def test_a_plain_triangle_split_into_parts():
    q, k, v = (rows(1, 2600, 32, 64, seed=s, device="cuda") for s in (88, 89, 90))
    out = window_attention(q, k, v)
    check_sampled(out[0], q[0], k, v, [2600], (0, 1, 127, 1000, 2047, 2048, 2599))


def test_two_streams_at_once():
    # Calls that split their keys, side by side on two streams, each with partial states of its own.
    seqs = [Sequences(n, m, heads=2, dim=64, page_size=16, seed=91 + i)
            for i, (n, m) in enumerate((([4000, 90], [130, 1]), ([5000, 3800], [1, 1])))]
    q = [rows(sum(s.new), 4, 64, seed=93, device="cuda") for s in seqs]
    good = [check(s, x) for s, x in zip(seqs, q)]
    streams = [torch.cuda.Stream() for _ in seqs]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_attention(q[i], seqs[i].cache, seqs[i].plan))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, good[i]) for x in outs[i])


def test_thousands_of_sequences():
    # More than the workgroup's threads, several times; single tokens, then some of two.
    lengths = [1 + (11 * i) % 40 for i in range(5000)]
    for new in ([1] * 5000, [1 + (i % 7 == 3) * (lengths[i] > 1) for i in range(5000)]):
        seqs = Sequences(lengths, new, heads=1, dim=64, page_size=16, seed=95)
        check(seqs, rows(sum(new), 1, 64, seed=96, device="cuda"))


@pytest.mark.parametrize("tq,tk", [(1, 40), (3, 9000), (70, 6000)])
@pytest.mark.parametrize("batch", [1, 5, 300])
def test_window_over_many_entries(batch, tq, tk):
    if batch == 300:
        tk = min(tk, 700)
    q, k, v = rows(batch, tq, 2, 64, seed=97), rows(batch, tk, 1, 64, seed=98), rows(batch, tk, 1, 64, seed=99)
    out = window_attention(q.cuda(), k.cuda(), v.cuda())
    for b in sorted({0, batch // 2, batch - 1}):
        assert_within(out[b], *attend(q[b], k[b], v[b]))


def test_scale_strides_and_misaligned_queries():
    seqs = Sequences([100, 30], [20, 3], heads=2, dim=64, seed=18)
    wide = rows(23, 8, 64, seed=19, device="cuda")
    check(seqs, wide[:, ::2], scale=0.3)
    odd = torch.zeros(23 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(23, 4, 64)
    odd.copy_(wide[:, 1::2])
    check(seqs, odd)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_small_and_large_scores(fmt, size):
    # Scores of a few thousand: the running maximum jumps, most probabilities vanish.
    seqs = Sequences([400, 130], [140, 1], heads=1, dim=64, fmt=fmt, page_size=16, seed=20)
    q = (rows(141, 2, 64, seed=21).float() * size).to(torch.bfloat16).cuda()
    check(seqs, q)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_scores_that_rise_or_fall_along_the_keys(order):
    n = 2000
    seqs = Sequences([n], [4], heads=1, dim=64, page_size=16, seed=22)
    ramp = torch.linspace(-40, 40, n) if order == "rising" else torch.linspace(40, -40, n)
    seqs.k[0][:, 0, 0] = ramp.to(torch.bfloat16)
    seqs.store()
    q = rows(4, 2, 64, seed=23)
    q[..., 0] = 16
    check(seqs, q.cuda())


@pytest.mark.parametrize("causal,window,sinks", [(True, None, 0), (True, 40, 3), (False, 40, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_never_reach_a_result(causal, window, sinks, bad):
    # A few keys and values are NaN or infinite: queries that do not see them are as if they were not there.
    lengths, new = [150, 300], [150, 40]
    seqs = Sequences(lengths, new, heads=2, dim=64, page_size=16, seed=24, fill=math.nan)
    for s, at in ((0, 77), (0, 140), (1, 2), (1, 230), (1, 290)):
        seqs.v[s][at, s] = bad
        if bad != bad:
            seqs.k[s][at, s] = bad
    seqs.store()
    q = rows(190, 4, 64, seed=25, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan, causal=causal, window=window, sink_tokens=sinks)
    expected, bound = seqs.expected(q, causal=causal, window=window, sinks=sinks)
    fine = torch.isfinite(torch.from_numpy(expected)).numpy()
    assert fine.any() and not fine.all()
    got = out.double().cpu().numpy()
    assert not (abs(got - expected)[fine] > bound[fine]).any()
    assert not torch.isfinite(torch.from_numpy(got[~fine])).any()


@pytest.mark.parametrize("fmt", ("int8", "fp8"))
def test_a_stored_row_that_is_nan_hides_behind_the_mask(fmt):
    seqs = Sequences([90], [60], heads=1, dim=64, fmt=fmt, page_size=16, seed=26, fill=math.nan)
    seqs.k[0][70, 0, 3] = math.inf
    seqs.v[0][70, 0, 9] = math.nan
    seqs.store()
    q = rows(60, 2, 64, seed=27, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan)
    assert torch.isfinite(out[:40]).all() and out[40:].isnan().all()
    assert_within(out[:40], *(x[:40] for x in seqs.expected(q)))


def hand_made(table, lengths, offsets):
    i32 = dict(dtype=torch.int32, device="cuda")
    return PagedPlan(torch.tensor(table, **i32), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_see_nothing_are_zeros_and_rows_behind_stay(fmt):
    seqs = Sequences([40, 8], [12, 2], heads=2, dim=64, fmt=fmt, page_size=16, seed=28)
    q = rows(20, 4, 64, seed=29, device="cuda")
    out = torch.full_like(q, 7.0)
    assert paged_attention(q, seqs.cache, seqs.plan, out=out) is out
    assert_within(out[:14], *seqs.expected(q[:14]))
    assert (out[14:] == 7.0).all()
    # Fewer keys than new rows: the first ones have positions before the first key.
    out = torch.full_like(q, 7.0)
    plan = hand_made([seqs.table[0]], [5], [0, 12])
    paged_attention(q, seqs.cache, plan, out=out)
    assert not out[:7].any() and (out[12:] == 7.0).all()
    k, v = (x[0] for x in cache_read(seqs.cache, hand_made([seqs.table[0]], [5], [0, 0]), 5))
    if fmt == "bf16":
        assert_within(out[7:12], *attend(q[7:12], k, v))
    out = torch.full_like(q, 7.0)
    paged_attention(q, seqs.cache, hand_made([seqs.table[0]], [0], [0, 12]), out=out, causal=False)
    assert not out[:12].any() and (out[12:] == 7.0).all()


def test_pages_outside_the_cache_are_not_attended():
    seqs = Sequences([100], [9], heads=2, dim=64, page_size=16, seed=30)
    q = rows(9, 4, 64, seed=31, device="cuda")
    for gone in ([1], [0, 3], [6], [0, 1, 2, 3, 4, 5, 6]):
        table = list(seqs.table[0])
        present = torch.ones(100, dtype=torch.bool).numpy()
        for i, g in enumerate(gone):
            table[g] = (-1, seqs.pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
            present[16 * g:16 * g + 16] = False
        out = paged_attention(q, seqs.cache, hand_made([table], [100], [0, 9]))
        assert_within(out, *attend(q, seqs.k[0], seqs.v[0], present=present))


def test_offsets_outside_their_range():
    seqs = Sequences([40, 8], [12, 2], heads=1, dim=64, page_size=16, seed=32)
    q = rows(14, 2, 64, seed=33, device="cuda")
    good = paged_attention(q, seqs.cache, seqs.plan)
    table = seqs.plan.page_table.tolist()
    out = torch.full_like(q, 7.0)
    paged_attention(q, seqs.cache, hand_made(table, [40, 8], [-5, 12, 2 ** 31 - 1]), out=out)
    assert torch.equal(out, good)
    for offsets in ([0, 0, 0], [14, 3, 0], [50, 60, 70], [-9, -8, -7]):
        out = torch.full_like(q, 7.0)
        paged_attention(q, seqs.cache, hand_made(table, [2 ** 31 - 1, -4], offsets), out=out)
        torch.cuda.synchronize()
        if offsets != [14, 3, 0]:
            assert (out == 7.0).all()


def test_empty_calls():
    seqs = Sequences([40], [0], heads=1, dim=64, seed=34)
    assert paged_attention(rows(0, 2, 64, device="cuda"), seqs.cache, seqs.plan).shape == (0, 2, 64)
    none = PagedPlan.create([], [], [], pages=4, page_size=16).to("cuda")
    out = torch.full((3, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    paged_attention(rows(3, 2, 64, device="cuda"), seqs.cache, none, out=out)
    assert (out == 7.0).all()


def test_offsets_past_32_bits():
    pages = (1 << 19) + 40
    cache = PagedCache.create(pages, 64, 1, 128)
    far = [pages - 1, 3, pages - 7]
    plan = PagedPlan.create([far], [150], [150], pages=pages, page_size=64).to("cuda")
    k, v = rows(150, 1, 128, seed=35, device="cuda"), rows(150, 1, 128, seed=36, device="cuda")
    cache_write(k, v, cache, plan)
    q = rows(150, 2, 128, seed=37, device="cuda")
    assert_within(paged_attention(q, cache, plan), *attend(q, k, v))
    one = hand_made([far], [150], [0, 1])
    assert_within(paged_attention(q[:1], cache, one), *attend(q[:1], k, v))


def run_window(q, k, v, **how):
    named = dict(how)
    named["sink_tokens"] = named.pop("sinks", 0)
    out = window_attention(q, k, v, **named)
    for b in range(q.shape[0]):
        assert_within(out[b], *attend(q[b], k[b], v[b], **how))
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 300), (5, 64), (64, 65), (193, 317), (200, 200), (300, 40)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (33, 2), (64, 100)])
def test_window(dim, tq, tk, causal, window, sinks):
    q, k, v = rows(2, tq, 4, dim, seed=1), rows(2, tk, 2, dim, seed=2), rows(2, tk, 2, dim, seed=3)
    run_window(q.cuda(), k.cuda(), v.cuda(), causal=causal, window=window, sinks=sinks)


def test_window_over_strided_heads_and_batches():
    q, k, v = rows(3, 130, 6, 64, seed=4), rows(3, 260, 6, 64, seed=5), rows(3, 260, 6, 64, seed=6)
    q, k, v = q.cuda()[:, :, ::2], k.cuda()[:, ::2, ::2], v.cuda()[:, 1::2, 1::2]
    run_window(q, k, v, causal=False, window=20, sinks=4)
    run_window(q, k, v)
    odd = torch.zeros(3 * 130 * 3 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 130, 3, 64)
    odd.copy_(k)
    run_window(q, odd, v, window=20)


def test_window_of_everything_is_dense_attention():
    q, k, v = (rows(1, n, 2, 128, seed=s, device="cuda") for s, n in ((7, 150), (8, 400), (9, 400)))
    out = run_window(q, k, v, causal=False)
    torch.testing.assert_close(out, dense_attention(q, k, v), rtol=2 ** -6, atol=2 ** -7)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_window_hides_values(bad):
    q, k, v = rows(1, 200, 2, 64, seed=10), rows(1, 200, 1, 64, seed=11), rows(1, 200, 1, 64, seed=12)
    v[0, 90, 0, 5] = bad
    v[0, 199, 0, 60] = -bad
    if bad != bad:
        k[0, 90] = bad
    out = window_attention(q.cuda(), k.cuda(), v.cuda(), window=30, sink_tokens=2).double().cpu().numpy()[0]
    expected, bound = attend(q[0], k[0], v[0], window=30, sinks=2)
    fine = torch.isfinite(torch.from_numpy(expected)).numpy()
    assert not (abs(out - expected)[fine] > bound[fine]).any()
    assert not torch.isfinite(torch.from_numpy(out[~fine])).any()
    assert fine[:90].all() and not fine[90:120].all()


def test_side_stream():
    seqs = Sequences([500, 90], [70, 1], heads=2, dim=128, page_size=64, seed=38)
    q = rows(71, 4, 128, seed=39, device="cuda")
    good = paged_attention(q, seqs.cache, seqs.plan)
    step = hand_made(seqs.plan.page_table.tolist(), [500, 90], [0, 1, 2])
    one = paged_attention(q[:2], seqs.cache, step)
    plain = window_attention(q[None], q[None], q[None], window=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = (paged_attention(q, seqs.cache, seqs.plan), paged_attention(q[:2], seqs.cache, step),
                window_attention(q[None], q[None], q[None], window=9))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(outs, (good, one, plain)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 37])
def test_captured_steps_follow_the_plan(fmt, new):
    # A step (write, attend) captured once and replayed as the sequences grow, against eager calls on a second cache;
    # a second graph shares nothing with it.
    heads, dim, page = 2, 64, 16
    make = lambda: PagedCache.create(40, page, heads, dim, format=fmt)  # noqa: E731
    table = [list(range(20)), list(range(20, 40))]
    first = [new + 60, new]
    plan = PagedPlan.create(table, first, [new, new], pages=40, page_size=page).to("cuda")
    history = rows(60, heads, dim, seed=40, device="cuda")
    start = PagedPlan.create(table, [60, 0], [60, 0], pages=40, page_size=page).to("cuda")
    caches = [make(), make(), make()]
    for c in caches:
        cache_write(history, history, c, start)
    q, k, v = (rows(2 * new, n, dim, seed=s, device="cuda") for s, n in ((41, 6), (42, heads), (43, heads)))

    def step(cache):
        cache_write(k, v, cache, plan)
        return paged_attention(q, cache, plan, window=50, sink_tokens=4), paged_attention(q, cache, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in caches[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for i in range(4):
        for x, s in ((q, 50), (k, 60), (v, 70)):
            x.copy_(rows(*x.shape, seed=s + i))
        for out in outs:
            for o in out:
                o.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        eager = step(caches[2])
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
        plan.context_lengths.add_(new)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_sequence_generated_piece_by_piece(fmt):
    # As a model runs them: a prompt, frames whose tokens see one another, single tokens; then the whole sequence is
    # read back and attended by the plain operators.
    heads, group, dim, page = 2, 2, 128, 64
    cache = PagedCache.create(16, page, heads, dim, format=fmt)
    k, v = rows(500, heads, dim, seed=80, device="cuda"), rows(500, heads, dim, seed=81, device="cuda")
    q = rows(500, heads * group, dim, seed=82, device="cuda")
    table = [[5, 9, 0, 3, 11, 2, 7, 1]]
    at = 0
    from paged_testlib import values
    kv = [values(x, fmt) for x in (k, v)]
    for n, causal in ((130, True), (84, False), (84, False), (84, False), (1, True), (1, True), (97, True)):
        plan = PagedPlan.create(table, [at + n], [n], pages=16, page_size=page).to("cuda")
        cache_write(k[at:at + n], v[at:at + n], cache, plan)
        how = dict(causal=causal, window=200, sinks=64)
        out = paged_attention(q[at:at + n], cache, plan, causal=causal, window=200, sink_tokens=64)
        assert_within(out, *attend(q[at:at + n], kv[0][:at + n], kv[1][:at + n], **how))
        at += n
    back = cache_read(cache, plan, at)
    assert all(x.shape == (1, at, heads, dim) for x in back)
    qh = q[None, :at, ::group].contiguous()
    dense = dense_attention(qh, *back)
    assert_within(dense[0], *attend(qh[0], back[0][0], back[1][0], causal=False))
    torch.testing.assert_close(sol_attention(qh, *back, beta=-math.inf), dense)
    assert_within(window_attention(q[None, :at], *back, window=200, sink_tokens=64)[0],
                  *attend(q[:at], back[0][0], back[1][0], window=200, sinks=64))
