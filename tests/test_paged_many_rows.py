"""GPU tests of paged_attention and window_attention at sizes that take tiles of 128 rows: more than 1,024 tiles of 16
rows over all heads.  A few of the heads are compared with the 64-bit forms."""

import math

import pytest
import torch

from paged_testlib import Sequences, assert_within, attend, rows, values
from sol_attn_amd import PagedPlan, paged_attention, window_attention
from sol_testlib import HAS_GPU

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not HAS_GPU, reason="AMD ROCm GPU required")]

FORMATS = ("bf16", "int8", "fp8")


def some(heads):
    return sorted({0, heads // 3, heads - 1})


def of_heads(q, heads, group):
    """The query heads of the K/V heads that are compared."""
    return torch.cat([q[..., h * group:(h + 1) * group, :] for h in some(heads)], -2)


def expected(q, ks, vs, new, group, **how):
    """(O, bound) of the compared heads, sequence by sequence."""
    at, outs = 0, []
    heads = ks[0].shape[1]
    for k, v, n in zip(ks, vs, new):
        if n:
            outs.append(attend(of_heads(q[at:at + n], heads, group), k[:, some(heads)], v[:, some(heads)], **how))
        at += n
    return tuple(torch.cat([torch.from_numpy(o[i]) for o in outs]).numpy() for i in (0, 1))


def check(seqs, q, heads, group, **how):
    named = dict(how)
    named["sink_tokens"] = named.pop("sinks", 0)
    out = paged_attention(q, seqs.cache, seqs.plan, **named)
    kv = [[values(x, seqs.fmt) for x in side] for side in (seqs.k, seqs.v)]
    assert_within(of_heads(out, heads, group), *expected(q, *kv, seqs.new, group, **how))
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,page,heads,group", [(64, 16, 60, 1), (128, 64, 24, 3)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 3), (100, 1), (65, 200)])
def test_chunks_under_a_window(fmt, dim, page, heads, group, causal, window, sinks):
    lengths, new = [150, 1, 0, 200, 64, 333, 130], [70, 1, 0, 77, 64, 33, 129]
    seqs = Sequences(lengths, new, heads=heads, dim=dim, fmt=fmt, page_size=page, seed=3, fill=math.nan)
    check(seqs, rows(sum(new), heads * group, dim, seed=4, device="cuda"), heads, group, causal=causal, window=window,
          sinks=sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_whole_tiles(fmt, dim, causal):
    # Key tiles that all rows of a wave see, some of them only of one wave.
    seqs = Sequences([700, 450], [389, 450], heads=24, dim=dim, fmt=fmt, page_size=64, seed=5)
    q = rows(839, 24, dim, seed=6, device="cuda")
    check(seqs, q, 24, 1, causal=causal)
    check(seqs, q, 24, 1, causal=causal, window=150, sinks=70)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_small_and_large_scores(fmt, size):
    # Scores of a few thousand: the running maximum jumps, most probabilities vanish.
    seqs = Sequences([400, 130], [280, 100], heads=48, dim=64, fmt=fmt, page_size=16, seed=20)
    q = (rows(380, 48, 64, seed=21).float() * size).to(torch.bfloat16).cuda()
    check(seqs, q, 48, 1)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_scores_that_rise_or_fall_along_the_keys(order):
    n = 900
    seqs = Sequences([n], [300], heads=64, dim=64, page_size=16, seed=22)
    ramp = torch.linspace(-40, 40, n) if order == "rising" else torch.linspace(40, -40, n)
    seqs.k[0][:, :, 0] = ramp.to(torch.bfloat16)[:, None]
    seqs.store()
    q = rows(300, 64, 64, seed=23)
    q[..., 0] = 16
    check(seqs, q.cuda(), 64, 1)


@pytest.mark.parametrize("causal,window,sinks", [(True, None, 0), (True, 40, 3), (False, 40, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_never_reach_a_result(causal, window, sinks, bad):
    lengths, new = [150, 300], [150, 140]
    seqs = Sequences(lengths, new, heads=60, dim=64, page_size=16, seed=24, fill=math.nan)
    for s, at in ((0, 77), (0, 140), (1, 2), (1, 230), (1, 290)):
        seqs.v[s][at, 20 * s] = bad
        if bad != bad:
            seqs.k[s][at, 20 * s] = bad
    seqs.store()
    q = rows(290, 60, 64, seed=25, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan, causal=causal, window=window, sink_tokens=sinks)
    want, bound = expected(q, seqs.k, seqs.v, new, 1, causal=causal, window=window, sinks=sinks)
    fine = torch.isfinite(torch.from_numpy(want)).numpy()
    assert fine.any() and not fine.all()
    got = of_heads(out, 60, 1).double().cpu().numpy()
    assert not (abs(got - want)[fine] > bound[fine]).any()
    assert not torch.isfinite(torch.from_numpy(got[~fine])).any()


@pytest.mark.parametrize("fmt", ("int8", "fp8"))
def test_a_stored_row_that_is_nan_hides_behind_the_mask(fmt):
    seqs = Sequences([290], [260], heads=64, dim=64, fmt=fmt, page_size=16, seed=26, fill=math.nan)
    seqs.k[0][170, 0, 3] = math.inf
    seqs.v[0][170, 0, 9] = math.nan
    seqs.store()
    q = rows(260, 64, 64, seed=27, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan)
    assert torch.isfinite(out[:140]).all() and out[140:, 0].isnan().all() and torch.isfinite(out[140:, 1:]).all()
    kv = [[values(x, fmt) for x in side] for side in (seqs.k, seqs.v)]
    assert_within(of_heads(out, 64, 1), *expected(q, *kv, [260], 1))


def hand_made(table, lengths, offsets):
    i32 = dict(dtype=torch.int32, device="cuda")
    return PagedPlan(torch.tensor(table, **i32), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_see_nothing_are_zeros_and_rows_behind_stay(fmt):
    seqs = Sequences([300, 8], [290, 2], heads=60, dim=64, fmt=fmt, page_size=16, seed=28)
    q = rows(300, 60, 64, seed=29, device="cuda")
    out = torch.full_like(q, 7.0)
    assert paged_attention(q, seqs.cache, seqs.plan, out=out) is out
    kv = [[values(x, fmt) for x in side] for side in (seqs.k, seqs.v)]
    assert_within(of_heads(out[:292], 60, 1), *expected(q[:292], *kv, seqs.new, 1))
    assert (out[292:] == 7.0).all()
    # Fewer keys than new rows: the first ones have positions before the first key.
    out = torch.full_like(q, 7.0)
    paged_attention(q, seqs.cache, hand_made([seqs.table[0]], [150], [0, 290]), out=out)
    assert not out[:140].any() and (out[290:] == 7.0).all()
    assert_within(of_heads(out[140:290], 60, 1), *expected(q[140:290], [kv[0][0][:150]], [kv[1][0][:150]], [150], 1))
    out = torch.full_like(q, 7.0)
    paged_attention(q, seqs.cache, hand_made([seqs.table[0]], [0], [0, 290]), out=out, causal=False)
    assert not out[:290].any() and (out[290:] == 7.0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_outside_the_cache_are_not_attended(fmt):
    seqs = Sequences([300], [270], heads=64, dim=64, fmt=fmt, page_size=16, seed=30)
    q = rows(270, 64, 64, seed=31, device="cuda")
    k, v = (values(x[0], fmt) for x in (seqs.k, seqs.v))
    for gone in ([1], [0, 3], [18], list(range(19))):
        table = list(seqs.table[0])
        present = torch.ones(300, dtype=torch.bool).numpy()
        for i, g in enumerate(gone):
            table[g] = (-1, seqs.pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
            present[16 * g:16 * g + 16] = False
        out = paged_attention(q, seqs.cache, hand_made([table], [300], [0, 270]))
        assert_within(of_heads(out, 64, 1), *expected(q, [k], [v], [270], 1, present=present))


def test_offsets_outside_their_range():
    seqs = Sequences([300, 8], [290, 2], heads=60, dim=64, page_size=16, seed=32)
    q = rows(292, 60, 64, seed=33, device="cuda")
    good = paged_attention(q, seqs.cache, seqs.plan)
    table = seqs.plan.page_table.tolist()
    out = torch.full_like(q, 7.0)
    paged_attention(q, seqs.cache, hand_made(table, [300, 8], [-5, 290, 2 ** 31 - 1]), out=out)
    assert torch.equal(out, good)
    for offsets in ([0, 0, 0], [292, 30, 0], [500, 600, 700], [-9, -8, -7]):
        out = torch.full_like(q, 7.0)
        paged_attention(q, seqs.cache, hand_made(table, [2 ** 31 - 1, -4], offsets), out=out)
        torch.cuda.synchronize()
        if offsets != [292, 30, 0]:
            assert (out == 7.0).all()


def window_expected(q, k, v, group, **how):
    heads = k.shape[1]
    return attend(of_heads(q, heads, group), k[:, some(heads)], v[:, some(heads)], **how)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tq,tk", [(193, 317), (257, 257), (300, 40)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (33, 2), (64, 100)])
def test_window(dim, tq, tk, causal, window, sinks):
    q, k, v = rows(2, tq, 48, dim, seed=1), rows(2, tk, 24, dim, seed=2), rows(2, tk, 24, dim, seed=3)
    out = window_attention(q.cuda(), k.cuda(), v.cuda(), causal=causal, window=window, sink_tokens=sinks)
    for b in range(2):
        assert_within(of_heads(out[b], 24, 2), *window_expected(q[b], k[b], v[b], 2, causal=causal, window=window,
                                                                sinks=sinks))


def test_window_over_strided_heads_and_batches():
    q, k, v = rows(2, 260, 96, 64, seed=4), rows(2, 600, 96, 64, seed=5), rows(2, 600, 96, 64, seed=6)
    q, k, v = q.cuda()[:, :, ::2], k.cuda()[:, ::2, ::2], v.cuda()[:, 1::2, 1::2]
    for how in (dict(causal=False, window=20, sinks=4), dict()):
        named = {("sink_tokens" if n == "sinks" else n): x for n, x in how.items()}
        out = window_attention(q, k, v, **named)
        for b in range(2):
            assert_within(of_heads(out[b], 48, 1), *window_expected(q[b], k[b], v[b], 1, **how))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_window_hides_values(bad):
    q, k, v = rows(1, 300, 64, 64, seed=10), rows(1, 300, 64, 64, seed=11), rows(1, 300, 64, 64, seed=12)
    v[0, 90, 0, 5] = bad
    v[0, 299, 0, 60] = -bad
    if bad != bad:
        k[0, 90, 0] = bad
    out = window_attention(q.cuda(), k.cuda(), v.cuda(), window=30, sink_tokens=2)[0]
    want, bound = window_expected(q[0], k[0], v[0], 1, window=30, sinks=2)
    got = of_heads(out, 64, 1).double().cpu().numpy()
    fine = torch.isfinite(torch.from_numpy(want)).numpy()
    assert not (abs(got - want)[fine] > bound[fine]).any()
    assert not torch.isfinite(torch.from_numpy(got[~fine])).any()
    assert fine[:90].all() and not fine[90:120].all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_captured_chunk_follows_the_plan(fmt):
    seqs = Sequences([900, 400], [260, 120], heads=48, dim=64, fmt=fmt, page_size=16, seed=34)
    q = rows(380, 48, 64, seed=35, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_attention(q, seqs.cache, seqs.plan)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, seqs.cache, seqs.plan)
    for lengths in ([900, 400], [300, 350], [260, 400], [777, 121]):
        seqs.plan.context_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, seqs.cache, seqs.plan))
