"""GPU tests of paged_attention and window_attention at their limits: lengths past the page table, values that are not
finite, and calls whose keys are split over workgroups."""

import math

import numpy as np
import pytest
import torch

from paged_testlib import Sequences, assert_within, attend, rows, values
from sol_attn_amd import PagedPlan, paged_attention, window_attention
from sol_testlib import HAS_GPU

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not HAS_GPU, reason="AMD ROCm GPU required")]

FORMATS = ("bf16", "int8", "fp8")


def hand_made(table, lengths, offsets):
    i32 = dict(dtype=torch.int32, device="cuda")
    return PagedPlan(torch.tensor(table, **i32), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32))


def longer(x, length):
    """Rows x [T, H, D] with zeros up to ``length``."""
    return torch.cat([x, x.new_zeros((length - len(x),) + x.shape[1:])])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,new", [(2, 9), (2, 1), (64, 270)])
@pytest.mark.parametrize("causal,window,sinks", [(True, None, 0), (True, 7, 2), (True, 100, 20), (False, 30, 0),
                                                 (False, None, 0)])
def test_a_length_past_the_table(fmt, heads, new, causal, window, sinks):
    # The new tokens keep their positions, and see what the table names of the keys before them.
    seqs = Sequences([288], [0], heads=heads, dim=64, fmt=fmt, page_size=16, seed=1, fill=math.nan)
    length = 288 + 5
    q = rows(new, heads, 64, seed=2, device="cuda")
    out = paged_attention(q, seqs.cache, hand_made([seqs.table[0]], [length], [0, new]), causal=causal, window=window,
                          sink_tokens=sinks)
    some = sorted({0, heads // 3, heads - 1})
    k, v = (longer(values(x[0], fmt)[:, some], length) for x in (seqs.k, seqs.v))
    assert_within(out[:, some], *attend(q[:, some], k, v, causal=causal, window=window, sinks=sinks,
                                        present=np.arange(length) < 288))


@pytest.mark.parametrize("heads,new", [(2, 9), (64, 270)])
def test_the_largest_length(heads, new):
    seqs = Sequences([288], [0], heads=heads, dim=64, page_size=16, seed=3)
    q = rows(new, heads, 64, seed=4, device="cuda")
    plan = hand_made([seqs.table[0]], [2 ** 31 - 1], [0, new])
    some = sorted({0, heads // 3, heads - 1})
    k, v = (x[0][:, some] for x in (seqs.k, seqs.v))
    for causal in (True, False):
        out = paged_attention(q, seqs.cache, plan, causal=causal)
        assert_within(out[:, some], *attend(q[:, some], k, v, causal=False))
        assert not paged_attention(q, seqs.cache, plan, causal=causal, window=1 << 29).any()
        out = paged_attention(q, seqs.cache, plan, causal=causal, window=1 << 29, sink_tokens=33)
        assert_within(out[:, some], *attend(q[:, some], k[:33], v[:33], causal=False))


def assert_same_where_infinite(got, want):
    """Infinities of the same sign, and NaN, in the same places."""
    got = got.detach().cpu().double().numpy()
    assert not np.isfinite(want).all()
    odd = ~np.isfinite(want)
    assert np.array_equal(np.where(odd, got, 0.0), np.where(odd, want, 0.0), equal_nan=True)
    assert np.isfinite(got[~odd]).all()


# Keys whose values are infinite, by feature: in tiles that a query sees whole and in those it sees in part.
INFINITE = ((2, 0, math.inf), (70, 1, -math.inf), (200, 2, math.inf), (210, 2, math.inf), (140, 3, math.inf),
            (90, 3, -math.inf), (299, 4, -math.inf))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,new,heads", [([300, 300], [1, 1], 2), ([300, 300], [9, 40], 2), ([300, 300], [150, 200], 48),
                                               ([9000], [1], 1), ([9000], [300], 2)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 30)])
def test_a_visible_infinity_stays_one(dim, lengths, new, heads, window, sinks):
    # Of the scores here no probability vanishes: every query that sees an infinite value gets it, or NaN for two of
    # opposite signs, whatever the tile.
    seqs = Sequences(lengths, new, heads=heads, dim=dim, page_size=16, seed=5)
    for x in seqs.v:
        for at, feature, bad in INFINITE:
            x[len(x) - 300 + at, 0, feature] = bad
    seqs.store()
    q = rows(sum(new), heads, dim, seed=6, device="cuda")
    out = paged_attention(q, seqs.cache, seqs.plan, window=window, sink_tokens=sinks)
    at = 0
    for k, v, n in zip(seqs.k, seqs.v, new):
        want, _ = attend(q[at:at + n, :1], k[:, :1], v[:, :1], window=window, sinks=sinks)
        assert_same_where_infinite(out[at:at + n, :1], want)
        at += n


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [2, 64])
def test_a_visible_infinity_stays_one_over_plain_keys(dim, heads):
    q, k, v = (rows(1, 300, heads, dim, seed=s) for s in (7, 8, 9))
    for at, feature, bad in INFINITE:
        v[0, at, 0, feature] = bad
    for how in (dict(), dict(causal=False), dict(window=150, sinks=30)):
        named = {("sink_tokens" if n == "sinks" else n): x for n, x in how.items()}
        out = window_attention(q.cuda(), k.cuda(), v.cuda(), **named)[0, :, :1]
        assert_same_where_infinite(out, attend(q[0, :, :1], k[0, :, :1], v[0, :, :1], **how)[0])


def workspace(seqs, q, *, causal=True, window=None, sinks=0):
    """Bytes of partial states that the call takes: more than none where keys are split over workgroups."""
    from sol_attn_amd import _native
    s, width = seqs.plan.page_table.shape
    return _native._paged_size(q.shape[0], s, width, seqs.page_size, q.shape[1], seqs.cache.k.shape[1], q.shape[2],
                               _native.CACHE_FORMATS[seqs.cache.k.dtype], causal, window or 0, sinks)


def check_some(out, q, seqs, picks, heads, **how):
    """Rows ``picks`` of each sequence, K/V heads ``heads``, against the 64-bit form: a causal row is the last of its
    first keys, and without a mask a row's place does not matter."""
    group = q.shape[1] // seqs.cache.k.shape[1]
    cols = [h * group + g for h in heads for g in range(group)]
    at = 0
    for k, v, n in zip(seqs.k, seqs.v, seqs.new):
        k, v = values(k[:, heads], seqs.fmt), values(v[:, heads], seqs.fmt)
        for i in sorted({min(x, n - 1) for x in picks} if n else ()):
            end = len(k) - n + i + 1 if how.get("causal", True) else len(k)
            assert_within(out[at + i:at + i + 1, cols], *attend(q[at + i:at + i + 1, cols], k[:end], v[:end], **how))
        at += n


PICKS = (0, 31, 63, 64, 150, 200, 298, 309)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("how", [dict(), dict(window=3000, sinks=70), dict(causal=False)])
def test_ragged_chunks_in_no_one_and_several_parts(fmt, dim, how):
    # Parts of 24 key tiles: three, one, none, two, one, two and one per row tile.
    seqs = Sequences([3600, 700, 0, 1900, 300, 2300, 1200], [300, 250, 0, 310, 300, 1, 299], heads=16, dim=dim, fmt=fmt,
                     page_size=16, seed=10)
    q = rows(sum(seqs.new), 32, dim, seed=11, device="cuda")
    assert workspace(seqs, q, **how) > 0
    named = {("sink_tokens" if n == "sinks" else n): x for n, x in how.items()}
    check_some(paged_attention(q, seqs.cache, seqs.plan, **named), q, seqs, PICKS, [0, 7, 15], **how)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_one_chunk_in_many_parts(fmt, dim, heads, causal):
    # Row tiles of 128 rows: 300 of a head over 9,000 keys are more than calls of 16-row tiles read.
    seqs = Sequences([9000], [300], heads=heads, dim=dim, fmt=fmt, page_size=64, seed=12)
    q = rows(300, heads, dim, seed=13, device="cuda")
    assert workspace(seqs, q, causal=causal) >= 2 * 3 * heads * 128 * (dim + 4) * 4
    check_some(paged_attention(q, seqs.cache, seqs.plan, causal=causal), q, seqs, (0, 127, 128, 256, 299),
               list(range(heads)), causal=causal)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new,group", [(1, 3), (40, 2)])
def test_a_few_long_sequences_among_hundreds(fmt, new, group):
    # More sequences than a workgroup has threads, of which some in their middle and the last one are split.
    lengths = [new + (37 * i) % 60 for i in range(300)]
    for at in (3, 4, 100, 255, 256, 299):
        lengths[at] = 3000 + 11 * at
    seqs = Sequences(lengths, [new] * 300, heads=2, dim=64, fmt=fmt, page_size=16, seed=14)
    q = rows(300 * new, 2 * group, 64, seed=15, device="cuda")
    assert workspace(seqs, q) > 0
    check_some(paged_attention(q, seqs.cache, seqs.plan), q, seqs, (0, 39), [0, 1])


@pytest.mark.parametrize("new,heads", [(1, 2), (300, 16)])
def test_replays_that_split_other_sequences(new, heads):
    # One captured call: its lengths change, and with them which sequences are split, all or none of them.
    most = [3600, 3400, 3200]
    whole = Sequences(most, [new] * 3, heads=heads, dim=64, page_size=16, seed=16)
    q = rows(3 * new, 2 * heads, 64, seed=17, device="cuda")
    assert workspace(whole, q) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_attention(q, whole.cache, whole.plan)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, whole.cache, whole.plan)
    kv = whole.k, whole.v
    for lengths in (most, [310, 305, 300], [310, 3400, 300], [3600, 300, 300], [300, 300, 3200], [0, 0, 0], most):
        whole.plan.context_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention(q, whole.cache, whole.plan))
        torch.cuda.synchronize()
        if lengths == [0, 0, 0]:
            assert not out.any()
            continue
        whole.k, whole.v = ([x[:n] for x, n in zip(of, lengths)] for of in kv)
        check_some(out, q, whole, (0, 150, 299), [0, heads - 1])
