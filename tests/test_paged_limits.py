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
