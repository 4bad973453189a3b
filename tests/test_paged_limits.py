"""GPU tests of paged_attention and window_attention at their limits: lengths past the page table, values that are not
finite, and calls whose keys are split over workgroups."""

import math

import numpy as np
import pytest
import torch

from paged_testlib import Sequences, assert_within, attend, rows, values
from sol_attn_amd import PagedPlan, paged_attention
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
