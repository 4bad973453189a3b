"""The operators together, as a program that generates with drafts uses them: rows normed and turned, stored, attended
as a tree, the accepted ones kept, the sequences continued and branched, and attended again, eager and replayed,
against the sequences written out plainly in 64 bits."""

import numpy as np
import pytest
import torch

from paged_testlib import assert_within, attend, rows, values
from sol_attn_amd import (PagedCache, PagedPlan, PagePool, RotaryAxes, cache_fork, cache_keep, cache_write,
                          paged_attention, rotate_heads, tree_attention)
from tree_testlib import attend_seen, seen_by

HQ, H, D, PAGE = 4, 2, 64, 16


class Model:
    """Rows of Q, K and V for tokens of a small vocabulary (a token's rows do not depend on its place before they are
    turned)."""

    def __init__(self, fmt):
        self.fmt = fmt
        self.q, self.k, self.v = (rows(50, heads, D, seed=seed, device="cuda") for heads, seed in ((HQ, 1), (H, 2), (H, 3)))
        g = torch.Generator().manual_seed(4)
        self.norms = [(1 + 0.2 * torch.randn(D, generator=g)).cuda() for _ in range(2)]
        self.rotary = RotaryAxes.create(D, D // 2)

    def rows_of(self, tokens, positions):
        q, k = rotate_heads(self.q[tokens], self.k[tokens], positions[:, None], self.rotary, q_norm=self.norms[0],
                            k_norm=self.norms[1])
        return q, k, self.v[tokens]

    def plainly(self, tokens):
        """(q, k, v) of a whole sequence, as the cache holds them."""
        ids = torch.tensor(tokens, device="cuda")
        q, k, v = self.rows_of(ids, torch.arange(len(tokens), dtype=torch.int32, device="cuda"))
        return q, values(k, self.fmt), values(v, self.fmt)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_step_of_drafts_and_the_next(fmt, captured):
    model = Model(fmt)
    prompts = [[(7 * i + j) % 50 for j in range(n)] for i, n in enumerate((21, 33, 48))]
    cache = PagedCache.create(64, PAGE, H, D, format=fmt)
    plan, pool = PagedPlan.create([], [], [], pages=64, page_size=PAGE).to("cuda"), PagePool.create(cache)
    plan, pool = cache_fork(cache, pool, plan, ints([-1] * 3), ints([len(p) for p in prompts]), width=8)
    ids = torch.tensor(sum(prompts, []), device="cuda")
    positions = ints(sum((list(range(len(p))) for p in prompts), []))
    q, k, v = model.rows_of(ids, positions)
    cache_write(k, v, cache, plan)
    o = paged_attention(q, cache, plan)
    at = 0
    for p in prompts:
        assert_within(o[at:at + len(p)], *attend(*model.plainly(p)))
        at += len(p)

    # Trees of drafts, three times: tokens, parents, and the path that is accepted (its numbers ascend).
    trees = [[-1, 0, 0, 1, 1, 2, 4, 6], [-1, -1, 1, 2, 2, 4, 4, 3], [-1, 0, 1, 2, 3, 4, 5, 6]]
    paths = [[0, 1, 4, 6], [1, 2, 4, 5], [0, 1, 2]]
    most = 8
    drafts = torch.zeros(3 * most, dtype=torch.long, device="cuda")
    parents, kept = ints(sum(trees, [])), ints([p + [-1] * (most - len(p)) for p in paths])
    depths = [[0] * most for _ in trees]
    for t, d in zip(trees, depths):
        for i, p in enumerate(t):
            d[i] = d[p] + 1 if p >= 0 else 0
    depth = ints(sum(depths, []))
    branches, tokens = ints([0, 2, 1, 2]), ints([1, 1, 1, 1])
    last = torch.zeros(4, dtype=torch.long, device="cuda")

    def step(plan, pool):
        """Drafts of every sequence, then one token more of the branches: both calls' outputs, and what holds then."""
        plan, pool = cache_fork(cache, pool, plan, ints_3, eight)
        base = (plan.context_lengths - most).repeat_interleave(most)
        q, k, v = model.rows_of(drafts, base + depth)
        cache_write(k, v, cache, plan)
        o = tree_attention(q, cache, plan, parents)
        lengths = cache_keep(cache, plan, kept)
        plan, pool = cache_fork(cache, pool, plan, branches, tokens, lengths=lengths)
        q2, k2, v2 = model.rows_of(last, plan.context_lengths - 1)
        cache_write(k2, v2, cache, plan)
        return q, o, paged_attention(q2, cache, plan), plan, pool

    ints_3, eight = ints([0, 1, 2]), ints([most] * 3)
    if captured:
        start = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8))]
        scales = [x.clone() for x in (cache.k_scales, cache.v_scales) if x is not None]
        step(plan, pool)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step(plan, pool)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        drafts.copy_(torch.randint(0, 50, (3 * most,), generator=g))
        last.copy_(torch.randint(0, 50, (4,), generator=g))
        if captured:
            for x, y in zip((cache.k.view(torch.int8), cache.v.view(torch.int8)), start):
                x.copy_(y)
            for x, y in zip([x for x in (cache.k_scales, cache.v_scales) if x is not None], scales):
                x.copy_(y)
            graph.replay()
        else:
            results = step(plan, pool)
        q, o, o2, after, left = results
        ids, ends = drafts.tolist(), last.tolist()
        outs = []
        for i, (p, tree) in enumerate(zip(prompts, trees)):
            mine = ids[i * most:(i + 1) * most]
            _, k, v = model.plainly(p)
            base = len(p)
            at = torch.tensor([base + d for d in depths[i]], dtype=torch.int32, device="cuda")
            _, kd, vd = model.rows_of(torch.tensor(mine, device="cuda"), at)
            outs.append(attend_seen(q[i * most:(i + 1) * most], torch.cat([k, values(kd, fmt)]),
                                    torch.cat([v, values(vd, fmt)]), seen_by(tree, base, base + most)))
        assert_within(o, *(np.concatenate([x[i] for x in outs]) for i in (0, 1)))
        # The branches, written out: their prompts, the accepted drafts, one token more.
        grown = [p + [ids[i * most + j] for j in path] for i, (p, path) in enumerate(zip(prompts, paths))]
        outs = []
        for b, parent in enumerate((0, 2, 1, 2)):
            q2, k, v = model.plainly(grown[parent] + [ends[b]])
            outs.append(attend(q2[-1:], k, v))
        assert_within(o2, *(np.concatenate([x[i] for x in outs]) for i in (0, 1)))
        assert after.context_lengths.tolist() == [len(grown[p]) + 1 for p in (0, 2, 1, 2)] and left.missing.item() == 0
        counts = [0] * 64
        for row, n in zip(after.page_table.tolist(), after.context_lengths.tolist()):
            for page in row[:-(-n // PAGE)]:
                counts[page] += 1
        assert left.refs.tolist() == counts
