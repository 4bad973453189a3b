"""Attention of trees of drafts over the paged cache on the GPU, against 64 bits (tolerances in ``paged_testlib``), and
its refusals."""

import ctypes
import random

import numpy as np
import pytest
import torch

from paged_testlib import Sequences, assert_within, rows, values
from sol_attn_amd import PagedCache, PagedPlan, _native, paged_attention, tree_attention
from tree_testlib import attend_seen, seen_by, shape


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def expected(b, q, trees, *, window=None, sinks=0, scale=None, hide=None):
    outs, at = [], 0
    for s, (n, length) in enumerate(zip(b.new, b.lengths)):
        seen = seen_by(trees[s], length - n, length, window, sinks)
        if hide:
            seen[:, [j for t, j in hide if t == s]] = False
        outs.append(attend_seen(q[at:at + n], values(b.k[s], b.fmt), values(b.v[s], b.fmt), seen, scale))
        at += n
    return tuple(np.concatenate([o[i] for o in outs]) for i in (0, 1))


def run(lengths, new, kinds, *, group=1, window=None, sinks=0, scale=None, seed=0, **how):
    b = Sequences(lengths, new, seed=seed, **how)
    trees = [shape(kind, n, seed + i) for i, (kind, n) in enumerate(zip(kinds, new))]
    q = rows(sum(new), how.get("heads", 2) * group, how.get("dim", 64), seed=seed + 50, device="cuda")
    o = tree_attention(q, b.cache, b.plan, ints([p for t in trees for p in t]), window=window, sink_tokens=sinks,
                       scale=scale)
    assert_within(o, *expected(b, q, trees, window=window, sinks=sinks, scale=scale))
    return b, q, trees, o


SHAPES = ["chain", "star", "roots", "level", "any", "odd"]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_drafts(dim, fmt):
    run([33, 70, 18, 7, 130, 1, 64, 45], [5, 7, 6, 7, 3, 1, 0, 4], SHAPES + ["any", "level"], dim=dim, fmt=fmt, group=3)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_drafts(dim, fmt):
    run([200, 150, 97, 140, 300, 131], [100, 150, 90, 77, 64, 33], SHAPES, dim=dim, fmt=fmt, group=4, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("page_size", [16, 64, 512])
@pytest.mark.parametrize("base", [0, 1, 31, 32, 33, 63, 100])
def test_bases_across_tiles_and_pages(base, page_size):
    run([base + 40, base + 67], [40, 67], ["any", "level"], page_size=page_size, group=2, seed=base)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [6, 90])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 3), (5, 0), (17, 40), (33, 4), (64, 300), (40, 129), (1000, 8)])
def test_windows_and_first_tokens_go_by_depths(window, sinks, new):
    run([120 + new, new, 33 + new, 64 + new], [new] * 4, ["chain", "chain", "any", "level"], window=window, sinks=sinks,
        seed=window, heads=1, group=2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 300)])
def test_large_trees(window, sinks, fmt):
    run([450, 700, 333], [400, 601, 333], ["chain", "any", "odd"], window=window, sinks=sinks, heads=1, fmt=fmt, seed=8,
        dim=128)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 80), (900, 2000)])
def test_parts_that_begin_and_end_among_the_nodes(window, sinks, fmt):
    run([2300, 1500, 17 + 300], [700, 650, 300], ["chain", "odd", "any"], window=window, sinks=sinks, heads=2, group=2,
        fmt=fmt, dim=128, page_size=32, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "any", "star"])
def test_trees_of_more_nodes_than_a_workgroup_holds(kind):
    run([1300, 1110], [1200, 1030], [kind, "level"], heads=1, seed=9)
    run([1300, 1110], [1200, 1030], [kind, "any"], heads=1, seed=9, window=200, sinks=50)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_keys_split_over_workgroups(fmt):
    run([9000], [7], ["level"], fmt=fmt, heads=1, group=2, dim=128, page_size=64)
    run([5000, 300, 7000], [60, 20, 41], ["any", "chain", "level"], fmt=fmt, heads=1, group=2, dim=128, page_size=64)
    run([7000], [40], ["any"], fmt=fmt, heads=2, group=4, dim=64, page_size=32, window=3000, sinks=100, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,fmt", [(64, "fp8"), (128, "bf16"), (128, "int8")])
def test_few_rows_over_many_keys(dim, fmt):
    run([20300, 19001], [40, 33], ["any", "chain"], fmt=fmt, heads=2, group=4, dim=dim, page_size=64)
    run([20300], [35], ["level"], fmt=fmt, heads=2, group=4, dim=dim, page_size=64, window=19500, sinks=30)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dim", [("bf16", 128), ("fp8", 64)])
@pytest.mark.parametrize("kind", ["chain", "level", "odd"])
def test_trees_much_larger_than_their_window(kind, fmt, dim):
    # Every row tile streams all the nodes before its last one, and sees few of them.
    run([2050], [2000], [kind], fmt=fmt, heads=4, dim=dim, page_size=64, window=64, sinks=5, seed=3)
    run([900, 1100, 40], [700, 1100, 40], [kind, "any", kind], fmt=fmt, heads=2, group=3, dim=dim, window=16, seed=4)


def test_the_choice_of_kernel_goes_by_the_nodes_that_a_tile_streams():
    # Row tiles of 128 rows whose keys are cut into parts, which take a workspace; by the window alone there are too few
    # keys to cut, and tiles of 16 rows.
    size = _native.library().sol_tree_attention_workspace_size
    for n, heads in ((2000, 8), (4000, 4)):
        assert size(n, 1, 64, 128, heads, heads, 128, 0, 64, 0) > 0
    assert size(24, 4, 64, 128, 8, 8, 128, 0, 64, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("new", [5, 80])
def test_a_chain_is_causal_attention(new):
    b = Sequences([200, 90 + new], [new, new], heads=2, dim=128)
    q = rows(2 * new, 4, 128, seed=5, device="cuda")
    for window, sinks in ((None, 0), (30, 7)):
        how = dict(window=window, sink_tokens=sinks)
        o = tree_attention(q, b.cache, b.plan, ints(list(range(-1, new - 1)) * 2), **how)
        assert_within(o, *b.expected(q, window=window, sinks=sinks))
        assert_within(paged_attention(q, b.cache, b.plan, **how), *b.expected(q, window=window, sinks=sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("new", [6, 70])
def test_nodes_that_are_not_seen_do_not_matter(new, fmt):
    b = Sequences([50 + new, 33 + new], [new, new], dim=64, fmt=fmt)
    tree = [-1, 0, 0, 1, 2, 3] + [4 + i % 2 for i in range(new - 6)]
    parents = ints(tree * 2)
    q = rows(2 * new, 4, 64, seed=5, device="cuda")
    clean = tree_attention(q, b.cache, b.plan, parents)
    # Node 3's key and value become infinite or NaN: nodes 3 and 5, and what follows 5, change, and no others.
    for s, base in ((0, 50), (1, 33)):
        page, slot = b.table[s][(base + 3) // 16], (base + 3) % 16
        for x, scales in ((b.cache.k, b.cache.k_scales), (b.cache.v, b.cache.v_scales)):
            if fmt == "bf16":
                x[page, :, slot] = float("nan")
                x[page, :, slot, ::2] = float("inf")
            else:
                scales[page, :, slot] = float("nan")
    after = tree_attention(q, b.cache, b.plan, parents)
    touched = [i in (3, 5) or (i >= 6 and tree[i] == 5) for i in range(new)] * 2
    same = torch.tensor([not x for x in touched], device="cuda")
    assert torch.equal(after[same], clean[same])
    assert after[~same].isnan().any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [6, 70])
def test_places_without_a_page_and_rows_behind_the_last(new):
    b = Sequences([50 + new, 33 + new], [new, new], dim=64)
    trees = [shape("any", new, 1), shape("level", new, 2)]
    q = rows(2 * new + 9, 2, 64, seed=5, device="cuda")
    parents = ints(trees[0] + trees[1] + [3] * 9)
    table = b.plan.page_table.clone()
    table[0, 3] = 1 << 20  # nodes among them
    table[1, 0] = -1
    plan = PagedPlan(table, b.plan.context_lengths, b.plan.query_offsets)
    out = torch.full_like(q, 7.0)
    hide = [(0, j) for j in range(48, 64) if j < 50 + new] + [(1, j) for j in range(16)]
    assert tree_attention(q, b.cache, plan, parents, out=out) is out
    assert_within(out[:2 * new], *expected(b, q, trees, hide=hide))
    assert bool((out[2 * new:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [4, 50])
def test_lengths_shorter_than_their_drafts_or_longer_than_the_table(new):
    b = Sequences([64, 64], [0, 0], dim=64, heads=1)
    q = rows(2 * new, 1, 64, seed=5, device="cuda")
    tree = shape("any", new, 3)
    for lengths in ([new - 2, 64 + 3], [0, 2 ** 31 - 1], [-5, 64 + new]):
        plan = PagedPlan(b.plan.page_table, ints(lengths), ints([0, new, 2 * new]))
        for window, sinks in ((None, 0), (20, 6)):
            o = tree_attention(q, b.cache, plan, ints(tree * 2), window=window, sink_tokens=sinks)
            outs = []
            for s, length in enumerate(lengths):
                end = max(length, 0)
                if end > 1 << 20:
                    # Every key is further away than the window, or is seen whole.
                    seen = np.zeros((new, 64), dtype=bool)
                    seen[:, :sinks if window else 64] = True
                else:
                    seen = seen_by(tree, end - new, min(end, 64), window, sinks)
                outs.append(attend_seen(q[s * new:(s + 1) * new], b.k[s][:seen.shape[1]], b.v[s][:seen.shape[1]], seen))
            assert_within(o, *(np.concatenate([x[i] for x in outs]) for i in (0, 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [6, 40])
def test_replays_follow_the_tree(new):
    b = Sequences([100 + new, 31 + new], [new, new], heads=2, dim=128, fmt="int8")
    q = rows(2 * new, 8, 128, seed=5, device="cuda")
    parents = ints(shape("any", new, 0) * 2)
    tree_attention(q, b.cache, b.plan, parents, window=60, sink_tokens=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = tree_attention(q, b.cache, b.plan, parents, window=60, sink_tokens=4)
    for seed in range(1, 4):
        parents.copy_(ints(shape("any", new, seed) + shape("level", new, seed)))
        q.copy_(rows(2 * new, 8, 128, seed=60 + seed, device="cuda"))
        graph.replay()
        eager = tree_attention(q, b.cache, b.plan, parents, window=60, sink_tokens=4)
        torch.cuda.synchronize()
        assert torch.equal(held, eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tree_attention(q, b.cache, b.plan, parents, window=60, sink_tokens=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, eager)


@pytest.mark.gpu
def test_offsets_that_make_no_sense_stay_inside_the_tensors():
    b = Sequences([80, 60, 40], [20, 20, 20], heads=1)
    q = rows(60, 1, 64, seed=5, device="cuda")
    parents = ints(shape("odd", 60, 4))
    for offsets in ([0, 70, 20, 60], [-9, 20, 40, 2 ** 31 - 1], [50, 10, 30, 60]):
        plan = PagedPlan(b.plan.page_table, b.plan.context_lengths, ints(offsets))
        tree_attention(q, b.cache, plan, parents)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,fmt,past,group", [(64, "bf16", 60, 1), (128, "int8", 60, 4), (128, "bf16", 6000, 4),
                                                (64, "fp8", 9000, 1)])
@pytest.mark.parametrize("offsets", [[0, 70, 20, 60], [-9, 20, 40, 2 ** 31 - 1], [50, 10, 30, 60],
                                     [-2 ** 31, 2 ** 31 - 1, 0, 61], [60, 60, 99, -1]])
def test_offsets_that_make_no_sense_write_nothing_around_the_output(offsets, dim, fmt, past, group):
    # One row tile and many, keys in one part and in several, whose states a second launch joins.
    b = Sequences([past + 20, past // 2 + 20, 40], [20, 20, 20], heads=2, dim=dim, fmt=fmt, page_size=64)
    q = rows(60, 2 * group, dim, seed=5, device="cuda")
    around = torch.full((60 + 2 * 300, 2 * group, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    parents = ints(shape("odd", 60, 4))
    plan = PagedPlan(b.plan.page_table, b.plan.context_lengths, ints(offsets))
    stored = [x.clone() for x in (b.cache.k.view(torch.int8), b.cache.v.view(torch.int8))]
    for how in (dict(), dict(window=30, sink_tokens=3)):
        tree_attention(q, b.cache, plan, parents, out=around[300:360], **how)
    assert bool((around[:300] == 7).all()) and bool((around[360:] == 7).all())
    assert all(torch.equal(x.view(torch.int8), y) for x, y in zip((b.cache.k, b.cache.v), stored))


@pytest.mark.gpu
def test_empty_calls_and_refusals():
    b = Sequences([40], [3], heads=2, dim=64)
    q = rows(3, 4, 64, seed=1, device="cuda")
    parents = ints([-1, 0, 0])
    assert tree_attention(q[:0], b.cache, b.plan, parents[:0]).shape == (0, 4, 64)
    none = PagedPlan.create([], [], [], pages=4, page_size=16).to("cuda")
    assert tree_attention(q, b.cache, none, parents).shape == q.shape
    with pytest.raises(ValueError, match="parents must be on"):
        tree_attention(q, b.cache, b.plan, parents.cpu())
    with pytest.raises(ValueError, match="must not share memory"):
        tree_attention(q, b.cache, b.plan, parents, out=q)


@pytest.mark.parametrize("parents,match", [
    (torch.zeros(3), "int32"), ([0, 0, 0], "int32"), (torch.zeros(4, dtype=torch.int32), "each row"),
    (torch.zeros((3, 1), dtype=torch.int32), "each row"), (torch.zeros(6, dtype=torch.int32)[::2], "contiguous"),
    (torch.zeros(3, dtype=torch.int32), "AMD ROCm GPU"),
])
def test_refusals(parents, match):
    cache = PagedCache.create(4, 16, 2, 64, device="cpu")
    plan = PagedPlan.create([[0, 1], [2]], [20, 5], (1, 2), pages=4, page_size=16)
    with pytest.raises(ValueError, match=match):
        tree_attention(torch.zeros((3, 4, 64), dtype=torch.bfloat16), cache, plan, parents)


def test_the_c_entry_refuses():
    lib = _native.library()
    here, strides = ctypes.c_void_p(1 << 20), (ctypes.c_int64 * 3)(256, 256, 64)
    good = [here, strides, 3, here, here, None, None, here, here, here, here, 2, 2, 4, 16, 4, 2, 64, 0, 0.125, 0, 0, None,
            0, here, None]
    for at, value in ((0, None), (7, None), (9, None), (10, None), (14, 24), (15, 3), (17, 96), (19, 0.0), (20, -1),
                      (24, None), (24, ctypes.c_void_p(8)), (11, 1 << 17)):
        args = list(good)
        args[at] = value
        assert lib.sol_tree_attention(*args) < 0, at
        assert lib.sol_last_error().startswith(b"sol_tree_attention"), at
