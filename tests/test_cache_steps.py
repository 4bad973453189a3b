"""Kept drafts, forks, pages shared, copied, taken and freed, against plain Python; whole numbers and moved rows are
equal, bit for bit."""

import ctypes
import random

import pytest
import torch

from sol_attn_amd import PagedCache, PagedPlan, PagePool, _native, cache_fork, cache_keep


def filled(pages, heads, page_size, dim, fmt, seed=0):
    """A cache whose every byte says where it is from."""
    g = torch.Generator().manual_seed(seed)
    cache = PagedCache.create(pages, page_size, heads, dim, format=fmt)
    for x in tensors(cache):
        if x.dtype == torch.float32 or x.dtype == torch.bfloat16:
            x.copy_(torch.randn(x.shape, generator=g))
        else:
            x.view(torch.int8).copy_(torch.randint(-120, 120, x.shape, generator=g))
    return cache


def tensors(cache):
    return [x for x in (cache.k, cache.v, cache.k_scales, cache.v_scales) if x is not None]


def plain(cache):
    return [(x.view(torch.int8) if x.dtype == torch.float8_e4m3fn else x).cpu().clone() for x in tensors(cache)]


def assert_same(cache, want):
    for x, y in zip(plain(cache), want):
        assert torch.equal(x, y)


def ints(values, shape=None):
    x = torch.tensor(values, dtype=torch.int32)
    return (x if shape is None else x.reshape(shape)).cuda()


# ---- keep ---------------------------------------------------------------------------------------------------


def keep_in_python(store, table, lengths, new, kept, page_size, pages):
    """The cache's tensors and the lengths after cache_keep."""
    before, out = [x.clone() for x in store], []
    for row, length, n, picks in zip(table, lengths, new, kept):
        base, count, last = length - n, 0, -1
        for x in picks:
            if not last < x < n:
                break
            last, count = x, count + 1
        out.append(max(0, base + count))
        for j, x in enumerate(picks[:count]):
            a, b = base + x, base + j
            if min(a, b) < 0 or b // page_size >= len(row):
                continue
            row = row + [-1] * (a // page_size + 1)
            p, q = row[a // page_size], row[b // page_size]
            if 0 <= q < pages and a != b:
                for x2, y2 in zip(store, before):
                    x2[q, :, b % page_size] = y2[p, :, a % page_size] if 0 <= p < pages else 0
    return store, out


def run_keep(lengths, new, kept, *, heads=2, dim=64, fmt="bf16", page_size=16, seed=0, spoil=()):
    rng = random.Random(seed)
    used = [-(-n // page_size) for n in lengths]
    pages = sum(used) + 2
    order = rng.sample(range(pages), pages)
    table = [[order.pop() for _ in range(n)] for n in used]
    width = max(used + [1])
    table = [row + [0] * (width - len(row)) for row in table]
    for s, e, page in spoil:
        table[s][e] = page
    cache = filled(pages, heads, page_size, dim, fmt, seed)
    most = max([len(x) for x in kept] + [0])
    kept = [x + [-1] * (most - len(x)) for x in kept]
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    plan = PagedPlan(ints(table), ints(lengths), ints(offsets))
    want, out = keep_in_python(plain(cache), table, lengths, new, kept, page_size, pages)
    got = cache_keep(cache, plan, ints(kept, (len(lengths), most)))
    assert got.dtype == torch.int32 and got.tolist() == out
    assert_same(cache, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_keep_of_a_batch_of_trees(dim, fmt):
    # A path that begins late, one whose targets are its own later sources, none, all, one token, no token.
    run_keep([37, 60, 21, 90, 5, 33, 16], [9, 26, 7, 5, 1, 0, 16],
             [[2, 3, 8], [0, 1, 2, 4, 5, 6, 7, 8, 20], [], [0, 1, 2, 3, 4], [0], [], [15]], dim=dim, fmt=fmt, heads=3)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("n,gap", [(700, 1), (1500, 2), (4032, 1), (2500, 700)])
def test_keep_of_long_runs_whose_targets_are_sources(n, gap, fmt):
    # Every row moves ``gap`` places forward, over many batches of rows.
    run_keep([n + 41, n], [n, n], [list(range(gap, n)), [x for x in range(n) if x % 3]], dim=128, fmt=fmt, heads=2,
             page_size=64)


@pytest.mark.gpu
@pytest.mark.parametrize("page_size", [16, 128, 4096])
def test_keep_across_page_sizes(page_size):
    rng = random.Random(page_size)
    lengths, new = [5000, 200, 77], [300, 150, 77]
    run_keep(lengths, new, [sorted(rng.sample(range(n), n // 2)) for n in new], page_size=page_size)


@pytest.mark.gpu
def test_keep_ends_its_list_at_the_first_entry_that_does_not_ascend():
    run_keep([40, 40, 40, 40, 40], [8] * 5, [[1, 1, 2], [3, 2, 7], [4, 8, 9], [2, 5, -1, 7], [0, 2, 5, 2147483647]])


@pytest.mark.gpu
def test_keep_leaves_what_has_no_page():
    # Pages outside the cache, among the sources and among the targets; a length that the table does not reach.
    run_keep([64, 64], [30, 30], [[5, 9, 20, 29], [1, 2, 17]], spoil=((0, 3, 99), (1, 2, -1)))
    cache = filled(4, 2, 16, 64, "bf16")
    want = plain(cache)
    plan = PagedPlan(ints([[0, 1], [2, 3]]), ints([3, 100]), ints([0, 9, 15]))
    # 9 new tokens of 3: positions -6 .. 2; and 6 of a sequence whose last pages are not in the table.
    # Token 7 of the first is position 1, which stays empty of it: token 1's place is before the sequence.
    assert cache_keep(cache, plan, ints([[0, 7], [1, 3]])).tolist() == [0, 96]
    assert_same(cache, want)
    # The second's tokens 0 and 1 have a page, the others none: they move as zeros.
    plan = PagedPlan(ints([[0, 1], [2, 3]]), ints([3, 36]), ints([0, 0, 6]))
    assert cache_keep(cache, plan, ints([[-1, -1], [1, 3]])).tolist() == [3, 32]
    for x, y in zip(plain(cache), want):
        assert torch.equal(x[3, :, 14], y[3, :, 15]) and not x[3, :, 15].any()
        x[3, :, 14:], y[3, :, 14:] = 0, 0
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_keep_of_nothing():
    cache = filled(4, 2, 16, 64, "int8")
    want = plain(cache)
    plan = PagedPlan(ints([[0, 1], [2, 3]]), ints([20, 30]), ints([0, 4, 9]))
    assert cache_keep(cache, plan, torch.empty((2, 0), dtype=torch.int32, device="cuda")).tolist() == [16, 25]
    empty = PagedPlan.create([], [], [], pages=4, page_size=16).to("cuda")
    assert cache_keep(cache, empty, torch.empty((0, 3), dtype=torch.int32, device="cuda")).shape == (0,)
    # Offsets that descend: no new tokens.
    down = PagedPlan(ints([[0, 1], [2, 3]]), ints([20, 30]), ints([9, 4, 9]))
    assert cache_keep(cache, down, ints([[0, 2], [0, 1]])).tolist() == [20, 27]
    assert_same(cache, want)


# ---- fork ---------------------------------------------------------------------------------------------------


def fork_in_python(store, refs, table, lengths, parents, new, page_size, continued=None, width=None):
    """(tensors, refs, table, lengths, offsets, missing) after cache_fork."""
    pages, before = len(refs), [x.clone() for x in store]
    old_width = len(table[0]) if table else 0
    width = width or old_width
    free = [p for p, n in enumerate(refs) if n <= 0]
    out, seen, missing = list(refs), set(), 0
    held = [min(-(-max(n, 0) // page_size), old_width) for n in lengths]
    for row, n in zip(table, held):
        for page in row[:n]:
            if 0 <= page < pages:
                out[page] -= 1
    rows, news, offsets = [], [], [0]
    for p, n in zip(parents, new):
        p = p if 0 <= p < len(table) else -1
        length = max(lengths[p], 0) if p >= 0 else 0
        kept = min(max((continued or lengths)[p], 0), length) if p >= 0 else 0
        after = min(kept + max(n, 0), 2 ** 31 - 1)
        first = p >= 0 and p not in seen
        seen.add(p)
        row = []
        for e in range(min(-(-after // page_size), width)):
            old = table[p][e] if p >= 0 and e < old_width else -1
            alone = 0 <= old < pages and refs[old] == 1
            begun = e == kept // page_size and kept % page_size
            if e < kept // page_size or (first and e < held[p] and alone):
                page = old
            elif begun and not (e < held[p] and 0 <= old < pages):
                page = -1
                missing += 1
            else:
                page = free.pop(0) if free else -1
                missing += page < 0
                if begun and page >= 0:
                    for x, y in zip(store, before):
                        x[page, :, :kept % page_size] = y[old, :, :kept % page_size]
            row.append(page)
            if 0 <= page < pages:
                out[page] += 1
        rows.append(row + [-1] * (width - len(row)))
        news.append(after)
        offsets.append(offsets[-1] + after - kept)
    return store, out, rows, news, offsets, missing


class Batch:
    """Sequences over a cache, with their pool, in Python and on the GPU."""

    def __init__(self, lengths, *, heads=2, dim=64, fmt="bf16", page_size=16, width=None, spare=20, shared=0, seed=0):
        rng = random.Random(seed)
        self.page_size, used = page_size, [-(-n // page_size) for n in lengths]
        pages = sum(used) + spare
        order = rng.sample(range(pages), pages)
        front = [order.pop() for _ in range(shared)]
        width = width or max(used + [1])
        self.table = [front + [order.pop() for _ in range(n - shared)] + [7] * (width - n) for n in used]
        self.lengths, self.width = list(lengths), width
        self.cache = filled(pages, heads, page_size, dim, fmt, seed)
        self.plan = PagedPlan(ints(self.table, (len(lengths), width)), ints(self.lengths), ints([0] * (len(lengths) + 1)))
        self.pool = PagePool.create(self.cache, self.plan)
        self.refs = [0] * pages
        for row, n in zip(self.table, used):
            for page in row[:n]:
                self.refs[page] += 1
        assert self.pool.refs.tolist() == self.refs

    def fork(self, parents, new, continued=None, width=None):
        want = fork_in_python(plain(self.cache), self.refs, self.table, self.lengths, parents, new, self.page_size,
                              continued, width or self.width)
        before = self.plan.page_table.clone(), self.pool.refs.clone()
        plan, pool = cache_fork(self.cache, self.pool, self.plan, ints(parents, (len(parents),)), ints(new, (len(new),)),
                                lengths=None if continued is None else ints(continued, (len(continued),)), width=width)
        assert torch.equal(before[0], self.plan.page_table) and torch.equal(before[1], self.pool.refs)
        store, self.refs, self.table, self.lengths, offsets, missing = want
        self.width = width or self.width
        assert plan.page_table.shape == (len(parents), self.width)
        assert plan.page_table.tolist() == self.table
        assert plan.context_lengths.tolist() == self.lengths and plan.query_offsets.tolist() == offsets
        assert pool.refs.tolist() == self.refs and pool.missing.tolist() == [missing]
        assert_same(self.cache, store)
        self.plan, self.pool = plan, pool
        return missing


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 64), (128, 4096)])
def test_beams_go_on_branch_and_end(dim, page_size, fmt):
    b = Batch([page_size * 3 + 5, page_size, 1, page_size * 2 - 1, 17], dim=dim, page_size=page_size, fmt=fmt, width=6,
              heads=3)
    b.fork([3, 0, 0, 4, 3], [1, 1, 1, 1, 1])
    b.fork([0, 1, 2, 3, 4], [1, 2, page_size, 0, 3])
    b.fork([2, 2, 2, 2, 1], [1, 1, 1, 1, 1])
    b.fork([4], [1])
    b.fork([], [])
    assert not any(b.refs)


@pytest.mark.gpu
def test_a_loop_of_random_steps_keeps_its_books():
    rng = random.Random(5)
    b = Batch([], width=30, spare=200)
    for step in range(40):
        n = rng.randint(0, 12)
        parents = [rng.randint(-1, max(len(b.lengths) - 1, 0)) for _ in range(n)]
        new = [rng.choice((0, 1, 1, rng.randint(0, 60))) for _ in range(n)]
        continued = [x - rng.randint(0, min(x, 40)) if rng.random() < 0.5 else x for x in b.lengths]
        # Sequences stay inside their tables.
        new = [min(x, 30 * 16 - (continued[p] if 0 <= p < len(continued) else 0)) for p, x in zip(parents, new)]
        b.fork(parents, new, continued)
        counts = [0] * len(b.refs)
        for row, length in zip(b.table, b.lengths):
            for page in row[:-(-length // 16)]:
                if page >= 0:
                    counts[page] += 1
        assert counts == b.refs


@pytest.mark.gpu
def test_samples_of_a_shared_prompt_and_a_wider_table():
    b = Batch([100, 120, 96], shared=5, spare=64)
    b.fork([0] * 9 + [2, 1, 2], [1] * 12, width=20)
    b.fork([11, 10, -1, -7, 99, 10], [3, 200, 31, 0, 16, 5])
    b.fork([0, 1, 2, 3, 4, 5], [1] * 6, width=2)  # a table too narrow for its sequences


@pytest.mark.gpu
def test_sequences_continued_from_a_part_of_their_tokens():
    b = Batch([100, 120, 90, 64], shared=2, spare=40)
    b.fork([0, 1, 2, 2, 3, 3], [30, 1, 5, 60, 1, 20], continued=[50, 33, 200, 48], width=12)
    b.fork([0, 0, 1, 2, 3, 4], [1] * 6, continued=[0, -5, 60, 10, 1, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [0, 33])
def test_long_sequences_that_go_back_far(shared):
    # Hundreds of the first children's pages lie behind what is kept, and some of them are other sequences' too.
    b = Batch([16 * 1400 + 3, 16 * 700, 16 * 650 + 9, 16 * 620, 16 * 33 + 1], width=1500, spare=1500, shared=shared)
    b.fork([0, 0, 1, 2, 2, 3, 4], [16 * 300, 5, 16 * 500, 1, 0, 7, 16 * 40], continued=[16 * 200 + 7, 16 * 600, 3, 0, 1])
    b.fork([0, 2, 0, 2, 6], [16 * 900, 16 * 450, 16 * 20, 1, 300], continued=[16 * 400, 0, 16 * 400 + 1, 0, 0, 0, 2])
    b.fork([1, 0, 3, 0], [16 * 1000, 16 * 1200, 0, 1], continued=[5, 16 * 20 + 2, 0, 0, 0])


@pytest.mark.gpu
def test_pages_that_run_out():
    b = Batch([40, 35], spare=3, width=9)
    assert b.fork([0, 0, 1, -1], [30, 30, 1, 40]) > 0
    assert b.fork([0, 1, 2, 3], [20, 20, 20, 20]) > 0
    b.fork([2], [1])
    assert b.fork([0, -1], [1, 30]) == 1  # the page that the first one had begun without
    assert b.fork([1, -1], [1, 30]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [4094, 4096, 9000])
def test_pools_of_several_slices(spare):
    b = Batch([300 * 16, 7], spare=spare, width=400, heads=1)
    b.fork([0, 1, 0] + [-1] * 40, [1000, 2000, 1500] + [90 * 16] * 40)
    b.fork([1, 2, 1, 5, 30], [1] * 5)


@pytest.mark.gpu
def test_more_sequences_than_threads():
    rng = random.Random(2)
    b = Batch([rng.randint(1, 40) for _ in range(2100)], spare=4000, width=5, heads=1)
    b.fork([rng.randrange(-100, 2100) for _ in range(2300)], [rng.randint(0, 20) for _ in range(2300)])
    b.fork(list(range(2300)), [1] * 2300)


@pytest.mark.gpu
@pytest.mark.parametrize("old", [4096, 4097])
def test_more_sequences_than_a_workgroup_holds(old):
    rng = random.Random(3)
    b = Batch([rng.randint(1, 20) for _ in range(old)], spare=3000, width=2, heads=1)
    b.fork([rng.choice((rng.randrange(old), old - 1 - i % 7)) for i in range(2500)], [rng.randint(0, 9) for _ in range(2500)])


@pytest.mark.gpu
def test_lengths_and_pages_that_make_no_sense_stay_inside_the_tensors():
    b = Batch([40, 35, 90], spare=10, width=6)
    b.table[0][1], b.table[1][2], b.table[2][5] = -3, 9999, 2147483647
    b.lengths = [500, -20, 2147483647]
    b.plan = PagedPlan(ints(b.table), ints(b.lengths), ints([0] * 4))
    b.refs[b.table[0][0]] = 0
    b.refs[b.table[0][2]] = -4
    b.pool = PagePool(ints(b.refs), b.pool.missing)
    b.fork([0, 0, 1, 2, -2147483648, 2147483647], [2147483647, 1, 5, 2147483647, -9, 3])


def absent(b):
    """Pages that a batch's tokens need and its tables do not name."""
    return sum(-(-max(n, 0) // b.page_size) - sum(0 <= x < len(b.refs) for x in row[:-(-max(n, 0) // b.page_size)])
               for row, n in zip(b.table, b.lengths))


@pytest.mark.gpu
def test_pages_past_the_tables_width_are_counted():
    b = Batch([100, 120, 96], shared=5, spare=64)
    assert b.pool.absent.dtype == torch.int64 and b.pool.absent.tolist() == [0]
    assert b.fork([0, 1, 2], [12, 8, 16]) == 0 and b.pool.absent.tolist() == [0]  # 7, 8 and 7 of 8 pages
    assert b.fork([0, 1, 2], [16, 1, 0]) == 0 and b.pool.absent.tolist() == [1]  # the second one's 9th page
    assert b.fork([0, 1, 2, 1, -1], [300, 0, 0, 0, 40]) == 0 and b.pool.absent.tolist() == [absent(b)] == [21]
    assert b.fork([0, 2, 4], [0, 0, 0], width=1) == 0 and b.pool.absent.tolist() == [absent(b)] == [34]
    assert b.fork([], []) == 0 and b.pool.absent.tolist() == [0]


@pytest.mark.gpu
def test_whole_pages_that_a_parent_lacks_are_counted():
    b = Batch([40, 35], spare=3, width=9)
    missing = b.fork([0, 0, 1, -1], [30, 30, 1, 40])
    assert b.pool.absent.tolist() == [absent(b)] == [missing] and missing > 0
    for parents, new in (([0, 1, 2, 3], [20] * 4), ([0, 1, 2, 3], [0] * 4), ([3, 1, 1], [9, 0, 50])):
        b.fork(parents, new)
        assert b.pool.absent.tolist() == [absent(b)] and absent(b) > 0
    b.fork([2], [0], continued=[0, 0, 20])
    assert b.pool.absent.tolist() == [absent(b)]


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [40, 14000, 70001])
def test_a_plan_and_a_pool_keep_no_large_workspace(pages):
    cache = PagedCache.create(pages, 16, 1, 64, format="int8")
    plan, pool = PagedPlan.create([], [], [], pages=pages, page_size=16).to("cuda"), PagePool.create(cache)
    for parents, new in (([-1] * 3, [20, 300, 7]), ([0, 0, 1, 2], [1] * 4)):
        plan, pool = cache_fork(cache, pool, plan, ints(parents), ints(new), width=21)
        results = 4 * (len(new) * 21 + 2 * len(new) + 1 + pages + 1) + 8
        kept = {x.untyped_storage().data_ptr(): x.untyped_storage().nbytes()
                for x in (plan.page_table, plan.context_lengths, plan.query_offsets, pool.refs, pool.missing, pool.absent)}
        assert sum(kept.values()) <= results + (1 << 18) + 512 * len(kept)
        assert pool.refs.sum() == sum(-(-n // 16) for n in plan.context_lengths.tolist())
        assert pool.missing.item() == pool.absent.item() == 0


@pytest.mark.gpu
def test_absent_pages_of_many_and_of_lengths_that_make_no_sense():
    rng = random.Random(6)
    b = Batch([rng.randint(1, 400) for _ in range(900)], spare=50, width=25, heads=1)
    b.fork([rng.randrange(-9, 900) for _ in range(700)], [rng.randint(0, 90) for _ in range(700)])
    assert b.pool.absent.tolist() == [absent(b)]
    # (Not in Python whole: the offsets of so many new tokens stop at what int32 holds.)
    parents, most = [rng.randrange(700) for _ in range(800)], 2 ** 31 - 1
    plan, pool = cache_fork(b.cache, b.pool, b.plan, ints(parents), ints([most] * 800), width=30)
    assert plan.context_lengths.tolist() == [most] * 800 and plan.query_offsets.tolist()[-1] == most
    b.table, b.lengths = plan.page_table.tolist(), [most] * 800
    assert pool.absent.tolist() == [absent(b)] and absent(b) > 2 ** 31
    b = Batch([40, 35, 90], spare=10, width=6)
    b.table[0][1], b.table[1][2], b.table[2][0] = -3, 9999, 2147483647
    b.lengths = [80, 35, 90]
    b.plan = PagedPlan(ints(b.table), ints(b.lengths), ints([0] * 4))
    b.fork([0, 1, 2, 2], [1, 5, 10, 0])
    assert b.pool.absent.tolist() == [absent(b)] and absent(b) >= 3


@pytest.mark.gpu
def test_replays_follow_their_tensors():
    b = Batch([33, 50, 70], spare=30, width=8)
    parents, new = ints([0, 0, 2]), ints([1, 1, 1])
    kept = ints([[0, 2], [1, 3], [0, 1]])
    plan = PagedPlan(b.plan.page_table, b.plan.context_lengths, ints([0, 4, 8, 12]))

    def step():
        lengths = cache_keep(b.cache, plan, kept)
        return lengths, *cache_fork(b.cache, b.pool, plan, parents, new, lengths=lengths)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for changes in ([0, 0, 2], [1, 1, 1], [-1, 2, 0]):
        parents.copy_(ints(changes))
        start = [x.clone() for x in tensors(b.cache)]
        graph.replay()
        after = plain(b.cache)
        for x, y in zip(tensors(b.cache), start):
            x.copy_(y)
        eager = step()
        torch.cuda.synchronize()
        assert_same(b.cache, after)
        assert torch.equal(held[0], eager[0]) and torch.equal(held[2].refs, eager[2].refs)
        assert all(torch.equal(x, y) for x, y in zip(vars(held[1]).values(), vars(eager[1]).values()))


@pytest.mark.gpu
def test_another_stream():
    b = Batch([33, 50, 70], spare=30, width=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.fork([2, 2, 0], [1, 5, 9])
    torch.cuda.current_stream().wait_stream(side)


# ---- refusals -----------------------------------------------------------------------------------------------


def parts(fmt="bf16"):
    cache = PagedCache.create(4, 16, 2, 64, format=fmt, device="cpu")
    plan = PagedPlan.create([[0, 1], [2]], [20, 5], [1, 2], pages=4, page_size=16)
    return cache, plan


def test_a_pool_counts_the_tables_that_name_a_page():
    cache, plan = parts()
    assert PagePool.create(cache).refs.tolist() == [0] * 4
    pool = PagePool.create(cache, PagedPlan.create([[0, 1], [0, 3]], [20, 30], [0, 0], pages=4, page_size=16))
    assert pool.refs.tolist() == [2, 1, 0, 1] and pool.refs.dtype == torch.int32 and pool.missing.tolist() == [0]
    with pytest.raises(ValueError, match="outside the cache"):
        PagePool.create(cache, PagedPlan(torch.tensor([[5]]), torch.tensor([3]), torch.tensor([0, 0])))
    for args in ((None,), (cache, 3)):
        with pytest.raises(ValueError, match="explicit"):
            PagePool.create(*args)


def test_everything_is_checked_before_the_device():
    cache, plan = parts()
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="AMD ROCm GPU"):
        cache_keep(cache, plan, i32.view(2, 1))
    with pytest.raises(ValueError, match="AMD ROCm GPU"):
        cache_fork(cache, PagePool.create(cache), plan, i32, i32)
    with pytest.raises(ValueError, match="PagedCache"):
        cache_keep(None, plan, i32.view(2, 1))
    with pytest.raises(ValueError, match="PagedPlan"):
        cache_fork(cache, PagePool.create(cache), None, i32, i32)


@pytest.mark.gpu
def test_refusals():
    cache = PagedCache.create(4, 16, 2, 64)
    plan = PagedPlan.create([[0, 1], [2]], [20, 5], [1, 2], pages=4, page_size=16).to("cuda")
    pool = PagePool.create(cache, plan)
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    for kept, match in ((i32, "entry for each"), (i32.long().view(2, 1), "int32"), (i32.cpu().view(2, 1), "device"),
                        (torch.zeros((3, 1), dtype=torch.int32, device="cuda"), "entry for each"),
                        (torch.zeros((3, 2), dtype=torch.int32, device="cuda").t(), "contiguous"), ([[0]], "int32")):
        with pytest.raises(ValueError, match=match):
            cache_keep(cache, plan, kept)
    with pytest.raises(ValueError, match="must not share memory"):
        cache_keep(PagedCache(cache.k, cache.k), plan, i32.view(2, 1))
    with pytest.raises(ValueError, match="must not share memory"):
        cache_fork(PagedCache(cache.k, cache.k), pool, plan, i32, i32)
    for change, match in ((dict(parents=i32.view(1, 2)), "entry for each"), (dict(new_tokens=i32[:1]), "entry for each"),
                          (dict(parents=i32.cpu()), "device"), (dict(lengths=i32[:1]), "entry for each"),
                          (dict(lengths=i32.long()), "int32"), (dict(width=0), "width"), (dict(width=-1), "nonnegative"),
                          (dict(width=1 << 27), "width"), (dict(pool=None), "PagePool"),
                          (dict(pool=PagePool(i32, i32)), "Invalid pool"),
                          (dict(pool=PagePool(pool.refs.cpu(), pool.missing)), "pool must be on")):
        args = dict(pool=pool, parents=i32, new_tokens=i32)
        args.update(change)
        with pytest.raises(ValueError, match=match):
            cache_fork(cache, args.pop("pool"), plan, args.pop("parents"), args.pop("new_tokens"), **args)


def test_the_c_entries_refuse():
    lib = _native.library()
    here = ctypes.c_void_p(1 << 20)
    assert lib.sol_cache_fork_workspace_size(-1, 1, 1) == -1 and lib.sol_cache_fork_workspace_size(1, 1, 0) == -1
    assert lib.sol_cache_fork_workspace_size(0, 0, 1) > 0
    keep = [here, here, here, 1, 1, 4, 16, 2, 64, 0, here, here, None, None, here, 1, here, None]
    for at, value in ((2, None), (6, 24), (8, 96), (9, 3), (10, None), (14, None), (16, None), (15, -1)):
        args = list(keep)
        args[at] = value
        assert lib.sol_cache_keep(*args) < 0, at
    assert lib.sol_cache_keep(*keep[:9], 1, *keep[10:]) < 0  # INT8 without scales
    big = list(keep)
    big[3], big[7] = 1 << 20, 60000
    assert lib.sol_cache_keep(*big) < 0 and b"grid" in lib.sol_last_error()
    size = lib.sol_cache_fork_workspace_size(1, 1, 4)
    fork = [here, here, None, 1, 1, here, here, 1, 1, here, 4, 16, 2, 64, 0, here, here, None, None, here, here, here,
            ctypes.c_void_p(2 << 20), here, here, size, None]
    for at, value in ((0, None), (1, None), (5, None), (6, None), (8, 0), (8, 1 << 27), (9, None), (11, 24), (13, 32),
                      (15, None), (19, None), (21, None), (22, None), (22, here), (23, None), (24, None),
                      (24, ctypes.c_void_p(8)), (25, size - 1), (7, -1), (7, 1 << 21)):
        args = list(fork)
        args[at] = value
        assert lib.sol_cache_fork(*args) < 0, at


def memory(n):
    """Addresses apart from each other's by far (nothing is read there: the calls are refused)."""
    return [ctypes.c_void_p((1 + i) << 32) for i in range(n)]


def test_the_c_entries_refuse_outputs_that_meet_something():
    lib = _native.library()
    table, lengths, offsets, k, v, ks, vs, kept, out = memory(9)
    # 70 sequences of 3 pages, 40 pages of 16 rows of 2 heads of 64 codes.
    keep = [table, lengths, offsets, 70, 3, 40, 16, 2, 64, 1, k, v, ks, vs, kept, 5, out, None]
    near = [(16, x.value + far) for x, far in ((table, 4 * 70 * 3 - 4), (lengths, 0), (lengths, 4 * 69), (lengths, -4 * 69),
                                               (offsets, 4 * 70), (kept, 4 * 70 * 5 - 4), (k, 40 * 2 * 16 * 64 - 4),
                                               (vs, 40 * 2 * 16 * 4 - 4))]
    for at, value in near + [(11, k.value + 40 * 2 * 16 * 64 - 16), (13, ks.value), (14, k.value), (0, vs.value)]:
        args = list(keep)
        args[at] = ctypes.c_void_p(value)
        assert lib.sol_cache_keep(*args) < 0 and b"memory of their own" in lib.sol_last_error(), (at, value)
    (table, lengths, continued, parents, new, refs, k, v, ks, vs, new_table, new_lengths, new_offsets, new_refs, missing,
     workspace) = memory(16)
    size = lib.sol_cache_fork_workspace_size(70, 90, 40)
    fork = [table, lengths, continued, 70, 3, parents, new, 90, 4, refs, 40, 16, 2, 64, 1, k, v, ks, vs, new_table,
            new_lengths, new_offsets, new_refs, missing, workspace, size, None]
    near = [(19, table.value), (19, table.value - 4 * 90 * 4 + 4), (20, lengths.value), (20, lengths.value + 4 * 69),
            (20, continued.value), (20, new.value + 4 * 89), (21, parents.value - 4 * 90), (22, refs.value + 4 * 39),
            (22, refs.value), (23, refs.value + 4 * 39), (23, new_table.value + 4 * 90 * 4 - 4), (23, missing.value + 0),
            (24, table.value), (24, k.value - (size - 16)), (23, workspace.value + size - 4), (16, k.value), (18, ks.value)]
    for at, value in near:
        args = list(fork)
        args[at] = ctypes.c_void_p(value)
        if value == missing.value:
            args[21] = ctypes.c_void_p(value - 4 * 90)
        assert lib.sol_cache_fork(*args) < 0 and b"memory of their own" in lib.sol_last_error(), (at, value)


@pytest.mark.gpu
def test_neighbours_in_memory_are_not_refused():
    # All of a batch's whole numbers one after another in one allocation, outputs between inputs.
    b = Batch([33, 50, 70], spare=30, width=8)
    want_plan, want_pool = cache_fork(b.cache, b.pool, b.plan, ints([0, 0, 2]), ints([1, 2, 3]))
    pages, lib = b.pool.refs.numel(), _native.library()
    size = lib.sol_cache_fork_workspace_size(3, 3, pages)
    parts = dict(work=size // 4, table=24, lengths=3, new_lengths=3, parents=3, new_table=24, new=3, offsets=4, refs=pages,
                 new_refs=pages, missing=1, keep_offsets=4, keep_lengths=3, kept=6)
    at, flat = {}, torch.full((sum(parts.values()),), 99, dtype=torch.int32, device="cuda")
    for name, n in parts.items():
        at[name] = flat[sum(x.numel() for x in at.values()):][:n]
    for name, x in (("table", b.plan.page_table.view(-1)), ("lengths", b.plan.context_lengths), ("parents", ints([0, 0, 2])),
                    ("new", ints([1, 2, 3])), ("refs", b.pool.refs), ("keep_offsets", ints([0, 4, 8, 12])),
                    ("kept", ints([0, 2, 1, 3, 0, 1]))):
        at[name].copy_(x)
    p = {name: x.data_ptr() for name, x in at.items()}
    k, v = b.cache.k.data_ptr(), b.cache.v.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.sol_cache_fork(p["table"], p["lengths"], None, 3, 8, p["parents"], p["new"], 3, 8, p["refs"], pages, 16, 2,
                              64, 0, k, v, None, None, p["new_table"], p["new_lengths"], p["offsets"], p["new_refs"],
                              p["missing"], p["work"], size, stream) == 0
    for name, x in (("new_table", want_plan.page_table.view(-1)), ("new_lengths", want_plan.context_lengths),
                    ("offsets", want_plan.query_offsets), ("new_refs", want_pool.refs), ("missing", want_pool.missing),
                    ("table", b.plan.page_table.view(-1)), ("lengths", b.plan.context_lengths)):
        assert torch.equal(at[name], x)
    assert lib.sol_cache_keep(p["table"], p["lengths"], p["keep_offsets"], 3, 8, pages, 16, 2, 64, 0, k, v, None, None,
                              p["kept"], 2, p["keep_lengths"], stream) == 0
    assert at["keep_lengths"].tolist() == [31, 48, 68]


def test_a_pool_counts_the_pages_that_its_tables_have_no_room_for():
    cache, plan = parts()
    assert PagePool.create(cache).absent.tolist() == [0] and PagePool.create(cache, plan).absent.tolist() == [0]
    long = PagedPlan(plan.page_table[:, :1], torch.tensor([50, 5], dtype=torch.int32), plan.query_offsets)
    assert PagePool.create(cache, long).absent.tolist() == [3]


def test_the_counting_c_entry_refuses():
    lib = _native.library()
    (table, lengths, parents, new, refs, k, v, new_table, new_lengths, new_offsets, new_refs, missing, absent,
     workspace) = memory(14)
    size = lib.sol_cache_fork_workspace_size(7, 9, 40)
    fork = [table, lengths, None, 7, 3, parents, new, 9, 4, refs, 40, 16, 2, 64, 0, k, v, None, None, new_table,
            new_lengths, new_offsets, new_refs, missing, absent, workspace, size, None]
    for at, value, match in ((24, absent.value + 4, b"aligned"), (24, missing.value - 4, b"aligned"),
                             (24, refs.value + 8, b"own"), (24, lengths.value - 0, b"own"), (23, absent.value + 4, b"own"),
                             (26, size - 1, b"workspace"), (5, None, b"parents")):
        args = list(fork)
        args[at] = value if at == 26 else ctypes.c_void_p(value)
        assert lib.sol_cache_fork_counted(*args) < 0 and match in lib.sol_last_error(), (at, value)
