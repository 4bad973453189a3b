"""A paged K/V cache and attention over it, for sequences generated piece by piece.

The new tokens' K and V rows are stored by :func:`cache_write`, in BF16 or
quantised to INT8 or FP8 (e4m3) with one scale per token and head;
:func:`paged_attention` attends the new tokens to everything stored, causally
or (a video frame) with the new tokens seeing one another, over all keys or a
sliding window with first tokens that stay visible; :func:`cache_read` gathers
stored rows back into plain BTHD tensors, as :func:`sol_attention` and
:func:`dense_attention` take them.  Not in the reference.
"""

from dataclasses import dataclass
import torch

from . import _native
from .attention import _nonnegative_integer, _on, _visibility

CACHE_FORMATS = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
MAX_POSITIONS = 1 << 30  # positions of one sequence that a page table may name
MAX_ATTENDED = 1 << 16  # sequences of one attention call: every workgroup finds its place among all of them by itself


@dataclass(frozen=True)
class PagedCache:
    """Stored K and V rows, in pages that sequences take as they grow.

    ``k``/``v``: contiguous ``[pages, heads, page_size, head_dim]`` of BF16,
    int8 or ``float8_e4m3fn``; ``k_scales``/``v_scales``: contiguous fp32
    ``[pages, heads, page_size]`` (value = code * scale), None for BF16.  Use
    :meth:`create`, or give tensors of your own.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scales: "torch.Tensor | None" = None
    v_scales: "torch.Tensor | None" = None

    @classmethod
    def create(cls, pages, page_size, heads, head_dim, *, format="bf16", device="cuda"):
        """A cache of zeros: ``format`` "bf16", "int8" or "fp8"; ``page_size`` a
        power of two from 16 to 4096; ``head_dim`` 64 or 128."""
        for name, value in (("pages", pages), ("page_size", page_size), ("heads", heads), ("head_dim", head_dim)):
            _nonnegative_integer(name, value)
        if format not in CACHE_FORMATS:
            raise ValueError("format must be 'bf16', 'int8' or 'fp8'")
        if pages == 0 or heads == 0:
            raise ValueError("pages and heads must be positive")
        if head_dim not in (64, 128):
            raise ValueError("Only head dimensions 64 and 128 are implemented")
        _page_size(page_size)
        shape = (pages, heads, page_size, head_dim)
        store = [torch.zeros(shape, device=device, dtype=torch.int8 if format == "fp8" else CACHE_FORMATS[format])
                 for _ in range(2)]
        if format == "bf16":
            return cls(*store)
        return cls(*(x.view(CACHE_FORMATS[format]) for x in store),
                   *(torch.zeros(shape[:3], device=device, dtype=torch.float32) for _ in range(2)))


def _page_size(page_size):
    if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two from 16 to 4096")


def _integers(name, values):
    values = values.tolist() if isinstance(values, torch.Tensor) else list(values)
    for x in values:
        _nonnegative_integer(name, x)
    return values


@dataclass(frozen=True)
class PagedPlan:
    """Where a batch's sequences lie in a cache, and which rows are their new tokens.

    ``page_table``: contiguous int32 ``[sequences, width]``: position p of
    sequence s is row ``p % page_size`` of page ``page_table[s, p //
    page_size]``.  ``context_lengths``: int32 ``[sequences]``, each sequence's
    keys, its new tokens included.  ``query_offsets``: int32 ``[sequences +
    1]``: rows ``query_offsets[s]`` .. ``query_offsets[s + 1] - 1`` of a call's
    K, V and Q are sequence s's new tokens, its last positions.

    :meth:`create` checks a plan on the host.  A program whose plan stays on
    the GPU may give tensors of its own and change them between calls (a
    captured launch follows what they hold at replay); the kernels read them
    there and check every entry against the tensors they address, so that no
    content makes them leave those: a page number outside the cache is no page
    (not written, read as zeros, not attended), and a new token whose position
    is past the table (a length that has outgrown it) is not written.  What
    else :meth:`create` refuses is then up to the program: offsets that do not
    ascend, and new tokens that name one row of one page twice, of which either
    one or a mix stays.
    """

    page_table: torch.Tensor
    context_lengths: torch.Tensor
    query_offsets: torch.Tensor

    @classmethod
    def create(cls, page_table, context_lengths, new_tokens, *, pages, page_size):
        """A checked plan on the CPU; transfer it with :meth:`to`.

        ``page_table``: an int matrix (CPU tensor) or a sequence of each
        sequence's page numbers; ``context_lengths``, ``new_tokens``: integers
        per sequence, ``new_tokens`` at most its ``context_lengths``;
        ``pages``, ``page_size``: the cache's.
        """
        _nonnegative_integer("pages", pages)
        _nonnegative_integer("page_size", page_size)
        _page_size(page_size)
        lengths, new = _integers("context_lengths", context_lengths), _integers("new_tokens", new_tokens)
        if isinstance(page_table, torch.Tensor) and page_table.ndim != 2:
            raise ValueError("page_table must hold one row of page numbers per sequence")
        rows = page_table.tolist() if isinstance(page_table, torch.Tensor) else [list(r) for r in page_table]
        if not len(rows) == len(lengths) == len(new):
            raise ValueError("page_table, context_lengths and new_tokens must have the same batch size")
        written = set()
        for row, length, n in zip(rows, lengths, new):
            if n > length:
                raise ValueError("new_tokens must not exceed context_lengths")
            used = -(-length // page_size)
            if used > len(row):
                raise ValueError("page_table has no page for a sequence's last tokens")
            for page in row[:used]:
                if not isinstance(page, int) or not 0 <= page < pages:
                    raise ValueError("page_table names a page outside the cache")
            if n:
                last = row[(length - n) // page_size:used]
                if len(set(last)) < len(last) or not written.isdisjoint(last):
                    raise ValueError("Two new tokens must not share a page of different places")
                written.update(last)
        width = max([len(r) for r in rows] + [1])
        if width > MAX_POSITIONS // page_size:
            raise ValueError(f"Sequences longer than {MAX_POSITIONS} tokens are not supported")
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32).reshape(len(rows), width)
        return cls(table, torch.tensor(lengths, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32))

    def to(self, device):
        return PagedPlan(self.page_table.to(device), self.context_lengths.to(device), self.query_offsets.to(device))


@dataclass(frozen=True)
class PagePool:
    """How many sequences hold each page of a cache; pages of none are free.

    ``refs``: contiguous int32 ``[pages]``, how many of the plan's tables name the
    page among their sequence's first ``ceil(context_lengths / page_size)``
    pages; ``missing``: int32 ``[1]``, the pages that the call which made the pool
    was to take, or to go on in, and could not; ``absent``: int64 ``[1]``, the pages
    that the plan's tokens need and its tables do not name, for whatever reason
    (missing now or before, or past the tables' width): 0 while every token has its
    place; None where nobody counted.  :func:`cache_fork` takes a pool's ``refs`` and
    returns the next pool.
    """

    refs: torch.Tensor
    missing: torch.Tensor
    absent_words: "torch.Tensor | None" = None  # int32 [2], absent's: a view of another type takes 0.6 us of a call

    @property
    def absent(self):
        return None if self.absent_words is None else self.absent_words.view(torch.int64)

    @classmethod
    def create(cls, cache, plan=None):
        """The pool of a cache whose pages are all free, or held by ``plan``, a
        :class:`PagedPlan` on any device."""
        if not isinstance(cache, PagedCache):
            raise ValueError("An explicit PagedCache is required")
        pages, _, page_size, _ = cache.k.shape
        refs, absent = torch.zeros(pages, dtype=torch.int32), 0
        if plan is not None:
            if not isinstance(plan, PagedPlan):
                raise ValueError("An explicit PagedPlan is required")
            for row, length in zip(plan.page_table.tolist(), plan.context_lengths.tolist()):
                needed = -(-max(length, 0) // page_size)
                absent += max(needed - len(row), 0)
                for page in row[:needed]:
                    if not 0 <= page < pages:
                        raise ValueError("page_table names a page outside the cache")
                    refs[page] += 1
        device = cache.k.device
        return cls(refs.to(device), torch.zeros(1, dtype=torch.int32, device=device),
                   torch.tensor([absent], dtype=torch.int64, device=device).view(torch.int32))


def _validate(cache, plan, device):
    """Checks a cache and a plan, and that they lie on ``device``; returns the cache's ``(heads, head_dim)``."""
    if not isinstance(cache, PagedCache):
        raise ValueError("An explicit PagedCache is required")
    if not isinstance(plan, PagedPlan):
        raise ValueError("An explicit PagedPlan is required")
    k, v, table, lengths, offsets = cache.k, cache.v, plan.page_table, plan.context_lengths, plan.query_offsets
    shape, dtype = k.shape, k.dtype
    if (len(shape) != 4 or v.shape != shape or dtype not in _native.CACHE_FORMATS or v.dtype != dtype
            or k.numel() == 0 or not (k.is_contiguous() and v.is_contiguous()) or (k.data_ptr() | v.data_ptr()) & 15):
        raise ValueError("Invalid cache tensors; use PagedCache.create")
    if k.requires_grad or v.requires_grad:
        raise ValueError("Inference only: the cache must not require gradients")
    _, heads, page_size, dim = shape
    if dim != 128 and dim != 64:
        raise ValueError("Only head dimensions 64 and 128 are implemented")
    if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
        _page_size(page_size)
    at = k.get_device()  # (integers compare in half the time of devices)
    if dtype != torch.bfloat16:
        rows = shape[:3]
        for x in (cache.k_scales, cache.v_scales):
            if (not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.shape != rows
                    or not x.is_contiguous() or x.get_device() != at):
                raise ValueError("INT8 and FP8 caches need contiguous fp32 scales [pages, heads, page_size]")
    if (table.ndim != 2 or lengths.ndim != 1 or offsets.ndim != 1
            or not table.dtype == lengths.dtype == offsets.dtype == torch.int32
            or not (table.is_contiguous() and lengths.is_contiguous() and offsets.is_contiguous())):
        raise ValueError("Invalid paged descriptor; use PagedPlan.create")
    sequences, width = table.shape
    if lengths.numel() != sequences or offsets.numel() != sequences + 1:
        raise ValueError("Invalid paged descriptor; use PagedPlan.create")
    if sequences and not 0 < width <= MAX_POSITIONS // page_size:
        raise ValueError(f"page_table must name 1 to {MAX_POSITIONS} positions of each sequence")
    if torch.version.hip is None or device.type != "cuda" or at != device.index or at != v.get_device():
        raise ValueError("The HIP backend requires the tensors and the cache on the same AMD ROCm GPU")
    if at != table.get_device() or at != lengths.get_device() or at != offsets.get_device():
        raise ValueError("Transfer the plan to the cache's device first")
    return heads, dim


def _overlap(x, y):
    """Whether two tensors' address ranges meet."""
    ends = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
            for t in (x, y)]
    return x.numel() > 0 and y.numel() > 0 and ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]


def _alike_overlap(x, y):
    """The same of two contiguous tensors of one shape and type."""
    return abs(x.data_ptr() - y.data_ptr()) < x.numel() * x.element_size()


def _separate(cache):
    """Refuses a cache that a call writes, where K and V are one."""
    if _alike_overlap(cache.k, cache.v) or (cache.k.dtype != torch.bfloat16
                                            and _alike_overlap(cache.k_scales, cache.v_scales)):
        raise ValueError("The cache's K and V, and their scales, must not share memory")


def _check_rows(name, x):
    if x.ndim != 3:
        raise ValueError(f"{name} must have NHD rank-3 layout")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"Only BF16 {name} are implemented")
    if x.requires_grad:
        raise ValueError(f"Inference only: {name} must not require gradients")
    if x.stride(2) != 1 or min(x.stride()) <= 0:
        raise ValueError(f"{name} need positive strides and contiguous head dimension")


def cache_write(k, v, cache, plan):
    """Stores the new tokens' K and V rows, BF16 ``[N, heads, head_dim]``, in ``cache``.

    Row ``plan.query_offsets[s] + i`` goes to sequence s's position
    ``context_lengths[s] - new + i``; rows at and past the last offset are not
    stored, and everything else in the cache is left as it was.  Per token and
    head, INT8 stores ``round(x * 127 / max|x|)`` (half to even) and FP8 the
    e4m3 value nearest ``x * 448 / max|x|``, with the scale ``max|x| / 127``
    (``/ 448``); a row with an infinity or a NaN reads back as NaN.  ``k`` and
    ``v`` may be views of a BF16 cache (a page copied to another), but not of
    rows that the call writes.
    """
    _check_rows("K/V", k)
    _check_rows("K/V", v)
    if k.shape != v.shape or k.device != v.device:
        raise ValueError("K and V must have the same shape and device")
    if k.shape[1:] != _validate(cache, plan, k.device):
        raise ValueError("K/V heads and head dimension must be the cache's")
    _separate(cache)
    with _on(k.device):
        _native.launch_cache_write(k, v, cache, plan)


def cache_read(cache, plan, tokens, *, start=0):
    """``(k, v)``: positions ``start`` .. ``start + tokens - 1`` of every sequence as
    contiguous BF16 ``[sequences, tokens, heads, head_dim]``, zeros at and past
    its ``context_lengths``.  Codes times scale in FP32, rounded once."""
    _nonnegative_integer("tokens", tokens)
    _nonnegative_integer("start", start)
    if tokens >= MAX_POSITIONS or start >= MAX_POSITIONS:
        raise ValueError(f"Sequences longer than {MAX_POSITIONS} tokens are not supported")
    device = cache.k.device if isinstance(cache, PagedCache) else None
    _validate(cache, plan, device)
    with _on(device):
        return _native.launch_cache_read(cache, plan, start, tokens)


def paged_attention(q, cache, plan, *, causal=True, window=None, sink_tokens=0, scale=None, out=None):
    """BF16 attention of the new tokens ``q`` ``[N, Hq, D]`` over what ``cache`` stores.

    Row ``plan.query_offsets[s] + i`` is the query at sequence s's position
    ``context_lengths[s] - new + i``; its K and V rows are stored first
    (:func:`cache_write`).  Query heads, causality, window and first tokens as in
    :func:`window_attention`: with ``causal=False`` the new tokens see one
    another (a video frame), with one new token per sequence the call is a
    decoding step.  FP32 scores, softmax and accumulation on the stored values
    (code times scale).  For its product with a value (a code) a probability
    (times the value's scale) is rounded to BF16, by at most 2^-8 of itself, in
    calls of chunks, and keeps 16 bits in decoding steps and small calls.  A
    query that sees no key gets zeros; infinities and NaN as in
    :func:`window_attention`.

    ``out``: an optional contiguous BF16 tensor shaped like ``q``.  Rows at and
    past the last offset are not computed: they are left as they were in
    ``out``, and are unspecified without it.
    """
    return _attend(q, cache, plan, causal, window, sink_tokens, scale, out)


def tree_attention(q, cache, plan, parents, *, window=None, sink_tokens=0, scale=None, out=None):
    """BF16 attention of new tokens that are trees of drafts, over what ``cache`` stores.

    As :func:`paged_attention`, but new token i of a sequence (row
    ``plan.query_offsets[s] + i``, its K and V rows stored at position
    ``context_lengths[s] - new + i`` first) need not follow the one before it:
    ``parents`` (contiguous int32 ``[N]``, a number per row of ``q``) names the
    new token of its sequence, one before it, that it continues; anything else,
    -1 say, makes it a root, which continues the stored tokens.  It sees the
    tokens before the new ones, its ancestors and itself.  With a ``window`` it
    sees those whose position is less than ``window`` before its own, and the
    first ``sink_tokens``; a draft's position is the number of stored tokens
    plus its depth (0 for a root), which is also where :func:`rotate_heads` has
    to turn it to.  Probabilities are rounded as there: to BF16 in calls of many
    new tokens per sequence, times the query heads that share a head, and not
    before 16 bits in those of few and in small calls.  :func:`cache_keep` keeps
    the accepted ones.
    """
    if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int32 or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous int32 tensor")
    if parents.shape != q.shape[:1]:
        raise ValueError("parents must have an entry for each row of Q")
    return _attend(q, cache, plan, True, window, sink_tokens, scale, out, parents)


def _attend(q, cache, plan, causal, window, sink_tokens, scale, out, parents=None):
    _check_rows("Q", q)
    heads, dim = _validate(cache, plan, q.device)
    if q.shape[2] != dim or q.shape[1] == 0 or q.shape[1] % heads:
        raise ValueError("Q heads must be a multiple of the cache's, of its head dimension")
    if plan.context_lengths.shape[0] > MAX_ATTENDED:
        raise ValueError(f"More than {MAX_ATTENDED} sequences in one call are not supported")
    scale = dim ** -0.5 if scale is None else float(scale)
    window = _visibility(scale, causal, window, sink_tokens)
    if out is not None and (out.dtype != torch.bfloat16 or out.shape != q.shape or not out.is_contiguous()
                            or out.device != q.device or out.data_ptr() & 15):
        raise ValueError("out must be a contiguous BF16 tensor shaped like Q on its device")
    if out is not None and out.requires_grad:
        raise ValueError("Inference only: out must not require gradients")
    if out is not None:
        scales = () if cache.k.dtype == torch.bfloat16 else (cache.k_scales, cache.v_scales)
        if any(_overlap(out, x) for x in (q, cache.k, cache.v, *scales)):
            raise ValueError("out must not share memory with Q or the cache")
    if parents is not None and parents.get_device() != q.get_device():
        raise ValueError("parents must be on Q's device")
    with _on(q.device):
        return _native.launch_paged(q, cache, plan, scale, causal, window, min(sink_tokens, MAX_POSITIONS), out, parents)


def _check_integers(name, x, shape, device):
    """Checks an int32 tensor on the GPU ``device`` (its index); None in ``shape``: any number."""
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor")
    sizes = x.shape
    if len(sizes) != len(shape) or (sizes[0] != shape[0] and shape[0] is not None):
        raise ValueError(f"{name} must have an entry for each sequence")
    if x.get_device() != device:
        raise ValueError(f"{name} must be on the cache's device")


def cache_keep(cache, plan, kept):
    """Moves the kept ones of the new tokens together: the accepted drafts of a tree
    (:func:`tree_attention`), or what is left of a frame that is thinned out.

    ``kept``: int32 ``[sequences, most]``: which of sequence s's new tokens stay,
    their numbers (0 .. new - 1) in ascending order; the first entry that does
    not ascend or is not one of them (-1, say) ends the list.  The K and V rows
    of new token ``kept[s, j]`` (of position ``context_lengths[s] - new +
    kept[s, j]``) move to that of new token j, in place; rows behind the kept
    ones stay as they are, and a row that has no page moves as zeros.  Stored
    values move as they are: keys that were turned by their positions keep those
    (:func:`rotate_heads` turns a draft by its depth, which is its place once it is
    kept).

    Returns the sequences' lengths then, int32 ``[sequences]``: what
    :func:`cache_fork` continues from, or the lengths of a plan of your own.
    """
    device = cache.k.device if isinstance(cache, PagedCache) else None
    _validate(cache, plan, device)
    _separate(cache)
    _check_integers("kept", kept, (plan.page_table.shape[0], None), device.index)
    with _on(device):
        return _native.launch_cache_keep(cache, plan, kept)


def cache_fork(cache, pool, plan, parents, new_tokens, *, lengths=None, width=None):
    """``(plan, pool)`` of the next call: sequences go on, branch, end or begin, on the GPU.

    New sequence i continues sequence ``parents[i]`` of ``plan`` (int32
    ``[new_sequences]``; outside of it, -1 say: none, the sequence begins) and has
    ``new_tokens[i]`` (int32, too) more tokens behind, whose rows
    :func:`cache_write` stores next.  A sequence that is no one's parent ends,
    and one that several continue branches: beams, samples of one prompt.
    ``lengths`` (int32 ``[sequences]``, from :func:`cache_keep`) continues from the
    first so many of a sequence's tokens instead of all.

    Whole pages are shared; a sequence's first child goes on in the pages behind
    them that no other sequence holds; the other children take pages of their
    own, and a copy of the rows that the first one begins with.  Pages are taken
    from those that ``pool`` has free, the lowest first, and freed pages are
    free for the next call.  Where none is left a table has -1, which is no page
    (not written, not attended), for the children that go on in it too, and
    ``missing`` of the new pool counts them.  ``absent`` of the new pool counts all
    pages that the new sequences' tokens lack, those of later calls' whole pages and
    those past ``width`` too: a program that generates without asking the host for
    lengths looks at this one.

    ``width``: pages that a new table has room for, by default the old one's; the
    lengths go on past it, the tokens there are not stored or attended.
    ``plan`` and ``pool`` stay as they were, but the sequences they describe must
    not be written any more: their pages have new owners.  (Two calls on one pool
    take the same pages: only one of the results can be gone on with.)
    """
    device = cache.k.device if isinstance(cache, PagedCache) else None
    _validate(cache, plan, device)
    _separate(cache)
    if not isinstance(pool, PagePool):
        raise ValueError("An explicit PagePool is required")
    at, table, store = device.index, plan.page_table.shape, cache.k.shape
    _check_integers("parents", parents, (None,), at)
    branches = parents.shape
    _check_integers("new_tokens", new_tokens, branches, at)
    if lengths is not None:
        _check_integers("lengths", lengths, table[:1], at)
    refs = pool.refs
    if refs.dtype != torch.int32 or refs.ndim != 1 or refs.shape[0] != store[0] or not refs.is_contiguous():
        raise ValueError("Invalid pool; use PagePool.create with this cache")
    if refs.get_device() != at:
        raise ValueError("The pool must be on the cache's device")
    if width is None:
        width = table[1]
    else:
        _nonnegative_integer("width", width)
    if not 0 < width <= MAX_POSITIONS // store[2]:
        raise ValueError(f"width must name 1 to {MAX_POSITIONS} positions of each sequence")
    if max(table[0], branches[0]) > MAX_ATTENDED:
        raise ValueError(f"More than {MAX_ATTENDED} sequences in one call are not supported")
    with _on(device):
        table, lengths, offsets, *left = _native.launch_cache_fork(cache, refs, plan, parents, new_tokens, lengths, width)
    return PagedPlan(table, lengths, offsets), PagePool(*left)
