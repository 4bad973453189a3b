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


def _validate(cache, plan, device):
    """Checks a cache and a plan, and that they lie on ``device``; returns the cache's ``(heads, head_dim)``."""
    if not isinstance(cache, PagedCache):
        raise ValueError("An explicit PagedCache is required")
    if not isinstance(plan, PagedPlan):
        raise ValueError("An explicit PagedPlan is required")
    k, v, table, lengths, offsets = cache.k, cache.v, plan.page_table, plan.context_lengths, plan.query_offsets
    shape, dtype = k.shape, k.dtype
    if (len(shape) != 4 or v.shape != shape or dtype not in _native.CACHE_FORMATS or v.dtype != dtype
            or min(shape) <= 0 or not k.is_contiguous() or not v.is_contiguous()
            or (k.data_ptr() | v.data_ptr()) & 15):
        raise ValueError("Invalid cache tensors; use PagedCache.create")
    if k.requires_grad or v.requires_grad:
        raise ValueError("Inference only: the cache must not require gradients")
    if shape[3] not in (64, 128):
        raise ValueError("Only head dimensions 64 and 128 are implemented")
    _page_size(shape[2])
    if dtype != torch.bfloat16:
        for x in (cache.k_scales, cache.v_scales):
            if (not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.shape != shape[:3]
                    or not x.is_contiguous() or x.get_device() != k.get_device()):
                raise ValueError("INT8 and FP8 caches need contiguous fp32 scales [pages, heads, page_size]")
    if (table.ndim != 2 or lengths.ndim != 1 or offsets.ndim != 1 or lengths.shape[0] != table.shape[0]
            or offsets.shape[0] != table.shape[0] + 1
            or not table.dtype == lengths.dtype == offsets.dtype == torch.int32
            or not (table.is_contiguous() and lengths.is_contiguous() and offsets.is_contiguous())):
        raise ValueError("Invalid paged descriptor; use PagedPlan.create")
    if table.shape[0] and not 0 < table.shape[1] <= MAX_POSITIONS // shape[2]:
        raise ValueError(f"page_table must name 1 to {MAX_POSITIONS} positions of each sequence")
    at = k.get_device()  # (integers compare in half the time of devices)
    if torch.version.hip is None or device.type != "cuda" or at != device.index or at != v.get_device():
        raise ValueError("The HIP backend requires the tensors and the cache on the same AMD ROCm GPU")
    if at != table.get_device() or at != lengths.get_device() or at != offsets.get_device():
        raise ValueError("Transfer the plan to the cache's device first")
    return shape[1], shape[3]


def _overlap(x, y):
    """Whether two tensors' address ranges meet."""
    ends = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
            for t in (x, y)]
    return x.numel() > 0 and y.numel() > 0 and ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]


def _alike_overlap(x, y):
    """The same of two contiguous tensors of one shape and type."""
    return abs(x.data_ptr() - y.data_ptr()) < x.numel() * x.element_size()


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
    if _alike_overlap(cache.k, cache.v) or (cache.k.dtype != torch.bfloat16
                                            and _alike_overlap(cache.k_scales, cache.v_scales)):
        raise ValueError("The cache's K and V, and their scales, must not share memory")
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
    with _on(q.device):
        return _native.launch_paged(q, cache, plan, scale, causal, window, min(sink_tokens, MAX_POSITIONS), out)
