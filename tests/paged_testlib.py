"""Plain 64-bit forms of the paged-cache and windowed-attention operators, and what the kernels may be off by.

Tolerance of an attention output O = sum p_j v_j (p the softmax, A = sum p_j |v_j|):
  - the output's rounding to BF16: half a step, 2^-8 |O|;
  - each probability's rounding to BF16 before its product with v (times its scale): 2^-8 A; the denominator sums
    the unrounded ones;
  - scores in FP32: D + 2 roundings of at most Q = max sum |q k| scale, each 2^-24; a score off by e moves p by 2 e A
    (its own and the denominator's);
  - FP32 sums, exp2 and the rescaling: a few 2^-23 of A per step, covered by 2^-12 A;
  - what FP32 and BF16 cannot hold: a probability (relative to the largest) or a result below their smallest normal
    number, 2^-126, may be taken for 0: 2^-126 (1 + sum |v_j|), as the denominator is at least 1.
"""

import math

import numpy as np
import torch

LEVELS = {"int8": 127.0, "fp8": 448.0}


def stored(x, fmt):
    """(codes, scales) a cache of format ``fmt`` holds for BF16 rows x [..., D], in 64 bits."""
    x = x.detach().cpu().double()
    if fmt == "bf16":
        return x, None
    most = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    codes = torch.where((most > 0)[..., None], x * LEVELS[fmt] / torch.where(most > 0, most, 1.0)[..., None], 0.0)
    codes = torch.where(bad[..., None], 0.0, codes)
    codes = codes.round() if fmt == "int8" else codes.float().to(torch.float8_e4m3fn).double()
    scale = (most / LEVELS[fmt]).float()
    return codes, torch.where(bad, math.nan, scale)


def values(x, fmt):
    """The values BF16 rows x [..., D] stand for once stored, in 64 bits."""
    codes, scale = stored(x, fmt)
    return codes if scale is None else codes * scale.double()[..., None]


def visible(pos, length, causal, window, sinks):
    """Keys 0 .. length - 1 that position ``pos`` sees (truth values)."""
    j = np.arange(length)
    seen = np.ones(length, dtype=bool)
    if causal:
        seen &= j <= pos
    if window:
        seen &= (np.abs(pos - j) < window) | (j < sinks)
    return seen


def attend(q, k, v, *, causal=True, window=None, sinks=0, scale=None, present=None):
    """One sequence: q [n, Hq, D], k / v [L, H, D] -> (O, bound), [n, Hq, D] in 64 bits; only visible keys are touched."""
    q, k, v = (np.asarray(x.detach().cpu().double()) for x in (q, k, v))
    n, heads, dim = q.shape
    length, kv = k.shape[:2]
    scale = dim ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        seen = visible(length - n + i, length, causal, window, sinks)
        if present is not None:
            seen &= present
        if not seen.any():
            continue
        ks, vs = k[seen], v[seen]
        for h in range(kv):
            qs = q[i, h * (heads // kv):(h + 1) * (heads // kv)]
            with np.errstate(invalid="ignore", over="ignore"):
                s = qs @ ks[:, h].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                o, a = p @ vs[:, h], p @ np.abs(vs[:, h])
                most = (np.abs(qs) @ np.abs(ks[:, h]).T).max() * scale
            out[i, h * (heads // kv):(h + 1) * (heads // kv)] = o
            bound[i, h * (heads // kv):(h + 1) * (heads // kv)] = (
                2 ** -8 * np.abs(o) + (2 ** -8 + 2 ** -12 + 2 * (dim + 2) * 2 ** -24 * most) * a
                + 2.0 ** -126 * (1 + np.abs(vs[:, h]).sum(0)))
    return out, bound


def assert_within(actual, expected, bound):
    a = np.asarray(actual.detach().cpu().double())
    assert a.shape == expected.shape
    nan = np.isnan(expected)
    assert np.array_equal(np.isnan(a), nan), "NaN in other places"
    off = np.where(nan, 0.0, np.abs(a - expected)) - np.where(nan, 0.0, bound)
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off.max() <= 0, f"{a[worst]} for {expected[worst]} at {worst}, bound {bound[worst]}"


def rows(*shape, seed=0, device="cpu"):
    """BF16 rows of different sizes, a few features larger than the others."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g))
    x[..., ::17] *= 2
    return x.to(torch.bfloat16).to(device)


class Sequences:
    """A batch of sequences with their K and V rows (CPU), and a cache and plan (GPU) that hold them."""

    def __init__(self, lengths, new, *, heads=2, dim=64, fmt="bf16", page_size=16, seed=0, spare=3, fill=0.0):
        from sol_attn_amd import PagedCache, PagedPlan
        self.lengths, self.new, self.fmt, self.page_size = list(lengths), list(new), fmt, page_size
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page_size) for n in lengths]
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=g).tolist()
        table, at = [], 0
        for n in used:
            table.append(order[at:at + n])
            at += n
        self.table, self.pages = table, pages
        self.k = [rows(n, heads, dim, seed=seed * 100 + 2 * i + 1) for i, n in enumerate(lengths)]
        self.v = [rows(n, heads, dim, seed=seed * 100 + 2 * i + 2) for i, n in enumerate(lengths)]
        self.cache = PagedCache.create(pages, page_size, heads, dim, format=fmt)
        if fill != 0.0:
            stores = (self.cache.k, self.cache.v) if fmt == "bf16" else (self.cache.k_scales, self.cache.v_scales)
            for x in stores:
                x.fill_(fill)
        self.plan = PagedPlan.create(table, lengths, new, pages=pages, page_size=page_size).to("cuda")
        self.store()

    def store(self):
        """Puts the rows into the cache with plain indexing."""
        for s, table in enumerate(self.table):
            for name, x in (("k", self.k[s]), ("v", self.v[s])):
                if not len(x):
                    continue
                pos = torch.arange(len(x))
                page = torch.tensor(table)[pos // self.page_size].cuda()
                slot = (pos % self.page_size).cuda()
                codes, scale = stored(x, self.fmt)
                dst = getattr(self.cache, name)
                if self.fmt == "fp8":
                    dst.view(torch.int8)[page, :, slot] = codes.float().to(torch.float8_e4m3fn).view(torch.int8).cuda()
                else:
                    dst[page, :, slot] = codes.to(dst.dtype).cuda()
                if scale is not None:
                    getattr(self.cache, name + "_scales")[page, :, slot] = scale.float().cuda()

    def expected(self, q, **how):
        """(O, bound) of the new tokens' queries q [N, Hq, D]."""
        outs, at = [], 0
        for s, n in enumerate(self.new):
            outs.append(attend(q[at:at + n], values(self.k[s], self.fmt), values(self.v[s], self.fmt), **how))
            at += n
        return tuple(np.concatenate([o[i] for o in outs]) for i in (0, 1))
