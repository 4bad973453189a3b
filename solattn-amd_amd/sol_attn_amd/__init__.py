"""Inference-only SOL-style BF16 routed attention, MI355X-native (gfx950 HIP kernels)."""

from .attention import SolStats, dense_attention, sol_attention, window_attention
from .indexed import IndexedPlan, sol_attention_indexed
from .rotary import RotaryAxes, rotate_heads
from .paged import (PagedCache, PagedPlan, PagePool, cache_fork, cache_keep, cache_read, cache_write,
                    paged_attention, tree_attention)

__all__ = ["SolStats", "dense_attention", "sol_attention", "IndexedPlan", "sol_attention_indexed",
           "window_attention", "PagedCache", "PagedPlan", "cache_write", "cache_read", "paged_attention", "RotaryAxes",
           "rotate_heads", "PagePool", "cache_keep", "cache_fork", "tree_attention"]
