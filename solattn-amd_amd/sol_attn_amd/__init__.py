"""Inference-only SOL-style BF16 routed attention, MI355X-native (gfx950 HIP kernels)."""

from .attention import SolStats, dense_attention, sol_attention, window_attention
from .indexed import IndexedPlan, sol_attention_indexed
from .paged import PagedCache, PagedPlan, cache_read, cache_write, paged_attention

__all__ = ["SolStats", "dense_attention", "sol_attention", "IndexedPlan", "sol_attention_indexed",
           "window_attention", "PagedCache", "PagedPlan", "cache_write", "cache_read", "paged_attention"]
