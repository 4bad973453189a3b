"""Norms of the heads of Q and K, and their rotation by the tokens' positions.

What a model does to Q and K before they are attended (:func:`sol_attention`,
:func:`dense_attention`, :func:`window_attention`) or stored
(:func:`cache_write`): :func:`rotate_heads` norms each head's row and turns its
pairs of elements by angles that grow with the token's position, along one axis
(a text) or several (time, height and width of a video's tokens), in one pass.
Not in the reference.
"""

from dataclasses import dataclass
import math

import torch

from . import _native
from .attention import _nonnegative_integer, _on

LAYOUTS = ("halves", "pairs")
NORM_TYPES = (torch.float32, torch.bfloat16)


@dataclass(frozen=True)
class RotaryAxes:
    """How the pairs of a head's row turn with a token's position.

    ``frequencies``: contiguous fp64 ``[head_dim / 2]``, radians per position;
    ``axes``: contiguous int32 ``[head_dim / 2]``, the axis of the position that
    a pair turns with (outside the positions' axes: it does not turn).
    ``layout``: pair j is elements j and ``j + head_dim / 2`` ("halves"), or ``2 j``
    and ``2 j + 1`` ("pairs").  Use :meth:`create`, or give tensors of your own
    (scaled frequencies, axes in another order); a captured launch follows what
    they hold at replay.
    """

    frequencies: torch.Tensor
    axes: torch.Tensor
    layout: str = "halves"

    @classmethod
    def create(cls, head_dim, pairs, *, base=10000.0, shared=False, layout="halves", device="cuda"):
        """``pairs``: how many pairs turn with each axis, in their order (an integer: one axis);
        pairs left over do not turn.  Pair j of an axis's n has the frequency
        ``base ** (-j / n)``; with ``shared`` one ladder runs over all axes'
        pairs."""
        if head_dim not in (64, 128):
            raise ValueError("Only head dimensions 64 and 128 are implemented")
        counts = [pairs] if isinstance(pairs, int) else list(pairs)
        for n in counts:
            _nonnegative_integer("pairs", n)
        if not counts or sum(counts) > head_dim // 2:
            raise ValueError("pairs must name an axis, and at most head_dim / 2 pairs in all")
        base = float(base)
        if not 0 < base < math.inf:
            raise ValueError("base must be finite and positive")
        if layout not in LAYOUTS:
            raise ValueError("layout must be 'halves' or 'pairs'")
        turning, left = sum(counts), head_dim // 2 - sum(counts)
        if shared:
            ladder = [base ** (-j / turning) for j in range(turning)]
        else:
            ladder = [base ** (-j / n) for n in counts for j in range(n)]
        axes = [a for a, n in enumerate(counts) for _ in range(n)]
        return cls(torch.tensor(ladder + [0.0] * left, dtype=torch.float64, device=device),
                   torch.tensor(axes + [-1] * left, dtype=torch.int32, device=device), layout)


def _meet(x, y):
    """Whether two BF16 row tensors may share memory.  Views of one projection do not: alike in all strides, each with
    its own heads of every token."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    lo, hi = (x, y) if x.data_ptr() <= y.data_ptr() else (y, x)
    reach = [1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) for t in (lo, hi)]
    apart = (hi.data_ptr() - lo.data_ptr()) // 2
    if apart >= reach[0]:
        return False
    if lo.stride()[:-2] != hi.stride()[:-2]:
        return True
    token = lo.stride(-3)
    heads = [(t.shape[-2] - 1) * t.stride(-2) + t.shape[-1] for t in (lo, hi)]
    # Tokens apart by whole multiples of their stride: heads [0, h) and [at, at + h) of it.
    if any(s % token for s in lo.stride()[:-3]):
        return True
    at = apart % token
    return not (heads[0] <= at and at + heads[1] <= token)


def _same(x, y):
    return x.data_ptr() == y.data_ptr() and x.stride() == y.stride()


def _meets_itself(x):
    """Whether a tensor's elements may share memory among themselves."""
    reach = 1
    for stride, size in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride < reach:
            return True
        reach = stride * (size - 1) + reach
    return False


def _check_out(inputs, outs):
    """Outputs are new memory, or their own inputs."""
    for i, (x, out) in enumerate(zip(inputs, outs)):
        if not isinstance(out, torch.Tensor) or out.dtype != torch.bfloat16 or out.shape != x.shape or out.device != x.device:
            raise ValueError("out must be BF16 tensors shaped like Q and K on their device")
        if out.requires_grad:
            raise ValueError("Inference only: out must not require gradients")
        if out.numel() and (min(out.stride()) <= 0 or out.stride(-1) != 1 or not _native._aligned(out)):
            raise ValueError("out needs positive strides, contiguous head dimension and 16-byte aligned rows")
        if _meets_itself(out):
            raise ValueError("out must not share memory with itself")
        if not _same(x, out) and _meet(x, out):
            raise ValueError("out must be Q and K themselves or share no memory with them")
        for j, other in enumerate(inputs):
            if j != i and _meet(other, out):
                raise ValueError("out must be Q and K themselves or share no memory with them")
    if len(outs) == 2 and _meet(*outs):
        raise ValueError("The two outputs must not share memory")


def rotate_heads(q, k, positions, rotary, *, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """``(q, k)`` with their heads' rows normed and turned by the tokens' positions.

    ``q``/``k``: BF16 ``[B, T, H, D]`` or ``[N, H, D]``, of the same tokens but any
    numbers of heads, views of one projection for instance; ``k`` may be None,
    and the result is Q's alone.  ``positions``: int32 ``[B, T, axes]`` or ``[N,
    axes]`` (expanded ones too), negative ones turn back.  ``rotary``: a
    :class:`RotaryAxes`.  With ``q_norm`` (``k_norm``), contiguous FP32 or BF16
    weights ``[D]``, a row x becomes ``x * weight / sqrt(mean(x ** 2) + eps)``
    before it turns.  A pair (a, b) at angle t becomes ``(a cos t - b sin t, a
    sin t + b cos t)``.  Angles in FP64, everything else in FP32, rounded once:
    stored keys turn on by ``positions`` that say by how much.

    ``out``: None for new contiguous tensors, or two tensors ``(q_out, k_out)``
    (one where ``k`` is None) of any positive strides, which may be Q and K
    themselves.
    """
    alone = k is None
    if q is None or q.ndim not in (3, 4) or (not alone and k.ndim != q.ndim):
        raise ValueError("Q and K must have BTHD rank-4 or NHD rank-3 layout")
    if q.dtype != torch.bfloat16 or (not alone and k.dtype != torch.bfloat16):
        raise ValueError("Only BF16 Q and K are implemented")
    shape, strides = q.shape, q.stride()
    tokens, dim = shape[:-2], shape[-1]
    if not alone and (k.shape[:-2] != tokens or k.shape[-1] != dim):
        raise ValueError("Q and K must be rows of the same tokens and head dimension")
    if dim != 128 and dim != 64:
        raise ValueError("Only head dimensions 64 and 128 are implemented")
    if shape[-2] == 0 or (not alone and k.shape[-2] == 0) or (len(shape) == 4 and shape[0] == 0):
        raise ValueError("Q and K need a batch entry and a head")
    if q.requires_grad or (not alone and k.requires_grad):
        raise ValueError("Inference only: Q and K must not require gradients")
    if strides[-1] != 1 or min(strides) <= 0 or (not alone and (k.stride(-1) != 1 or min(k.stride()) <= 0)):
        raise ValueError("Q and K need positive strides and contiguous head dimension")
    at = positions.shape
    if positions.dtype != torch.int32 or at[:-1] != tokens or at[-1] == 0:
        raise ValueError("positions must be int32, an entry per axis for every token")
    if at[-1] != 1 and positions.stride(-1) != 1:
        raise ValueError("positions need contiguous axes")
    if not isinstance(rotary, RotaryAxes):
        raise ValueError("An explicit RotaryAxes is required")
    freq, axes = rotary.frequencies, rotary.axes
    if (freq.dtype != torch.float64 or axes.dtype != torch.int32 or not freq.ndim == axes.ndim == 1
            or not freq.numel() == axes.numel() == dim // 2 or not (freq.is_contiguous() and axes.is_contiguous())
            or rotary.layout not in LAYOUTS):
        raise ValueError("Invalid rotary descriptor; use RotaryAxes.create for this head dimension")
    if freq.requires_grad:
        raise ValueError("Inference only: frequencies must not require gradients")
    if alone and k_norm is not None:
        raise ValueError("k_norm needs K")
    device = q.get_device()
    same = (positions.get_device() == device and freq.get_device() == device and axes.get_device() == device
            and (alone or k.get_device() == device))
    for w in (q_norm, k_norm):
        if w is None:
            continue
        if w.dtype not in NORM_TYPES or w.ndim != 1 or w.numel() != dim or not w.is_contiguous():
            raise ValueError("Norm weights must be contiguous FP32 or BF16 of the head dimension")
        if w.requires_grad:
            raise ValueError("Inference only: norm weights must not require gradients")
        same = same and w.get_device() == device
    if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
        raise ValueError("Norm weights must have one type")
    if not 2.0 ** -126 <= eps < 2.0 ** 127:
        raise ValueError("eps must be a positive FP32 number")
    if torch.version.hip is None or device < 0 or not same:
        raise ValueError("The HIP backend requires all tensors on the same AMD ROCm GPU")
    q_out = k_out = None
    if out is not None:
        outs = [out] if alone else list(out)
        if len(outs) != 1 + (not alone):
            raise ValueError("out must be one tensor for Q and one for K")
        _check_out([q] if alone else [q, k], outs)
        q_out, k_out = outs[0], None if alone else outs[1]
    with _on(q.device):
        q_out, k_out = _native.launch_rotate(q, k, positions, rotary, q_norm, k_norm, float(eps), q_out, k_out)
    return q_out if alone else (q_out, k_out)
