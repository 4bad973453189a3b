"""The heads' norms and rotation in 64 bits, and what the kernel may be off by.

Tolerance of an element a cos t - b sin t (a, b the normed pair, exact):
  - its rounding to BF16: half a step, 2^-8 of it (2^-134 below BF16's normal numbers);
  - the norm in FP32: a sum of squares of 16 elements per lane and three sums over lanes, 19 roundings, halved by the
    root; the mean, eps, root, quotient, three products: under 16 roundings of 2^-24 in all, 2^-20 of a and b;
  - cos and sin: the angle in FP64 (three roundings of 2^-53 of it), its part of a turn rounded to FP32 (2^-26 of a
    turn, 2^-23.3), sincospi's own few units of 2^-24: under 2^-21 + |t| 2^-51 each;
  - two products and a sum in FP32: 3 roundings of 2^-24 of |a| + |b|;
together 2^-8 |y| + (2^-19 + |t| 2^-51) (|a| + |b|).
"""

import numpy as np
import torch


def rotated(x, positions, frequencies, axes, layout, norm=None, eps=1e-6):
    """x [..., H, D], positions [..., A] -> (y, bound) in 64 bits (numpy)."""
    x = x.detach().cpu().double().numpy()
    positions = positions.detach().cpu().double().numpy()
    frequencies, axes = frequencies.detach().cpu().numpy(), axes.detach().cpu().numpy()
    with np.errstate(all="ignore"):
        if norm is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.detach().cpu().double().numpy()
        turns = (axes >= 0) & (axes < positions.shape[-1])
        angle = np.where(turns, positions[..., np.where(turns, axes, 0)] * frequencies, 0.0)[..., None, :]
        half = x.shape[-1] // 2
        a, b = (x[..., :half], x[..., half:]) if layout == "halves" else (x[..., 0::2], x[..., 1::2])
        y = np.empty_like(x)
        bound = np.empty_like(x)
        parts = (a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle))
        slack = (2.0 ** -19 + np.abs(angle) * 2.0 ** -51) * (np.abs(a) + np.abs(b)) + 2.0 ** -133
        for i, part in enumerate(parts):
            place = (slice(i * half, (i + 1) * half),) if layout == "halves" else (slice(i, None, 2),)
            y[(..., *place)] = part
            bound[(..., *place)] = 2.0 ** -8 * np.abs(part) + slack
    return y, bound


def check(actual, x, positions, rotary, norm=None, eps=1e-6):
    y, bound = rotated(x, positions, rotary.frequencies, rotary.axes, rotary.layout, norm, eps)
    a = actual.detach().cpu().double().numpy()
    assert a.shape == y.shape
    nan = np.isnan(y)
    assert np.array_equal(np.isnan(a), nan), "NaN in other places"
    off = np.where(nan, 0.0, np.abs(a - y) - bound)
    assert off.size == 0 or off.max() <= 0, f"off by {off.max()} over the bound at {np.unravel_index(np.argmax(off), off.shape)}"


def positions_of(*shape, axes, reach, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-reach, reach, shape + (axes,), generator=g).to(torch.int32)
