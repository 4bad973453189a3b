"""Norms of the heads' rows and their rotation on the GPU, against the formulas in 64 bits (tolerances in
``rotary_testlib``), and the host contract on the CPU."""

import pytest
import torch

from paged_testlib import rows
from rotary_testlib import check, positions_of
from sol_attn_amd import RotaryAxes, rotate_heads


def weights(dim, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).cuda()


def axes_of(dim, axes, layout, left=0, device="cuda"):
    turning = dim // 2 - left
    counts = turning if axes == 1 else [turning - (axes - 1) * (turning // axes)] + [turning // axes] * (axes - 1)
    return RotaryAxes.create(dim, counts, layout=layout, device=device)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,hq,hk,axes,norm", [
    (1, 1, 1, 1, None), (7, 3, 1, 1, torch.float32), (8, 8, 2, 3, torch.bfloat16), (17, 5, 5, 2, None),
    (129, 12, 3, 3, torch.float32), (1000, 2, 1, 4, torch.bfloat16), (33, 40, 8, 3, torch.float32),
])
def test_rows_of_new_tokens(tokens, hq, hk, axes, norm, dim, layout):
    q, k = rows(tokens, hq, dim, seed=1, device="cuda"), rows(tokens, hk, dim, seed=2, device="cuda")
    positions = positions_of(tokens, axes=axes, reach=5000, seed=3).cuda()
    rotary = axes_of(dim, axes, layout)
    wq, wk = (None, None) if norm is None else (weights(dim, 4, norm), weights(dim, 5, norm))
    q2, k2 = rotate_heads(q, k, positions, rotary, q_norm=wq, k_norm=wk)
    assert q2.is_contiguous() and k2.is_contiguous() and q2.dtype == torch.bfloat16
    check(q2, q, positions, rotary, wq)
    check(k2, k, positions, rotary, wk)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("reach", [1 << 20, 1 << 30])
def test_far_positions_keep_their_angles(reach, dim):
    q = rows(50, 4, dim, seed=1, device="cuda")
    positions = positions_of(50, axes=1, reach=reach, seed=2).cuda()
    rotary = axes_of(dim, 1, "halves")
    check(rotate_heads(q, None, positions, rotary), q, positions, rotary)
    ends = torch.tensor([[-(1 << 31)], [(1 << 31) - 1], [0], [1]], dtype=torch.int32, device="cuda")
    check(rotate_heads(q[:4], None, ends, rotary), q[:4], ends, rotary)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_batches_of_a_projections_views_with_shared_positions(layout):
    both = rows(3, 61, 8 + 2 + 1, 128, seed=7, device="cuda")
    q, k = both[:, :, :8], both[:, :, 8:10]
    positions = positions_of(61, axes=3, reach=100, seed=8).cuda().expand(3, -1, -1)
    rotary = RotaryAxes.create(128, [20, 22, 22], layout=layout, shared=True)
    wk = weights(128, 9)
    q2, k2 = rotate_heads(q, k, positions, rotary, k_norm=wk)
    check(q2, q, positions, rotary)
    check(k2, k, positions, rotary, wk)
    # In place, and into every other row of something larger.
    want = q2.clone(), k2.clone()
    target = torch.full((3, 61, 2, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    q3, k3 = rotate_heads(q, k, positions, rotary, k_norm=wk, out=(target[:, :, 1], torch.empty_like(k2)))
    assert torch.equal(q3, want[0]) and torch.equal(k3, want[1]) and bool((target[:, :, 0] == 5).all())
    rest = both[:, :, 10].clone()
    q4, k4 = rotate_heads(q, k, positions, rotary, k_norm=wk, out=(q, k))
    assert q4.data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(both[:, :, 10], rest)


@pytest.mark.gpu
def test_misaligned_rows_and_pairs_without_an_axis():
    flat = rows(9 * 3 * 64 + 1, 1, seed=1, device="cuda").view(-1)
    q = flat[1:].view(9, 3, 64)
    positions = positions_of(9, axes=2, reach=50, seed=2).cuda()
    rotary = RotaryAxes.create(64, [7, 5], layout="pairs")
    q2 = rotate_heads(q, None, positions, rotary)
    check(q2, q, positions, rotary)
    assert torch.equal(q2[..., 24:], q[..., 24:])
    # An axis that the positions do not have turns nothing.
    odd = RotaryAxes(rotary.frequencies, torch.full_like(rotary.axes, 2), "halves")
    assert torch.equal(rotate_heads(q, None, positions, odd), q)
    # Whatever its frequency.
    odd = RotaryAxes(torch.full_like(rotary.frequencies, float("inf")), odd.axes, "pairs")
    assert torch.equal(rotate_heads(q, None, positions, odd), q)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim", [64, 128])
def test_pairs_without_an_axis_stay_as_they_are_whatever_they_hold(dim, layout):
    q = rows(21, 3, dim, seed=4, device="cuda")
    half = dim // 2
    # The last eight pairs have no axis: infinities, NaN and zeros of both signs beside ordinary partners and each other.
    first, second = ((slice(half - 8, half), slice(dim - 8, dim)) if layout == "halves"
                     else (slice(dim - 16, None, 2), slice(dim - 15, None, 2)))
    inf, nan = float("inf"), float("nan")
    q[..., first] = torch.tensor([inf, 1.5, -inf, inf, nan, -0.0, 2.0, -0.0], dtype=torch.bfloat16, device="cuda")
    q[..., second] = torch.tensor([0.5, -inf, inf, -3.0, 1.0, -1.0, nan, 0.0], dtype=torch.bfloat16, device="cuda")
    rotary = RotaryAxes.create(dim, half - 8, layout=layout)
    positions = positions_of(21, axes=1, reach=5000, seed=5).cuda()
    got = rotate_heads(q, None, positions, rotary)
    for part in (first, second):
        x, y = q[..., part], got[..., part]
        assert torch.equal(x.isnan(), y.isnan())
        assert torch.equal(x.view(torch.int16)[~x.isnan()], y.view(torch.int16)[~x.isnan()])
    # The others turn as ever.
    clean = q.clone()
    clean[..., first] = clean[..., second] = 1.0
    got[..., first] = got[..., second] = 1.0
    check(got, clean, positions, rotary)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("tokens,hq,hk,dim", [(32793, 5, 2, 64), (8203, 13, 3, 128), (8205, 3, 11, 128),
                                              (33001, 6, 0, 64)])
def test_calls_so_large_that_a_wave_takes_more_heads_than_it_loads_at_once(tokens, hq, hk, dim, layout):
    # Heads that neither four nor eight divide, Q's end inside a wave's, tokens that end inside a wave's.
    both = rows(tokens, hq + hk, dim, seed=6, device="cuda")
    q, k = both[:, :hq], both[:, hq:] if hk else None
    positions = positions_of(tokens, axes=3, reach=300, seed=7).cuda()
    rotary = axes_of(dim, 3, layout, left=3)
    norms = dict(q_norm=weights(dim, 8), k_norm=weights(dim, 9) if hk else None)
    got = rotate_heads(q, k, positions, rotary, **norms)
    for x, y, w in zip((q, k), got if hk else (got,), norms.values()):
        check(y, x, positions, rotary, w)
    rotate_heads(q, k, positions, rotary, out=(q, k) if hk else q, **norms)
    assert torch.equal(both, torch.cat(got, 1) if hk else got)


@pytest.mark.gpu
def test_turning_on_and_back():
    q = rows(40, 2, 128, seed=1, device="cuda")
    rotary = axes_of(128, 1, "halves")
    positions = positions_of(40, axes=1, reach=1 << 20, seed=2).cuda()
    there = rotate_heads(q, None, positions, rotary)
    check(rotate_heads(there, None, -positions, rotary), there, -positions, rotary)
    assert torch.equal(rotate_heads(q, None, torch.zeros_like(positions), rotary), q)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-6, 1e-30, 2e-38])
def test_rows_outside_the_range_of_their_squares(eps):
    q = rows(12, 4, 128, seed=3).float()
    for i, f in enumerate((1e-38, 1e-30, 1e-20, 1e-10, 1e10, 1e18, 1e19, 1e20, 1e30, 3e37)):
        q[i] *= f / q[i].abs().amax(-1, keepdim=True)
    q[10] = 0.0
    q = q.to(torch.bfloat16).cuda()
    w = weights(128, 4)
    positions = positions_of(12, axes=1, reach=100, seed=5).cuda()
    rotary = axes_of(128, 1, "pairs")
    check(rotate_heads(q, None, positions, rotary, q_norm=w, eps=eps), q, positions, rotary, w, eps)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rows_that_are_not_finite_stay_among_themselves(layout):
    q = rows(16, 3, 64, seed=3, device="cuda")
    clean = q.clone()
    q[3, 1, 5] = float("nan")
    q[7, 0, 63] = float("inf")
    q[9, 2] = float("-inf")
    positions = positions_of(16, axes=1, reach=100, seed=5).cuda()
    rotary = axes_of(64, 1, layout)
    w = weights(64, 6)
    for norm in (None, w):
        got = rotate_heads(q, None, positions, rotary, q_norm=norm)
        want = rotate_heads(clean, None, positions, rotary, q_norm=norm)
        other = torch.ones(16, 3, dtype=torch.bool)
        other[3, 1] = other[7, 0] = other[9, 2] = False
        assert torch.equal(got[other.cuda()], want[other.cuda()])
        assert not torch.isfinite(got.float())[9, 2].any() and got[3, 1].isnan().any()


@pytest.mark.gpu
def test_empty_calls_other_streams_and_replays():
    rotary = axes_of(128, 1, "halves")
    none = torch.empty((0, 4, 128), dtype=torch.bfloat16, device="cuda")
    q2, k2 = rotate_heads(none, none[:, :1], torch.empty((0, 1), dtype=torch.int32, device="cuda"), rotary)
    assert q2.shape == (0, 4, 128) and k2.shape == (0, 1, 128)
    q, k = rows(30, 4, 128, seed=1, device="cuda"), rows(30, 2, 128, seed=2, device="cuda")
    positions = positions_of(30, axes=1, reach=1000, seed=3).cuda()
    want = rotate_heads(q, k, positions, rotary)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate_heads(q, k, positions, rotary)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotate_heads(q, k, positions, rotary)
    for step in range(3):
        positions += 17
        q.copy_(rows(30, 4, 128, seed=10 + step, device="cuda"))
        graph.replay()
        eager = rotate_heads(q, k, positions, rotary)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.gpu
def test_gpu_refusals():
    rotary = axes_of(128, 1, "halves")
    q = rows(6, 4, 128, seed=1, device="cuda")
    positions = torch.zeros((6, 1), dtype=torch.int32, device="cuda")
    for out, match in (((q, q), "shaped like"), (q[:5], "shaped like"), (q.float(), "shaped like")):
        with pytest.raises(ValueError, match=match):
            rotate_heads(q, None, positions, rotary, out=out)
    k = rows(6, 4, 128, seed=2, device="cuda")
    wide = rows(7, 4, 128, seed=3, device="cuda")
    for out in ((k, q), (q, q), (torch.empty_like(q), q), (wide[:6], wide[1:])):
        with pytest.raises(ValueError, match="share no memory|share memory"):
            rotate_heads(q, k, positions, rotary, out=out)
    with pytest.raises(ValueError, match="share no memory"):
        rotate_heads(wide[:6], None, positions, rotary, out=wide[1:])
    rolling = torch.as_strided(wide, (6, 4, 128), (128, 128, 1))  # rows that tokens have in common
    with pytest.raises(ValueError, match="with itself"):
        rotate_heads(rolling, None, positions, rotary, out=rolling)
    check(rotate_heads(rolling, None, positions, rotary), rolling, positions, rotary)
    with pytest.raises(ValueError, match="16-byte aligned"):
        rotate_heads(q, None, positions, rotary,
                     out=torch.empty(6 * 4 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 4, 128))
    with pytest.raises(ValueError, match="same AMD ROCm GPU"):
        rotate_heads(q, None, positions.cpu(), rotary)


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def call(**change):
    args = dict(q=bf16(3, 4, 64), k=bf16(3, 2, 64), positions=torch.zeros((3, 1), dtype=torch.int32),
                rotary=RotaryAxes.create(64, 32, device="cpu"))
    args.update(change)
    return rotate_heads(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("rotary"), **args)


@pytest.mark.parametrize("change,match", [
    (dict(q=bf16(3, 64)), "rank-4"), (dict(k=bf16(1, 3, 2, 64)), "rank-4"), (dict(q=bf16(3, 4, 64).float()), "Only BF16"),
    (dict(k=bf16(2, 2, 64)), "same tokens"), (dict(k=bf16(3, 2, 128)), "same tokens"),
    (dict(q=bf16(3, 4, 32), k=None), "head dimensions"), (dict(q=bf16(3, 0, 64)), "a head"),
    (dict(q=bf16(3, 4, 64).requires_grad_()), "Inference only"),
    (dict(q=bf16(3, 64, 4).transpose(1, 2)), "contiguous head"), (dict(q=bf16(3, 1, 64).expand(3, 4, 64)), "positive strides"),
    (dict(positions=torch.zeros((3, 1))), "int32"), (dict(positions=torch.zeros((2, 1), dtype=torch.int32)), "every token"),
    (dict(positions=torch.zeros((3, 0), dtype=torch.int32)), "every token"),
    (dict(positions=torch.zeros((2, 3), dtype=torch.int32).t()), "contiguous axes"),
    (dict(rotary=None), "RotaryAxes"), (dict(rotary=RotaryAxes.create(128, 64, device="cpu")), "Invalid rotary"),
    (dict(rotary=RotaryAxes(torch.zeros(32), torch.zeros(32, dtype=torch.int32))), "Invalid rotary"),
    (dict(rotary=RotaryAxes(torch.zeros(32, dtype=torch.float64), torch.zeros(32, dtype=torch.int32), "thirds")), "Invalid"),
    (dict(rotary=RotaryAxes(torch.zeros(32, dtype=torch.float64, requires_grad=True), torch.zeros(32, dtype=torch.int32))),
     "Inference only"),
    (dict(q_norm=torch.ones(32)), "Norm weights"), (dict(k_norm=torch.ones(64, dtype=torch.float16)), "Norm weights"),
    (dict(q_norm=torch.ones(64), k_norm=torch.ones(64, dtype=torch.bfloat16)), "one type"),
    (dict(q_norm=torch.ones(64, requires_grad=True)), "Inference only"), (dict(k=None, k_norm=torch.ones(64)), "needs K"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(), "AMD ROCm GPU"),
])
def test_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        call(**change)


@pytest.mark.parametrize("kwargs,match", [
    (dict(head_dim=96), "head dimensions"), (dict(pairs=33), "at most"), (dict(pairs=[20, 20]), "at most"),
    (dict(pairs=-1), "nonnegative"), (dict(pairs=[]), "at most"), (dict(base=0), "base"), (dict(layout="thirds"), "layout"),
])
def test_axes_refuse(kwargs, match):
    args = dict(head_dim=64, pairs=32)
    args.update(kwargs)
    with pytest.raises(ValueError, match=match):
        RotaryAxes.create(args.pop("head_dim"), args.pop("pairs"), device="cpu", **args)


def test_axes_hold_the_ladders():
    rotary = RotaryAxes.create(64, [2, 3], base=100.0, device="cpu")
    want = [1.0, 0.1, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]
    assert rotary.frequencies[:5].tolist() == pytest.approx(want) and not rotary.frequencies[5:].any()
    assert rotary.axes.tolist() == [0, 0, 1, 1, 1] + [-1] * 27 and rotary.layout == "halves"
    shared = RotaryAxes.create(64, [2, 2], base=16.0, shared=True, device="cpu")
    assert shared.frequencies[:4].tolist() == pytest.approx([1.0, 0.5, 0.25, 0.125])
