"""CPU tests of the paged cache's and the windowed attention's host contract: refusals, plans, C-ABI checks."""

import ctypes
import os

import pytest
import torch

from sol_attn_amd import (PagedCache, PagedPlan, _native, cache_read, cache_write, paged_attention, window_attention)


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def parts(format="bf16", dim=64, new=(1, 2)):
    cache = PagedCache.create(4, 16, 2, dim, format=format, device="cpu")
    plan = PagedPlan.create([[0, 1], [2]], [20, 5], new, pages=4, page_size=16)
    return cache, plan


def test_plan_holds_the_lengths_tables_and_offsets():
    _, plan = parts()
    assert plan.page_table.tolist() == [[0, 1], [2, 0]] and plan.page_table.dtype == torch.int32
    assert plan.context_lengths.tolist() == [20, 5] and plan.query_offsets.tolist() == [0, 1, 3]
    moved = plan.to("cpu")
    assert moved.page_table.is_contiguous() and moved.query_offsets.tolist() == [0, 1, 3]
    table = torch.tensor([[3, 9], [1, -1]])  # entries past a sequence's pages are not looked at
    assert PagedPlan.create(table, torch.tensor([16, 0]), [0, 0], pages=4, page_size=16).page_table.shape == (2, 2)
    empty = PagedPlan.create([], [], [], pages=4, page_size=16)
    assert empty.page_table.shape == (0, 1) and empty.query_offsets.tolist() == [0]


@pytest.mark.parametrize("table,lengths,new,match", [
    ([[0], [1]], [16], [1], "same batch size"),
    ([[0]], [5], [6], "must not exceed"),
    ([[0]], [17], [1], "no page for"),
    ([[4]], [3], [1], "outside the cache"),
    ([[-1]], [3], [1], "outside the cache"),
    ([[0, 0]], [20], [18], "share a page"),
    ([[0], [0]], [3, 3], [1, 1], "share a page"),
    ([[0]], [-1], [0], "nonnegative integer"),
    ([[0]], [1], [True], "nonnegative integer"),
    (torch.zeros(3, dtype=torch.int64), [1], [1], "one row of page numbers"),
])
def test_plan_refuses(table, lengths, new, match):
    with pytest.raises(ValueError, match=match):
        PagedPlan.create(table, lengths, new, pages=4, page_size=16)


def test_plan_allows_a_shared_prefix():
    plan = PagedPlan.create([[0, 1], [0, 2]], [20, 30], [4, 3], pages=4, page_size=16)
    assert plan.page_table.tolist() == [[0, 1], [0, 2]]


@pytest.mark.parametrize("kwargs,match", [
    (dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"), (dict(page_size=8192), "power of two"),
    (dict(head_dim=96), "head dimensions"), (dict(format="fp4"), "format must be"), (dict(pages=0), "positive"),
    (dict(heads=0), "positive"), (dict(pages=-1), "nonnegative integer"),
])
def test_cache_refuses(kwargs, match):
    args = dict(pages=4, page_size=16, heads=2, head_dim=64, format="bf16")
    args.update(kwargs)
    with pytest.raises(ValueError, match=match):
        PagedCache.create(args["pages"], args["page_size"], args["heads"], args["head_dim"], format=args["format"],
                          device="cpu")


def test_cache_is_zeros_of_its_format():
    for format, dtype in (("bf16", torch.bfloat16), ("int8", torch.int8), ("fp8", torch.float8_e4m3fn)):
        cache = PagedCache.create(3, 32, 2, 128, format=format, device="cpu")
        assert cache.k.shape == (3, 2, 32, 128) and cache.k.dtype == cache.v.dtype == dtype
        assert not cache.k.float().any() and not cache.v.float().any()
        if format == "bf16":
            assert cache.k_scales is None and cache.v_scales is None
        else:
            assert cache.k_scales.shape == (3, 2, 32) and not cache.v_scales.any()


def test_everything_is_checked_before_the_device():
    cache, plan = parts()
    for call in (lambda: cache_write(bf16(3, 2, 64), bf16(3, 2, 64), cache, plan), lambda: cache_read(cache, plan, 4),
                 lambda: paged_attention(bf16(3, 4, 64), cache, plan),
                 lambda: window_attention(bf16(1, 3, 4, 64), bf16(1, 5, 2, 64), bf16(1, 5, 2, 64), window=2)):
        with pytest.raises(ValueError, match="AMD ROCm GPU"):
            call()


@pytest.mark.parametrize("change,match", [
    (dict(k=bf16(3, 128)), "NHD rank-3"), (dict(k=bf16(3, 2, 64).float()), "Only BF16"),
    (dict(k=bf16(2, 2, 64)), "same shape"), (dict(k=bf16(3, 2, 64).requires_grad_()), "Inference only"),
    (dict(k=bf16(3, 3, 64), v=bf16(3, 3, 64)), "must be the cache's"),
    (dict(k=bf16(3, 2, 128), v=bf16(3, 2, 128)), "must be the cache's"),
    (dict(k=bf16(3, 64, 2).transpose(1, 2)), "contiguous head dimension"),
    (dict(k=bf16(1, 2, 64).expand(3, 2, 64)), "positive strides"),
    (dict(cache=None), "PagedCache is required"), (dict(plan=None), "PagedPlan is required"),
])
def test_write_refuses(change, match, monkeypatch):
    cache, plan = parts()
    args = dict(k=bf16(3, 2, 64), v=bf16(3, 2, 64), cache=cache, plan=plan)
    args.update(change)
    if "must be the cache's" in match:  # that check follows the device's
        from sol_attn_amd import paged
        monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    with pytest.raises(ValueError, match=match):
        cache_write(**args)


@pytest.mark.parametrize("change,match", [
    (dict(q=bf16(3, 4, 128)), "multiple of the cache's"), (dict(q=bf16(3, 3, 64)), "multiple of the cache's"),
    (dict(window=0), "window must be"), (dict(window=-1), "window must be"), (dict(window=2.0), "window must be"),
    (dict(window=True), "window must be"), (dict(sink_tokens=-1), "sink_tokens must be"),
    (dict(causal=1), "causal must be"), (dict(scale=0.0), "scale must be"), (dict(scale=float("nan")), "scale must be"),
    (dict(out=bf16(3, 4, 64).float()), "out must be"), (dict(out=bf16(2, 4, 64)), "out must be"),
    (dict(out=bf16(3, 8, 64)[:, ::2]), "out must be"), (dict(out="q"), "share memory"),
    (dict(q=bf16(3, 4, 64).requires_grad_()), "Inference only"),
])
def test_paged_attention_refuses(change, match, monkeypatch):
    from sol_attn_amd import paged
    cache, plan = parts()
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))  # everything is on the CPU here
    args = dict(q=bf16(3, 4, 64), cache=cache, plan=plan)
    args.update(change)
    if args.get("out") == "q":
        args["out"] = args["q"]
    with pytest.raises(ValueError, match=match):
        paged_attention(**args)


@pytest.mark.parametrize("change,match", [
    (dict(k=bf16(4, 2, 16, 32), v=bf16(4, 2, 16, 32)), "head dimensions"),
    (dict(k=bf16(4, 2, 24, 64), v=bf16(4, 2, 24, 64)), "power of two"),
    (dict(v=bf16(3, 2, 16, 64)), "Invalid cache tensors"), (dict(v=bf16(4, 2, 16, 64).char()), "Invalid cache tensors"),
    (dict(k=bf16(4, 2, 16, 64).float(), v=bf16(4, 2, 16, 64).float()), "Invalid cache tensors"),
    (dict(k=bf16(4, 16, 2, 64).transpose(1, 2)), "Invalid cache tensors"),
    (dict(k=bf16(4, 2, 16, 64).char(), v=bf16(4, 2, 16, 64).char()), "need contiguous fp32 scales"),
    (dict(k=bf16(8193 * 64)[4:4 + 8192].view(4, 2, 16, 64)), "Invalid cache tensors"),  # 8 bytes off a 16-byte row
    (dict(page_table=torch.zeros(2, 2)), "Invalid paged descriptor"),
    (dict(context_lengths=torch.zeros(3, dtype=torch.int32)), "Invalid paged descriptor"),
    (dict(query_offsets=torch.zeros(2, dtype=torch.int32)), "Invalid paged descriptor"),
    (dict(page_table=torch.zeros((2, 4), dtype=torch.int32)[:, ::2]), "Invalid paged descriptor"),
    (dict(page_table=torch.zeros((2, 0), dtype=torch.int32)), "page_table must name"),
])
def test_read_refuses_hand_made_descriptors(change, match):
    cache, plan = parts()
    c = {x: change.get(x, getattr(cache, x)) for x in ("k", "v", "k_scales", "v_scales")}
    p = {x: change.get(x, getattr(plan, x)) for x in ("page_table", "context_lengths", "query_offsets")}
    with pytest.raises(ValueError, match=match):
        cache_read(PagedCache(**c), PagedPlan(**p), 4)


@pytest.mark.parametrize("kwargs,match", [
    (dict(tokens=-1), "tokens must be"), (dict(tokens=1.5), "tokens must be"), (dict(tokens=4, start=-1), "start must be"),
    (dict(tokens=1 << 30), "Sequences longer"), (dict(tokens=4, start=1 << 30), "Sequences longer"),
])
def test_read_refuses_ranges(kwargs, match):
    with pytest.raises(ValueError, match=match):
        cache_read(*parts(), **kwargs)


@pytest.mark.parametrize("q,k,kwargs,match", [
    ((1, 3, 3, 64), (1, 5, 2, 64), {}, "must agree and be nonempty"), ((1, 3, 4, 64), (2, 5, 2, 64), {}, "must agree"),
    ((1, 3, 4, 64), (1, 5, 2, 128), {}, "must agree"), ((1, 3, 4, 96), (1, 5, 2, 96), {}, "head dimensions"),
    ((3, 4, 64), (1, 5, 2, 64), {}, "BTHD rank-4"), ((1, 0, 4, 64), (1, 5, 2, 64), {}, "nonempty"),
    ((1, 3, 4, 64), (1, 5, 2, 64), dict(scale=-1.0), "scale must be"),
])
def test_window_attention_refuses_shapes(q, k, kwargs, match):
    with pytest.raises(ValueError, match=match):
        window_attention(bf16(*q), bf16(*k), bf16(*k), **kwargs)


def test_window_arguments_are_keywords():
    with pytest.raises(TypeError):
        window_attention(bf16(1, 3, 2, 64), bf16(1, 5, 2, 64), bf16(1, 5, 2, 64), True)
    with pytest.raises(TypeError):
        paged_attention(bf16(3, 2, 64), *parts(), True)


def test_grouped_heads_stay_refused_elsewhere():
    from sol_attn_amd import dense_attention
    with pytest.raises(ValueError, match="must agree"):
        dense_attention(bf16(1, 3, 4, 64), bf16(1, 5, 2, 64), bf16(1, 5, 2, 64))


def test_c_abi_refuses_without_launching():
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libsol_attn_amd.so not built")
    lib = _native.library()
    fake = ctypes.c_void_p(1 << 20)  # never dereferenced: validation fails first
    odd = ctypes.c_void_p((1 << 20) + 8)
    ok, bad = (ctypes.c_int64 * 3)(0, 128, 64), (ctypes.c_int64 * 3)(0, 127, 64)

    def write(strides=ok, rows=3, table=fake, offsets=fake, seqs=2, width=2, pages=4, page=16, heads=2, dim=64, fmt=0,
              store=fake, scales=None):
        return lib.sol_cache_write(fake, strides, fake, ok, rows, table, fake, offsets, seqs, width, pages, page, heads,
                                   dim, fmt, store, fake, scales, scales, None)

    def read(start=0, tokens=4, out=fake, fmt=0, scales=None):
        return lib.sol_cache_read(fake, fake, scales, scales, fake, fake, 2, 2, 4, 16, 2, 64, fmt, start, tokens, out,
                                  fake, None)

    def attend(q=fake, rows=3, hq=4, heads=2, scale=0.125, window=0, sinks=0, out=fake, offsets=fake, width=2,
               ws=None, size=0):
        return lib.sol_paged_attention(q, ok, rows, fake, fake, None, None, fake, fake, offsets, 2, width, 4, 16, hq,
                                       heads, 64, 0, scale, 1, window, sinks, ws, size, out, None)

    def plain(strides=ok, tq=3, tk=5, hq=4, heads=2, dim=64, out=fake, ws=None):
        s = (ctypes.c_int64 * 3)(128 * 5, strides[1], strides[2])
        return lib.sol_window_attention(fake, s, fake, s, fake, s, 1, tq, tk, hq, heads, dim, 0.125, 1, 0, 0, ws, 16,
                                        out, None)

    refused = [
        (lambda: write(bad), b"aligned"),
        (lambda: write(rows=-1), b"invalid shape"),
        (lambda: write(table=None), b"required"),
        (lambda: write(offsets=None), b"query_offsets"),
        (lambda: write(seqs=0), b"invalid shape"),
        (lambda: write(width=1 << 29), b"invalid shape"),
        (lambda: write(pages=1 << 31), b"invalid shape"),
        (lambda: write(page=24), b"power of two"),
        (lambda: write(dim=96), b"head_dim"),
        (lambda: write(fmt=3), b"format"),
        (lambda: write(store=odd), b"aligned"),
        (lambda: write(fmt=1), b"scales"),
        (lambda: read(start=-1), b"token range"),
        (lambda: read(tokens=1 << 30), b"token range"),
        (lambda: read(out=odd), b"aligned"),
        (lambda: read(fmt=2), b"scales"),
        (lambda: attend(q=odd), b"aligned"),
        (lambda: attend(hq=3), b"multiple"),
        (lambda: attend(scale=float("inf")), b"scale"),
        (lambda: attend(window=-1), b"negative"),
        (lambda: attend(sinks=-1), b"negative"),
        (lambda: attend(out=None), b"aligned"),
        (lambda: attend(offsets=None), b"query_offsets"),
        (lambda: attend(rows=1 << 30), b"invalid shape"),
        (lambda: plain(bad), b"aligned"),
        (lambda: plain(tq=0), b"shape"),
        (lambda: plain(tk=0), b"shape"),
        (lambda: plain(hq=5), b"multiple"),
        (lambda: plain(dim=32), b"head_dim"),
        (lambda: plain(out=odd), b"aligned"),
        (lambda: attend(width=200), b"workspace"),
        (lambda: attend(width=200, ws=odd, size=1 << 40), b"workspace"),
        (lambda: attend(width=200, ws=fake, size=16), b"workspace"),
        (lambda: plain(tk=5000, ws=fake), b"workspace"),
        (lambda: plain((ctypes.c_int64 * 3)(0, 1 << 24, 64)), b"2^24"),
    ]
    for call, word in refused:
        assert call() < 0 and word in lib.sol_last_error(), (word, lib.sol_last_error())
    assert write(rows=0) == 0 and read(tokens=0) == 0 and attend(rows=0) == 0  # nothing to do, nothing launched
    # Partial states of the calls that split their keys: none for short sequences.
    paged, window = lib.sol_paged_attention_workspace_size, lib.sol_window_attention_workspace_size
    assert paged(3, 2, 2, 16, 4, 2, 64, 0, 1, 0, 0) == 0 and paged(0, 2, 200, 16, 4, 2, 64, 0, 1, 0, 0) == 0
    assert paged(3, 2, 200, 16, 4, 2, 64, 0, 1, 0, 0) > 0 and paged(3, 2, 200, 16, 4, 2, 64, 0, 1, 10, 0) == 0
    assert paged(3, 2, 200, 16, 4, 2, 96, 0, 1, 0, 0) == -1 and paged(3, 2, 200, 16, 3, 2, 64, 0, 1, 0, 0) == -1
    assert window(1, 3, 5, 4, 2, 64, 1, 0, 0) == 0 and window(1, 3, 5000, 4, 2, 64, 1, 0, 0) > 0
    assert window(1, 0, 5, 4, 2, 64, 1, 0, 0) == -1 and window(1, 3, 5, 4, 2, 64, 1, -1, 0) == -1


def test_c_abi_refuses_launches_of_too_many_threads():
    # 2^24 workgroups of 256 threads and more.
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libsol_attn_amd.so not built")
    lib = _native.library()
    fake, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)  # never dereferenced
    ok = (ctypes.c_int64 * 3)(1 << 40, 128, 64)

    def write(rows, heads, dim):
        return lib.sol_cache_write(fake, ok, fake, ok, rows, fake, fake, fake, 2, 2, 4, 16, heads, dim, 0, fake, fake,
                                   None, None, None)

    def read(seqs, tokens, heads, dim):
        return lib.sol_cache_read(fake, fake, None, None, fake, fake, seqs, 2, 4, 16, heads, dim, 0, 0, tokens, fake,
                                  fake, None)

    def attend(rows, seqs, heads, width=2, ws=None):
        return lib.sol_paged_attention(fake, ok, rows, fake, fake, None, None, fake, fake, fake, seqs, width, 4, 16,
                                       heads, heads, 64, 0, 0.125, 1, 0, 0, ws, 16, fake, None)

    def plain(batch, tq, heads):
        return lib.sol_window_attention(fake, ok, fake, ok, fake, ok, batch, tq, 20, heads, heads, 64, 0.125, 1, 0, 0,
                                        odd, 16, fake, None)

    for call in (lambda: write(1 << 24, 16, 128), lambda: write(1 << 24, 32, 64), lambda: read(1 << 14, 1 << 10, 16, 128),
                 lambda: read(1 << 14, 1 << 10, 32, 64), lambda: read(1 << 20, (1 << 30) - 1, (1 << 16) - 1, 128),
                 lambda: attend(1 << 21, 1 << 16, 192), lambda: attend(1, 1 << 16, (1 << 16) - 1),
                 lambda: plain(1 << 20, 32, 15)):
        assert call() == -2 and b"grid too large" in lib.sol_last_error()
    assert attend(1, (1 << 16) + 1, 2) == -2 and b"65,536 sequences" in lib.sol_last_error()
    paged, window = lib.sol_paged_attention_workspace_size, lib.sol_window_attention_workspace_size
    assert paged(3, 1 << 16, 2, 16, 4, 2, 64, 0, 1, 0, 0) == 0 and paged(3, (1 << 16) + 1, 2, 16, 4, 2, 64, 0, 1, 0, 0) == -1
    assert paged((1 << 30) - 1, 2, 1 << 25, 16, 65534, 2, 64, 0, 1, 0, 0) == -1
    assert window(1 << 20, 1 << 10, 5, 4, 2, 64, 1, 0, 0) == -1


def test_too_many_sequences_are_refused(monkeypatch):
    from sol_attn_amd import paged
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    cache, _ = parts()
    n = paged.MAX_ATTENDED + 1
    plan = PagedPlan(torch.zeros(n, 1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32),
                     torch.zeros(n + 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="More than 65536 sequences"):
        paged_attention(bf16(3, 4, 64), cache, plan)


@pytest.mark.parametrize("shift", [0, 64])
def test_write_refuses_a_cache_whose_sides_share_memory(shift, monkeypatch):
    from sol_attn_amd import paged
    _, plan = parts()
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    store = bf16(4 * 2 * 16 * 64 + shift)
    cache = PagedCache(*(x.view(4, 2, 16, 64) for x in (store[:8192], store[shift:])))
    with pytest.raises(ValueError, match="share memory"):
        cache_write(bf16(3, 2, 64), bf16(3, 2, 64), cache, plan)


@pytest.mark.parametrize("name", ["k", "v", "out"])
def test_gradients_of_the_cache_and_the_output_are_refused(name, monkeypatch):
    from sol_attn_amd import paged
    cache, plan = parts()
    q, out = bf16(3, 4, 64), bf16(3, 4, 64)
    if name == "out":
        monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
        out.requires_grad_()
    else:
        getattr(cache, name).requires_grad_()
    with pytest.raises(ValueError, match="Inference only"):
        paged_attention(q, cache, plan, out=out)


def test_partial_states_do_not_grow_with_the_rows():
    # At most 2 target records (parts of split row tiles) per head, target 1.5 x 512 workgroups over all heads for chunks
    # and 512, or twice that, for single tokens, a little more by rounding up per head.
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libsol_attn_amd.so not built")
    lib = _native.library()
    paged, window = lib.sol_paged_attention_workspace_size, lib.sol_window_attention_workspace_size
    for dim in (64, 128):
        for heads, group in ((8, 4), (1, 1), (24, 1)):
            record = heads * 128 * (dim + 4) * 4
            for rows, seqs, keys in ((8192, 2, 131072), (262144, 2, 131072), (1 << 19, 64, 8192), (1 << 19, 4096, 65536)):
                for fmt in (0, 1, 2):
                    size = paged(rows, seqs, keys // 64, 64, heads * group, heads, dim, fmt, 1, 0, 0)
                    target = -(-3 * 256 // heads)
                    assert 0 <= size <= 2 * target * (record + 32 * heads) + 16, (rows, seqs, keys, heads, dim, fmt)
            step = heads * 16 * (dim + 4) * 4
            for seqs in (64, 4096, 65536):
                size = paged(seqs, seqs, 1024, 64, heads * group, heads, dim, 0, 1, 0, 0)
                assert 0 < size <= 2 * -(-1024 // heads) * (step + 32 * heads) + 16
            assert window(1, 131072, 131072, heads * group, heads, dim, 1, 0, 0) <= 2 * target * (record + 32 * heads) + 16


@pytest.mark.parametrize("shift", [0, 16])
def test_write_refuses_a_cache_whose_scales_share_memory(shift, monkeypatch):
    from sol_attn_amd import paged
    cache, plan = parts("int8")
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    scales = torch.zeros(4 * 2 * 16 + shift)
    shared = PagedCache(cache.k, cache.v, *(x.view(4, 2, 16) for x in (scales[:128], scales[shift:])))
    with pytest.raises(ValueError, match="share memory"):
        cache_write(bf16(3, 2, 64), bf16(3, 2, 64), shared, plan)


@pytest.mark.parametrize("side", [0, 1])
def test_attention_refuses_an_output_in_the_scales(side, monkeypatch):
    from sol_attn_amd import paged
    cache, plan = parts("int8")
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    store = torch.zeros(1024)
    scales = [cache.k_scales, cache.v_scales]
    scales[side] = store[:128].view(4, 2, 16)
    with pytest.raises(ValueError, match="share memory"):
        paged_attention(bf16(3, 4, 64), PagedCache(cache.k, cache.v, *scales), plan,
                        out=store.view(torch.bfloat16)[:768].view(3, 4, 64))


@pytest.mark.parametrize("scale", [2.0 ** 127, 1e39, 1e300, float("inf")])
def test_scales_past_fp32_are_refused(scale, monkeypatch):
    from sol_attn_amd import attention, paged
    cache, plan = parts()
    monkeypatch.setattr(paged, "_validate", lambda c, p, d: (2, 64))
    with pytest.raises(ValueError, match="scale must be"):
        paged_attention(bf16(3, 4, 64), cache, plan, scale=scale)
    monkeypatch.setattr(attention, "_validate", lambda q, k, v, scale, grouped: scale)
    with pytest.raises(ValueError, match="scale must be"):
        window_attention(bf16(1, 3, 4, 64), bf16(1, 5, 2, 64), bf16(1, 5, 2, 64), scale=scale)
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libsol_attn_amd.so not built")
    lib, fake, ok = _native.library(), ctypes.c_void_p(1 << 20), (ctypes.c_int64 * 3)(640, 128, 64)
    assert lib.sol_paged_attention(fake, ok, 3, fake, fake, None, None, fake, fake, fake, 2, 2, 4, 16, 4, 2, 64, 0, scale,
                                   1, 0, 0, None, 0, None, None) < 0 and b"scale" in lib.sol_last_error()
    assert lib.sol_window_attention(fake, ok, fake, ok, fake, ok, 1, 3, 5, 4, 2, 64, scale, 1, 0, 0, None, 0, None,
                                    None) < 0 and b"scale" in lib.sol_last_error()
