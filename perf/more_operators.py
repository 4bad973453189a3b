"""A step of drafted or branching sequences over the paged cache: the operators' cases, and their plain forms.

What surrounds the paged cache's writes and its attention in a program that generates with it: ``rotate_heads`` norms
the heads' rows of Q and K and rotates them by their positions (one axis for text, three for video), before rows are
stored or attended; ``tree_attention`` attends new tokens that are a tree of drafts; ``cache_keep`` moves the accepted
drafts' rows together; ``cache_fork`` makes the next step's plan on the GPU: sequences continue, branch, end or begin,
whole pages are shared, pages about to be written are copied, pages are taken and freed.  The package is inference
only, so there is no backward direction, and BF16 is the type of its activations.

A case holds sizes and a number ``mix``, from which its lengths, trees and branches are drawn on the host; values and
the order of the pages come from the seed.  Sizes are those of this repository's benchmark and tests, or odd ones
between them.
"""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LEVELS = {"int8": 127.0, "fp8": 448.0}
STORAGE = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
EPS = 1e-6


def listed():
    return [
        # One decoding step of 48 sequences at far positions: norms and rotation, latency alone.
        dict(name="rotate step 48 h24/8 d128", op="rotate", batch=0, tokens=48, heads=24, kv_heads=8, dim=128, axes=1,
             layout="halves", norm=True, part=1.0, reach=1 << 20, mix=1),
        # Packed prompts, half of each head rotated, no norm, heads of 64.
        dict(name="rotate prompts 19003 h12/3 d64", op="rotate", batch=0, tokens=19003, heads=12, kv_heads=3, dim=64,
             axes=1, layout="halves", norm=False, part=0.5, reach=8192, mix=2),
        # A video clip of 21 x 48 x 84 tokens before routed attention: norms, three axes.
        dict(name="rotate clip 84672 h24 d128", op="rotate", batch=1, tokens=84672, heads=24, kv_heads=24, dim=128,
             axes=3, layout="pairs", norm=True, part=1.0, reach=64, mix=3),
        # The smallest tree: three short sequences, seven drafts each.
        dict(name="tree 3x7 over 317 bf16 h2 d64", op="tree", seqs=3, new=7, branch=2, past=317, ragged=True,
             format="bf16", heads=2, kv_heads=2, dim=64, page=16, window=0, sinks=0, mix=4),
        # A served batch with drafts of odd numbers, grouped heads, full precision.
        dict(name="tree 16x26 over 19003 bf16 h24/8", op="tree", seqs=16, new=26, branch=3, past=19003, ragged=True,
             format="bf16", heads=24, kv_heads=8, dim=128, page=64, window=0, sinks=0, mix=5),
        # One long sequence over an 8-bit cache.
        dict(name="tree 1x64 over 84672 int8 h24/8", op="tree", seqs=1, new=64, branch=4, past=84672, ragged=False,
             format="int8", heads=24, kv_heads=8, dim=128, page=64, window=0, sinks=0, mix=6),
        # Large trees under a window with first tokens, 8-bit floating point.
        dict(name="tree 6x701 over 8191 fp8 h16/4", op="tree", seqs=6, new=701, branch=2, past=8191, ragged=True,
             format="fp8", heads=16, kv_heads=4, dim=128, page=32, window=4096, sinks=64, mix=7),
        # The accepted drafts of a batch.
        dict(name="keep 48 of 26 int8 h8 d128", op="keep", seqs=48, new=26, past=317, ragged=True, format="int8",
             kv_heads=8, dim=128, page=64, mix=8),
        # A video frame thinned out once it has been attended.
        dict(name="keep 2 of 4032 bf16 h24 d128", op="keep", seqs=2, new=4032, past=1024, ragged=False, format="bf16",
             kv_heads=24, dim=128, page=64, mix=9),
        # Beams: each of 48 continues one of 48, with one token more.
        dict(name="fork beams 48 int8 h8 d128", op="fork", seqs=48, children=48, past=1501, ragged=True, new=1, trim=0,
             begin=0.0, format="int8", kv_heads=8, dim=128, page=64, mix=10),
        # Samples of one prompt in full precision.
        dict(name="fork 1 to 16 bf16 h24 d128", op="fork", seqs=1, children=16, past=9001, ragged=False, new=1, trim=0,
             begin=0.0, format="bf16", kv_heads=24, dim=128, page=64, mix=11),
        # A large batch's turnover: drafts dropped, sequences that end and begin, new drafts for all; small pages.
        dict(name="fork batch 300 fp8 h2 d64", op="fork", seqs=300, children=317, past=4801, ragged=True, new=26,
             trim=26, begin=0.1, format="fp8", kv_heads=2, dim=64, page=16, mix=12),
    ]


# (query, key) pairs x heads that the plain form of the largest listed case forms.
_MOST = 6 * 701 * 8892 * 16


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "rotate", "tree", "tree", "tree", "keep", "fork", "fork"))
    kv = rng.choice((1, 2, 3, 4, 8, 12, 16, 24))
    case = dict(op=op, kv_heads=kv, dim=rng.choice((64, 128, 128)), mix=rng.randrange(1 << 30))
    if op == "rotate":
        case.update(heads=kv * rng.choice((1, 1, 2, 3, 4, 8)), batch=rng.choice((0, 0, 1, 2, 3)), axes=rng.choice((1, 1, 3)),
                    layout=rng.choice(("halves", "pairs")), norm=rng.random() < 0.6, tokens=_log_int(rng, 1, 84672),
                    part=rng.choice((1.0, 1.0, 0.5)), reach=_log_int(rng, 64, 1 << 24))
        while max(1, case["batch"]) * case["tokens"] * (case["heads"] + kv) * case["dim"] > 84672 * 48 * 128:
            case["tokens"] //= 2
        return case
    case.update(format=rng.choice(("bf16", "int8", "fp8")), page=rng.choice((16, 32, 64, 128)),
                seqs=_log_int(rng, 1, 64), ragged=rng.random() < 0.7)
    if op == "tree":
        case.update(heads=kv * rng.choice((1, 1, 2, 3, 4, 8)), new=_log_int(rng, 1, 701), branch=rng.choice((1, 2, 3, 4, 8)),
                    past=_log_int(rng, 1, 40000), window=rng.choice((0, 0, _log_int(rng, 1, 8192))),
                    sinks=rng.choice((0, 4, 64, 129)))
        while (case["seqs"] * case["new"] * (case["new"] + case["past"]) * max(4, case["heads"]) > _MOST
               or case["seqs"] * (case["new"] + case["past"]) * kv * case["dim"] > 3e8):
            case["seqs"], case["past"] = max(1, case["seqs"] // 2), max(1, case["past"] * 3 // 4)
    elif op == "keep":
        case.update(new=_log_int(rng, 1, 4032), past=rng.choice((0, _log_int(rng, 1, 2048))))
    else:
        case.update(seqs=_log_int(rng, 1, 300), children=_log_int(rng, 1, 317), past=_log_int(rng, 1, 4801),
                    new=rng.choice((1, _log_int(rng, 1, 256))), trim=rng.choice((0, 0, _log_int(rng, 1, 100))),
                    begin=rng.choice((0.0, 0.1, 0.5)))
    if op in ("keep", "fork"):
        while (case["seqs"] + case.get("children", 0)) * (case["new"] + case["past"]) * kv * case["dim"] > 1.5e8:
            case["seqs"], case["past"] = max(1, case["seqs"] // 2), case["past"] * 3 // 4
            case["new"] = max(1, case["new"] * 3 // 4)
            if op == "fork":
                case["children"], case["past"] = max(1, case["children"] // 2), max(1, case["past"])
    return case


# ---- what a case's number decides -------------------------------------------------------------------------


def _lengths(case):
    """Per sequence: the new tokens (none before a fork), and the keys with them."""
    rng = random.Random(case["mix"])
    new, keys = [], []
    for _ in range(case["seqs"]):
        n, past = (0 if case["op"] == "fork" else case["new"]), case["past"]
        if case["ragged"]:
            n = n if n <= 1 else rng.randint(1, n)
            past = _log_int(rng, max(1, past // 16), past) if past else 0
        new.append(n)
        keys.append(n + past)
    return new, keys


def _trees(case):
    """Per sequence a list of parents (-1: a root) in level order, about ``branch`` children each."""
    rng = random.Random(case["mix"] + 1)
    return [[-1 if i == 0 else max(-1 if rng.random() < 0.05 else 0, (i - 1) // case["branch"] - rng.randint(0, 1))
             for i in range(n)] for n in _lengths(case)[0]]


def _depths(tree):
    at = []
    for p in tree:
        at.append(0 if p < 0 else at[p] + 1)
    return at


def _accepted(case):
    """Per sequence the kept ones of its new tokens, ascending: first ones that stay in place, then some of the rest,
    further back than those places (levels of a tree wider than a path is long; a frame thinned to less than half)."""
    rng = random.Random(case["mix"] + 2)
    out = []
    for n in _lengths(case)[0]:
        count = rng.randint(1 if n else 0, max(1, n // 2) if n < 64 else n // 2)
        stay = rng.randint(1, max(1, count // 4))
        out.append((list(range(min(stay, count)))
                    + sorted(rng.sample(range(count, n), max(0, min(count - stay, n - count)))))[:count])
    return out


def _branches(case):
    """Per old sequence the length it is continued from; per new one the old one it continues (-1: none), and its new
    tokens; and how many pages at the front all old ones share."""
    rng = random.Random(case["mix"] + 3)
    keys = _lengths(case)[1]
    lengths = [max(0, n - (rng.randint(0, case["trim"]) if case["trim"] else 0)) for n in keys]
    parents = [-1 if rng.random() < case["begin"] else rng.randrange(case["seqs"]) for _ in range(case["children"])]
    new = [rng.randint(1, case["new"]) for _ in range(case["children"])]
    return lengths, parents, new, min(lengths) // case["page"] // 2


# ---- inputs -----------------------------------------------------------------------------------------------


def _rows(gen, *shape):
    """BF16 rows as a projection gives them: a scale per row and a few features that are larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))
    x[..., ::17] *= 2.0
    return x.to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ladder(case):
    """The pairs' frequencies (64 bits) and axes."""
    half = case["dim"] // 2
    turned = int(half * case["part"])
    counts = [turned] if case["axes"] == 1 else [turned - 2 * (turned // 3), turned // 3, turned // 3]
    freq = [10000.0 ** (-j / n) for n in counts for j in range(n)] + [0.0] * (half - turned)
    axis = [a for a, n in enumerate(counts) for _ in range(n)] + [0] * (half - turned)
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), _ints(axis)


def _prepare_rotate(case, gen):
    shape = ((case["batch"],) if case["batch"] else ()) + (case["tokens"],)
    hq, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    # Q, K and V come out of one projection; Q and K are views of it.
    both = _rows(gen, *shape, hq + hk + 1, dim)
    if case["axes"] == 1:
        # Places of several sequences: runs that begin anywhere.
        starts = torch.randint(0, case["reach"], shape[:-1] + (-(-case["tokens"] // 317),), generator=gen, device="cuda")
        at = torch.arange(case["tokens"], device="cuda")
        positions = (starts[..., at // 317] + at % 317)[..., None]
    else:
        first = int(torch.randint(0, case["reach"], (1,), generator=gen, device="cuda"))
        at = torch.arange(case["tokens"], device="cuda")
        positions = torch.stack([first + at // 4032, at // 84 % 48, at % 84], -1).expand(*shape, 3)
    frequencies, axis = _ladder(case)
    norms = [1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda") for _ in range(2)] if case["norm"] else [None, None]
    return dict(case=case, q=both[..., :hq, :], k=both[..., hq:hq + hk, :], positions=positions.to(torch.int32).contiguous(),
                frequencies=frequencies, axis=axis, q_norm=norms[0], k_norm=norms[1])


def _quantise(x, format):
    """(codes as 32-bit values, 32-bit scales) of rows x [..., D]: the larger of a row at the last level, the others
    rounded half to even."""
    x = x.float()
    most = x.abs().amax(-1)
    codes = x * LEVELS[format] / torch.where(most > 0, most, 1.0)[..., None]
    codes = codes.round() if format == "int8" else codes.to(torch.float8_e4m3fn).float()
    return codes, most / LEVELS[format]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotate":
        return _prepare_rotate(case, gen)
    new, keys = _lengths(case)
    page, kv, dim, format = case["page"], case["kv_heads"], case["dim"], case["format"]
    used, shared, more, wide = [-(-n // page) for n in keys], 0, 0, 1
    if case["op"] == "fork":
        lengths, parents, fresh, shared = _branches(case)
        after = [n + (lengths[p] if p >= 0 else 0) for p, n in zip(parents, fresh)]
        more = sum(-(-n // page) + 1 for n in fresh)
        wide = max(-(-n // page) for n in after)
    pages = shared + sum(n - shared for n in used) + more + 3  # a pool with a few pages to spare
    wide = max(used + [wide])
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(keys), wide), dtype=torch.int32, device="cuda")
    table[:, :shared] = order[:shared]
    at = shared
    for s, n in enumerate(used):
        table[s, shared:n] = order[at:at + n - shared]
        at += n - shared
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    state = dict(case=case, table=table, most=max(keys), most_new=max(new), lengths=_ints(keys), offsets=_ints(offsets))
    for name in ("cache_k", "cache_v"):
        rows = _rows(gen, pages, kv, page, dim)
        codes, scale = (rows, None) if format == "bf16" else _quantise(rows, format)
        state[name], state[name + "_scale"] = codes.to(STORAGE[format]), scale
        del rows, codes
    if case["op"] == "tree":
        state["q"] = _rows(gen, offsets[-1], case["heads"], dim)
        state["parents"] = _ints([p for tree in _trees(case) for p in tree])
    elif case["op"] == "keep":
        kept = _accepted(case)
        most = max(1, max(len(x) for x in kept))
        state["kept"] = _ints([x + [-1] * (most - len(x)) for x in kept])
    else:
        state.update(from_lengths=_ints(lengths), parents=_ints(parents), fresh=_ints(fresh))
        held = torch.arange(wide, device="cuda") < _ints(used)[:, None]
        state["refs"] = torch.bincount(table[held].long(), minlength=pages).to(torch.int32)
        state["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return state


# ---- one pass ---------------------------------------------------------------------------------------------


def _package(found=[]):
    if not found:
        path = os.path.join(ROOT, "solattn-amd_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import sol_attn_amd
        found.append(sol_attn_amd)
    return found[0]


def _handles(state):
    """The cache, plan and rotation objects over the state's tensors, which a program keeps."""
    if "handles" not in state:
        sol = _package()
        if state["case"]["op"] == "rotate":
            state["handles"] = sol.RotaryAxes(state["frequencies"], state["axis"], state["case"]["layout"])
        else:
            cache = sol.PagedCache(state["cache_k"], state["cache_v"], state["cache_k_scale"], state["cache_v_scale"])
            plan = sol.PagedPlan(state["table"], state["lengths"], state["offsets"])
            pool = sol.PagePool(state["refs"], state["missing"]) if "refs" in state else None
            state["handles"] = (cache, plan, pool)
    return state["handles"]


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        return {"rotate": _plain_rotate, "tree": _plain_tree, "keep": _plain_keep, "fork": _plain_fork}[op](state)
    sol = _package()
    if op == "rotate":
        return sol.rotate_heads(state["q"], state["k"], state["positions"], _handles(state), q_norm=state["q_norm"],
                                k_norm=state["k_norm"], eps=EPS)
    cache, plan, pool = _handles(state)
    if op == "tree":
        return sol.tree_attention(state["q"], cache, plan, state["parents"], window=case["window"] or None,
                                  sink_tokens=case["sinks"])
    if op == "keep":
        return dict(_stored(state), lengths=sol.cache_keep(cache, plan, state["kept"]))
    after, left = sol.cache_fork(cache, pool, plan, state["parents"], state["fresh"], lengths=state["from_lengths"])
    return dict(_stored(state), table=after.page_table, lengths=after.context_lengths, offsets=after.query_offsets,
                refs=left.refs, missing=left.missing)


def _stored(state):
    return {name: state[name] for name in ("cache_k", "cache_v", "cache_k_scale", "cache_v_scale")
            if state[name] is not None}


def _plain_rotate(state):
    angle = state["positions"].double()[..., state["axis"].long()] * state["frequencies"]
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        if state["case"]["layout"] == "halves":
            a, b = x.chunk(2, -1)
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(torch.bfloat16)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(torch.bfloat16)

    return turned(state["q"], state["q_norm"]), turned(state["k"], state["k_norm"])


def _gathered(state, name, tokens):
    """[sequences, tokens, heads, dim] of 32-bit values, zero past each sequence's keys."""
    x = state[name].float()
    if state[name + "_scale"] is not None:
        x = x * state[name + "_scale"][..., None]
    x = x[state["table"].long()].transpose(2, 3).flatten(1, 2)[:, :tokens]
    past = torch.arange(tokens, device="cuda") >= state["lengths"][:, None]
    return x.masked_fill_(past[:, :, None, None], 0.0)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(D)) v over what is seen, 0 for a row that sees nothing; q [B, T, Hq, D] in 32 bits, k and
    v [B, L, H, D], seen [B, T, L]."""
    b, t, heads, dim = q.shape
    kv = k.shape[2]
    rows = q.view(b, t, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim) * dim ** -0.5
    s = torch.matmul(rows, k.permute(0, 2, 3, 1).contiguous()).view(b, kv, heads // kv, t, -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, kv, -1, s.shape[-1]), v.permute(0, 2, 1, 3).contiguous()).view(b, kv, heads // kv, t, dim)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, heads, dim)


def _plain_tree(state):
    case, q, most_new = state["case"], state["q"], state["most_new"]
    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    seqs, new = lengths.shape[0], offsets[1:] - offsets[:-1]
    row = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    at = row - offsets[seq]
    padded = torch.zeros((seqs, most_new) + q.shape[1:], device="cuda")
    padded[seq, at] = q.float()
    # Ancestors: the paths of at most 1, 2, 4, ... steps along the tree, a last column for what has no parent.
    step = torch.zeros((seqs, most_new + 1, most_new + 1), device="cuda")
    step[seq, at, torch.where(state["parents"] < 0, most_new, state["parents"].long())] = 1.0
    above = (step + torch.eye(most_new + 1, device="cuda")).clamp_(max=1.0)
    for _ in range(most_new.bit_length()):
        above = torch.matmul(above, above).clamp_(max=1.0)
    above = above[:, :-1, :-1] > 0
    depth = above.sum(-1) - 1
    # A key's position: its place, and for a draft the base's length and its depth.
    base = (lengths - new)[:, None]
    j = torch.arange(state["most"], device="cuda")[None]
    draft = (j - base).clamp(0, most_new - 1)
    position = torch.where(j < base, j, base + depth.gather(1, draft))
    seen = (j < base)[:, None] | above.gather(2, draft[:, None].expand(-1, most_new, -1))
    seen &= (j < lengths[:, None])[:, None]
    if case["window"]:
        away = (base + depth)[:, :, None] - position[:, None]
        seen &= (away < case["window"]) | (position < case["sinks"])[:, None]
    o = _attend(padded, _gathered(state, "cache_k", state["most"]), _gathered(state, "cache_v", state["most"]), seen)
    return o[seq, at].to(torch.bfloat16)


def _bytes_of(x):
    return x.view(torch.int8) if x.dtype == torch.float8_e4m3fn else x


def _plain_keep(state):
    page, kept = state["case"]["page"], state["kept"].long()
    lengths, offsets, table = state["lengths"].long(), state["offsets"].long(), state["table"].long()
    new = offsets[1:] - offsets[:-1]
    base = lengths - new
    before = torch.cat([torch.full_like(kept[:, :1], -1), kept[:, :-1]], 1)
    good = ((kept > before) & (kept < new[:, None])).long().cumprod(1)
    seq, j = good.nonzero(as_tuple=True)
    source, target = base[seq] + kept[seq, j], base[seq] + j
    for x in _stored(state).values():
        x = _bytes_of(x)
        x[table[seq, target // page], :, target % page] = x[table[seq, source // page], :, source % page]
    return dict(_stored(state), lengths=(base + good.sum(1)).to(torch.int32))


def _plain_fork(state):
    page, table, refs = state["case"]["page"], state["table"].long(), state["refs"].long()
    seqs, wide = table.shape
    pages, parents = refs.shape[0], state["parents"].long()
    continues = parents >= 0
    parent = parents.clamp(min=0)
    held = torch.where(continues, (state["lengths"].long()[parent] + page - 1) // page, 0)[:, None]
    kept = torch.where(continues, state["from_lengths"].long()[parent], 0)
    after = kept + state["fresh"]
    full, used = (kept // page)[:, None], ((after + page - 1) // page)[:, None]
    # The first child of a sequence writes on in the pages that are its alone.
    child = torch.arange(parents.shape[0], device="cuda")
    firsts = torch.full((seqs,), parents.shape[0], device="cuda").scatter_reduce(
        0, parent, torch.where(continues, child, parents.shape[0]), "amin")
    first = continues & (firsts[parent] == child)
    e = torch.arange(wide, device="cuda")
    old = table[parent]
    stays = (e < used) & ((e < full) | (first[:, None] & (e < held) & (refs[old] == 1)))
    takes = (e < used) & ~stays
    rank = takes.flatten().long().cumsum(0).view(takes.shape) - 1
    free = torch.argsort((refs > 0).int(), stable=True)
    count = (refs <= 0).sum()
    taken = torch.where(rank < count, free[rank.clamp(0, pages - 1)], -1)
    result = torch.where(stays, old, torch.where(takes, taken, -1))
    used_before = (state["lengths"].long() + page - 1) // page
    refs = refs - torch.bincount(table[e < used_before[:, None]], minlength=pages)
    refs = refs + torch.bincount(result[result >= 0], minlength=pages)
    # Pages begun: the rows so far go along.
    copies = ((kept % page > 0)[:, None] & (e == full) & takes & (taken >= 0)).nonzero()
    source, target = old[copies[:, 0], copies[:, 1]], result[copies[:, 0], copies[:, 1]]
    rows = torch.arange(page, device="cuda") < (kept % page)[copies[:, 0], None]
    for x in _stored(state).values():
        x = _bytes_of(x)
        along = rows[:, None, :, None] if x.ndim == 4 else rows[:, None, :]
        x[target] = torch.where(along, x[source], x[target])
    offsets = torch.cat([torch.zeros_like(parents[:1]), state["fresh"].long().cumsum(0)])
    return dict(_stored(state), table=result.to(torch.int32), lengths=after.to(torch.int32),
                offsets=offsets.to(torch.int32), refs=refs.to(torch.int32),
                missing=(takes.sum() - count).clamp(min=0).to(torch.int32).view(1))


# ---- what a pass cannot do without ------------------------------------------------------------------------


def _row_bytes(case):
    """Of a token's K and V in the cache."""
    return 2.0 * case["kv_heads"] * (case["dim"] * 2 if case["format"] == "bf16" else case["dim"] + 4)


def work(case):
    if case["op"] == "rotate":
        tokens = case["tokens"] * max(1, case["batch"])
        rows = tokens * (case["heads"] + case["kv_heads"])
        return {"bytes": rows * case["dim"] * 4.0 + tokens * case["axes"] * 4.0,
                "flops": rows * case["dim"] * (7.0 if case["norm"] else 3.0)}
    new, keys = _lengths(case)
    if case["op"] == "tree":
        pairs = used = 0
        for n, length, tree in zip(new, keys, _trees(case)):
            depths, base = _depths(tree), length - n
            window = case["window"] or 1 << 60
            for d in depths:
                lo = max(0, base + d - window + 1)
                pairs += max(0, base - lo) + min(d + 1, window) + (min(case["sinks"], lo) if case["window"] else 0)
            lo = max(0, base - window + 1)
            used += length - lo + (min(case["sinks"], lo) if case["window"] else 0)
        return {"bytes": used * _row_bytes(case) + sum(new) * (4.0 * case["heads"] * case["dim"] + 4),
                "flops": 4.0 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "keep":
        moved = sum(sum(x != j for j, x in enumerate(kept)) for kept in _accepted(case))
        return {"bytes": moved * (2.0 * _row_bytes(case) + 4) + 8.0 * case["seqs"], "flops": 0.0}
    lengths, parents, fresh, shared = _branches(case)
    page, seen, rows, entries = case["page"], set(), 0, sum(-(-n // case["page"]) for n in keys)
    for p, n in zip(parents, fresh):
        if p >= 0 and p in seen:
            rows += lengths[p] % page
        entries += -(-(n + (lengths[p] if p >= 0 else 0)) // page)
        seen.add(p)
    pages = shared + sum(-(-n // page) - shared for n in keys)
    return {"bytes": 2.0 * rows * _row_bytes(case) + 4.0 * entries + 8.0 * pages + 12.0 * len(parents), "flops": 0.0}


# ---- the same in 64 bits ----------------------------------------------------------------------------------


def _exact_rotate(state):
    case = state["case"]
    turn = torch.polar(torch.ones_like(state["frequencies"]).expand(state["positions"].shape[:-1] + (case["dim"] // 2,)),
                       state["positions"].to(torch.float64)[..., state["axis"].tolist()] * state["frequencies"])
    out = []
    for x, weight in ((state["q"], state["q_norm"]), (state["k"], state["k_norm"])):
        y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for h in range(x.shape[-2]):
            row = x[..., h, :].double()
            if weight is not None:
                row = row / (row.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
            shape = row.shape[:-1]
            row = row.view(*shape, 2, -1).transpose(-1, -2) if case["layout"] == "halves" else row.view(*shape, -1, 2)
            row = torch.view_as_real(torch.view_as_complex(row.contiguous()) * turn)
            y[..., h, :] = (row.transpose(-1, -2) if case["layout"] == "halves" else row).reshape(*shape, -1)
        out.append(y)
    return tuple(out)


def _value64(state, name, s, length):
    """The first `length` rows of sequence s in 64 bits, [heads, length, dim]."""
    page = state["case"]["page"]
    pages = state["table"][s, :-(-length // page)].long()
    x = state[name][pages].to(torch.float64)
    if state[name + "_scale"] is not None:
        x *= state[name + "_scale"][pages].to(torch.float64).unsqueeze(-1)
    return x.movedim(1, 0).reshape(x.shape[1], -1, x.shape[-1])[:, :length]


def _exact_tree(state):
    case, out, at = state["case"], torch.empty(state["q"].shape, dtype=torch.float64, device="cuda"), 0
    heads, dim = case["heads"], case["dim"]
    for s, (n, length, tree) in enumerate(zip(*_lengths(case), _trees(case))):
        base, depths = length - n, _depths(tree)
        hidden = torch.ones((n, length), dtype=torch.bool)
        for i in range(n):
            p, window = base + depths[i], case["window"] or length + 1
            hidden[i, max(0, p - window + 1):base] = False
            if case["window"]:
                hidden[i, :min(base, case["sinks"])] = False
            a = i
            while a >= 0:
                hidden[i, base + a] = not (depths[i] - depths[a] < window
                                           or (case["window"] and base + depths[a] < case["sinks"]))
                a = tree[a]
        hidden = hidden.cuda()
        q, k, v = state["q"][at:at + n].double(), _value64(state, "cache_k", s, length), _value64(state, "cache_v", s, length)
        for h in range(heads):
            kv = h // (heads // case["kv_heads"])
            scores = (q[:, h] @ k[kv].t().contiguous()) / math.sqrt(dim)
            scores[hidden] = -math.inf
            out[at:at + n, h] = torch.nan_to_num(torch.softmax(scores, 1)) @ v[kv]
        at += n
    return out


def _moved(state, moves):
    """The stored tensors in 64 bits (None for whole numbers) after ``moves``: (source page, first row, target page,
    first row, rows) each, all read before any is written."""
    out = {}
    for name, x in _stored(state).items():
        if x.dtype == torch.int8:
            out[name] = None
            continue
        before = x.double()
        after = before.clone()
        for sp, sr, tp, tr, n in moves:
            after[tp, :, tr:tr + n] = before[sp, :, sr:sr + n]
        out[name] = after
    return out


def _exact_keep(state):
    page, table, moves = state["case"]["page"], state["table"].tolist(), []
    for row, n, length, kept in zip(table, *_lengths(state["case"]), _accepted(state["case"])):
        for j, x in enumerate(kept):
            a, b = length - n + x, length - n + j
            if a != b:
                moves.append((row[a // page], a % page, row[b // page], b % page, 1))
    return dict(_moved(state, moves), lengths=None)


def _exact_fork(state):
    case, page, table = state["case"], state["case"]["page"], state["table"].tolist()
    lengths, parents, fresh, _ = _branches(case)
    held = [-(-n // page) for n in _lengths(case)[1]]
    refs = state["refs"].tolist()
    free = [p for p, n in enumerate(refs) if n == 0]
    moves, seen, at = [], set(), 0
    for p, n in zip(parents, fresh):
        kept = lengths[p] if p >= 0 else 0
        for e in range(kept // page, -(-(kept + n) // page)):
            if p >= 0 and p not in seen and e < held[p] and refs[table[p][e]] == 1:
                continue
            if e == kept // page and kept % page:
                moves.append((table[p][e], 0, free[at], 0, kept % page))
            at += 1
        seen.add(p)
    return dict(_moved(state, moves), table=None, lengths=None, offsets=None, refs=None, missing=None)


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotate": _exact_rotate, "tree": _exact_tree, "keep": _exact_keep, "fork": _exact_fork}[case["op"]](state)
