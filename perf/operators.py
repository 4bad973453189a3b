"""The paged-cache and windowed-attention operators: cases, and their plain forms.

Operators of a model that generates its sequence piece by piece (a video frame by frame, a text token by
token): ``cache_write`` stores the new tokens' K and V rows in a paged cache, in BF16 or quantised to INT8 or
FP8 (e4m3) with one scale per token and head; ``cache_read`` gathers a cache's rows back into plain BTHD BF16;
``paged_attention`` attends the new tokens to the cache; ``window_attention`` attends plain BTHD tensors under a
sliding window with first tokens that stay visible.  The package is inference only, so there is no backward
direction, and BF16 is the type of its activations.

Query heads share a K/V head in groups (``heads`` / ``kv_heads``).  Row i of sequence s's ``n`` new tokens has
position ``L - n + i``, L the keys of the sequence (the new ones included).  Key j is visible to position p if
``j < L``, ``j <= p`` where causal, and, with a window, ``|p - j| < window`` or ``j < sinks``.

Sequence lengths are part of a case (drawn from its ``mix``), values and the order of the pages come from the
seed.  Lengths, heads and dimensions are those of this repository's benchmark and tests, or odd ones between.
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


def listed():
    return [
        # One decoding step of 48 sequences: every sequence stores one token, latency alone.
        dict(name="write step 48 int8 h8 d128", op="write", seqs=48, new=1, past=4096, ragged=True, format="int8",
             kv_heads=8, dim=128, page=64, mix=1),
        # A video model appends one frame (48 x 84 tokens) in full precision.
        dict(name="write frame 4032 bf16 h24 d128", op="write", seqs=1, new=4032, past=8064, ragged=False,
             format="bf16", kv_heads=24, dim=128, page=64, mix=2),
        # A batch of prompts of odd lengths, stored in 8-bit floating point, small pages.
        dict(name="write prompts 9x4801 fp8 h12 d64", op="write", seqs=9, new=4801, past=0, ragged=True, format="fp8",
             kv_heads=12, dim=64, page=16, mix=3),
        # A short video clip read back for routed attention over plain tensors.
        dict(name="read 19003 int8 h16 d128", op="read", seqs=1, past=19003, ragged=False, format="int8", kv_heads=16,
             dim=128, page=64, mix=4),
        # Several short sequences of different lengths, padded to the longest.
        dict(name="read 7x1501 fp8 h3 d64", op="read", seqs=7, past=1501, ragged=True, format="fp8", kv_heads=3, dim=64,
             page=32, mix=5),
        # The smallest step: three short sequences, two heads.
        dict(name="step 3x317 bf16 h2 d64", op="paged", seqs=3, new=1, past=317, ragged=True, format="bf16", heads=2,
             kv_heads=2, dim=64, page=16, causal=True, window=0, sinks=0, mix=6),
        # An ordinary decoding step of a served batch: 48 sequences of very different lengths, grouped heads.
        dict(name="step 48x19003 bf16 h24/8 d128", op="paged", seqs=48, new=1, past=19003, ragged=True, format="bf16",
             heads=24, kv_heads=8, dim=128, page=64, causal=True, window=0, sinks=0, mix=7),
        # One long sequence's step over an 8-bit cache: few rows, all of the work along the keys.
        dict(name="step 1x84672 int8 h24/8 d128", op="paged", seqs=1, new=1, past=84672, ragged=False, format="int8",
             heads=24, kv_heads=8, dim=128, page=64, causal=True, window=0, sinks=0, mix=8),
        # The next chunks of several sequences of odd lengths, causal, window and first tokens, 8-bit floating point.
        dict(name="chunks 6x701 fp8 h16/4 d128", op="paged", seqs=6, new=701, past=8191, ragged=True, format="fp8",
             heads=16, kv_heads=4, dim=128, page=32, causal=True, window=4096, sinks=64, mix=9),
        # A video model's next frame: its tokens see one another and the ten frames stored so far.
        dict(name="frame 4032x40320 bf16 h24 d128", op="paged", seqs=1, new=4032, past=36288, ragged=False,
             format="bf16", heads=24, kv_heads=24, dim=128, page=64, causal=False, window=0, sinks=0, mix=10),
        # The smallest plain call: odd lengths, both sides of the window.
        dict(name="window 193x317 h2 d64", op="window", batch=1, tq=193, tk=317, heads=2, kv_heads=2, dim=64,
             causal=False, window=64, sinks=5, mix=11),
        # A clip's prompt: each token sees one frame's worth of tokens before it, and the first 128.
        dict(name="window 19003 h16 d128", op="window", batch=1, tq=19003, tk=19003, heads=16, kv_heads=16, dim=128,
             causal=True, window=4032, sinks=128, mix=12),
    ]


# (query, key) pairs x heads that the plain form of the largest listed case forms.
_MOST = 19003 ** 2 * 16


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "write", "read", "paged", "paged", "paged", "window"))
    kv = rng.choice((1, 2, 3, 4, 8, 12, 16, 24))
    case = dict(op=op, kv_heads=kv, dim=rng.choice((64, 128, 128)), mix=rng.randrange(1 << 30))
    if op != "window":
        case.update(format=rng.choice(("bf16", "int8", "fp8")), page=rng.choice((16, 32, 64, 128)),
                    seqs=_log_int(rng, 1, 64), ragged=rng.random() < 0.7)
    if op in ("paged", "window"):
        case.update(heads=kv * rng.choice((1, 1, 2, 3, 4, 8)), causal=rng.random() < 0.7,
                    window=rng.choice((0, 0, _log_int(rng, 1, 8192))), sinks=rng.choice((0, 4, 64, 129)))
    if op == "write":
        case.update(new=rng.choice((1, _log_int(rng, 2, 8192))), past=rng.choice((0, _log_int(rng, 1, 8192))))
        while case["seqs"] * case["new"] * kv * case["dim"] > 4e8:
            case["seqs"] = max(1, case["seqs"] // 2)
        while case["seqs"] * (case["new"] + case["past"]) * kv * case["dim"] > 4e8:
            case["past"] //= 2
    elif op == "read":
        case.update(past=_log_int(rng, 100, 40000))
        while case["seqs"] * case["past"] * kv * case["dim"] > 2e8:
            case["seqs"], case["past"] = max(1, case["seqs"] // 2), max(100, case["past"] // 2)
    elif op == "paged":
        case.update(new=rng.choice((1, 1, _log_int(rng, 2, 2048))), past=_log_int(rng, 1, 40000))
        while (case["seqs"] * case["new"] * (case["new"] + case["past"]) * max(4, case["heads"]) > _MOST
               or case["seqs"] * (case["new"] + case["past"]) * kv * case["dim"] > 1e9):
            case["seqs"], case["past"] = max(1, case["seqs"] // 2), max(1, case["past"] * 3 // 4)
    else:
        tk = _log_int(rng, 100, 19003)
        case.update(batch=rng.choice((1, 1, 2, 3)), tk=tk, tq=rng.choice((1, tk, tk, _log_int(rng, 1, tk))))
        while case["batch"] * case["tq"] * tk * max(4, case["heads"]) > _MOST:
            case["batch"], case["tq"] = max(1, case["batch"] // 2), max(1, case["tq"] // 2)
    return case


def _lengths(case):
    """Per sequence: the new tokens, and the keys with them."""
    rng = random.Random(case["mix"])
    new, keys = [], []
    for _ in range(case["seqs"]):
        n, past = case.get("new", 0), case["past"]
        if case["ragged"]:
            n = n if n <= 1 else rng.randint(1, n)
            past = _log_int(rng, max(1, past // 16), past) if past else 0
        new.append(n)
        keys.append(n + past)
    return new, keys


# ---- inputs -----------------------------------------------------------------------------------------------


def _rows(gen, *shape):
    """BF16 rows as a projection gives them: a scale per row and a few features that are larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))
    x[..., ::17] *= 2.0
    return x.to(torch.bfloat16)


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
    dim = case["dim"]
    if case["op"] == "window":
        q = _rows(gen, case["batch"], case["tq"], case["heads"], dim)
        k, v = (_rows(gen, case["batch"], case["tk"], case["kv_heads"], dim) for _ in range(2))
        return dict(case=case, q=q, k=k, v=v)
    new, keys = _lengths(case)
    page, kv, format = case["page"], case["kv_heads"], case["format"]
    wide = -(-max(keys) // page)
    used = [-(-n // page) for n in keys]
    pages = sum(used) + 3  # a pool with a few pages to spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(keys), wide), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    state = dict(case=case, table=table, most=max(keys), most_new=max(new),
                 lengths=torch.tensor(keys, dtype=torch.int32, device="cuda"),
                 offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    shape = (pages, kv, page, dim)
    if case["op"] == "write":
        for name in ("cache_k", "cache_v"):
            state[name] = torch.zeros(shape, dtype=STORAGE[format], device="cuda")
            state[name + "_scale"] = None if format == "bf16" else torch.zeros(shape[:-1], device="cuda")
        # K and V come out of one projection: every other head row of it is the other operand's.
        both = _rows(gen, offsets[-1], 2, kv, dim)
        state["k"], state["v"] = both[:, 0], both[:, 1]
        return state
    for name in ("cache_k", "cache_v"):
        rows = _rows(gen, *shape)
        codes, scale = (rows, None) if format == "bf16" else _quantise(rows, format)
        state[name], state[name + "_scale"] = codes.to(STORAGE[format]), scale
        del rows, codes
    if case["op"] == "paged":
        state["q"] = _rows(gen, offsets[-1], case["heads"], dim)
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
    """The cache and plan objects over the state's tensors, which a program keeps."""
    if "handles" not in state:
        sol = _package()
        state["handles"] = (sol.PagedCache(state["cache_k"], state["cache_v"], state["cache_k_scale"],
                                           state["cache_v_scale"]),
                            sol.PagedPlan(state["table"], state["lengths"], state["offsets"]))
    return state["handles"]


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        sol = _package()
        if op == "window":
            return sol.window_attention(state["q"], state["k"], state["v"], window=case["window"] or None,
                                        sink_tokens=case["sinks"], causal=case["causal"])
        cache, plan = _handles(state)
        if op == "write":
            sol.cache_write(state["k"], state["v"], cache, plan)
            return _stored(state)
        if op == "read":
            return sol.cache_read(cache, plan, state["most"])
        return sol.paged_attention(state["q"], cache, plan, causal=case["causal"], window=case["window"] or None,
                                   sink_tokens=case["sinks"])
    if op == "window":
        return _plain_window(state)
    return {"write": _plain_write, "read": _plain_read, "paged": _plain_paged}[op](state)


def _stored(state):
    return {name: state[name] for name in ("cache_k", "cache_v", "cache_k_scale", "cache_v_scale")
            if state[name] is not None}


def _plain_write(state):
    format, page = state["case"]["format"], state["case"]["page"]
    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    row = torch.arange(state["k"].shape[0], device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    position = lengths[seq] - offsets[seq + 1] + row
    where = state["table"].long()[seq, position // page]
    for name, x in (("cache_k", state["k"]), ("cache_v", state["v"])):
        if format == "bf16":
            state[name][where, :, position % page] = x
            continue
        codes, scale = _quantise(x, format)
        state[name].view(torch.int8)[where, :, position % page] = codes.to(STORAGE[format]).view(torch.int8)
        state[name + "_scale"][where, :, position % page] = scale
    return _stored(state)


def _gathered(state, name, tokens):
    """[sequences, tokens, heads, dim] of 32-bit values, zero past each sequence's keys."""
    x = state[name].float()
    if state[name + "_scale"] is not None:
        x = x * state[name + "_scale"][..., None]
    x = x[state["table"].long()].transpose(2, 3).flatten(1, 2)[:, :tokens]
    past = torch.arange(tokens, device="cuda") >= state["lengths"][:, None]
    return x.masked_fill_(past[:, :, None, None], 0.0)


def _plain_read(state):
    return tuple(_gathered(state, name, state["most"]).to(torch.bfloat16) for name in ("cache_k", "cache_v"))


def _visible(case, position, keys, key_lengths):
    """[batch, queries, keys] truth values; position [batch, queries], key_lengths [batch]."""
    j = torch.arange(keys, dtype=torch.int32, device="cuda")
    seen = j < key_lengths[:, None, None]
    away = position.to(torch.int32)[:, :, None] - j
    if case["causal"]:
        seen = seen & (away >= 0)
    if case["window"]:
        seen = seen & ((away.abs() < case["window"]) | (j < case["sinks"]))
    return seen


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


def _plain_paged(state):
    case, q = state["case"], state["q"]
    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    new = offsets[1:] - offsets[:-1]
    row = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    at = row - offsets[seq]
    padded = torch.zeros((lengths.shape[0], state["most_new"]) + q.shape[1:], device="cuda")
    padded[seq, at] = q.float()
    position = (lengths - new)[:, None] + torch.arange(state["most_new"], device="cuda")
    seen = _visible(case, position, state["most"], lengths)
    o = _attend(padded, _gathered(state, "cache_k", state["most"]), _gathered(state, "cache_v", state["most"]), seen)
    return o[seq, at].to(torch.bfloat16)


def _plain_window(state):
    case, b = state["case"], state["case"]["batch"]
    tk = torch.full((b,), case["tk"], device="cuda")
    position = torch.arange(case["tk"] - case["tq"], case["tk"], device="cuda").expand(b, -1)
    seen = _visible(case, position, case["tk"], tk)
    return _attend(state["q"].float(), state["k"].float(), state["v"].float(), seen).to(torch.bfloat16)


# ---- what a pass cannot do without ------------------------------------------------------------------------


def _seen_count(case, first, n, length):
    """Visible (query, key) pairs of n queries at positions first .. first + n - 1 over `length` keys, and the keys
    that one of them sees at least."""
    window = case["window"] or 1 << 60
    sinks = min(case["sinks"], length) if case["window"] else 0

    def near(p):
        return max(0, p - window + 1), min(length - 1, p if case["causal"] else p + window - 1)

    pairs = 0
    for p in range(first, first + n):
        lo, hi = near(p)
        pairs += hi - lo + 1 + min(sinks, lo) + (0 if case["causal"] else max(0, sinks - hi - 1))
    lo, hi = near(first)[0], near(first + n - 1)[1]
    return pairs, hi - lo + 1 + min(sinks, lo) + (0 if case["causal"] else max(0, sinks - hi - 1))


def work(case):
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "window":
        pairs, used = _seen_count(case, case["tk"] - case["tq"], case["tq"], case["tk"])
        return {"bytes": case["batch"] * dim * 4.0 * (case["tq"] * case["heads"] + used * kv),
                "flops": 4.0 * case["batch"] * pairs * case["heads"] * dim}
    new, keys = _lengths(case)
    stored = 2.0 * kv * (dim * (2 if case["format"] == "bf16" else 1) + (0 if case["format"] == "bf16" else 4))
    if case["op"] == "write":
        return {"bytes": sum(new) * (4.0 * kv * dim + stored), "flops": 0.0}
    if case["op"] == "read":
        return {"bytes": sum(keys) * stored + len(keys) * max(keys) * 4.0 * kv * dim, "flops": 0.0}
    counts = [_seen_count(case, m - n, n, m) for n, m in zip(new, keys)]
    return {"bytes": sum(used for _, used in counts) * stored + sum(new) * 4.0 * case["heads"] * dim,
            "flops": 4.0 * sum(pairs for pairs, _ in counts) * case["heads"] * dim}


# ---- the same in 64 bits ----------------------------------------------------------------------------------


def _value64(state, name, s, length):
    """The first `length` rows of sequence s in 64 bits, [heads, length, dim]."""
    page = state["case"]["page"]
    pages = state["table"][s, :-(-length // page)].long()
    x = state[name][pages].to(torch.float64)
    if state[name + "_scale"] is not None:
        x *= state[name + "_scale"][pages].to(torch.float64).unsqueeze(-1)
    return x.movedim(1, 0).reshape(x.shape[1], -1, x.shape[-1])[:, :length]


def _attend64(case, q, k, v, first):
    """One sequence: q [n, Hq, D], k and v [H, L, D] in 64 bits, queries at positions first .. first + n - 1."""
    out = torch.zeros_like(q)
    n, heads, dim = q.shape
    length, group = k.shape[1], heads // k.shape[0]
    j = torch.arange(length, device="cuda")[None]
    step = max(1, (1 << 28) // length)
    for a in range(0, n, step):
        p = torch.arange(first + a, first + min(n, a + step), device="cuda")[:, None]
        hidden = (j > p) if case["causal"] else torch.zeros((p.shape[0], length), dtype=torch.bool, device="cuda")
        if case["window"]:
            hidden |= ((j <= p - case["window"]) | (j >= p + case["window"])) & (j >= case["sinks"])
        for h in range(heads):
            s = (q[a:a + step, h] @ k[h // group].t().contiguous()) / math.sqrt(dim)
            s[hidden] = -math.inf
            out[a:a + step, h] = torch.nan_to_num(torch.softmax(s, 1)) @ v[h // group]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "window":
        out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            out[b] = _attend64(case, state["q"][b].double(), state["k"][b].double().movedim(1, 0),
                               state["v"][b].double().movedim(1, 0), case["tk"] - case["tq"])
        return out
    new, keys = _lengths(case)
    if case["op"] == "paged":
        out, at = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda"), 0
        for s, (n, length) in enumerate(zip(new, keys)):
            out[at:at + n] = _attend64(case, state["q"][at:at + n].double(), _value64(state, "cache_k", s, length),
                                       _value64(state, "cache_v", s, length), length - n)
            at += n
        return out
    if case["op"] == "read":
        shape = (case["seqs"], max(keys), case["kv_heads"], case["dim"])
        out = [torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        for x, name in zip(out, ("cache_k", "cache_v")):
            for s, length in enumerate(keys):
                x[s, :length] = _value64(state, name, s, length).movedim(0, 1)
        return tuple(out)
    # Writing: the stored rows; FP8 codes have no exact value, and whole numbers need none.
    out = {}
    for name, rows in (("cache_k", state["k"]), ("cache_v", state["v"])):
        store = torch.zeros(state[name].shape if case["format"] == "bf16" else state[name].shape[:-1],
                            dtype=torch.float64, device="cuda")
        at = 0
        for s, (n, length) in enumerate(zip(new, keys)):
            p = torch.arange(length - n, length, device="cuda")
            x = rows[at:at + n].double()
            x = x if case["format"] == "bf16" else x.abs().max(-1).values / LEVELS[case["format"]]
            store[state["table"][s].long()[p // case["page"]], :, p % case["page"]] = x
            at += n
        out[name] = store if case["format"] == "bf16" else None
        if case["format"] != "bf16":
            out[name + "_scale"] = store
    return out
