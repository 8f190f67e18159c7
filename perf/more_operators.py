"""Operators of a serving step with drafted tokens, for timing and for comparing outputs.

A server that drafts tokens takes pages for them and learns their slots and positions (`reserve`), turns queries and keys to those positions
(`rotary`; in training, where the same turn stands in front of the attention, its gradients too), attends to the cache with each drafted
token seeing its own branch of the tree only (`tree`), accepts a branch by the target's and the draft's probabilities with given random numbers
(`verify`), and moves the rows of the accepted tokens together in the cache (`keep`).  Row 0 of a sequence's new tokens is the
last accepted token; `parents[row]` is the row of the same sequence that it follows, -1 for none.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}            # largest code


def _tree(name, new, before, hq, hkv, dim, page, store, dtype="bfloat16", spread=8, append=True, lse=False):
    """`new`, `before`: new tokens of each sequence and tokens in its pages already, as texts "a,b,c" or "a,bxN" (N times over).  A row's
    parent is one of the `spread` rows before it (1: a chain)."""
    return _named(name, {"kind": "tree", "new": new, "before": before, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "store": store,
                         "dtype": dtype, "spread": spread, "append": append, "lse": lse})


def _verify(name, new, vocabulary, dtype="float32", spread=1, draft=True):
    return _named(name, {"kind": "verify", "new": new, "vocabulary": vocabulary, "dtype": dtype, "spread": spread, "draft": draft})


def _rotary(name, rows, hq, hkv, dim, turned, form="half", scaling="none", far=4096, dtype="bfloat16", train=False):
    """`turned`: dims of a head that are turned; `far`: positions are below it."""
    return _named(name, {"kind": "rotary", "rows": rows, "hq": hq, "hkv": hkv, "dim": dim, "turned": turned, "form": form, "scaling": scaling,
                         "far": far, "dtype": dtype, "train": train})


def _reserve(name, new, before, page, spread=1):
    return _named(name, {"kind": "reserve", "new": new, "before": before, "page": page, "spread": spread})


def _keep(name, new, before, hkv, dim, page, store, dtype="bfloat16", spread=8):
    return _named(name, {"kind": "keep", "new": new, "before": before, "hkv": hkv, "dim": dim, "page": page, "store": store, "dtype": dtype,
                         "spread": spread})


def _named(name, c):
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # a tree of eight drafted tokens of one request: latency of a layer's step
        _tree("tree-8-d64", "8", "4001", 16, 4, 64, 16, "same", "float16", spread=4),
        # trees of 32 in a ragged batch of 12 over 8-bit pages
        _tree("tree-12x32-e4m3", "32x12", "4097,900,20011,6144,12345,333x2", 32, 8, 128, 64, "e4m3", lse=True),
        # trees of 63 drafted tokens behind the last one of 24 requests: the largest call
        _tree("tree-24x64", "64x24", "8191,1023,16000,5000,2047,12000x4", 32, 8, 128, 64, "same", append=False),
        # five drafted tokens behind the last one of one request, in a line: latency
        _verify("verify-1x6", "6", 32000),
        # the same of a batch of 64 requests, a large vocabulary
        _verify("verify-64x5", "5x64", 128000),
        # trees whose tokens are the likeliest of the draft, without its probabilities; 16 bits, rows that begin at odd addresses
        _verify("verify-trees-16x40", "40x16", 100003, "bfloat16", spread=6, draft=False),
        # a decode step of 64 requests, far positions, scaled for them, in place
        _rotary("rotary-64-far", 64, 32, 8, 128, 128, scaling="parts", far=1 << 20),
        # the turn in front of the attention of a training step, and back: half of a head, pairs side by side
        _rotary("rotary-train-16k", 16384, 32, 8, 128, 64, form="pairs", train=True),
        # pages, slots and positions of a decode step of 64 requests
        _reserve("reserve-64x1", "1x64", "1023,16,4000,777,0,12345,63,64x8", 64),
        # the same of prompts, drafted tokens and decode steps in small pages
        _reserve("reserve-mixed-16", "40000,17,1,64,5,2048,1,7777x4", "0,100,16,5000,31,4096,20000,1x4", 16, spread=6),
        # trees of eight of six requests written, and an accepted branch of each moved together: latency
        _keep("keep-6x8", "8x6", "4001,333,64,70,1000,15", 4, 64, 16, "same", "float16", spread=4),
        # trees of 64 of 64 requests over 8-bit pages
        _keep("keep-64x64-e4m3", "64x64", "129,1023,60,5000,700,90,2047,31x8", 8, 128, 64, "e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(x):
    return ",".join(str(v) for v in x)


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "verify", "rotary", "reserve", "keep"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 6, 8] if hkv <= 4 else [1, 2, 4])
    dim = rng.choice([64, 96, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    page = rng.choice([16, 32, 64, 128])
    spread = rng.choice([1, 3, 6, 12])
    store = rng.choice(["same", "e4m3", "int8"])
    if kind == "tree":
        b = rng.choice([1, 1, 2, 4, 9, 20])
        new = [_log(rng, 1, 96 if b < 9 else 48) for _ in range(b)]
        before = [_log(rng, 1, 100000 // (b * max(1, hkv * dim // 256)) + 64) - 1 for _ in range(b)]
        return _tree(None, _text(new), _text(before), hq, hkv, dim, page, store, dtype, spread, rng.random() < 0.5, rng.random() < 0.4)
    if kind == "verify":
        b = rng.choice([1, 2, 5, 16, 48])
        new = [_log(rng, 1, 48 if b < 16 else 12) for _ in range(b)]
        most = min(200000, int(4e7 / sum(new)))
        return _verify(None, _text(new), _log(rng, 100, most), rng.choice(["float32", "float32", "bfloat16", "float16"]), spread,
                       rng.random() < 0.6)
    if kind == "rotary":
        turned = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rotary(None, _log(rng, 1, 16384 * 40 * 128 // ((hq + hkv) * dim)), hq, hkv, dim, turned, rng.choice(["half", "half", "pairs"]),
                       rng.choice(["none", "linear", "base", "parts"]), _log(rng, 64, 1 << 20), dtype, rng.random() < 0.4)
    if kind == "reserve":
        b = rng.choice([1, 2, 7, 33, 256, 1000])
        new = [_log(rng, 1, 30000 if b < 7 else 600 if b < 256 else 40) for _ in range(b)]
        before = [_log(rng, 1, 30000) - 1 for _ in range(b)]
        return _reserve(None, _text(new), _text(before), page, spread)
    b = rng.choice([1, 3, 10, 40])
    new = [_log(rng, 1, 96) for _ in range(b)]
    before = [_log(rng, 1, 3000) - 1 for _ in range(b)]
    return _keep(None, _text(new), _text(before), hkv, dim, page, store, dtype, spread)


def _numbers(text):
    """"a,bxN": the numbers of a list, repeated N times over."""
    body, _, times = text.partition("x")
    return [int(v) for v in body.split(",")] * (int(times) if times else 1)


def _lens(case):
    """(new, total) tokens of each sequence."""
    new, before = _numbers(case["new"]), _numbers(case["before"])
    assert len(new) == len(before)
    return new, [n + b for n, b in zip(new, before)]


def _parents(new, spread, seed):
    """Parents of all packed rows, sequence by sequence; long ones are blocks of prompts, without branches."""
    r = random.Random(seed)
    out = []
    for n in new:
        if n > 128:
            out += range(-1, n - 1)
            continue
        out += [-1] + [i - 1 - r.randrange(min(i, spread)) for i in range(1, n)] if n else []
    return out


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _ends(new):
    return [0] + [sum(new[:i + 1]) for i in range(len(new))]


# ---- inputs ----------------------------------------------------------------------------------

def _two(e):
    """2^e in 64 bits, without a rounding (a power function has one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes(x, store):
    """(codes, exponent bytes) of rows of fp32 values [..., D] of ordinary size: the least power of two whose product with the largest code reaches
    the row's largest magnitude."""
    amax = x.abs().amax(-1).double()
    e = torch.frexp(amax.float() / TOP[store])[1].clamp(-96, 127)
    for _ in range(2):                                        # the quotient is rounded: settled by comparing
        e = torch.where(TOP[store] * _two(e - 1) >= amax, e - 1, e).clamp(min=-96)
    e = torch.where(TOP[store] * _two(e) < amax, e + 1, e)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = x.double() * _two(-e)[..., None]
    codes = y.round().to(torch.int8) if store == "int8" else y.float().to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, exps):
    """What codes stand for, in 32 bits.  codes [..., D], exps [...]."""
    return codes.float() * (exps.to(torch.int32) << 23).view(torch.float32)[..., None]


def _prepare_pages(case, g, rows, total):
    """Pools, table and lengths; pages in no order, some of them other requests'."""
    dtype, store, hkv, dim, page = DTYPES[case["dtype"]], case["store"], case["hkv"], case["dim"], case["page"]
    need = [-(-n // page) for n in total]
    pages = sum(need) + 5
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(total), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    state = {"table": table, "lens": _i32(total), "max_len": max(total)}
    shift = torch.randn(hkv, dim, device="cuda", generator=g) * 0.5        # channels of keys have means of their own
    for name, mean in (("k", shift), ("v", torch.zeros_like(shift))):
        if store == "same":                                   # stored head by head within a page
            x = torch.randn(pages, hkv, page, dim, device="cuda", dtype=dtype, generator=g)
            state[name] = x.add_(mean.to(dtype)[:, None]).transpose(1, 2)
            state[name + "_scale"] = None
        else:
            codes = torch.empty(pages, hkv, page, dim, dtype=CODES[store], device="cuda")
            exps = torch.empty(pages, hkv, page, dtype=torch.uint8, device="cuda")
            for lo in range(0, pages, 512):
                x = torch.randn(min(512, pages - lo), hkv, page, dim, device="cuda", generator=g) + mean[:, None]
                codes[lo:lo + 512], exps[lo:lo + 512] = _codes(x, store)
            state[name], state[name + "_scale"] = codes.transpose(1, 2), exps
    return state


def _prepare_tree(case, seed, g):
    new, total = _lens(case)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    rows = sum(new)
    state = _prepare_pages(case, g, rows, total)
    # what a fused projection leaves: q, k and v of a token side by side
    qkv = torch.randn(rows, hq + 2 * hkv, dim, device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
    state.update(q=qkv[:, :hq], k_new=qkv[:, hq:hq + hkv], v_new=qkv[:, hq + hkv:], rows=rows, max_new=max(new), cu=_i32(_ends(new)),
                 parents=_i32(_parents(new, case["spread"], seed)))
    return state


def _prepare_keep(case, seed, g):
    new, total = _lens(case)
    rows = sum(new)
    state = _prepare_pages(case, g, rows, total)
    kv = torch.randn(rows, 2 * case["hkv"], case["dim"], device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
    parents, r, paths = _parents(new, case["spread"], seed), random.Random(seed + 1), []
    for n, lo in zip(new, _ends(new)):
        at, path = r.randrange(n), []
        while at >= 0:
            path.insert(0, at)
            at = parents[lo + at]
        paths.append(path[:1 + r.randrange(len(path))])
    wide = torch.full((len(new), max(new)), -1, dtype=torch.int32)
    for i, path in enumerate(paths):
        wide[i, :len(path)] = torch.tensor(path, dtype=torch.int32)
    state.update(k_new=kv[:, :case["hkv"]], v_new=kv[:, case["hkv"]:], rows=rows, cu=_i32(_ends(new)), path=wide.cuda(),
                 count=_i32([len(path) for path in paths]))
    return state


def _prepare_verify(case, seed, g):
    new, v, dtype = _numbers(case["new"]), case["vocabulary"], DTYPES[case["dtype"]]
    rows, parents = sum(new), _parents(new, case["spread"], seed)
    target = torch.empty(rows, v, dtype=dtype, device="cuda")
    draft = torch.empty_like(target)
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    common = 2.0 * torch.randn(v, device="cuda", generator=g)             # some tokens are frequent everywhere
    ends = _ends(new)
    sequence = torch.tensor([lo for lo, n in zip(ends, new) for _ in range(n)])
    follows = torch.tensor(parents)
    parent_row = torch.where(follows < 0, torch.full_like(follows, -1), follows + sequence)
    seen, nth = {}, []
    for p in parent_row.tolist():                             # which child of its parent a row is
        nth.append(seen.get(p, 0))
        seen[p] = nth[-1] + 1
    nth, most = torch.tensor(nth), max(seen.values())
    chunk = max(1, 50_000_000 // v)
    picks = torch.zeros(rows, most, dtype=torch.int64, device="cuda")     # tokens that a row's children may have
    for lo in range(0, rows, chunk):
        n = min(chunk, rows - lo)
        x = common + 2.5 * torch.randn(n, v, device="cuda", generator=g)
        target[lo:lo + n] = torch.softmax(x, -1)
        x += 0.7 * torch.randn(n, v, device="cuda", generator=g)
        p = torch.softmax(x, -1)
        draft[lo:lo + n] = p
        if case["draft"]:                                     # drawn from the draft, one by one
            picks[lo:lo + n] = torch.multinomial(p, most, replacement=True, generator=g)
        else:                                                 # its likeliest ones
            picks[lo:lo + n, :min(most, v)] = p.topk(min(most, v), -1).indices
    has = (parent_row >= 0).cuda()
    tokens[has] = picks[parent_row.cuda()[has], nth.cuda()[has]]
    return {"target": target, "draft": draft if case["draft"] else None, "tokens": tokens, "cu": _i32(ends), "max_new": max(new),
            "accept": torch.rand(rows, device="cuda", generator=g), "sample": torch.rand(len(new), device="cuda", generator=g),
            "parents": None if case["spread"] == 1 else _i32(parents), "new": new}


def _frequencies(case):
    """Radians that a position turns each pair by (64 bits)."""
    d, base, kind, factor, original = case["turned"], 10000.0, case["scaling"], 16.0, 4096.0
    if kind == "base" and d > 2:
        base *= factor ** (d / (d - 2))
    f = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if kind == "linear":
        f = f / factor
    if kind == "parts":                                       # what turns often within the original length stays, the rest is stretched
        stay = ((original * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * stay + f / factor * (1 - stay)
    return f


def _prepare_rotary(case, seed, g):
    rows, hq, hkv, dim = case["rows"], case["hq"], case["hkv"], case["dim"]
    qkv = torch.randn(rows, hq + 2 * hkv, dim, device="cuda", dtype=DTYPES[case["dtype"]], generator=g)
    state = {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "positions": torch.randint(case["far"], (rows,), device="cuda", generator=g).int(),
             "magnitude": 1.0 + 0.1 * math.log(16.0) if case["scaling"] == "parts" else 1.0, "frequencies": _frequencies(case)}
    if case["train"]:
        state["dq"], state["dk"] = (torch.randn(rows, h, dim, device="cuda", dtype=qkv.dtype, generator=g) for h in (hq, hkv))
        state["q"], state["k"] = (x.detach().requires_grad_() for x in (state["q"], state["k"]))
    else:                                                     # (the turned rows go to tensors that the program keeps)
        state["q_out"], state["k_out"] = (torch.empty(rows, h, dim, device="cuda", dtype=qkv.dtype) for h in (hq, hkv))
    if own:                                                   # kept by a program for all layers and calls
        from baselinebenchmark_b200 import RotaryTable
        state["table"] = RotaryTable(state["frequencies"], interleaved=case["form"] == "pairs", magnitude=state["magnitude"], device="cuda")
    state["device_frequencies"] = state["frequencies"].cuda()
    return state


def _prepare_reserve(case, seed, g):
    new, total = _lens(case)
    page = case["page"]
    held = [-(-(t - n) // page) for n, t in zip(new, total)]
    need = [-(-t // page) for t in total]
    pages = sum(need) + 7
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(new), max(need) + 2), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[:pages - at] = order[at:]
    parents = None if case["spread"] == 1 else _i32(_parents(new, case["spread"], seed))
    return {"table": table, "cu": _i32(_ends(new)), "lens": _i32(total), "before": _i32([t - n for n, t in zip(new, total)]), "free": free,
            "free_count": _i32([pages - at]), "parents": parents, "rows": sum(new)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"tree": _prepare_tree, "keep": _prepare_keep, "verify": _prepare_verify, "rotary": _prepare_rotary,
             "reserve": _prepare_reserve}[case["kind"]](case, seed, g)
    state["case"] = dict(case)
    return state


# ---- plain forms -----------------------------------------------------------------------------

def _places(state):
    """(sequence, index in it, position by index) of each packed row."""
    row = torch.arange(state["rows"], device="cuda", dtype=torch.int32)
    cu = state["cu"]
    seq = torch.bucketize(row, cu[1:], right=True)
    at = (row - cu[seq]).long()
    return seq, at, state["lens"][seq].long() - (cu[seq + 1] - cu[seq]) + at


def _slots(state):
    seq, _, pos = _places(state)
    page = state["case"]["page"]
    return state["table"][seq, pos // page].long(), pos % page


def _plain_store(state):
    where, at = _slots(state)
    for name in ("k", "v"):
        x = state[name + "_new"]
        if state[name + "_scale"] is None:
            state[name][where, at] = x
        else:
            codes, exps = _codes(x.float(), state["case"]["store"])
            state[name].view(torch.int8)[where, at] = codes.view(torch.int8)
            state[name + "_scale"].transpose(1, 2)[where, at] = exps


def _ancestors(state):
    """[rows, max_new]: row's index is a row's own or one of its ancestors'."""
    seq, at, _ = _places(state)
    first, n = state["cu"][seq].long(), state["max_new"]
    seen = torch.zeros(state["rows"], n, dtype=torch.bool, device="cuda")
    here = at
    row = torch.arange(state["rows"], device="cuda")
    for _ in range(n):
        live = here >= 0
        seen[row, here.clamp(min=0)] |= live
        here = torch.where(live, state["parents"][first + here.clamp(min=0)].long(), here)
    return seen


def _plain_tree(state):
    """Softmax attention of a batch padded to its longest sequence and most new tokens, in 32 bits."""
    case = state["case"]
    if case["append"]:
        _plain_store(state)
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    cu, lens, table = state["cu"], state["lens"], state["table"]
    b, n, wide = lens.numel(), state["max_new"], -(-state["max_len"] // page)
    ids = table[:, :wide].clamp(min=0).long()

    def rows(name):                                           # [B, Hkv, keys, D]
        pages, scale = state[name], state[name + "_scale"]
        if scale is None:
            x = pages[ids].float()
        else:
            x = _values(pages.view(torch.int8)[ids].view(pages.dtype), scale.transpose(1, 2)[ids])
        return x.reshape(b, wide * page, hkv, dim).transpose(1, 2)

    count = (cu[1:] - cu[:-1]).long()
    seq, at, _ = _places(state)
    key = torch.arange(wide * page, device="cuda")
    before = (lens.long() - count)[:, None]                   # tokens in front of the new ones
    rel = key[None] - before                                  # [B, keys]: index among the new ones
    pad = torch.zeros(b, n, n, dtype=torch.bool, device="cuda")
    pad[seq, at] = _ancestors(state)
    branch = torch.gather(pad, 2, rel.clamp(0, n - 1)[:, None].expand(b, n, -1))
    there = torch.arange(n, device="cuda")[None] < count[:, None]
    see = ((rel < 0)[:, None] | (branch & (rel >= 0)[:, None] & (rel < count[:, None])[:, None])) & there[..., None]
    q = torch.zeros(b, n, hq, dim, device="cuda")
    q[seq, at] = state["q"].float()
    q = q.reshape(b, n, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * (hq // hkv), dim)
    s = torch.matmul(q, rows("k").transpose(2, 3)).mul_(dim ** -0.5)
    s = s.view(b, hkv, n, hq // hkv, wide * page).masked_fill_(~see[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, -1, wide * page), rows("v")).view(b, hkv, n, hq // hkv, dim) / total
    out = o[seq, :, at].reshape(state["rows"], hq, dim).to(DTYPES[case["dtype"]])
    if not case["lse"]:
        return (out,)
    lse = (top + total.log())[..., 0]
    return out, lse[seq, :, at].reshape(state["rows"], hq).t().contiguous()


def _plain_keep(state):
    _plain_store(state)
    page = state["case"]["page"]
    path, count, cu = state["path"].long(), state["count"], state["cu"]
    step = torch.arange(path.shape[1], device="cuda")[None]
    live = step < count[:, None]
    before = (state["lens"] - (cu[1:] - cu[:-1])).long()[:, None]
    source = before + path.clamp(min=0)
    # (behind its end a path reads row 0, which stays where it is)
    source = torch.where(live, source, before)
    target = torch.where(live, before + step, before)
    seq = torch.arange(path.shape[0], device="cuda")[:, None].expand_as(path)
    place = lambda x: (state["table"][seq, x // page].long(), x % page)  # noqa: E731
    source, target = place(source), place(target)
    for name in ("k", "v"):
        pages = state[name] if state[name + "_scale"] is None else state[name].view(torch.int8)
        pages[target] = pages[source]
        if state[name + "_scale"] is not None:
            scale = state[name + "_scale"].transpose(1, 2)
            scale[target] = scale[source]
    return (state["lens"] - (cu[1:] - cu[:-1]) + count).int()


def _read_back(state):
    """The new tokens' places in the pools."""
    where, at = _slots(state)
    dtype = DTYPES[state["case"]["dtype"]]
    return tuple(_values(state[name].view(torch.int8)[where, at].view(state[name].dtype), state[name + "_scale"].transpose(1, 2)[where, at]).to(dtype)
                 for name in ("k", "v"))


def _plain_verify(state):
    """All sequences side by side, row by row in the order of the tree, in 64 bits."""
    target, draft, cu, n = state["target"], state["draft"], state["cu"], state["max_new"]
    b = cu.numel() - 1
    count = (cu[1:] - cu[:-1]).long()
    step = torch.arange(n, device="cuda")
    there = step[None] < count[:, None]
    row = torch.where(there, cu[:-1, None].long() + step, 0)
    parents = (step[None] - 1).expand(b, n) if state["parents"] is None else state["parents"].long()[row]
    tokens = state["tokens"][row]
    at = torch.zeros(b, dtype=torch.long, device="cuda")      # the branch's last row so far
    left = target[row[:, 0]].double()                         # what is left of its row's probabilities
    mass = torch.ones(b, dtype=torch.float64, device="cuda")
    path = torch.full((b, n), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    length = torch.ones(b, dtype=torch.long, device="cuda")
    every = torch.arange(b, device="cuda")
    for i in range(1, n):
        child = there[:, i] & (parents[:, i] == at)
        x = tokens[:, i]
        have = left[every, x]
        u = state["accept"][row[:, i]].double()
        q = draft[row[every, at]].double() if draft is not None else None
        bar = u * mass * (q[every, x] if draft is not None else 1.0)
        take = child & (have > 0) & (bar < have)
        miss = child & ~take
        if draft is not None:
            less = (left / mass.clamp(min=1e-300)[:, None] - q).clamp(min=0)
            left = torch.where(miss[:, None], less, left)
            mass = torch.where(miss, less.sum(-1), mass)
        else:
            mass = torch.where(miss, mass - have, mass)
            left[every[:, None], x[:, None]] = torch.where(miss, 0.0, have)[:, None]
        left = torch.where(take[:, None], target[row[:, i]].double(), left)
        mass = torch.where(take, 1.0, mass)
        path[every, length.clamp(max=n - 1)] = torch.where(take, i, path[every, length.clamp(max=n - 1)].long()).int()
        length = length + take.long()
        at = torch.where(take, i, at)
    none = left.sum(-1) <= 0
    left = torch.where(none[:, None], target[row[every, at]].double(), left)
    ends = left.cumsum(-1)
    token = (ends <= (state["sample"].double() * ends[:, -1])[:, None]).sum(-1)
    last = target.shape[1] - 1 - (left.flip(-1) > 0).int().argmax(-1)
    return path, length.int(), torch.minimum(token, last)


def _turn(x, cos, sin, case):
    """The first `turned` dims of x [rows, heads, D], in 32 bits."""
    d = case["turned"]
    y = x.detach().float()
    if case["form"] == "half":
        a, b = y[..., :d // 2], y[..., d // 2:d]
    else:
        a, b = y[..., 0:d:2], y[..., 1:d:2]
    cos, sin = cos[:, None], sin[:, None]
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([u, v], -1) if case["form"] == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, y[..., d:]], -1).to(x.dtype)


def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["device_frequencies"]
    cos, sin = ((f(angle) * state["magnitude"]).float() for f in (torch.cos, torch.sin))
    out = tuple(_turn(state[name], cos, sin, case) for name in ("q", "k"))
    if case["train"]:
        return out + tuple(_turn(state[name], cos, -sin, case) for name in ("dq", "dk"))
    state["q_out"].copy_(out[0])
    state["k_out"].copy_(out[1])
    return state["q_out"], state["k_out"]


def _plain_reserve(state):
    page, table, free = state["case"]["page"], state["table"], state["free"]
    have = state["free_count"].long()
    column = torch.arange(table.shape[1], device="cuda")[None]
    lens, before = state["lens"].long()[:, None], state["before"].long()[:, None]
    lack = (column >= before // page) & (column < -(-lens // page)) & ((table < 0) | (table >= free.numel()))
    rank = lack.flatten().long().cumsum(0).view_as(table) - 1
    take = lack & (rank < have)
    table.copy_(torch.where(take, free[(have - 1 - rank).clamp(0, free.numel() - 1)], table))
    missing = (lack.sum() - take.sum()).int().reshape(1)
    state["free_count"].sub_(take.sum().int())
    seq, at, pos = _places(state)
    entry = table[seq, pos // page].long()
    slots = torch.where(entry >= 0, entry * page + pos % page, -1)
    positions = pos
    if state["parents"] is not None:                          # depth below a row without a parent
        first = state["cu"][seq].long()
        up = state["parents"].long()
        hop, reach = torch.where(up >= 0, up + first, -1), (up >= 0).long()
        for _ in range(state["rows"].bit_length()):           # in doubled steps
            more = hop >= 0
            reach = reach + torch.where(more, reach[hop.clamp(min=0)], 0)
            hop = torch.where(more, hop[hop.clamp(min=0)], -1)
        positions = pos - at + reach
    # the step over, its pages go back: those behind the tokens that were there before
    back = (column >= -(-before // page)) & (table >= 0) & (table < free.numel())
    order = back.flatten().long().cumsum(0).view_as(table)
    total, base = order[-1, -1], state["free_count"].long()
    # (what does not go back is written behind the end)
    place = torch.where(back, base + total - order, free.numel())
    free.copy_(torch.cat([free, free[:1]]).scatter(0, place.flatten(), table.flatten())[:-1])
    state["free_count"].add_(total.int())
    table.masked_fill_(back, -1)
    return slots, positions.int(), missing, table, free, state["free_count"]


# ---- a pass ----------------------------------------------------------------------------------

def _pages(state):
    return (state["k"], state["v"], state["table"], state["cu"], state["lens"])


def _scales(state):
    return {"k_scales": state["k_scale"], "v_scales": state["v_scale"]}


def _own_tree(state):
    from baselinebenchmark_b200 import paged_append, paged_attention
    case = state["case"]
    new = (state["k_new"], state["v_new"]) if case["append"] else ()
    out = (paged_append if case["append"] else paged_attention)(state["q"], *new, *_pages(state), state["max_new"], parents=state["parents"],
                                                                return_lse=case["lse"], **_scales(state))
    return out if case["lse"] else (out,)


def _own_keep(state):
    from baselinebenchmark_b200 import paged_keep, paged_store
    paged_store(state["k_new"], state["v_new"], *_pages(state), **_scales(state))
    return paged_keep(*_pages(state), state["path"], state["count"], **_scales(state))


def _own_read_back(state):
    from baselinebenchmark_b200 import paged_load
    return paged_load(*_pages(state), state["rows"], dtype=DTYPES[state["case"]["dtype"]], **_scales(state))


def _own_verify(state):
    from baselinebenchmark_b200 import verify_drafts
    return verify_drafts(state["target"], state["draft"], state["tokens"], state["cu"], state["accept"], state["sample"], state["max_new"],
                         parents=state["parents"])


def _own_rotary(state):
    from baselinebenchmark_b200 import rotary
    if not state["case"]["train"]:
        return rotary(state["q"], state["k"], state["positions"], state["table"], out=(state["q_out"], state["k_out"]))
    out = rotary(state["q"], state["k"], state["positions"], state["table"])
    return tuple(out) + torch.autograd.grad(out, (state["q"], state["k"]), (state["dq"], state["dk"]))


def _own_reserve(state):
    from baselinebenchmark_b200 import paged_release, paged_reserve
    pool = (state["free"], state["free_count"], state["case"]["page"])
    slots, positions, missing = paged_reserve(state["table"], state["cu"], state["lens"], *pool, state["rows"], parents=state["parents"])
    paged_release(state["table"], state["before"], *pool)
    return slots, positions, missing, state["table"], state["free"], state["free_count"]


def run(state):
    kind = state["case"]["kind"]
    if kind == "keep":
        lens = _own_keep(state) if own else _plain_keep(state)
        if state["k_scale"] is None:
            return lens, state["k"], state["v"]
        return (lens, *(_own_read_back(state) if own else _read_back(state)))
    if kind == "tree":
        kept = (state["k"], state["v"]) if state["case"]["append"] and state["k_scale"] is None else ()
        return (*(_own_tree(state) if own else _plain_tree(state)), *kept)
    if own:
        return {"verify": _own_verify, "rotary": _own_rotary, "reserve": _own_reserve}[kind](state)
    return {"verify": _plain_verify, "rotary": _plain_rotary, "reserve": _plain_reserve}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "verify":                                      # one row of each distribution a sequence, and an element a row
        size, new = DTYPES[case["dtype"]].itemsize, _numbers(case["new"])
        sides = 2 if case["draft"] else 1
        return {"bytes": sides * size * (case["vocabulary"] * len(new) + sum(new)) + 16 * sum(new), "flops": 0}
    if kind == "rotary":
        elements = case["rows"] * (case["hq"] + case["hkv"]) * case["dim"]
        sides = 2 if case["train"] else 1
        return {"bytes": 4 * elements * sides + 4 * case["rows"], "flops": sides * 3 * elements * case["turned"] // case["dim"]}
    new, total = _lens(case)
    if kind == "reserve":                                     # pages taken and put back, a slot and a position a row
        pages = sum(-(-t // case["page"]) - -(-(t - n) // case["page"]) for n, t in zip(new, total))
        return {"bytes": 16 * pages + sum(new) * (12 + (4 if case["spread"] > 1 else 0)) + 16 * len(new), "flops": 0}
    row = case["dim"] * (2 if case["store"] == "same" else 1) + (0 if case["store"] == "same" else 1)   # bytes of a stored row
    values, stored = 4 * case["hkv"] * sum(new) * case["dim"], 2 * case["hkv"] * sum(new) * row
    if kind == "keep":                                        # rows in, codes out, some of them moved, 8-bit ones read back
        return {"bytes": values + stored + (stored + values if case["store"] != "same" else 0), "flops": 0}
    move = 2 * case["hkv"] * sum(total) * row + 4 * sum(new) * case["hq"] * case["dim"] + (4 * sum(new) * case["hq"] if case["lse"] else 0)
    if case["append"]:
        move += values + stored
    # each row sees the tokens in front and its branch; of the drafted ones that is a few
    return {"bytes": move, "flops": 4 * case["dim"] * case["hq"] * sum(n * (t - n + 1) for n, t in zip(new, total))}


# ---- from the definitions, in 64 bits ----------------------------------------------------------

def _exact_codes(x, store):
    """What the rows [..., D] stand for once stored."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / TOP[store])).clamp(-96, 127)
    for d in (1, -1):                                         # log2 is rounded: the neighbours decide
        near = (e + d).clamp(-96, 127)
        e = torch.where((TOP[store] * _two(near) >= amax) & ((near < e) | (TOP[store] * _two(e) < amax)), near, e)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = x / _two(e)
    if store == "int8":
        return y.round() * _two(e)
    step = _two(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)   # e4m3: an eighth of the power of two below, 2^-9 under 2^-6
    return (y / step).round() * step * _two(e)


def _exact_tree(case, s):
    new, total = _lens(case)
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    group, parents = hq // hkv, s["parents"].tolist()
    if 4 * dim * hq * sum(n * t for n, t in zip(new, total)) > 4e13:
        return None
    kept = [s["k"].double(), s["v"].double()] if case["append"] and case["store"] == "same" else []
    out, lse, lo = [], [], 0
    for i, n in enumerate(new):
        kv = []
        for name in ("k", "v"):
            used = s["table"][i, :-(-total[i] // page)].long()
            if case["store"] == "same":
                x = s[name][used].double()
            else:
                x = s[name].view(torch.int8)[used].view(s[name].dtype).double() * _two(s[name + "_scale"][used].transpose(1, 2).int() - 127)[..., None]
            x = x.reshape(-1, hkv, dim)[:total[i]]
            if case["append"]:
                fresh = s[name + "_new"][lo:lo + n].double()
                x[total[i] - n:] = fresh if case["store"] == "same" else _exact_codes(fresh, case["store"])
            kv.append(x)
        for x, y in zip(kept, kv):
            at = torch.arange(total[i] - n, total[i], device="cuda")
            x[s["table"][i, at // page].long(), at % page] = y[at]
        hidden = torch.ones(n, total[i], dtype=torch.bool)
        hidden[:, :total[i] - n] = False
        for r in range(n):
            up = r
            while up >= 0:
                hidden[r, total[i] - n + up] = False
                up = parents[lo + up]
        hidden = hidden.cuda()
        o, m = [], []
        for h in range(hq):
            score = s["q"][lo:lo + n, h].double() @ kv[0][:, h // group].t() / math.sqrt(dim)
            score = score.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(score, -1)
            o.append(torch.exp(score - z[:, None]) @ kv[1][:, h // group])
            m.append(z)
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(m))
        lo += n
    return (torch.cat(out), *([torch.cat(lse, 1)] if case["lse"] else []), *kept)


def _exact_keep(case, s):
    new, total = _lens(case)
    page, same = case["page"], case["store"] == "same"
    pools = [s[name].double() for name in ("k", "v")] if same else []
    back = [[], []]
    lens, lo = [], 0
    for i, n in enumerate(new):
        path = s["path"][i, :int(s["count"][i])].tolist()
        lens.append(total[i] - n + len(path))
        for w, name in enumerate(("k", "v")):
            fresh = s[name + "_new"][lo:lo + n].double()
            fresh = fresh if same else _exact_codes(fresh, case["store"])
            after = fresh.clone()
            after[:len(path)] = fresh[path]
            back[w].append(after)
            if same:
                at = torch.arange(total[i] - n, total[i], device="cuda")
                pools[w][s["table"][i, at // page].long(), at % page] = after
        lo += n
    return (_i32(lens), *(pools if same else (torch.cat(x) for x in back)))


def _exact_verify(case, s):
    out, tokens, accept = [], s["tokens"].tolist(), s["accept"].double().tolist()
    ends = _ends(s["new"])
    parents = s["parents"].tolist() if s["parents"] is not None else [r - lo - 1 for lo, n in zip(ends, s["new"]) for r in range(lo, lo + n)]
    most = max(s["new"])
    for b, (lo, n) in enumerate(zip(ends, s["new"])):
        at, path, end = 0, [0], False
        while not end:
            left, mass = s["target"][lo + at].double(), 1.0
            children = [r for r in range(1, n) if parents[lo + r] == at]
            end = True
            for r in children:
                x = tokens[lo + r]
                have = float(left[x])
                drawn = float(s["draft"][lo + at, x]) if s["draft"] is not None else 1.0
                if have > 0 and accept[lo + r] * drawn * mass < have:
                    at, end = r, False
                    path.append(r)
                    break
                if s["draft"] is not None:
                    left = (left / max(mass, 1e-300) - s["draft"][lo + at].double()).clamp(min=0)
                    mass = float(left.sum())
                else:
                    mass -= have
                    left[x] = 0.0
        if float(left.sum()) <= 0:
            left = s["target"][lo + at].double()
        ends_of = left.cumsum(0)
        over = torch.nonzero(ends_of > s["sample"][b].double() * ends_of[-1])
        out.append((path, int(over[0]) if over.numel() else int(torch.nonzero(left > 0)[-1])))
    path = torch.tensor([p + [-1] * (most - len(p)) for p, _ in out], dtype=torch.int32)
    return path, torch.tensor([len(p) for p, _ in out], dtype=torch.int32), torch.tensor([t for _, t in out])


def _exact_rotary(case, s):
    if case["rows"] * (case["hq"] + case["hkv"]) * case["dim"] > 2e8:
        return None
    d = case["turned"]
    z = torch.polar(torch.full((case["rows"], d // 2), s["magnitude"], dtype=torch.float64, device="cuda"),
                    s["positions"].double()[:, None] * s["frequencies"].cuda())[:, None]
    out = []
    for name in ("q", "k") + (("dq", "dk") if case["train"] else ()):
        x = s[name].detach().double().clone()
        first, second = (slice(0, d // 2), slice(d // 2, d)) if case["form"] == "half" else (slice(0, d, 2), slice(1, d, 2))
        y = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * (z.conj() if name[0] == "d" else z)
        x[..., first], x[..., second] = y.real, y.imag
        out.append(x)
    return tuple(out)


def _exact_reserve(case, s):
    new, total = _lens(case)
    page, cu = case["page"], _ends(new)
    table, count = s["table"].cpu(), int(s["free_count"])
    free = s["free"].cpu()
    after, left = table.clone(), count
    for b, (n, t) in enumerate(zip(new, total)):
        for i in range((t - n) // page, -(-t // page)):
            if after[b, i] < 0:
                left -= 1
                after[b, i] = free[left]
    slots, positions = [], []
    parents = s["parents"].tolist() if s["parents"] is not None else None
    for b, (n, t) in enumerate(zip(new, total)):
        pos = torch.arange(t - n, t)
        slots.append(after[b, pos // page].long() * page + pos % page)
        if parents is not None:
            depth = []
            for r in range(n):
                up = parents[cu[b] + r]
                depth.append(0 if up < 0 else depth[up] + 1)
            pos = t - n + torch.tensor(depth, dtype=torch.int64)
        positions.append(pos.int())
    # all of it goes back to where it was
    return torch.cat(slots), torch.cat(positions), torch.zeros(1, dtype=torch.int32), table, free, torch.tensor([count], dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "keep": _exact_keep, "verify": _exact_verify, "rotary": _exact_rotary, "reserve": _exact_reserve}[case["kind"]](case, s)
