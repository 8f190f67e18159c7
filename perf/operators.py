"""Operators over a cache of keys and values that is kept in pages, for timing and for comparing outputs.

A case is one call that a serving program makes between two layers' projections: new K and V rows written into the
pages of their sequences and read back (`write`), the rows of whole sequences read back as the packed batch that a
prefill takes (`read`), and attention of each sequence's new tokens over its pages (`attend`; with `append` the
new tokens' rows are written first, as in a decode step).  Pages hold 16-bit rows, or 8-bit codes with a power of two per
row and head: a code c with exponent byte e stands for c * 2^(e - 127).
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
STORES = {"same": None, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
#: largest code; its power of two's exponent and its significand: the smallest e with amax <= code * 2^e
TOP = {"e4m3": 448.0, "int8": 127.0}
#: the largest magnitude that a code may stand for: finite in the rows' 16-bit type
MOST = {("e4m3", "bfloat16"): 240.0 * 2.0 ** 120, ("int8", "bfloat16"): 63.0 * 2.0 ** 122,
        ("e4m3", "float16"): 240.0 * 2.0 ** 8, ("int8", "float16"): 63.0 * 2.0 ** 10}


def _case(name, kind, new, before, hq, hkv, dim, page, store, dtype="bfloat16", append=False, lse=False):
    """`new`, `before`: new tokens of each sequence and tokens that are in its pages already, as texts (one number
    for all of them, "nxcount", or a list).  `store`: what the pages hold."""
    c = {"kind": kind, "new": new, "before": before, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "store": store,
         "dtype": dtype, "append": append, "lse": lse}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # the rows of one decode step of 64 requests: latency of the write
        _case("write-64x1-e4m3", "write", "1x64", "700x64", 32, 8, 128, 64, "e4m3"),
        # three blocks of chunked prefills, ragged, fp16, into 8-bit integers
        _case("write-8k-int8", "write", "4097,1023,3071", "0,5000,12345", 32, 8, 128, 32, "int8", "float16"),
        # a small model's ragged batch into 16-bit pages
        _case("write-ragged-d96", "write", "127,513,2049", "33,0,1000", 8, 4, 96, 16, "same"),
        # a 128K-token prefix read back for a prefill that continues it
        _case("read-128k-e4m3", "read", "131072", "0", 32, 8, 128, 64, "e4m3"),
        # a ragged batch of prompts read back, head_dim 64
        _case("read-ragged-d64", "read", "1023,4097,8191", "0x3", 16, 4, 64, 16, "same", "float16"),
        # one decode token of one request: latency
        _case("decode-20011-d64", "attend", "1", "20011", 16, 4, 64, 16, "same", "float16", append=True),
        # a decode step of a batch of 48 ragged requests
        _case("decode-48", "attend", "1x48", "15,16,17,700,1023,4097,8191,11000,333,2560,6144,7168x4", 32, 8, 128, 64, "same", lse=True),
        # a decode step of 16 long requests over 8-bit pages: bytes of the cache
        _case("decode-16x32k-e4m3", "attend", "1x16", "32768,20011,16384,40000x4", 32, 8, 128, 64, "e4m3", append=True),
        # five drafted tokens of 12 requests checked at once, 8-bit integers
        _case("verify-5x12-int8", "attend", "5x12", "4097,900,20011,6144,12345,333x2", 16, 4, 128, 32, "int8", "float16", lse=True),
        # prompts without a prefix at the largest head dim
        _case("prompts-d256", "attend", "1023,4096,200", "0x3", 16, 16, 256, 64, "same"),
        # one block of a chunked prefill behind a ragged prefix
        _case("block-700", "attend", "700", "50021", 32, 8, 128, 64, "same"),
        # a long block over 8-bit pages: the largest call
        _case("block-2048-e4m3", "attend", "2048", "30720", 32, 8, 128, 64, "e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 6, 8] if hkv <= 4 else [1, 2, 4])
    dim = rng.choice([64, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    store = rng.choice(["same", "e4m3", "int8"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "write":
        b = rng.choice([1, 2, 3, 5, 16, 64])
        new = [_log(rng, 1, 2048 if b <= 5 else 64) for _ in range(b)]
        before = [_log(rng, 1, 8192) - 1 for _ in range(b)]
    elif kind == "read":
        b = rng.choice([1, 2, 3, 7])
        new = [_log(rng, 1, 32768 // b) for _ in range(b)]
        before = [0] * b
    else:
        form = rng.choice(["decode", "decode", "draft", "block", "prompts"])
        if form in ("decode", "draft"):
            b = rng.choice([1, 2, 4, 9, 16, 40])
            new = [1] * b if form == "decode" else [rng.choice([1, 2, 4, 5, 8]) for _ in range(b)]
            before = [_log(rng, 1, 262144 // (b * max(1, hkv * dim // 256)) + 64) - 1 for _ in range(b)]
        elif form == "block":
            b = rng.choice([1, 1, 2, 3])
            new = [_log(rng, 9, (700 if dim == 256 else 1500) // b) for _ in range(b)]
            before = [_log(rng, 1, 32768 // b) for _ in range(b)]
        else:
            b = rng.choice([1, 2, 3, 5])
            new = [_log(rng, 16, 4096 // b) for _ in range(b)]
            before = [0] * b
    text = lambda x: ",".join(str(v) for v in x)  # noqa: E731
    append = kind == "attend" and rng.random() < 0.4
    return _case(None, kind, text(new), text(before), hq, hkv, dim, page, store, dtype, append, kind == "attend" and rng.random() < 0.4)


def _numbers(text):
    """"a,bxN": the numbers of a list, repeated N times over."""
    body, _, times = text.partition("x")
    return [int(v) for v in body.split(",")] * (int(times) if times else 1)


def _lens(case):
    """(new, total) tokens of each sequence."""
    new, before = _numbers(case["new"]), _numbers(case["before"])
    assert len(new) == len(before)
    return new, [n + b for n, b in zip(new, before)]


def _two(e):
    """2^e in 64 bits, without a rounding (a power function has one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes(x, store, dtype):
    """(codes, exponent bytes) of rows of fp32 values [..., D]."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax / TOP[store])                    # amax / top = m * 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e).clamp(-96, 127)     # the smallest with top * 2^e >= amax; exact: see below
    # frexp of a rounded quotient may sit one off at the border: settled by comparing in 64 bits
    two = _two(e)
    e = torch.where(TOP[store] * two < amax.double(), e + 1, e)
    e = torch.where((TOP[store] * two * 0.5 >= amax.double()) & (e > -96), e - 1, e)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = x.clamp(-MOST[store, dtype], MOST[store, dtype]).double() * _two(-e)[..., None]
    codes = y.round().to(torch.int8) if store == "int8" else y.float().to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, exps):
    """What codes stand for, in 32 bits.  codes [..., D], exps [...]."""
    return codes.float() * (exps.to(torch.int32) << 23).view(torch.float32)[..., None]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, store = DTYPES[case["dtype"]], case["store"]
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    new, total = _lens(case)
    b, rows = len(new), sum(new)
    # what a fused projection leaves: q, k and v of a token side by side
    qkv = torch.randn(rows, hq + 2 * hkv, dim, device="cuda", dtype=dtype, generator=g)
    shift = torch.randn(hkv, dim, device="cuda", generator=g) * 0.5        # channels of keys have means of their own
    qkv[:, hq:hq + hkv] += shift.to(dtype)
    # pages in no order, some of them other requests'; behind a sequence's last page the table has none
    need = [-(-n // page) for n in total]
    pages = sum(need) + 5
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    state = {"case": dict(case), "q": qkv[:, :hq], "k_new": qkv[:, hq:hq + hkv], "v_new": qkv[:, hq + hkv:], "table": table,
             "cu": torch.tensor([0] + [sum(new[:i + 1]) for i in range(b)], dtype=torch.int32, device="cuda"),
             "lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "max_new": max(new), "rows": rows,
             # padded positions of the plain form's batch: host numbers that any program has
             "max_len": max(total)}
    for name, mean in (("k", shift), ("v", 0.0)):
        # stored head by head within a page
        if store == "same":
            x = torch.randn(pages, hkv, page, dim, device="cuda", dtype=dtype, generator=g)
            if name == "k":
                x += shift.to(dtype)[:, None]
            state[name] = x.transpose(1, 2)
            state[name + "_scale"] = None
        else:
            codes = torch.empty(pages, hkv, page, dim, dtype=STORES[store], device="cuda")
            exps = torch.empty(pages, hkv, page, dtype=torch.uint8, device="cuda")
            for lo in range(0, pages, 512):
                x = torch.randn(min(512, pages - lo), hkv, page, dim, device="cuda", generator=g)
                if name == "k":
                    x += shift[:, None]
                codes[lo:lo + 512], exps[lo:lo + 512] = _codes(x, store, case["dtype"])
            state[name], state[name + "_scale"] = codes.transpose(1, 2), exps
    return state


def _places(state):
    """(sequence, position) of each packed row."""
    row = torch.arange(state["rows"], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(row, state["cu"][1:], right=True)
    return seq, (state["lens"][seq] - (state["cu"][seq + 1] - row)).long()


def _slots(state):
    seq, pos = _places(state)
    page = state["case"]["page"]
    return state["table"][seq, pos // page].long(), pos % page


def _plain_store(state):
    where, at = _slots(state)
    for name in ("k", "v"):
        x = state[name + "_new"]
        if state[name + "_scale"] is None:
            state[name][where, at] = x
        else:
            codes, exps = _codes(x.float(), state["case"]["store"], state["case"]["dtype"])
            bits = state[name].view(torch.int8)
            bits[where, at] = codes.view(torch.int8)
            state[name + "_scale"].transpose(1, 2)[where, at] = exps


def _plain_load(state):
    where, at = _slots(state)
    dtype, out = DTYPES[state["case"]["dtype"]], []
    for name in ("k", "v"):
        pages, scale = state[name], state[name + "_scale"]
        if scale is None:
            out.append(pages[where, at])
        else:
            codes = pages.view(torch.int8)[where, at].view(pages.dtype)
            out.append(_values(codes, scale.transpose(1, 2)[where, at]).to(dtype))
    return tuple(out)


def _plain_attend(state):
    """Softmax attention of a batch padded to its longest sequence and most new tokens, in 32 bits."""
    case = state["case"]
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

    count = cu[1:] - cu[:-1]
    step = torch.arange(n, device="cuda")
    src = (cu[:-1, None] + step).clamp(max=state["rows"] - 1).long()
    q = state["q"][src].float().reshape(b, n, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * (hq // hkv), dim)
    s = torch.matmul(q, rows("k").transpose(2, 3)).mul_(dim ** -0.5)
    pos = (lens - count)[:, None] + step                      # position of each new token
    last = torch.where(step < count[:, None], pos, -1)
    hidden = torch.arange(wide * page, device="cuda")[None, None] > last[:, :, None]
    s = s.view(b, hkv, n, hq // hkv, wide * page).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    seq, pos = _places(state)
    at = torch.arange(state["rows"], device="cuda") - cu[seq]
    o = torch.matmul(s.view(b, hkv, -1, wide * page), rows("v")).view(b, hkv, n, hq // hkv, dim) / total
    out = o[seq, :, at].reshape(state["rows"], hq, dim).to(DTYPES[case["dtype"]])
    if not case["lse"]:
        return (out,)
    lse = (top + total.log())[..., 0]
    return out, lse[seq, :, at].reshape(state["rows"], hq).t().contiguous()


def _kept(state):
    """What an append leaves in 16-bit pages."""
    return (state["k"], state["v"]) if state["case"]["append"] and state["case"]["store"] == "same" else ()


def run(state):
    case = state["case"]
    if own:
        from baselinebenchmark_b200 import paged_append, paged_attention, paged_load, paged_store
        pages = (state["k"], state["v"], state["table"], state["cu"], state["lens"])
        scales = {"k_scales": state["k_scale"], "v_scales": state["v_scale"]}
        if case["kind"] == "write":
            paged_store(state["k_new"], state["v_new"], *pages, **scales)
        if case["kind"] in ("write", "read"):
            return paged_load(*pages, state["rows"], dtype=DTYPES[case["dtype"]], **scales)
        if case["append"]:
            out = paged_append(state["q"], state["k_new"], state["v_new"], *pages, state["max_new"], return_lse=case["lse"], **scales)
        else:
            out = paged_attention(state["q"], *pages, state["max_new"], return_lse=case["lse"], **scales)
        return (*(out if case["lse"] else (out,)), *_kept(state))
    if case["kind"] == "write":
        _plain_store(state)
    if case["kind"] in ("write", "read"):
        return _plain_load(state)
    if case["append"]:
        _plain_store(state)
    return (*_plain_attend(state), *_kept(state))


def work(case):
    new, total = _lens(case)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    row = dim * (2 if case["store"] == "same" else 1) + (0 if case["store"] == "same" else 1)   # bytes of a stored row
    stored = 2 * hkv * sum(new) * row
    values = 2 * hkv * sum(new) * dim * 2
    if case["kind"] == "write":                                # rows in, codes out, codes in, values out
        return {"bytes": values + 2 * stored + values, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": stored + values, "flops": 0}
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
    move = 2 * hkv * sum(total) * row + 2 * sum(new) * hq * dim * 2 + (sum(new) * hq * 4 if case["lse"] else 0)
    if case["append"]:
        move += values + stored
    return {"bytes": move, "flops": 4 * dim * hq * pairs}


def _exact_codes(x, store, dtype):
    """64 bits: what the rows [..., D] stand for once stored."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / TOP[store])).clamp(-96, 127)
    for d in (1, -1):                                         # log2 is rounded: the neighbours decide
        near = (e + d).clamp(-96, 127)
        e = torch.where((TOP[store] * _two(near) >= amax) & ((near < e) | (TOP[store] * _two(e) < amax)), near, e)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = x.clamp(-MOST[store, dtype], MOST[store, dtype]) / _two(e)
    if store == "int8":
        return y.round() * _two(e)
    # e4m3: steps of an eighth of the power of two below, of 2^-9 under 2^-6
    step = _two(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (y / step).round() * step * _two(e)


def exact(case, seed):
    s = prepare(case, seed)
    new, total = _lens(case)
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    group = hq // hkv

    def sequence(name, i):                                    # rows [tokens, Hkv, D] of a sequence before the call
        used = s["table"][i, :-(-total[i] // page)].long()
        if s[name + "_scale"] is None:
            x = s[name][used].double()
        else:
            codes = s[name].view(torch.int8)[used].view(s[name].dtype).double()
            x = codes * _two(s[name + "_scale"][used].transpose(1, 2).int() - 127)[..., None]
        return x.reshape(-1, hkv, dim)[:total[i]]

    def fresh(name, lo, n):
        x = s[name + "_new"][lo:lo + n].double()
        return x if case["store"] == "same" else _exact_codes(x, case["store"], case["dtype"])

    if case["kind"] == "write":
        return tuple(fresh(name, 0, sum(new)) for name in ("k", "v"))
    if case["kind"] == "read":
        return tuple(torch.cat([sequence(name, i)[total[i] - n:] for i, n in enumerate(new)]) for name in ("k", "v"))
    if 4 * dim * hq * sum(n * t for n, t in zip(new, total)) > 4e13:
        return None
    out, lse, lo = [], [], 0
    kept = [s["k"].double(), s["v"].double()] if case["append"] and case["store"] == "same" else []
    for i, n in enumerate(new):
        k, v = sequence("k", i), sequence("v", i)
        if case["append"] and n:
            k[total[i] - n:], v[total[i] - n:] = fresh("k", lo, n), fresh("v", lo, n)
        for x, y in zip(kept, (k, v)):
            at = torch.arange(total[i] - n, total[i], device="cuda")
            x[s["table"][i, at // page].long(), at % page] = y[at]
        visible = torch.arange(total[i], device="cuda")[None] <= torch.arange(total[i] - n, total[i], device="cuda")[:, None]
        o, m = [], []
        for h in range(hq):
            score = s["q"][lo:lo + n, h].double() @ k[:, h // group].t() / math.sqrt(dim)
            score = torch.where(visible, score, torch.full_like(score, -math.inf))
            z = torch.logsumexp(score, -1)
            o.append(torch.exp(score - z[:, None]) @ v[:, h // group])
            m.append(z)
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(m))
        lo += n
    return (torch.cat(out), *([torch.cat(lse, 1)] if case["lse"] else []), *kept)
