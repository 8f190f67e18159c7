"""GPU: the operators around drafted tokens as a server runs them: pages taken, positions turned to, trees attended to, tokens verified, rows kept,
pages given back, step after step."""
import pytest
import torch

from baselinebenchmark_b200 import (PagedKV, PagePool, RotaryTable, paged_attention, rotary, rotary_frequencies, verify_drafts)
from tests.paged_util import quantise, values
from tests.test_gpu_drafts import rule
from tests.tree_util import random_parents

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
V = 50


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """Tokens have fixed rows of q, k and v; what is behind a row depends on its token and depth only."""

    def __init__(self, hq, hkv, dim, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda h: torch.randn(V, h, dim, device="cuda", generator=g).to(dtype)  # noqa: E731
        self.q, self.k, self.v = rand(hq), rand(hkv), rand(hkv)
        self.target = torch.softmax(2 * torch.randn(V, V, device="cuda", generator=g), -1)
        self.draft = torch.softmax(self.target.log() + 0.5 * torch.randn(V, V, device="cuda", generator=g), -1)


def _attention(q, k, v, scale):
    """float64 (out, sum of p |v|, largest sum of |q k|) of rows q [n, Hq, D] that see all of k, v [m, Hkv, D]."""
    group = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(group, 1) for x in (k, v))
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    p = torch.softmax(s, -1)
    size = torch.einsum("nhd,mhd->hnm", q.double().abs(), k.abs()).amax(-1) * scale
    return torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs()), size.t()


@pytest.mark.parametrize("dim,dtype,store,with_draft,spread", [(64, BF16, None, True, 3), (128, FP16, INT8, False, 4), (128, BF16, E4M3, True, 1),
                                                                (256, BF16, None, False, 2), (96, FP16, None, True, 5)])
def test_a_server_that_drafts(dim, dtype, store, with_draft, spread):
    hq, hkv, page, requests, columns = 8, 2, 16, 5, 24
    m = Model(hq, hkv, dim, dtype, seed=1)
    table = RotaryTable(rotary_frequencies(dim // 2), interleaved=True)
    cache, pool = PagedKV(80, page, hkv, dim, dtype, store), PagePool(80, page)
    pages = torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    lens, text, last = _i32([0] * requests), [[] for _ in range(requests)], [0] * requests
    begun = []
    for step in range(14):
        # who comes, who leaves
        news, tokens, parents = [], [], []
        for b in range(requests):
            if step == 3 * b:                                 # a prompt of its own length, without branches; a last token is among its rows
                prompt = torch.randint(V, (20 + 17 * b,), generator=g).tolist()
                news.append(len(prompt))
                tokens += prompt
                parents += range(-1, len(prompt) - 1)
                begun.append(b)
            elif b in begun and not (b == 1 and step == 9):
                n = [1, 6, 9, 14][int(torch.randint(4, (1,), generator=g))]
                p = random_parents([n], spread, 100 * step + b)
                row = [last[b]]
                for i in range(1, n):
                    row.append(int(torch.multinomial(m.draft[row[p[i]]].cpu(), 1, generator=g)))
                news.append(n)
                tokens += row
                parents += p
            else:
                news.append(0)
        ends = [0] + [sum(news[:i + 1]) for i in range(requests)]
        cu, rows, most = _i32(ends), ends[-1], max(news)
        ids, up = torch.tensor(tokens, device="cuda"), _i32(parents)
        now = lens + (cu[1:] - cu[:-1])
        slots, positions, missing = pool.reserve(pages, cu, now, rows, parents=up)
        assert int(missing) == 0 and (slots >= 0).all()
        q, k = rotary(m.q[ids], m.k[ids], positions, table)
        out = cache.append(q, k, m.v[ids], pages, cu, now, most, parents=up)
        # ---- every row is attention over its branch
        drafting = [n if b in begun and step != 3 * b else 0 for b, n in enumerate(news)]
        u = torch.finfo(dtype).eps / 2
        for b in range(requests):
            for i in range(news[b]):
                branch, at = [], i
                while at >= 0:
                    branch.insert(0, at)
                    at = parents[ends[b] + at]
                assert int(positions[ends[b] + i]) == len(text[b]) + len(branch) - 1
                if i % 5 and i != news[b] - 1:
                    continue
                history = torch.tensor(text[b] + [tokens[ends[b] + r] for r in branch], device="cuda")
                kk = rotary(m.k[history], None, torch.arange(len(history), device="cuda").int(), table)[0]
                vv = m.v[history]
                if store:
                    kk, vv = (values(*quantise(x, store)) for x in (kk, vv))
                want, mass, size = _attention(q[ends[b] + i:ends[b] + i + 1], kk, vv, dim ** -0.5)
                e = 2 * ((dim + 8) * 2.0 ** -24 * size + 1e-4 + len(history) * 2.0 ** -24)
                assert ((out[ends[b] + i].double() - want[0]).abs() <= mass[0] * (u + e[0][:, None]) + u * want[0].abs() + 1e-7).all()
        # ---- verification: a prompt is a chain whose rows all stand
        accept, sample = torch.rand(rows, generator=g), torch.rand(requests, generator=g)
        for b in range(requests):
            if news[b] and not drafting[b]:
                accept[ends[b]:ends[b + 1]] = -1.0
        target, draft = m.target[ids], m.draft[ids] if with_draft else None
        path, count, following = verify_drafts(target, draft, ids, cu, accept.cuda(), sample.cuda(), most, parents=up)
        want = rule(target.cpu(), None if draft is None else draft.cpu(), tokens, news, accept.double().tolist(), sample.double().tolist(), most, parents)
        assert [path.tolist(), count.tolist(), following.tolist()] == list(want)
        lens = cache.keep(pages, cu, now, path, count)
        for b in range(requests):
            if news[b]:
                text[b] += [tokens[ends[b] + r] for r in want[0][b] if r >= 0]
                last[b] = want[2][b]
        if step == 8:                                         # a request is over
            text[1], begun = [], [b for b in begun if b != 1]
            lens[1] = 0
        pool.release(pages, lens)
        assert lens.tolist() == [len(t) for t in text]
        used = sum(-(-len(t) // page) for t in text)
        assert int(pool.free_count) == 80 - used and int((pages >= 0).sum()) == used
        owned = pages[pages >= 0].tolist() + pool.free_pages[:int(pool.free_count)].tolist()
        assert sorted(owned) == list(range(80))               # no page lost, none twice
        # ---- the cache holds the accepted texts, turned to their positions
        total = sum(len(t) for t in text)
        whole = _i32([0] + [sum(len(t) for t in text[:i + 1]) for i in range(requests)])
        ids = torch.tensor([x for t in text for x in t], device="cuda", dtype=torch.long)
        pos = torch.tensor([i for t in text for i in range(len(t))], device="cuda").int()
        kk = rotary(m.k[ids], None, pos, table)[0]
        got = cache.load(pages, whole, lens, total)
        for x, y in zip(got, (kk, m.v[ids])):
            assert torch.equal(x, y if store is None else values(*quantise(y, store)).to(dtype))
    assert max(len(t) for t in text) > 60


def test_a_captured_step():
    """Reserve, turn, append, verify and keep as one graph, replayed with other tokens and trees; each replay is what the eager calls give."""
    hq, hkv, dim, page, rows = 8, 2, 64, 16, 12
    m, table = Model(hq, hkv, dim, BF16, 3), RotaryTable(rotary_frequencies(dim))
    cu = _i32([0, 5, 12])

    def fresh():
        cache, pool = PagedKV(12, page, hkv, dim), PagePool(12, page)
        return cache, pool, torch.full((2, 5), -1, dtype=torch.int32, device="cuda"), _i32([5, 7])

    ids, up = torch.zeros(rows, dtype=torch.int64, device="cuda"), _i32([-1] * rows)
    accept, sample = torch.zeros(rows, device="cuda"), torch.zeros(2, device="cuda")

    def step(cache, pool, pages, now):
        slots, positions, missing = pool.reserve(pages, cu, now, rows, parents=up)
        q, k = rotary(m.q[ids], m.k[ids], positions, table)
        out = cache.append(q, k, m.v[ids], pages, cu, now, 7, parents=up)
        path, count, after = verify_drafts(m.target[ids], m.draft[ids], ids, cu, accept, sample, 7, parents=up)
        lens = cache.keep(pages, cu, now, path, count)
        now.copy_(lens + (cu[1:] - cu[:-1]))
        pool.release(pages, lens)
        return slots, positions, missing, out, path, count, after, lens

    held = fresh()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*fresh())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(*held)
    torch.cuda.current_stream().wait_stream(stream)
    again = fresh()
    g = torch.Generator().manual_seed(4)
    for i in range(6):
        ids.copy_(torch.randint(V, (rows,), generator=g))
        up.copy_(torch.tensor(random_parents([5, 7], 3, i), dtype=torch.int32))
        accept.copy_(torch.rand(rows, generator=g))
        sample.copy_(torch.rand(2, generator=g))
        graph.replay()
        want = step(*again)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(held[0].k, again[0].k) and torch.equal(held[2], again[2]) and torch.equal(held[1].free_pages, again[1].free_pages)
        assert torch.equal(held[3], again[3])


def test_trees_beside_other_rows_of_a_batch():
    """A prompt's block, a decode step and a tree in one call give what each gives alone."""
    m, page = Model(8, 2, 128, BF16, 5), 32
    cache = PagedKV(40, page, 2, 128)
    g = torch.Generator(device="cuda").manual_seed(7)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    news, lens = [40, 1, 13], [300, 77, 500]
    table = torch.full((3, 17), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b, i], at = at, at + 1
    table, ends = table.cuda(), [0, 40, 41, 54]
    parents = list(range(-1, 39)) + [-1] + random_parents([13], 4, 6)
    q = torch.randn(54, 8, 128, device="cuda", generator=g).to(BF16)
    largest = cache.v.float().abs().max().item()
    whole, lse = paged_attention(q, cache.k, cache.v, table, _i32(ends), _i32(lens), 40, parents=_i32(parents), return_lse=True)
    for b in range(3):
        rows = slice(ends[b], ends[b + 1])
        up = _i32(parents[rows]) if b == 2 else None
        alone, one = paged_attention(q[rows], cache.k, cache.v, table[b:b + 1], _i32([0, news[b]]), _i32(lens[b:b + 1]), news[b], parents=up, return_lse=True)
        # each is off by half a step of P times sum p |v| (the largest |v| at most), half a step of the output, and twice the exponentials' 1e-4 and the
        # scores' (128 + 8) 2^-24 sum |q k|, which 100 bounds here (128 products of normal values times 128^-0.5)
        off = 2.0 ** -8 * (largest + alone.double().abs()) + 2 * (1e-4 + 136 * 2.0 ** -24 * 100) * largest
        assert ((whole[rows].double() - alone.double()).abs() <= 2 * off).all()
        assert (lse[:, rows] - one).abs().max() <= 2 * (1e-4 + 136 * 2.0 ** -24 * 100 + 500 * 2.0 ** -24 + 2.0 ** -20)
