"""GPU: pages taken and given back, slots, positions, and rows of accepted branches moved together; whole numbers and copies, all exact."""
import pytest
import torch

from baselinebenchmark_b200 import PagedKV, PagePool, paged_keep, paged_release, paged_reserve, paged_store
from tests.paged_util import Batch
from tests.tree_util import branch, random_parents

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _ends(news):
    return [0] + [sum(news[:i + 1]) for i in range(len(news))]


def reserve_rule(table, news, lens, free, count, page, rows, parents=None):
    """Lists in, lists out: the table, the count, slots, positions, entries without a page.  `free` stays as it is."""
    pages, per = len(free), len(table[0])
    table, missing, slots, positions = [list(r) for r in table], 0, [-1] * rows, [-1] * rows
    is_page = lambda x: 0 <= x < pages  # noqa: E731
    left = max(min(count, pages), 0)
    for b, (n, length) in enumerate(zip(news, lens)):
        for i in range(max(length - n, 0) // page, -(-min(max(length, 0), per * page) // page)) if n > 0 else ():
            if not is_page(table[b][i]):
                if left:
                    left -= 1
                    table[b][i] = free[left]
                else:
                    missing += 1
    lo = 0
    for b, (n, length) in enumerate(zip(news, lens)):
        for i in range(n):
            pos = length - n + i
            if 0 <= pos < per * page and is_page(table[b][pos // page]):
                slots[lo + i] = table[b][pos // page] * page + pos % page
            depth = i if parents is None else len(branch(parents[lo:lo + n], i)) - 1
            positions[lo + i] = length - n + depth
        lo += n
    return table, left, slots, positions, missing


def release_rule(table, keep, free, count, page):
    pages = len(free)
    table, free = [list(r) for r in table], list(free)
    back = []
    for b, n in enumerate(keep):
        for i in range(-(-max(n, 0) // page), len(table[b])):
            if 0 <= table[b][i] < pages:
                back.append(table[b][i])
                table[b][i] = -1
    count = max(min(count, pages), 0)
    for r, x in enumerate(back):
        if count + len(back) - 1 - r < pages:
            free[count + len(back) - 1 - r] = x
    return table, free, min(count + len(back), pages)


def _start(lens, page, per, pages, seed=0, holes=()):
    """A table in which sequences of `lens` tokens have their pages, shuffled, and the stack of the others."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = [[(-1, pages, -9, 2 ** 31 - 1)[(b + i) % 4] for i in range(per)] for b in range(len(lens))]
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b][i] = order.pop()
    for b, i in holes:
        table[b][i] = -1
    free = order + [-1] * (pages - len(order))
    return table, free, len(order)


CASES = [
    # (new tokens, tokens before, page, columns, pages)
    ([1], [0], 16, 1, 1),
    ([1], [16], 16, 2, 40),
    ([1, 1, 0, 1, 5], [15, 16, 8, 0, 60], 16, 8, 40),
    ([40, 1, 200, 3], [7, 64, 0, 31], 32, 12, 60),
    ([64] * 9, [100 + i for i in range(9)], 64, 5, 64),
    ([3000, 1, 0, 700], [5, 1000, 3, 0], 16, 260, 400),                        # many rows: several launches
    ([1] * 1500, [i % 70 for i in range(1500)], 16, 6, 6000),
    ([2, 3] * 1200, [i % 40 for i in range(2400)], 16, 4, 9000),
    ([200000], [77], 16, 12600, 12700),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("tree", [False, True])
def test_reserve_and_back(case, tree):
    news, before, page, per, pages = CASES[case]
    if tree and sum(news) > 50000:
        news = [5000, 1200]
        before = [77, 3]
    lens = [n + b for n, b in zip(news, before)]
    table, free, count = _start(before, page, per, pages, seed=case)
    rows = sum(news) + 3
    parents = random_parents(news, 6 if case < 5 else 2, case, 0.05) if tree else None
    if tree and case == 5:
        parents[:3000] = range(-1, 2999)                     # as deep as it is long
    want = reserve_rule(table, news, lens, free, count, page, rows, parents)
    t, f, c = _i32(table), _i32(free), _i32([count])
    slots, positions, missing = paged_reserve(t, _i32(_ends(news)), _i32(lens), f, c, page, rows,
                                              parents=_i32(parents + [0] * 3) if tree else None)
    assert t.tolist() == want[0] and c.tolist() == [want[1]] and f.tolist() == free
    assert slots.dtype == torch.int64 and slots.tolist() == want[2] and positions.tolist() == want[3] and missing.tolist() == [want[4]]
    # again: nothing lacks
    again = paged_reserve(t, _i32(_ends(news)), _i32(lens), f, c, page, rows)
    assert t.tolist() == want[0] and c.tolist() == [want[1]] and again[0].tolist() == want[2]
    # what was taken goes back to where it was
    paged_release(t, _i32(before), f, c, page)
    kept = [[x if i < -(-n // page) else -1 if 0 <= y < pages else y for i, (x, y) in enumerate(zip(r, w))] for r, w, n in zip(table, want[0], before)]
    assert t.tolist() == kept and f.tolist() == free and c.tolist() == [count]


@pytest.mark.parametrize("many", [False, True])
def test_a_pool_that_runs_out(many):
    news = [30, 1, 50, 2, 40] + ([500] * 5 if many else [])
    before = [2, 16, 0, 31, 9] + ([0] * 5 if many else [])
    lens, page, per = [n + b for n, b in zip(news, before)], 16, 40
    table, free, count = _start(before, page, per, 30, seed=1)
    for have in (3, 0, -4, 10 ** 6):
        want = reserve_rule(table, news, lens, free, have, page, sum(news))
        t, f, c = _i32(table), _i32(free), _i32([have])
        slots, positions, missing = paged_reserve(t, _i32(_ends(news)), _i32(lens), f, c, page, sum(news))
        assert t.tolist() == want[0] and c.tolist() == [want[1]] and missing.tolist() == [want[4]]
        assert slots.tolist() == want[2] and positions.tolist() == want[3]


def test_lengths_that_make_no_sense():
    """Positions below 0 and behind the table, holes in what a sequence has, rows in front of the first sequence."""
    page, per = 16, 4
    table, free, count = _start([10, 40, 0], page, per, 20, seed=2, holes=[(1, 0), (1, 2)])
    news, lens = [12, 50, 3], [5, 90, -2]
    want = reserve_rule(table, news, lens, free, count, page, 65)
    t, c = _i32(table), _i32([count])
    slots, positions, missing = paged_reserve(t, _i32(_ends(news)), _i32(lens), _i32(free), c, page, 65)
    assert t.tolist() == want[0] and slots.tolist() == want[2] and positions.tolist() == want[3] and missing.tolist() == [want[4]]
    slots, positions, _ = paged_reserve(t, _i32([2, 4, 4, 5]), _i32([12, 50, 3]), _i32(free), c, page, 8)
    assert [x >= 0 for x in slots.tolist()] == [False, False, True, True, True, False, False, False]
    assert positions.tolist() == [-1, -1, 10, 11, 2, -1, -1, -1]


@pytest.mark.parametrize("batch,per", [(1, 1), (3, 5), (64, 64), (70, 3000), (9000, 7)])
def test_release(batch, per):
    page, pages = 16, max(batch * per // 2, 4)
    g = torch.Generator().manual_seed(batch)
    fill = torch.rand(batch, per, generator=g)
    order = torch.randperm(pages, generator=g).tolist()
    table = [[order.pop() if f < 0.3 and order else (-1, pages, -3)[i % 3] for i, f in enumerate(r)] for r in fill.tolist()]
    free = list(reversed(order)) + [-7] * (pages - len(order))
    keep = [(-5, 0, 1, 16, 17, 40, 10 ** 6)[b % 7] for b in range(batch)]
    want = release_rule(table, keep, free, len(order), page)
    t, f, c = _i32(table), _i32(free), _i32([len(order)])
    paged_release(t, _i32(keep), f, c, page)
    assert t.tolist() == want[0] and f.tolist() == want[1] and c.tolist() == [want[2]]


def test_a_captured_step_takes_and_gives_back():
    """One graph for many steps: requests grow, are cut and leave."""
    page, per, pages = 16, 20, 30
    table, free, count = _start([0, 0, 0], page, per, pages)
    t, f, c = _i32(table), _i32(free), _i32([count])
    cu, lens, keep = _i32([0, 3, 6, 9]), _i32([3, 3, 3]), _i32([0, 0, 0])
    call = lambda: (paged_reserve(t, cu, lens, f, c, page, 9), paged_release(t, keep, f, c, page))[0]  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            slots, positions, missing = call()
    torch.cuda.current_stream().wait_stream(stream)
    for now, kept in (([30, 3, 9], [30, 0, 8]), ([33, 3, 11], [17, 3, 11]), ([20, 6, 14], [0, 6, 0])):
        before = t.tolist(), f.tolist(), int(c)
        want = reserve_rule(before[0], [3, 3, 3], now, before[1], before[2], page, 9)
        after = release_rule(want[0], kept, before[1], want[1], page)
        lens.copy_(_i32(now))
        keep.copy_(_i32(kept))
        graph.replay()
        assert (t.tolist(), f.tolist(), int(c)) == (after[0], after[1], after[2])
        assert slots.tolist() == want[2] and positions.tolist() == want[3] and int(missing) == want[4]


def test_no_rows():
    """Nothing to place, or no sequence with a row: pages stay where they are."""
    table, free, count = _start([20, 3], 16, 4, 9)
    for rows, cu in ((0, [0, 0, 0]), (3, [0, 0, 0]), (0, [0, 2, 2])):
        t, c = _i32(table), _i32([count])
        slots, positions, missing = paged_reserve(t, _i32(cu), _i32([20, 3]), _i32(free), c, 16, rows)
        assert t.tolist() == table and c.tolist() == [count] and missing.tolist() == [0]
        assert slots.tolist() == [-1] * rows and positions.tolist() == [-1] * rows


def test_pool_refusals():
    table, free, count, cu, lens = _i32([[-1] * 4] * 2), _i32([0, 1, 2]), _i32([3]), _i32([0, 1, 2]), _i32([1, 1])
    reserve = lambda **kw: paged_reserve(*{**dict(table=table, cu=cu, lens=lens, free=free, count=count, size=16, rows=2), **kw}.values())  # noqa: E731
    for error, kw in ((ValueError, dict(table=table[0])), (TypeError, dict(table=table.long())), (NotImplementedError, dict(table=_i32([[-1] * 2] * 4).t())),
                      (ValueError, dict(table=table[:1].expand(2, 4))), (ValueError, dict(cu=cu[:2])), (TypeError, dict(cu=cu.long())),
                      (ValueError, dict(lens=lens[:1])), (TypeError, dict(lens=lens.cpu())), (ValueError, dict(free=free[:0])), (TypeError, dict(free=free.long())),
                      (ValueError, dict(count=_i32([3, 3]))), (NotImplementedError, dict(size=24)), (ValueError, dict(size=0)), (ValueError, dict(rows=-1))):
        with pytest.raises(error):
            reserve(**kw)
    with pytest.raises(ValueError, match="parents"):
        paged_reserve(table, cu, lens, free, count, 16, 2, parents=_i32([0]))
    with pytest.raises(RuntimeError, match="error -2"):                   # more sequences than a call takes
        paged_release(_i32([[-1]]).repeat(16385, 1), _i32([0]).repeat(16385), free, count, 16)
    with pytest.raises(ValueError, match="keep_lens"):
        paged_release(table, lens[:1], free, count, 16)
    assert table.tolist() == [[-1] * 4] * 2 and count.tolist() == [3]
    with torch.inference_mode():
        made = _i32([[-1] * 4] * 2)
    with pytest.raises(RuntimeError, match="inference"):
        paged_release(made, lens, free, count, 16)


def test_many_sequences():
    news, before = [1] * 16384, [(7 * i) % 50 for i in range(16384)]
    lens = [n + b for n, b in zip(news, before)]
    table, free, count = _start(before, 16, 4, 70000, seed=3)
    want = reserve_rule(table, news, lens, free, count, 16, 16384)
    t, c = _i32(table), _i32([count])
    slots, positions, missing = paged_reserve(t, _i32(list(range(16385))), _i32(lens), _i32(free), c, 16, 16384)
    assert t.tolist() == want[0] and c.tolist() == [want[1]] and slots.tolist() == want[2] and positions.tolist() == want[3]


def test_pool_of_a_cache():
    pool = PagePool(7, 32)
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    slots, positions, missing = pool.reserve(table, _i32([0, 40, 41]), _i32([40, 1]), 41)
    assert table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and pool.free_count.tolist() == [4] and missing.tolist() == [0]
    assert slots.tolist() == list(range(40)) + [64] and positions.tolist() == list(range(40)) + [0]
    pool.release(table, _i32([20, 0]))
    assert table.tolist() == [[0, -1, -1, -1], [-1] * 4] and pool.free_count.tolist() == [6]
    with pytest.raises(ValueError, match="num_pages"):
        PagePool(0, 16)
    with pytest.raises(NotImplementedError, match="page_size"):
        PagePool(3, 24)


# ---- rows moved together

BF16, FP16, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8


def _kept(b, paths):
    """Pools and lengths after the paths' rows have moved, by the definition."""
    k, v = (x.view(torch.int8).clone() if b.store != b.dtype else x.clone() for x in (b.k, b.v))
    ks, vs = (None if x is None else x.clone() for x in (b.ks, b.vs))
    lens = []
    for i, ((n, length), path) in enumerate(zip(b.seqs, paths)):
        good = 0
        while good < min(len(path), n) and path[good] < n and path[good] > (path[good - 1] if good else -1):
            good += 1
        lens.append(length - n + good)
        place = lambda r: (b.page_of(i, length - n + r), (length - n + r) % b.page)  # noqa: E731
        for j, r in enumerate(path[:good]):
            (p0, s0), (p1, s1) = place(r), place(j)
            if p0 < 0 or p1 < 0:
                continue
            for x in (k, v):
                x[p1, s1] = x[p0, s0]
            for x in (ks, vs):
                if x is not None:
                    x[p1, :, s1] = x[p0, :, s0]
    return k, v, ks, vs, lens


@pytest.mark.parametrize("hkv,dim,page,dtype,store", [(1, 64, 16, BF16, None), (3, 96, 16, FP16, None), (4, 128, 32, BF16, E4M3),
                                                      (2, 256, 64, FP16, INT8), (8, 128, 16, BF16, None), (2, 96, 16, BF16, INT8)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_keep(hkv, dim, page, dtype, store, layout):
    seqs = [(7, 50), (1, 1), (0, 9), (40, 40), (64, 300), (5, 3), (9, 9), (6, 20)]
    paths = [[0, 2, 3, 6], [0], [], [0, 1, 2, 3, 4, 5, 6, 7, 9, 12, 13, 15, 20, 33, 39], [0] + list(range(20, 64, 2)), [0, 2, 4], [3, 5, 8], [0, 4, 4, 5]]
    b = Batch(seqs, hkv, hkv, dim, page, dtype, store, seed=1, layout=layout, missing=[(3, 1)])
    paged_store(b.k_new, b.v_new, b.k, b.v, *b.where, **b.scales)
    want = _kept(b, paths)
    path = torch.full((8, 70), 77, dtype=torch.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    got = paged_keep(b.k, b.v, *b.where, path.cuda()[:, :64], _i32([len(p) for p in paths]), **b.scales)
    bits = lambda x: x.view(torch.int16) if store is None else x.view(torch.int8)  # noqa: E731
    assert got.tolist() == want[4] and b.lens.tolist() == [n for _, n in seqs]
    assert torch.equal(bits(b.k), bits(want[0])) and torch.equal(bits(b.v), bits(want[1]))
    assert store is None or (torch.equal(b.ks, want[2]) and torch.equal(b.vs, want[3]))


def test_keep_of_counts_that_make_no_sense():
    b = Batch([(4, 20), (4, 20), (4, 20)], 2, 2, 64, 16, seed=2)
    b.fill()
    path = _i32([[0, 2, 3], [0, 2, 3], [-1, 2, 3]])
    want = _kept(b, [[0, 2, 3], [], []])
    assert paged_keep(b.k, b.v, *b.where, path, _i32([99, -3, 2])).tolist() == want[4] == [19, 16, 16]
    assert torch.equal(b.k.view(torch.int16), want[0].view(torch.int16))


def test_keep_refusals():
    cache = PagedKV(4, 16, 2, 64)
    where = (_i32([[0]]), _i32([0, 2]), _i32([2]))
    with pytest.raises(ValueError, match="path"):
        cache.keep(*where, _i32([0, 1]), _i32([2]))
    with pytest.raises(TypeError, match="path"):
        cache.keep(*where, torch.zeros(1, 2, device="cuda"), _i32([2]))
    with pytest.raises(ValueError, match="count"):
        cache.keep(*where, _i32([[0, 1]]), _i32([2, 2]))
    with torch.inference_mode():
        assert cache.keep(*where, _i32([[0, 1]]), _i32([2])).tolist() == [2]
