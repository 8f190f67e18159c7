"""GPU: paged attention of trees of drafted tokens against softmax attention in 64 bits (bounds: Batch.check)."""
import pytest
import torch

from baselinebenchmark_b200 import PagedKV, paged_append, paged_attention
from tests.tree_util import TreeBatch

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8


def _attend(b, **kw):
    return paged_attention(b.q, b.k, b.v, *b.where, b.max_new, parents=b.parents, return_lse=True, **b.scales, **kw)


# (sequences (new, length), hq, hkv, dim, page, dtype, store): both kernels, row tiles that are half empty, trees that begin and end inside a page and a tile
CASES = [
    ([(1, 1)], 2, 2, 64, 16, BF16, None),
    ([(2, 2), (1, 40), (0, 30), (2, 19)], 4, 1, 128, 16, FP16, None),
    ([(8, 100), (5, 5), (7, 260)], 2, 2, 128, 32, BF16, None),
    ([(5, 77), (8, 300), (3, 3)], 2, 2, 96, 16, FP16, None),
    ([(8, 40), (6, 515)], 2, 1, 256, 64, BF16, None),
    ([(12, 150), (9, 31), (1, 64)], 4, 1, 128, 16, BF16, E4M3),
    ([(24, 220), (17, 17)], 2, 1, 64, 32, FP16, INT8),
    ([(16, 90), (3, 700)], 4, 2, 256, 16, BF16, INT8),
    ([(15, 100), (2, 129)], 3, 1, 96, 64, BF16, E4M3),
    # many rows: tcgen05
    ([(17, 300), (33, 33), (64, 129), (0, 5), (9, 9)], 8, 2, 128, 16, BF16, None),
    ([(63, 64), (40, 1000)], 16, 4, 64, 32, FP16, None),
    ([(130, 257), (20, 20)], 6, 3, 96, 64, BF16, None),
    ([(70, 400), (12, 12)], 4, 2, 256, 128, FP16, None),
    ([(64, 640), (31, 31), (1, 1)], 8, 2, 128, 64, BF16, E4M3),
    ([(100, 140)], 4, 2, 64, 16, FP16, INT8),
    ([(60, 333), (77, 77)], 8, 8, 256, 32, BF16, E4M3),
    ([(45, 45), (61, 1200)], 12, 4, 96, 16, FP16, INT8),
    ([(300, 777), (513, 513)], 4, 2, 128, 64, BF16, None),
]


@pytest.mark.parametrize("seqs,hq,hkv,dim,page,dtype,store", CASES)
@pytest.mark.parametrize("spread", [1, 5])
def test_branches(seqs, hq, hkv, dim, page, dtype, store, spread):
    b = TreeBatch(seqs, hq, hkv, dim, page, dtype, store, seed=7, spread=spread, roots=0.1 if spread > 1 else 0.0)
    b.fill()
    b.check(*_attend(b))


@pytest.mark.parametrize("new,store", [(2, None), (40, None), (10, E4M3), (40, INT8)])
def test_a_chain_is_causal_attention(new, store):
    """Parents that are the rows before give the bits of the call without them."""
    b = TreeBatch([(new, 200), (new, new), (1, 77)], 4, 1, 128, 16, store=store, spread=1, seed=3)
    b.fill()
    got, lse = _attend(b)
    want, want_lse = paged_attention(b.q, b.k, b.v, *b.where, b.max_new, return_lse=True, **b.scales)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("new,store", [(3, None), (24, None), (11, E4M3), (50, E4M3)])
def test_parents_that_are_none(new, store):
    """A row's own number, later rows and numbers far off stand for no parent; rows that follow nothing see the tokens in front and themselves."""
    odd = [0, 5000, -7, 2 ** 31 - 1, -2 ** 31, 1]
    parents = [odd[i % 6] if i % 2 else i for i in range(new)] * 2
    b = TreeBatch([(new, 90), (new, new)], 2, 1, 128, 16, store=store, parents=parents, seed=5)
    b.fill()
    b.check(*_attend(b))


@pytest.mark.parametrize("new,store", [(4, None), (40, None), (9, INT8), (50, INT8)])
def test_rows_that_see_nothing(new, store):
    """Missing pages, rows below position 0 and sequences without a token: zeros and -inf."""
    b = TreeBatch([(new, 2), (new, 0), (new, new), (new, 130)], 2, 1, 64, 16, store=store, seed=9, missing=[(2, 0), (3, 1), (3, 8)])
    b.fill()
    got, lse = _attend(b)
    b.check(got, lse)
    assert torch.isinf(lse).any() and (got[torch.isinf(lse).t()] == 0).all()


@pytest.mark.parametrize("store", [None, E4M3])
@pytest.mark.parametrize("new,told", [(30, 1), (3, 500), (60, 20)])
def test_the_most_rows_are_a_hint(new, told, store):
    b = TreeBatch([(new, 400), (1, 50)], 4, 1, 128, 32, store=store, seed=2)
    b.fill()
    b.check(*paged_attention(b.q, b.k, b.v, *b.where, told, parents=b.parents, return_lse=True, **b.scales))


@pytest.mark.parametrize("new,dim,store", [(6, 128, None), (30, 128, E4M3), (64, 64, None), (64, 256, INT8)])
def test_append_and_strides(new, dim, store):
    """Rows of a fused projection written and attended to, pages token by token, output into a wider tensor; rows behind the last sequence stay."""
    seqs = [(new, 100), (0, 7), (new, new)]
    b = TreeBatch(seqs, 4, 2, dim, 16, store=store, seed=4, layout="tokens")
    b.fill(new=False)
    rows = b.rows + 3
    qkv = torch.full((rows, 8, dim), 5.0, dtype=b.dtype, device="cuda")
    qkv[:b.rows, :4], qkv[:b.rows, 4:6], qkv[:b.rows, 6:] = b.q, b.k_new, b.v_new
    wide = torch.full((rows, 6, dim), 9.0, dtype=b.dtype, device="cuda")
    parents = torch.cat([b.parents, torch.zeros(3, dtype=torch.int32, device="cuda")])
    out, lse = paged_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], b.k, b.v, *b.where, new, parents=parents, return_lse=True, out=wide[:, 1:5],
                            **b.scales)
    b.check(out[:b.rows], lse[:, :b.rows])
    assert (wide[b.rows:] == 9).all() and (wide[:, 0] == 9).all() and (wide[:, 5] == 9).all()


@pytest.mark.parametrize("new,store", [(2, None), (40, None), (12, E4M3), (60, E4M3)])
def test_a_captured_call_follows_its_parents(new, store):
    b = TreeBatch([(new, 150), (new, 40 + new)], 4, 1, 128, 16, store=store, seed=6)
    b.fill()
    out = torch.zeros_like(b.q)
    call = lambda: paged_attention(b.q, b.k, b.v, *b.where, new, parents=b.parents, return_lse=True, out=out, **b.scales)  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, lse = call()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (1, 2):
        other = TreeBatch(b.seqs, 4, 1, 128, 16, store=store, seed=6)
        other.parent_list = TreeBatch(b.seqs, 4, 1, 128, 16, seed=seed, spread=7).parent_list
        b.parents.copy_(torch.tensor(other.parent_list, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        other.check(out, lse)


def test_many_sequences_and_two_streams():
    """More sequences than a launch takes, two calls side by side."""
    batches = [TreeBatch([(3, 20 + i % 50) for i in range(1100)], 2, 1, 64, 16, seed=s, store=st) for s, st in ((1, None), (2, E4M3))]
    batches += [TreeBatch([(20, 20 + i % 50) for i in range(60)], 8, 1, 64, 16, seed=3)]
    streams, got = [torch.cuda.Stream() for _ in batches], []
    for b in batches:
        b.fill()
    for b, s in zip(batches, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_attend(b))
    torch.cuda.synchronize()
    for b, (out, lse) in zip(batches, got):
        b.check(out, lse)


def test_a_long_tree():
    """Rows whose branches go back through several key tiles, to the first row and beyond it."""
    for store in (None, E4M3):
        b = TreeBatch([(1000, 1100), (700, 700)], 2, 1, 128, 64, store=store, seed=8, spread=40)
        b.fill()
        b.check(*_attend(b))


def test_parents_are_checked():
    cache = PagedKV(4, 16, 2, 64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    where, q = (i32([[0]]), i32([0, 2]), i32([2])), torch.ones(2, 4, 64, dtype=BF16, device="cuda")
    for parents, error in ((i32([0]), ValueError), (i32([[0, 0]]), ValueError), (torch.zeros(2, device="cuda"), TypeError),
                           (torch.zeros(2, dtype=torch.int32), TypeError), (i32([0, 0, 0, 0])[::2], NotImplementedError)):
        with pytest.raises(error, match="parents"):
            cache.attend(q, *where, 2, parents=parents)
    assert cache.attend(q, *where, 2, parents=i32([-1, 0])).shape == q.shape
    assert cache.attend(q[:0], *where, 2, parents=i32([])).shape == (0, 4, 64)


# The same calls in both kernels: a table with room for many pages, of which the batch has a few, puts trees of 9 to 64 rows on tcgen05.
@pytest.mark.parametrize("new,g,dim", [(3, 4, 64), (12, 4, 128), (16, 4, 256), (64, 1, 96), (9, 1, 128), (17, 3, 64)])
@pytest.mark.parametrize("wide", [False, True])
def test_both_kernels(new, g, dim, wide):
    b = TreeBatch([(new, 300), (new, new), (0, 40), (1, 130), (new, 1500)], 2 * g, 2, dim, 16, seed=10, spread=3)
    b.fill()
    table = torch.full((5, 200000), -1, dtype=torch.int32, device="cuda") if wide else b.table
    table[:, :b.table.shape[1]] = b.table
    b.check(*paged_attention(b.q, b.k, b.v, table, b.cu, b.lens, new, parents=b.parents, return_lse=True))


def test_even_and_uneven_batches_of_one_row_tile():
    """Items on a line of units: one key tile, many, more items than CTAs, fewer; sequences without rows between them."""
    for seqs in ([(40, 40)], [(33, 5000)], [(40, 200 + 37 * i) if i % 3 else (0, 50) for i in range(70)], [(64, 64)] * 90, [(50, 3000), (64, 100)] * 3):
        b = TreeBatch(seqs, 8, 2, 64, 64, seed=13, spread=6)
        b.fill()
        table = torch.full((len(seqs), 8000), -1, dtype=torch.int32, device="cuda")
        table[:, :b.table.shape[1]] = b.table
        b.check(*paged_attention(b.q, b.k, b.v, table, b.cu, b.lens, 64, parents=b.parents, return_lse=True))


@pytest.mark.parametrize("store", [None, E4M3])
@pytest.mark.parametrize("dim", [128, 256])
def test_prompts_beside_trees(dim, store):
    """Blocks without branches, one that has a single branch late, trees and decode steps in one call; and a prompt alone, with parents and without."""
    seqs = [(700, 900), (1, 300), (530, 530), (40, 100), (0, 9), (300, 800)]
    b = TreeBatch(seqs, 4, 2, dim, 32, store=store, seed=14, spread=5)
    ends, parents = b.cu_list, b.parent_list
    for i in (0, 2, 5):
        parents[ends[i]:ends[i + 1]] = range(-1, seqs[i][0] - 1)
    parents[ends[2] + 511] = 400
    b.parents.copy_(torch.tensor(parents, dtype=torch.int32))
    b.fill()
    b.check(*_attend(b))
    one = TreeBatch([(700, 900)], 4, 2, dim, 32, store=store, seed=14, spread=1)
    one.fill()
    got, lse = _attend(one)
    want, want_lse = paged_attention(one.q, one.k, one.v, *one.where, 700, return_lse=True, **one.scales)
    # (pieces of an item may be cut elsewhere: sums of other parts)
    one.check(got, lse)
    one.check(want, want_lse)
