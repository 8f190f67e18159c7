"""GPU: the paged cache as a program uses it: requests that come, grow and share pages, beside the MoBA operator, under
captured graphs, on several streams, in a pool beyond 32-bit offsets."""
import math

import pytest
import torch

from baselinebenchmark_b200 import PagedKV, paged_append, paged_attention, paged_load, paged_store, parallel_moba
from baselinebenchmark_b200.incremental import IncrementalMoba
from tests.paged_util import Batch, quantise, values

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,store,dim", [(torch.bfloat16, None, 128), (torch.float16, INT8, 64), (torch.bfloat16, E4M3, 256)])
def test_a_server_run(dtype, store, dim):
    """Four requests: prompts in blocks, then decode steps of whoever is there, one of them with drafted tokens.  Every step's rows are those
    of softmax attention over the whole history, in 64 bits."""
    hq, hkv, page = 8, 2, 16
    ends = [70, 33, 150, 5]
    whole = Batch([(n, n) for n in ends], hq, hkv, dim, page, dtype, store, seed=11)
    want = whole.attention()
    u, e = torch.finfo(dtype).eps / 2, 2 * (1e-4 + (dim + 8) * 2.0 ** -24 * want[3] + 150 * 2.0 ** -24)
    tol = want[2] * (u + e.t()[..., None]) + u * want[0].abs() + 1e-30
    cache = PagedKV(40, page, hkv, dim, dtype, store)
    free, table = list(range(39, -1, -1)), torch.full((4, 12), -1, dtype=torch.int32)
    at = [0, 0, 0, 0]
    # new tokens of each request in each step
    steps = [[40, 0, 100, 0], [27, 30, 47, 0], [1, 1, 1, 1], [1, 0, 1, 1], [1, 2, 1, 2], [0, 0, 0, 1]]
    assert [sum(s[i] for s in steps) for i in range(4)] == ends
    for new in steps:
        for i, n in enumerate(new):
            for p in range(-(-at[i] // page), -(-(at[i] + n) // page)):
                table[i, p] = free.pop()
            at[i] += n
        rows = torch.cat([torch.arange(whole.cu_list[i] + at[i] - n, whole.cu_list[i] + at[i]) for i, n in enumerate(new)]).cuda()
        cu = _i32([0] + [sum(new[:i + 1]) for i in range(4)])
        out, lse = cache.append(whole.q[rows], whole.k_new[rows], whole.v_new[rows], table.cuda(), cu, _i32(at), max(new), return_lse=True)
        assert ((out.double() - want[0][rows]).abs() <= tol[rows]).all()
        assert ((lse.double() - want[1][:, rows]).abs() <= e[:, rows] + 2.0 ** -22 * want[1][:, rows].abs()).all()
    # and the whole of it read back is what was written
    k, v = cache.load(table.cuda(), whole.cu, whole.lens, sum(ends))
    for got, new in ((k, whole.k_new), (v, whole.v_new)):
        assert torch.equal(got, values(*quantise(new, store)).to(dtype) if store else new)


def test_moba_over_rows_read_back():
    """16-bit pages give MoBA the rows that were written: a prefill of the batch, and the continuation of one request, are bit for bit what
    they are without the cache."""
    lens, hq, hkv, dim, chunk, topk = [700, 1300, 255], 8, 2, 128, 128, 3
    b = Batch([(n, n) for n in lens], hq, hkv, dim, 64, seed=12)
    paged_store(b.k_new, b.v_new, b.k, b.v, *b.where)
    k, v = paged_load(b.k, b.v, *b.where, b.rows)
    with torch.inference_mode():
        assert torch.equal(parallel_moba(b.q, k, v, b.cu, max(lens), chunk, topk), parallel_moba(b.q, b.k_new, b.v_new, b.cu, max(lens), chunk, topk))
    grown = IncrementalMoba(2000, hkv, dim, chunk, topk)
    first = slice(b.cu_list[1], b.cu_list[2])
    whole = grown.append(b.q[first], b.k_new[first], b.v_new[first])
    one = (b.table[1:2], _i32([0, 1300]), b.lens[1:2])
    k, v = paged_load(b.k, b.v, *one, 1300)
    again = IncrementalMoba(2000, hkv, dim, chunk, topk)
    again.append(b.q[first][:900], k[:900], v[:900])
    assert torch.equal(again.append(b.q[first][900:], k[900:], v[900:]), whole[900:])
    # one chunk for the whole sequence: MoBA is causal attention, and the two operators agree
    with torch.inference_mode():
        dense = parallel_moba(b.q, b.k_new, b.v_new, b.cu, max(lens), 2048, 1)
    b.fill()
    b.check(dense)
    b.check(paged_attention(b.q, b.k, b.v, *b.where, max(lens)))


@pytest.mark.parametrize("new,store", [(1, None), (1, E4M3), (60, None), (60, INT8)])
def test_captured_calls_follow_their_tensors(new, store):
    """Two graphs, replayed in turn with other tokens, lengths and pages in the same tensors."""
    shape = dict(hq=8, hkv=2, dim=128, page=32, dtype=torch.bfloat16, store=store)
    first = [[(new, 300), (new, 90), (0, 20)], [(new, 64), (new, 700), (0, 0)]]
    later = [[(new, 100), (0, 31), (new, 500)], [(0, 0), (new, 333), (new, 61)]]
    pools, graphs = [], []
    make = lambda seqs, seed: Batch(seqs, **shape, seed=seed, spare=80 - sum(-(-n // 32) for _, n in seqs))  # noqa: E731  (80 pages)
    for i, seqs in enumerate(first):
        b = make(seqs, 20 + i)
        b.fill(new=False)
        table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
        table[:, :b.table.shape[1]] = b.table
        out, lse = torch.zeros_like(b.q), None
        args = [b.q, b.k_new, b.v_new, b.k, b.v, table, b.cu, b.lens]
        call = lambda a=args, o=out, s=b.scales: paged_append(*a, new, out=o, return_lse=True, **s)  # noqa: E731
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                _, lse = call()
        torch.cuda.current_stream().wait_stream(stream)
        pools.append((b, args, out, lse))
        graphs.append(graph)
    for seqs_of in (first, later):
        now = []
        for i, (b, args, out, lse) in enumerate(pools):
            c = make(seqs_of[i], 20 + i if seqs_of is first else 30 + i)
            if seqs_of is later:                              # other rows, in other pages of the same pool
                c.fill(new=False)
                bits = lambda x: x.view(torch.int8) if store else x  # noqa: E731
                for x, y in ((b.k, c.k), (b.v, c.v)):
                    bits(x).copy_(bits(y))
                if store:
                    b.ks.copy_(c.ks)
                    b.vs.copy_(c.vs)
                for x, y in zip(args[:3], (c.q, c.k_new, c.v_new)):
                    x.copy_(y)
                args[5].fill_(-1)
                args[5][:, :c.table.shape[1] - 1] = c.table[:, :-1]
                args[6].copy_(c.cu)
                args[7].copy_(c.lens)
            now.append(c)
        for graph in (*graphs, *graphs):
            graph.replay()
        torch.cuda.synchronize()
        for c, (b, args, out, lse) in zip(now, pools):
            c.check(out, lse)


@pytest.mark.parametrize("store", [None, E4M3])
def test_calls_on_two_streams(store):
    """Calls that overlap on the GPU share nothing: each has its own scratch memory."""
    batches = [Batch(seqs, 8, 2, 128, 16, torch.bfloat16, store, seed=40 + i)
               for i, seqs in enumerate(([(1, 5000), (1, 900)], [(300, 4000)], [(1, 2000)] * 3, [(90, 90), (7, 3000)]))]
    for b in batches:
        b.fill()
    want = [paged_attention(b.q, b.k, b.v, *b.where, b.max_new, **b.scales) for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], []
    for _ in range(20):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                got.append(paged_attention(b.q, b.k, b.v, *b.where, b.max_new, **b.scales))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % len(batches)])


@pytest.mark.parametrize("store", [None, INT8])
def test_pool_beyond_32_bits(store):
    """Pages whose elements lie behind 2^32 bytes and 2^31 elements of their pool."""
    page, hkv, dim, dtype = 64, 8, 128, torch.bfloat16
    pages = 2 ** 31 // (page * hkv * dim) + 60
    small = Batch([(1, 400), (50, 700), (3, 3)], 16, hkv, dim, page, dtype, store, seed=50)
    big = PagedKV.__new__(PagedKV)
    make = lambda: torch.empty(pages, hkv, page, dim, dtype=torch.int8 if store else dtype, device="cuda")  # noqa: E731
    big.dtype, big.k, big.v, big.k_scales, big.v_scales = dtype, make().transpose(1, 2), make().transpose(1, 2), None, None
    if store:
        big.k_scales, big.v_scales = (torch.empty(pages, hkv, page, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.where((small.table >= 0) & (small.table < small.pages), pages - 1 - small.table, small.table)
    table[:, -1] = -1
    for lo in range(0, 700, 700):                             # the whole history, as rows of one call
        cu = _i32([0, 400, 1100, 1103])
        k, v = (torch.cat([h[i] for h in small.hist]).cuda() for i in range(2))
        big.store(k, v, table, cu, small.lens)
    got_k, got_v = big.load(table, cu, small.lens, 1103)
    assert torch.equal(got_k, values(*quantise(k, store)).to(dtype) if store else k)
    assert torch.equal(got_v, values(*quantise(v, store)).to(dtype) if store else v)
    for kernel in (1, 4096):
        out, lse = big.attend(small.q, table, small.cu, small.lens, kernel, return_lse=True)
        small.check(out, lse)


@pytest.mark.parametrize("kernel", [1, 4096])
def test_pages_shared_by_requests(kernel):
    """Two requests with one prefix, whose pages are in both tables."""
    b = Batch([(2, 100), (2, 100), (1, 64)], 4, 2, 64, 16, torch.float16, seed=60)
    b.hist[1][0][:64], b.hist[1][1][:64] = b.hist[0][0][:64], b.hist[0][1][:64]
    b.table[1, :4] = b.table[0, :4]
    b.table_list = b.table.tolist()
    b.fill()
    b.check(*paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True))


def test_nothing_to_do():
    cache = PagedKV(4, 16, 2, 64)
    where = (torch.zeros(2, 1, dtype=torch.int32, device="cuda"), _i32([0, 0, 0]), _i32([3, 0]))
    rows = lambda h: torch.empty(0, h, 64, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    cache.store(rows(2), rows(2), *where)
    assert [x.shape for x in cache.load(*where, 0)] == [(0, 2, 64)] * 2
    out, lse = cache.append(rows(4), rows(2), rows(2), *where, 1, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    # rows, and no sequence that has them
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 5)
    for kernel in (1, 4096):
        cache.attend(q, *where, kernel, out=out)
    cache.store(q[:, :2], q[:, 2:], *where)
    assert (out == 5).all() and (cache.k == 0).all() and (cache.v == 0).all()


def test_what_is_refused():
    cache = PagedKV(4, 16, 2, 64)
    where = (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _i32([0, 2]), _i32([2]))
    k, q = (torch.ones(2, h, 64, dtype=torch.bfloat16, device="cuda") for h in (2, 4))
    with pytest.raises(NotImplementedError, match="backward"):
        cache.attend(q.clone().requires_grad_(), *where, 1)
    with pytest.raises(NotImplementedError, match="backward"):
        cache.store(k.clone().requires_grad_(), k, *where)
    with torch.no_grad():
        cache.store(k.clone().requires_grad_(), k, *where)
    with pytest.raises(ValueError, match="divisible"):
        cache.attend(torch.ones(2, 3, 64, dtype=torch.bfloat16, device="cuda"), *where, 1)
    with pytest.raises(TypeError, match="dtype"):
        cache.attend(q.half(), *where, 1)
    with pytest.raises(ValueError, match="device"):
        cache.store(k.cpu(), k, *where)
    with pytest.raises(TypeError, match="seq_lens"):
        cache.load(where[0], where[1], where[2].cpu(), 2)
    with pytest.raises(ValueError, match="scales"):
        paged_load(cache.k, cache.v, *where, 2, k_scales=torch.zeros(4, 2, 16, dtype=torch.uint8, device="cuda"))
    with torch.inference_mode():
        frozen = PagedKV(4, 16, 2, 64)
        frozen.store(k, k, *where)
    with pytest.raises(RuntimeError, match="inference"):
        frozen.store(k, k, *where)
    assert frozen.attend(q, *where, 1).shape == q.shape
    # what autograd saved of the pages is stale after a write
    x = torch.ones(1, device="cuda", requires_grad=True)
    y = (cache.k * x).sum()
    cache.store(k, k, *where)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    assert not math.isnan(float(cache.k.float().sum()))
