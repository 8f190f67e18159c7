"""GPU: the paged cache against plain implementations in 64 bits."""
import math

import pytest
import torch

from baselinebenchmark_b200 import PagedKV, paged_append, paged_attention, paged_load, paged_store
from tests.paged_util import Batch, quantise, values

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
#: `max_new` decides between the kernel for few rows and the one for many, whatever the batch holds
FEW, MANY = 1, 4096
#: (new, length): a fresh sequence, one without new tokens, an empty one, one token, page borders from both sides
RAGGED = [(5, 5), (0, 40), (0, 0), (1, 1), (1, 17), (16, 64), (3, 65), (33, 100), (1, 128), (2, 129)]


def _same(x, y):
    """Equal bit for bit, NaN like NaN."""
    return x.dtype == y.dtype and x.shape == y.shape and torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(7), y.nan_to_num(7))


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("dim,dtype,store", [(64, torch.float16, E4M3), (96, torch.bfloat16, INT8), (128, torch.bfloat16, E4M3),
                                             (128, torch.float16, None), (256, torch.float16, INT8), (96, torch.bfloat16, None),
                                             (256, torch.bfloat16, E4M3)])
def test_rows_written_and_read_back(dim, dtype, store, layout):
    """The pages hold exactly the codes of the rule, the rows come back as what the codes stand for, nothing else is touched."""
    b = Batch(RAGGED, 4, 3 if dim != 128 else 8, dim, 16, dtype, store, seed=dim, layout=layout, missing=((5, 3), (7, 5)))
    b.hq = b.hkv
    ref = Batch(RAGGED, 4, b.hkv, dim, 16, dtype, store, seed=dim, layout=layout, missing=((5, 3), (7, 5)))
    ref.fill()
    old = Batch(RAGGED, 4, b.hkv, dim, 16, dtype, store, seed=dim, layout=layout, missing=((5, 3), (7, 5)))
    old.fill(new=False)
    paged_store(b.k_new, b.v_new, b.k, b.v, *b.where, **b.scales)
    for got, want, before in ((b.k, ref.k, old.k), (b.v, ref.v, old.v)):
        # what the call wrote is in `ref` and not in `old`; everywhere else b is as it was made (NaN)
        bits = lambda x: x.view(torch.int8 if store else torch.int16)  # noqa: E731
        fresh = (bits(want) != bits(before)).any(-1)
        assert torch.equal(bits(got)[fresh], bits(want)[fresh])
        assert torch.equal(bits(got)[~fresh], bits(Batch(RAGGED, 4, b.hkv, dim, 16, dtype, store, seed=dim, layout=layout,
                                                         missing=((5, 3), (7, 5))).k)[~fresh])
    if store:
        for got, want, before in ((b.ks, ref.ks, old.ks), (b.vs, ref.vs, old.vs)):
            assert torch.equal(got[want != before], want[want != before]) and (got[want == before] == 255).all()
    k, v = paged_load(b.k, b.v, *b.where, b.rows, dtype=dtype, **b.scales)
    for got, new in ((k, b.k_new), (v, b.v_new)):
        want = values(*quantise(new, store)).to(dtype) if store else new.clone()
        for i, (n, length) in enumerate(RAGGED):
            for j in range(n):
                if b.page_of(i, length - n + j) < 0:
                    want[b.cu_list[i] + j] = 0
        assert _same(got, want)


@pytest.mark.parametrize("store", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_of_unusual_rows(store, dtype):
    """Zeros, the type's largest and smallest values, borders of the power of two, halves between codes, infinities and NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [torch.zeros(64), torch.full((64,), big), torch.full((64,), -big), torch.full((64,), tiny), torch.full((64,), tiny / 2 ** 5),
            torch.linspace(-448, 448, 64), torch.linspace(-127, 127, 64), torch.arange(64) / 2 - 16, (torch.arange(64) / 2 - 16) * 2.0 ** -9,
            torch.cat([torch.tensor([math.inf]), torch.ones(63)]), torch.cat([torch.ones(63), torch.tensor([-math.inf])]),
            torch.cat([torch.ones(31), torch.tensor([math.nan]), torch.ones(32)])]
    for top in (127.0, 127.5, 128.0, 448.0, 450.0, 254.0, 255.0, 256.0, 1.75, 1.7578125, 1.984375, 1.9921875):
        rows.append(torch.cat([torch.tensor([top]), torch.linspace(-1, 1, 63) * top]))
    x = torch.stack(rows).to(dtype).cuda()[:, None]
    cache = PagedKV(3, 16, 1, 64, dtype, store)
    n = x.shape[0]
    where = (torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"),
             torch.tensor([n], dtype=torch.int32, device="cuda"))
    cache.store(x, -x, *where)
    k, v = cache.load(*where, n)
    for got, rows in ((k, x), (v, -x)):
        codes, byte = quantise(rows, store)
        assert _same(got, values(codes, byte).to(dtype))
    finite = torch.isfinite(x).all(-1)[:, 0]
    assert torch.isfinite(k[finite]).all() and torch.isnan(k[~finite]).all()


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (6, 2), (16, 1), (40, 1)])
@pytest.mark.parametrize("dim,page,dtype,store", [
    (64, 16, torch.float16, None), (64, 64, torch.bfloat16, E4M3), (64, 128, torch.float16, INT8),
    (96, 32, torch.bfloat16, None), (96, 16, torch.float16, E4M3), (96, 16, torch.bfloat16, INT8),
    (128, 64, torch.bfloat16, None), (128, 16, torch.bfloat16, E4M3), (128, 32, torch.float16, INT8), (128, 256, torch.float16, E4M3),
    (256, 16, torch.bfloat16, None), (256, 64, torch.float16, E4M3), (256, 32, torch.bfloat16, INT8)])
def test_attention_of_a_ragged_batch(dim, page, dtype, store, hq, hkv, kernel):
    b = Batch(RAGGED, hq, hkv, dim, page, dtype, store, seed=dim + hq, layout="heads" if hq % 3 else "tokens")
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    b.check(got, lse)
    again = paged_attention(b.q, b.k, b.v, *b.where, kernel, **b.scales)
    assert torch.equal(got, again)


@pytest.mark.parametrize("store", [None, E4M3, INT8])
@pytest.mark.parametrize("seqs", [[(1, n)] for n in (1, 2, 15, 16, 17, 127, 128, 129, 1000, 4097)] +
                         [[(1, 3000), (1, 1), (1, 700), (2, 2), (1, 5000)], [(7, 2500), (1, 9)], [(200, 200)], [(150, 1300), (1, 77)]])
@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_attention_over_lengths(seqs, store, kernel):
    b = Batch(seqs, 8, 2, 128, 16, torch.bfloat16, store, seed=len(seqs) + seqs[0][1])
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    b.check(got, lse)


@pytest.mark.parametrize("store", [None, E4M3])
@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_rows_that_see_nothing(store, new, kernel):
    """Positions below zero, pages that are not there (all of a sequence's, its first, one in the middle), a table too short."""
    seqs = [(new, new - 2), (new, 0), (new, -4), (new, 300), (new, 300), (new, 300), (1, 40)]
    missing = [(3, i) for i in range(19)] + [(4, 0)] + [(5, 7)]
    b = Batch(seqs, 4, 2, 64, 16, torch.float16, store, seed=new, missing=missing)
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    b.check(got, lse)
    empty = torch.isinf(lse).t()
    assert empty[:2].all() == (new > 2) and empty[new:3 * new].all() and (got[empty] == 0).all()
    assert empty[3 * new:4 * new].all()


@pytest.mark.parametrize("store", [None, INT8])
@pytest.mark.parametrize("new", [1, 40])
def test_append_and_rows_behind_the_batch(store, new):
    """A padded batch: rows behind the last sequence keep what `out` held, and nothing of them is written to the pages."""
    seqs = [(new, 90), (new, new), (0, 30), (new, 257)]
    b, ref = (Batch(seqs, 8, 4, 128, 32, torch.bfloat16, store, seed=3) for _ in range(2))
    b.fill(new=False)
    ref.fill()
    pad = lambda x: torch.cat([x, torch.full((5, *x.shape[1:]), math.nan, dtype=x.dtype, device="cuda")])  # noqa: E731
    out = torch.full((b.rows + 5, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    got, lse = paged_append(pad(b.q), pad(b.k_new), pad(b.v_new), b.k, b.v, *b.where, new, return_lse=True, out=out, **b.scales)
    assert got is out and (out[b.rows:] == 3.0).all()
    b.check(out[:b.rows], lse[:, :b.rows])
    bits = torch.int8 if store else torch.int16
    assert torch.equal(b.k.view(bits), ref.k.view(bits)) and torch.equal(b.v.view(bits), ref.v.view(bits))
    k, _ = paged_load(b.k, b.v, *b.where, b.rows + 5, dtype=torch.bfloat16, out=(out[:, :4], torch.empty_like(out[:, 4:])), **b.scales)
    assert (out[b.rows:] == 3.0).all() and torch.equal(k[:b.rows], paged_load(ref.k, ref.v, *b.where, b.rows, **ref.scales)[0])


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("store", [None, E4M3])
def test_pages_of_two_layouts(store, kernel):
    """K head by head, V token by token within a page; pages longer than a key tile; one page, one kv head."""
    k, v = (Batch(RAGGED, 8, 2, 128, 16, torch.bfloat16, store, seed=8, layout=x) for x in ("heads", "tokens"))
    k.fill()
    v.fill()
    k.check(*paged_attention(k.q, k.k, v.v, *k.where, kernel, return_lse=True, **k.scales))
    long = Batch([(40, 700), (1, 1500), (3, 3)], 8, 1, 64, 1024, torch.float16, store, seed=9)
    long.fill()
    long.check(*paged_attention(long.q, long.k, long.v, *long.where, kernel, return_lse=True, **long.scales))
    one = Batch([(2, 60)], 4, 1, 96, 64, torch.float16, store, seed=10, spare=0)
    one.fill()
    one.check(*paged_attention(one.q, one.k, one.v, *one.where, kernel, return_lse=True, **one.scales))


def test_strides_and_scale():
    """q, k and v side by side as a fused projection leaves them, an output inside a wider tensor, a table inside a wider one, a factor."""
    b = Batch(RAGGED, 8, 2, 128, 16, seed=9)
    b.fill()
    qkv = torch.cat([b.q, b.k_new, b.v_new], 1)
    wide = torch.zeros(b.rows, 11, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.full((len(RAGGED), b.table.shape[1] + 9), 10 ** 6, dtype=torch.int32, device="cuda")
    table[:, 2:2 + b.table.shape[1]] = b.table
    b.k.fill_(0)
    got = paged_append(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], b.k, b.v, table[:, 2:2 + b.table.shape[1]], b.cu, b.lens, b.max_new,
                       scale=0.2, out=wide[:, 2:10])
    assert (wide[:, :2] == 0).all() and (wide[:, 10:] == 0).all()
    c = Batch(RAGGED, 8, 2, 128, 16, seed=9)
    c.fill(new=False)
    c.k.fill_(0)
    paged_store(c.k_new, c.v_new, c.k, c.v, *c.where)
    assert torch.equal(b.k.view(torch.int16), c.k.view(torch.int16))
    # keys before the new tokens are zeros now
    for i, (n, length) in enumerate(RAGGED):
        b.hist[i][0][:max(length - n, 0)] = 0
    b.check(got, want=b.attention(0.2))


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("store", [None, E4M3])
def test_numbers_that_are_none(store, kernel):
    """A NaN in a token's query reaches its own row only; a key or value row with one reaches the rows that see it, and not the
    sequences that do not."""
    seqs = [(2, 200), (1, 77), (1, 40)]
    b = Batch(seqs, 4, 2, 64, 16, torch.bfloat16, store, seed=1)
    clean = Batch(seqs, 4, 2, 64, 16, torch.bfloat16, store, seed=1)
    clean.fill()
    want = paged_attention(clean.q, clean.k, clean.v, *clean.where, kernel, **clean.scales)
    b.q[2, 1, 5] = math.nan
    b.hist[0][0][30, 0, 3] = math.inf
    b.hist[2][1][7, 1] = math.nan
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    bad = torch.isnan(got).any(-1)
    # an infinite key scores +inf or -inf, as the query's element there has it: the first makes NaN (inf - inf), the second a weight
    # of 0.  Quantised, the key is NaN and so is every score of it.
    hit = b.q[:2, :2, 3] > 0 if store is None else torch.ones(2, 2, dtype=torch.bool, device="cuda")
    assert torch.equal(bad[:2, :2], hit) and not bad[:2, 2:].any()
    assert bad[2].tolist() == [False, True, False, False] and bad[3].tolist() == [False, False, True, True]
    bad[:2, :2] = True
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("store,scale", [(None, 1e3), (E4M3, 1e3), (E4M3, 1e-3), (INT8, 1e-3), (INT8, 3e4), (E4M3, 2.0 ** 60), (INT8, 2.0 ** -60)])
@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_large_and_small_values(store, scale, kernel):
    """Rows of any size, scores that run from one key to a single one: weights stay in range whatever the powers of two are."""
    b = Batch([(1, 500), (4, 900), (40, 300)], 4, 2, 128, 16, torch.bfloat16, store, seed=4, scale=scale, q_scale=1.0 / scale)
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    b.check(got, lse)


@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_v_rows_of_very_different_sizes(kernel):
    """Powers of two of V rows that differ by 2^20: the weights follow their product with the probabilities."""
    b = Batch([(1, 400), (3, 777)], 4, 2, 128, 16, torch.float16, E4M3, seed=5)
    for k, v in b.hist:
        v[::3] *= 2.0 ** -12
        v[1::3] *= 2.0 ** 8
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    b.check(got, lse)


@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_many_sequences(kernel):
    """More sequences than one launch adds up, most of them without new tokens."""
    seqs = [(1, 3 + i % 40) if i % 3 == 0 else (0, i % 7) for i in range(2500)]
    b = Batch(seqs, 2, 1, 64, 16, torch.float16, seed=6)
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True)
    b.check(got, lse)
    k, v = paged_load(b.k, b.v, *b.where, b.rows)
    assert torch.equal(k, b.k_new) and torch.equal(v, b.v_new)
