"""GPU: trees of drafted tokens, what lies in front of them: both attention kernels against softmax attention in 64 bits (bounds: Batch.check)."""
import pytest
import torch

from baselinebenchmark_b200 import paged_attention
from tests.tree_util import TreeBatch

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
#: `max_new` for the kernel for few rows and the one for many
KERNELS = [1, 4096]


# Packed rows behind the last position that the table has room for, in part or all of them, by little or by much; the room is no whole number of key tiles.
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dim,dtype,store", [(128, BF16, None), (64, FP16, INT8), (96, BF16, E4M3), (256, FP16, None), (256, BF16, E4M3)])
@pytest.mark.parametrize("spread", [1, 6])
@pytest.mark.parametrize("new", [30, 150])
def test_lengths_beyond_the_table(new, spread, dim, dtype, store, kernel):
    columns, room = 37, 37 * 16                              # 592: the last tile has 80 keys
    seqs = [(new, room + over) for over in (new // 2, new, new + 48, new + 300, new + 3000)] + [(new, 700 - new), (new, new)]
    b = TreeBatch(seqs, 4, 2, dim, 16, dtype, store, seed=21, spread=spread, roots=0.1 if spread > 1 else 0.0)
    b.table, b.table_list = b.table[:, :columns], [row[:columns] for row in b.table_list]
    b.fill()
    want = b.attention()
    call = lambda: paged_attention(b.q, b.k, b.v, *b.where, kernel, parents=b.parents, return_lse=True, **b.scales)  # noqa: E731
    b.check(*call(), want=want)
    b.lens[4] = 2 ** 31 - 1                                  # (its packed rows see the whole table either way)
    b.check(*call(), want=want)


STORES = [(128, BF16, None), (128, BF16, E4M3), (96, FP16, INT8), (64, FP16, None), (256, BF16, None), (256, FP16, E4M3)]
#: one row tile a sequence, and more
BLOCKS = [[(20, 1301), (30, 900), (0, 50)], [(20, 1301), (130, 900)]]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dim,dtype,store", STORES)
@pytest.mark.parametrize("spread", [1, 5])
@pytest.mark.parametrize("seqs", BLOCKS)
def test_pages_missing_in_front(seqs, spread, dim, dtype, store, kernel):
    """Single pages of a key tile, all of one, and the first and last of several, far in front of the packed rows."""
    missing = [(0, i) for i in (2, 8, 9, 10, 11, 12, 13, 14, 15, 23, 24, 40, 61)] + [(1, 0), (1, 20)]
    b = TreeBatch(seqs, 8, 2, dim, 16, dtype, store, seed=22, spread=spread, missing=missing)
    b.fill()
    b.check(*paged_attention(b.q, b.k, b.v, *b.where, kernel, parents=b.parents, return_lse=True, **b.scales))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dim,dtype,store", STORES)
@pytest.mark.parametrize("spread", [1, 5])
@pytest.mark.parametrize("seqs", BLOCKS)
def test_large_scores_and_nan_in_front(seqs, spread, dim, dtype, store, kernel):
    """One row whose scores are millions, of five keys in front, and one that is not a number, beside ordinary rows of the same tokens and heads."""
    b = TreeBatch(seqs, 8, 2, dim, 16, dtype, store, seed=23, spread=spread)
    keys = [200, 203, 210, 255, 300]
    for k, _ in b.hist[:2]:
        k[keys, :, 0] = 1024.0
    large, odd = [(0, 1), (19, 5), (25, 6)], [(3, 2), (28, 4)]   # (packed row, head)
    for row, head in large:
        b.q[row, head] = 0
        b.q[row, head, 0] = 32768.0                          # 2^25 scale log2 e: 3e6 at head dim 256
    for row, head in odd:
        b.q[row, head, 3] = torch.nan
    b.fill()
    clean = b.q.clone()
    b.q[[r for r, _ in odd], [h for _, h in odd], 3] = 0.0
    want = b.attention()
    got, lse = paged_attention(clean, b.k, b.v, *b.where, kernel, parents=b.parents, return_lse=True, **b.scales)
    for row, head in odd:
        assert torch.isnan(got[row, head]).all() and torch.isnan(lse[head, row])
        got[row, head], lse[head, row] = want[0][row, head].to(dtype), want[1][head, row].float()
    u = torch.finfo(dtype).eps / 2
    for row, head in large:
        # five equal weights: a rounding of P, sums and the quotient in 32 bits (6 roundings each and a reciprocal's 2), the output's rounding
        v, x = b.stored(0 if row < 20 else 1, 1)[0][keys, head // 4], got[row, head].double()
        assert ((x - v.mean(0)).abs() <= u * v.mean(0).abs() + (u + 14 * 2.0 ** -24) * v.abs().mean(0)).all()
        assert abs(lse[head, row].item() / want[1][head, row].item() - 1) <= 2.0 ** -20
    b.check(got, lse, want=want)
