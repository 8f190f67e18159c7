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
