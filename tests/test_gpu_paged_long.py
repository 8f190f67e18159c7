"""GPU: the kernel for many rows over long sequences: every phase of its rings, items cut into pieces and joined, the tiles of an item that
are asked for while the one before it runs."""
import pytest
import torch

from baselinebenchmark_b200 import paged_attention
from tests.paged_util import Batch

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("dim,dtype,store", [(256, torch.bfloat16, None), (256, torch.float16, E4M3), (256, torch.bfloat16, INT8), (96, torch.float16, None),
                                             (96, torch.bfloat16, E4M3), (96, torch.float16, INT8), (64, torch.bfloat16, INT8), (128, torch.float16, E4M3)])
@pytest.mark.parametrize("seqs,hq,hkv", [
    ([(16, 4100)], 4, 1),                                    # one item's rows against pieces of the keys
    ([(3, 2900), (70, 1500), (1, 1), (0, 300)], 8, 2),       # cut and uncut items, one row tile and both
    ([(1200, 1200)], 12, 12),                                # uncut, many items a CTA at most head dims
    ([(300, 1723), (0, 0), (129, 129)], 24, 8)])
def test_many_key_tiles(dim, dtype, store, seqs, hq, hkv):
    b = Batch(seqs, hq, hkv, dim, 64, dtype, store, seed=80 + dim)
    b.fill()
    got, lse = paged_attention(b.q, b.k, b.v, *b.where, 4096, return_lse=True, **b.scales)
    b.check(got, lse)
    assert torch.equal(got, paged_attention(b.q, b.k, b.v, *b.where, 4096, **b.scales))


@pytest.mark.parametrize("store", [None, E4M3])
@pytest.mark.parametrize("dim", [96, 256])
def test_pages_missing_in_long_sequences(dim, store):
    """Whole key tiles without a page, in the first piece, the last one and between, and a sequence that ends inside a page."""
    missing = [(0, i) for i in (0, 1, 2, 3, 9, 30, 31, 32, 33, 62)] + [(1, 2)]
    b = Batch([(20, 4001), (130, 900)], 8, 2, dim, 64, torch.bfloat16, store, seed=90, missing=missing)
    b.fill()
    b.check(*paged_attention(b.q, b.k, b.v, *b.where, 4096, return_lse=True, **b.scales))
