"""CPU: arguments of the paged cache's operators at the ends of their ranges.  No kernel is launched."""
import ctypes as C

import pytest
import torch

from baselinebenchmark_b200 import _lib, build, paged
from tests.test_paged_abi import _dev, _paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def test_factor_of_the_scores_is_a_number_of_32_bits(lib):
    """A factor that becomes 0 in 32 bits would stand for head_dim^-0.5, and one whose product with log2(e) is infinite for NaN rows."""
    pages, q = _dev(torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)), _dev(torch.zeros(7, 4, 64, dtype=torch.bfloat16))
    for scale in (1e-46, 7e-46, 2.5e38, 3.0e38, 1e300, float("inf"), -1e-46):
        with pytest.raises(ValueError, match="scale"):
            paged._check_attention(q, pages, 3, scale, None)
    for scale in (2e-45, 1e-38, 0.3, 2.2e38):
        paged._check_attention(q, pages, 3, scale, None)
    check = lambda x: lib.moba_paged_check(C.byref(_paged(softmax_scale=x)))  # noqa: E731
    assert [check(x) for x in (2.5e38, 3.0e38, 3.3e38)] == [-1] * 3
    assert [check(x) for x in (0.0, 2e-45, 2.2e38)] == [0] * 3


def test_tensors_that_autograd_follows_are_refused():
    """Pages, too, and tangents of forward mode (a dual tensor does not require grad)."""
    x, y = torch.zeros(3), torch.zeros(3, requires_grad=True)
    with pytest.raises(NotImplementedError, match="v_pages.*backward"):
        paged._check_not_followed(k_pages=x, v_pages=y)
    with torch.no_grad():
        paged._check_not_followed(k_pages=x, v_pages=y)
    paged._check_not_followed(k_pages=x, v_pages=x, out=None)
    with torch.autograd.forward_ad.dual_level():
        paged._check_not_followed(k_pages=x)
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(NotImplementedError, match="q has a tangent"):
            paged._check_not_followed(q=dual, k_pages=x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
            paged._check_not_followed(q=dual)


def test_sizes_beyond_32_bits():
    """`max_new` is a hint: any positive number is one.  Sizes that the structure has no room for are refused with a word of it."""
    g = paged._Pages.__new__(paged._Pages)
    g.shape, g.batch, g.per_seq, g.store, g.strides = (11, 16, 2, 64), 3, 9, 0, (8,) * 7
    field = lambda n: _lib.Paged.from_buffer_copy(g.pack(21, 4, n, torch.float16, 0.0)).max_new  # noqa: E731
    assert [field(n) for n in (1, 2 ** 31 - 1, 2 ** 31, 2 ** 70)] == [1] + [2 ** 31 - 1] * 3
    for name, x in (("shape", (2 ** 31, 16, 2, 64)), ("per_seq", 2 ** 31), ("batch", 2 ** 32)):
        kept = getattr(g, name)
        setattr(g, name, x)
        with pytest.raises(NotImplementedError, match="32 bits"):
            g.pack(21, 4, 1, torch.float16, 0.0)
        setattr(g, name, kept)


def test_scratch_follows_the_call(lib):
    """No more results of pieces than a call's row tiles, heads and table can come to: a few rows of one request do not take what a prompt does."""
    def size(**kw):
        need = C.c_size_t(0)
        assert lib.moba_paged_workspace_size(C.byref(_paged(**kw)), C.byref(need)) == 0
        return need.value
    one = dict(batch=1, num_kv_heads=1, num_q_heads=8, max_new=16)
    plan = size(total_tokens=16, pages_per_seq=8, **one)     # 512 keys are one piece: nothing to join
    assert plan < 1 << 16
    slot = 256 * (128 + 2) * 4                               # head dim 128: 256 rows of output, maximum and sum
    assert size(total_tokens=16, pages_per_seq=9, table_stride=9, **one) == plan + 2 * slot
    assert size(total_tokens=16, pages_per_seq=640, table_stride=640, **one) == plan + 80 * slot
    many = size(total_tokens=65536, pages_per_seq=2048, table_stride=2048, batch=3, max_new=30000)
    assert many == plan + 8 * 148 * slot
    assert size(total_tokens=2 ** 27, num_q_heads=8, batch=2000, max_new=2 ** 17, pages_per_seq=2 ** 14, table_stride=2 ** 14) == many
