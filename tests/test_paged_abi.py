"""CPU: argument checks of the paged cache, in the C ABI and in Python.  No kernel is launched."""
import ctypes as C

import pytest
import torch

import baselinebenchmark_b200 as moba
from baselinebenchmark_b200 import _lib, build, paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _paged(**kw):
    base = dict(total_tokens=10, batch=3, num_q_heads=8, num_kv_heads=2, head_dim=128, num_pages=50, page_size=64, pages_per_seq=9,
                max_new=4, dtype=0, store=0, q_stride_token=1024, q_stride_head=128, o_stride_token=1024, o_stride_head=128,
                k_stride_token=256, k_stride_head=128, v_stride_token=256, v_stride_head=128, k_page_stride=64 * 256,
                k_page_token=128, k_page_head=64 * 128, v_page_stride=64 * 256, v_page_token=128, v_page_head=64 * 128, table_stride=9)
    base.update(kw)
    return _lib.Paged(**base)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(store=1)), (0, dict(store=2, dtype=1)), (0, dict(head_dim=64)), (0, dict(batch=1, table_stride=0)),
    (0, dict(q_stride_token=0)), (0, dict(page_size=16, pages_per_seq=1, table_stride=1)), (0, dict(softmax_scale=0.3)),
    (-1, dict(total_tokens=0)), (-1, dict(batch=0)), (-1, dict(num_q_heads=7)), (-1, dict(max_new=0)), (-1, dict(num_pages=0)),
    (-1, dict(pages_per_seq=0)), (-1, dict(table_stride=8)), (-1, dict(softmax_scale=-1.0)), (-1, dict(softmax_scale=float("nan"))),
    (-1, dict(softmax_scale=float("inf"))), (-1, dict(k_page_token=0)), (-1, dict(q_stride_token=-8)),
    (-2, dict(head_dim=80)), (-2, dict(page_size=8)), (-2, dict(page_size=48)), (-2, dict(dtype=2)), (-2, dict(store=3)),
    (-2, dict(reserved=1)), (-2, dict(num_q_heads=258)), (-2, dict(total_tokens=2 ** 28)), (-2, dict(pages_per_seq=2 ** 24, table_stride=2 ** 24)),
    (-6, dict(q_stride_head=132)), (-6, dict(v_page_token=132)), (-6, dict(store=1, k_page_token=136))])
def test_check_codes(lib, code, kw):
    assert lib.moba_paged_check(C.byref(_paged(**kw))) == code


def test_pointers_are_checked_before_any_launch(lib):
    ok, off = 0x10000, 0x10008
    p, q = C.byref(_paged()), C.byref(_paged(store=1))
    need = C.c_size_t(0)
    assert lib.moba_paged_check(None) == -4 and lib.moba_paged_workspace_size(p, None) == -4
    assert lib.moba_paged_workspace_size(p, C.byref(need)) == 0 and need.value > 0
    store = lambda *a: lib.moba_paged_store(*a, None)  # noqa: E731
    load = lambda p, cu, lens, table, kp, vp, ks, vs, k, v: lib.moba_paged_load(p, cu, lens, table, kp, vp, ks, vs, k, v, None)  # noqa: E731
    attend = lambda p, q, cu, out=ok, lse=None, ws=ok, size=need.value, ks=None: lib.moba_paged_attention(  # noqa: E731
        p, q, cu, ok, ok, ok, ok, ks, ks, out, lse, ws, size, None)
    assert store(p, None, ok, ok, ok, ok, ok, ok, None, None) == -4
    assert store(p, ok, ok, ok, ok, None, ok, ok, None, None) == -4
    assert store(q, ok, ok, ok, ok, ok, ok, ok, None, ok) == -4                       # 8-bit pages have scales
    assert store(p, off, ok, ok, ok, ok, ok, ok, None, None) == -6
    assert store(p, ok, ok, ok, ok, ok, off, ok, None, None) == -6
    assert store(q, ok, ok, ok, ok, ok, ok, ok, ok, off) == -6
    assert store(p, ok, ok, 0x10002, ok, ok, ok, ok, None, None) == -6
    assert load(p, ok, ok, ok, ok, ok, None, None, ok, None) == -4
    assert load(p, ok, ok, ok, ok, ok, None, None, ok, off) == -6
    assert attend(p, None, ok) == -4 and attend(p, ok, None) == -4 and attend(q, ok, ok) == -4
    assert attend(p, off, ok) == -6 and attend(p, ok, ok, out=off) == -6 and attend(p, ok, ok, lse=0x10002) == -6
    assert attend(p, ok, ok, ws=None) == -3 and attend(p, ok, ok, size=need.value - 1) == -3
    assert attend(p, ok, ok, ws=0x10010) == -6
    assert attend(C.byref(_paged(o_stride_token=0)), ok, ok) == -1 and attend(C.byref(_paged(o_stride_head=0)), ok, ok) == -1
    assert load(C.byref(_paged(v_stride_token=0)), ok, ok, ok, ok, ok, None, None, ok, ok) == -1     # rows on one another


def _tensors(**kw):
    """A call's tensors on the CPU: everything that is looked at before the device is."""
    t = dict(k_pages=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16), v_pages=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16),
             page_table=torch.zeros(2, 3, dtype=torch.int32), cu_seqlens=torch.zeros(3, dtype=torch.int32),
             seq_lens=torch.zeros(2, dtype=torch.int32), k_scales=None, v_scales=None)
    t.update(kw)
    return t


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "accelerator", {}),
    (ValueError, "shape", dict(k_pages=torch.zeros(5, 16, 64))),
    (ValueError, "identical shapes", dict(v_pages=torch.zeros(5, 16, 1, 64, dtype=torch.bfloat16))),
    (TypeError, "same dtype", dict(v_pages=torch.zeros(5, 16, 2, 64, dtype=torch.float16))),
    (TypeError, "pages hold", dict(k_pages=torch.zeros(5, 16, 2, 64), v_pages=torch.zeros(5, 16, 2, 64))),
])
def test_pages_are_checked(error, match, kw):
    with pytest.raises(error, match=match):
        paged._check_pages(**_tensors(**kw))


class _OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a device: the checks behind the device's."""

    @property
    def device(self):
        return torch.device("cuda", 0)


def _dev(x):
    return x.as_subclass(_OnDevice)


@pytest.mark.parametrize("error,match,kw", [
    (NotImplementedError, "page_size", dict(k_pages=(5, 48, 2, 64), v_pages=(5, 48, 2, 64))),
    (NotImplementedError, "page_size", dict(k_pages=(5, 8, 2, 64), v_pages=(5, 8, 2, 64))),
    (NotImplementedError, "head_dim", dict(k_pages=(5, 16, 2, 80), v_pages=(5, 16, 2, 80))),
    (ValueError, "non-zero", dict(k_pages=(0, 16, 2, 64), v_pages=(0, 16, 2, 64))),
    (ValueError, "no scales", dict(k_scales=torch.zeros(5, 2, 16, dtype=torch.uint8))),
    (ValueError, "cu_seqlens", dict(cu_seqlens=torch.zeros(1, dtype=torch.int32))),
    (ValueError, "page_table", dict(page_table=torch.zeros(3, 3, dtype=torch.int32))),
    (ValueError, "seq_lens", dict(seq_lens=torch.zeros(3, dtype=torch.int32))),
    (TypeError, "cu_seqlens", dict(cu_seqlens=torch.zeros(3, dtype=torch.int64))),
    (TypeError, "page_table", dict(page_table=torch.zeros(2, 3, dtype=torch.int64))),
    (NotImplementedError, "page_table", dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t())),
])
def test_what_describes_the_batch_is_checked(error, match, kw):
    kw = {n: _dev(torch.zeros(*x, dtype=torch.bfloat16)) if isinstance(x, tuple) else _dev(x) for n, x in kw.items()}
    t = {n: _dev(x) if x is not None else None for n, x in _tensors().items()}
    t.update(kw)
    with pytest.raises(error, match=match):
        paged._check_pages(**t)


def test_scales_of_8_bit_pages_are_checked():
    t = {n: _dev(x) if x is not None else None for n, x in _tensors().items()}
    for n in ("k_pages", "v_pages"):
        t[n] = _dev(torch.zeros(5, 16, 2, 64, dtype=torch.int8))
    good = _dev(torch.zeros(5, 2, 16, dtype=torch.uint8))
    paged._check_pages(**{**t, "k_scales": good, "v_scales": good})
    for bad in (None, _dev(torch.zeros(5, 16, 2, dtype=torch.uint8)), _dev(torch.zeros(5, 2, 16)),
                _dev(torch.zeros(5, 16, 2, dtype=torch.uint8).transpose(1, 2))):
        with pytest.raises(ValueError, match="v_scales"):
            paged._check_pages(**{**t, "k_scales": good, "v_scales": bad})


def test_rows_are_checked():
    pages, codes = (_dev(torch.zeros(5, 16, 2, 64, dtype=d)) for d in (torch.bfloat16, torch.int8))
    rows = lambda *s, dtype=torch.bfloat16: _dev(torch.zeros(*s, dtype=dtype))  # noqa: E731
    paged._check_rows("k", rows(7, 2, 64), pages, 2, None)
    paged._check_rows("k", rows(7, 2, 64, dtype=torch.float16), codes, 2, 7)
    for error, match, x, heads, tokens in ((ValueError, "shape", rows(7, 2), 2, None), (ValueError, "shape", rows(7, 3, 64), 2, None),
                                           (ValueError, "shape", rows(7, 2, 128), 2, None), (ValueError, "shape", rows(7, 2, 64), 2, 8),
                                           (TypeError, "float16", rows(7, 2, 64, dtype=torch.float32), 2, None),
                                           (TypeError, "dtype of the pages", rows(7, 2, 64, dtype=torch.float16), 2, None),
                                           (ValueError, "device", torch.zeros(7, 2, 64, dtype=torch.bfloat16), 2, None),
                                           (ValueError, "heads", rows(7, 0, 64), None, None),
                                           (NotImplementedError, "contiguous", rows(7, 64, 2).transpose(1, 2), 2, None)):
        with pytest.raises(error, match=match):
            paged._check_rows("k", x, pages, heads, tokens)
    with pytest.raises(NotImplementedError, match="backward"):
        paged._check_rows("q", rows(7, 2, 64).requires_grad_(), pages, 2, None)
    with torch.no_grad():
        paged._check_rows("q", rows(7, 2, 64).requires_grad_(), pages, 2, None)


def test_attention_arguments_are_checked():
    pages, q = _dev(torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)), _dev(torch.zeros(7, 4, 64, dtype=torch.bfloat16))
    paged._check_attention(q, pages, 3, None, None)
    for error, args in ((ValueError, (_dev(torch.zeros(7, 3, 64, dtype=torch.bfloat16)), pages, 3, None, None)), (ValueError, (q, pages, 0, None, None)),
                        (ValueError, (q, pages, 1.5, None, None)), (ValueError, (q, pages, 3, 0.0, None)), (ValueError, (q, pages, 3, float("nan"), None)),
                        (TypeError, (q, pages, 3, None, _dev(torch.zeros(7, 4, 64, dtype=torch.float16))))):
        with pytest.raises(error):
            paged._check_attention(*args)


def test_packed_structure_is_the_declared_one():
    """The bytes that a call hands over, read back through the declared structure."""
    g = paged._Pages.__new__(paged._Pages)
    g.shape, g.batch, g.per_seq, g.store, g.strides = (11, 16, 2, 64), 3, 9, 2, (1, 2, 3, 4, 5, 6, 7)
    p = _lib.Paged.from_buffer_copy(g.pack(21, 4, 5, torch.float16, 0.25, (31, 32), (33, 34), (35, 36), (37, 38)))
    assert [getattr(p, n) for n, _ in _lib.Paged._fields_] == [21, 3, 4, 2, 64, 11, 16, 9, 5, 1, 2, 0.25, 0, *range(31, 39), *range(1, 8)]


def test_pool_arguments_are_checked():
    for error, args in ((TypeError, (4, 16, 2, 64, torch.float32)), (TypeError, (4, 16, 2, 64, torch.bfloat16, torch.float16)),
                        (ValueError, (0, 16, 2, 64)), (ValueError, (4, 16, 0, 64)), (NotImplementedError, (4, 48, 2, 64)),
                        (NotImplementedError, (4, 16, 2, 80))):
        with pytest.raises(error):
            moba.PagedKV(*args, device="cpu")
    pool = moba.PagedKV(4, 16, 2, 64, torch.float16, torch.float8_e4m3fn, device="cpu")
    assert pool.k.shape == (4, 16, 2, 64) and pool.k.stride() == (2048, 64, 1024, 1) and pool.k_scales.shape == (4, 2, 16)
