"""CPU: arguments of the operators around drafted tokens, in the C ABI and in Python, and the rotary tables.  No kernel is launched."""
import ctypes as C
import math

import pytest
import torch

from baselinebenchmark_b200 import RotaryTable, _lib, build, drafts, paged, rotary_frequencies
from tests.test_paged_abi import _paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _pool(**kw):
    base = dict(total_tokens=10, batch=3, pages_per_seq=9, num_pages=50, page_size=64, table_stride=9)
    base.update(kw)
    return _lib.PagePool(**base)


def _rotary(**kw):
    base = dict(total_tokens=10, num_q_heads=8, num_kv_heads=2, head_dim=128, rotary_dim=64, magnitude=1.0, q_stride_token=1024, q_stride_head=128,
                k_stride_token=256, k_stride_head=128, qo_stride_token=1024, qo_stride_head=128, ko_stride_token=256, ko_stride_head=128)
    base.update(kw)
    return _lib.Rotary(**base)


def _drafts(**kw):
    base = dict(total_tokens=10, vocabulary=1000, batch=3, max_new=5, dtype=2, token_bits=64, target_stride=1000, draft_stride=1000)
    base.update(kw)
    return _lib.Drafts(**base)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(total_tokens=0)), (0, dict(batch=1, table_stride=0)), (0, dict(batch=16384)),
    (-1, dict(batch=0)), (-1, dict(pages_per_seq=0)), (-1, dict(num_pages=0)), (-1, dict(page_size=0)), (-1, dict(total_tokens=-1)),
    (-1, dict(table_stride=8)), (-2, dict(page_size=8)), (-2, dict(page_size=48)), (-2, dict(batch=16385)), (-2, dict(reserved=1)),
    (-2, dict(total_tokens=2 ** 31)), (-2, dict(pages_per_seq=2 ** 24, table_stride=2 ** 24)), (-2, dict(batch=16384, pages_per_seq=2 ** 17, page_size=16, table_stride=2 ** 17))])
def test_pool_codes(lib, code, kw):
    assert lib.moba_page_pool_check(C.byref(_pool(**kw))) == code


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(num_kv_heads=0)), (0, dict(rotary_dim=2)), (0, dict(rotary_dim=128)), (0, dict(q_stride_token=0)), (0, dict(total_tokens=1, qo_stride_token=0)),
    (-1, dict(total_tokens=0)), (-1, dict(num_q_heads=0)), (-1, dict(rotary_dim=130)), (-1, dict(rotary_dim=3)), (-1, dict(rotary_dim=0)),
    (-1, dict(magnitude=0.0)), (-1, dict(magnitude=math.nan)), (-1, dict(magnitude=math.inf)), (-1, dict(q_stride_token=-8)), (-1, dict(qo_stride_token=0)),
    (-1, dict(ko_stride_head=0)), (-2, dict(head_dim=80)), (-2, dict(dtype=2)), (-2, dict(interleaved=2)), (-2, dict(inverse=-1)), (-2, dict(reserved=1)),
    (-2, dict(reserved2=1)), (-2, dict(total_tokens=2 ** 28)), (-6, dict(q_stride_head=132))])
def test_rotary_codes(lib, code, kw):
    assert lib.moba_rotary_check(C.byref(_rotary(**kw))) == code


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(dtype=0)), (0, dict(token_bits=32)), (0, dict(max_new=1024)), (0, dict(vocabulary=2 ** 22)), (0, dict(target_stride=0)),
    (-1, dict(total_tokens=0)), (-1, dict(batch=0)), (-1, dict(vocabulary=0)), (-1, dict(max_new=0)), (-1, dict(draft_stride=-1)),
    (-2, dict(dtype=3)), (-2, dict(token_bits=16)), (-2, dict(max_new=1025)), (-2, dict(vocabulary=2 ** 22 + 1)), (-2, dict(reserved=1)),
    (-2, dict(total_tokens=2 ** 31)), (-2, dict(batch=2 ** 27))])
def test_drafts_codes(lib, code, kw):
    assert lib.moba_drafts_check(C.byref(_drafts(**kw))) == code


def test_pointers_are_checked_before_any_launch(lib):
    ok, odd = 0x10000, 0x10002
    for check in (lib.moba_page_pool_check, lib.moba_rotary_check, lib.moba_drafts_check):
        assert check(None) == -4
    args = [ok] * 9
    def with_(i, x):  # noqa: E306
        a = list(args)
        a[i] = x
        return a
    reserve = lambda a: lib.moba_paged_reserve(C.byref(_pool()), *a, None)  # noqa: E731
    for i in (0, 1, 3, 4, 5, 6, 7, 8):
        assert reserve(with_(i, None)) == -4
    for i in range(9):
        assert reserve(with_(i, odd)) == -6
    assert reserve(with_(6, 0x10004)) == -6
    release = lambda a: lib.moba_paged_release(C.byref(_pool()), *a[:4], None)  # noqa: E731
    for i in range(4):
        assert release(with_(i, None)) == -4 and release(with_(i, odd)) == -6
    turn = lambda a, **kw: lib.moba_rotary(C.byref(_rotary(**kw)), *a[:6], None)  # noqa: E731
    for i in range(6):
        assert turn(with_(i, None)) == -4 and turn(with_(i, odd)) == -6
    assert turn(with_(0, 0x10008)) == -6 and turn(with_(3, 0x10004)) == -6
    verify = lambda a, **kw: lib.moba_verify_drafts(C.byref(_drafts(**kw)), *(a + [ok])[:10], None)  # noqa: E731
    for i in (0, 2, 3, 5, 6, 7, 8):
        assert verify(with_(i, None)) == -4
    for i in range(9):
        assert verify(with_(i, 0x10001)) == -6
    assert verify(with_(2, 0x10004)) == -6
    p = C.byref(_paged())
    keep = lambda path=ok, stride=4, columns=4, count=ok, lens=ok, k=ok: lib.moba_paged_keep(p, ok, ok, ok, path, stride, columns, count, k, ok, None, None, lens, None)  # noqa: E731
    assert keep(path=None) == -4 and keep(count=None) == -4 and keep(lens=None) == -4 and keep(k=None) == -4
    assert keep(path=odd) == -6 and keep(stride=3) == -1 and keep(columns=0) == -1
    need = C.c_size_t(0)
    assert lib.moba_paged_tree_workspace_size(p, C.byref(need)) == 0 and lib.moba_paged_tree_workspace_size(p, None) == -4
    tree = lambda size: lib.moba_paged_tree_attention(p, ok, ok, ok, ok, ok, ok, ok, None, None, ok, None, ok, size, None)  # noqa: E731
    assert tree(need.value - 1) == -3
    assert lib.moba_paged_tree_attention(p, ok, odd, ok, ok, ok, ok, ok, None, None, ok, None, ok, need.value, None) == -6


def test_python_refusals_on_the_cpu():
    """What is looked at before a device is needed, or because of it."""
    x, i = torch.ones(4, 9), torch.zeros(4, dtype=torch.int32)
    call = lambda **kw: drafts.verify_drafts(**{**dict(target=x, draft=None, tokens=i, cu_seqlens=i, accept=x[:, 0], sample=x[:3, 0], max_new=2), **kw})  # noqa: E731
    with pytest.raises(ValueError, match="accelerator"):
        call()
    with pytest.raises(ValueError, match="vocabulary"):
        call(target=x[0])
    with pytest.raises(TypeError, match="float32, bfloat16"):
        call(target=x.double())
    with pytest.raises(ValueError, match="accelerator"):
        paged.paged_reserve(i.view(2, 2), i[:3], i[:2], i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="accelerator"):
        paged.paged_release(i.view(2, 2), i[:2], i, i[:1], 16)


def test_turns_are_the_frequencies_to_half_a_unit():
    """Each turn is the frequency over 2 pi times 2^64, whole turns dropped (compared through double-double: 2^-11 of a 64-bit unit)."""
    f = torch.tensor([1.0, 0.5, 1e-4, 2 * math.pi * 0.75, 7.0, -0.25, 0.0], dtype=torch.float64)
    t = RotaryTable(f, device="cpu")
    assert t.rotary_dim == 14 and t.turns.dtype == torch.int64
    # 2^64 / (2 pi) = 2935890503282001226.71...
    unit = 2935890503282001227
    as_signed = lambda n: (n + 2 ** 63) % 2 ** 64 - 2 ** 63  # noqa: E731
    for got, x in zip(t.turns.tolist(), f.tolist()):
        from fractions import Fraction
        want = Fraction(x) * (unit - Fraction(1, 4))
        assert abs(as_signed(got - round(want))) <= max(abs(x), 1)
    assert t.turns[-1] == 0


def test_frequencies():
    f = rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1 and abs(f[31].item() - 10000.0 ** (-62 / 64)) < 1e-18
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=4.0), f / 4)
    g = rotary_frequencies(64, scaling="base", factor=4.0)
    assert g[0] == 1 and abs(g[31].item() * 4 / f[31].item() - 1) < 1e-13
    p = rotary_frequencies(64, scaling="parts", factor=4.0, original=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.allclose(p[turns <= 1], f[turns <= 1] / 4, rtol=1e-15, atol=0)
    assert ((p <= f) & (p >= f / 4 * (1 - 1e-15))).all()
    for kw in (dict(rotary_dim=0), dict(rotary_dim=5), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.0), dict(rotary_dim=2, scaling="base"),
               dict(rotary_dim=8, scaling="parts"), dict(rotary_dim=8, scaling="parts", original=9, fast=1.0), dict(rotary_dim=8, base=-1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**kw)
    for kw in (dict(frequencies=torch.zeros(0)), dict(frequencies=torch.zeros(2, 2)), dict(frequencies=[math.nan]), dict(frequencies=[1.0], magnitude=0.0),
               dict(frequencies=[1.0], magnitude=math.inf)):
        with pytest.raises(ValueError):
            RotaryTable(device="cpu", **kw)
