"""GPU: calls of the paged cache that are refused, and what they leave behind."""
import ctypes

import pytest
import torch

from baselinebenchmark_b200 import PagedKV, _lib, paged, paged_attention, paged_load, paged_store

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _call():
    cache = PagedKV(4, 16, 2, 64)
    where = (_i32([[0]]), _i32([0, 2]), _i32([2]))
    k, q = (torch.ones(2, h, 64, dtype=torch.bfloat16, device="cuda") for h in (2, 4))
    return cache, where, q, k


def test_pages_that_require_grad():
    cache, where, q, k = _call()
    for name in ("k", "v"):
        pages = [x.clone().requires_grad_(name == n) for n, x in (("k", cache.k), ("v", cache.v))]
        with pytest.raises(NotImplementedError, match="backward"):
            paged_load(*pages, *where, 2)
        with pytest.raises(NotImplementedError, match="backward"):
            paged_attention(q, *pages, *where, 2)
        with torch.no_grad():
            assert paged_attention(q, *pages, *where, 2).shape == q.shape and paged_load(*pages, *where, 2)[0].shape == k.shape


def test_tangents():
    cache, where, q, k = _call()
    forward = torch.autograd.forward_ad
    with forward.dual_level():
        dual = lambda x: forward.make_dual(x, torch.ones_like(x))  # noqa: E731
        with pytest.raises(NotImplementedError, match="tangent"):
            cache.attend(dual(q), *where, 2)
        with pytest.raises(NotImplementedError, match="tangent"):
            paged_attention(q, dual(cache.k), cache.v, *where, 2)
        with pytest.raises(NotImplementedError, match="tangent"):
            paged_load(cache.k, dual(cache.v), *where, 2)
        with pytest.raises(NotImplementedError, match="tangent"):
            cache.store(k, dual(k), *where)
        with pytest.raises(NotImplementedError, match="tangent"):
            paged_store(k, k, cache.k, dual(cache.v), *where)
        with pytest.raises(NotImplementedError, match="tangent"):
            cache.append(q, dual(k), k, *where, 2)
        assert (cache.k == 0).all() and (cache.v == 0).all()
        assert cache.append(q, k, k, *where, 2).shape == q.shape


@pytest.mark.parametrize("tokens", [2, 40])
def test_a_refused_append_writes_nothing(tokens, monkeypatch):
    """What only the attention refuses is found before the new rows are stored: an output whose rows lie on one another, addresses, no
    memory for scratch.  A call that goes through tells autograd of its writes."""
    cache = PagedKV(4, 16, 2, 64)
    where = (_i32([[0, 1, 2]]), _i32([0, tokens]), _i32([tokens]))
    k, q = (torch.ones(tokens, h, 64, dtype=torch.bfloat16, device="cuda") for h in (2, 4))
    shifted = torch.ones(tokens * 4 * 64 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(tokens, 4, 64)
    version = cache.k._version

    def refused(error, query=q, **options):
        with pytest.raises(error):
            cache.append(query, k, k, *where, tokens, **options)
        torch.cuda.synchronize()
        assert (cache.k == 0).all() and (cache.v == 0).all() and cache.k._version == version

    refused(_lib.MobaError, out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda").expand(tokens, 4, 64))
    refused(_lib.MobaError, out=torch.zeros(tokens, 1, 64, dtype=torch.bfloat16, device="cuda").expand(tokens, 4, 64))
    refused(_lib.MobaError, out=shifted)
    refused(_lib.MobaError, query=shifted)
    with monkeypatch.context() as m:
        def none(*_):
            raise torch.cuda.OutOfMemoryError("no memory")
        m.setattr(paged, "_workspace", none)
        refused(torch.cuda.OutOfMemoryError)
    assert cache.append(q, k, k, *where, tokens).shape == q.shape and cache.k._version > version and (cache.k[0, 0] == 1).all()


@pytest.mark.parametrize("dim,store", [(128, None), (256, torch.int8), (64, torch.float8_e4m3fn)])
def test_scratch_is_not_exceeded(dim, store):
    """Bytes behind the workspace that a call asks for are not touched, also where sequences that overlap make more items than it counts."""
    hq, hkv, tokens, pages = 8, 2, 60, 130
    cache = PagedKV(pages, 64, hkv, dim, torch.bfloat16, store)
    for batch, cu in ((1, [0, tokens]), (40, [0, tokens] * 20 + [0]), (3, [0, 20, 21, tokens])):
        table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)
        lens, cu = _i32([8000 - 64 * i for i in range(batch)]), _i32(cu)
        q = torch.randn(tokens, hq, dim, device="cuda").bfloat16()
        out = torch.empty_like(q)
        g = paged._Pages(cache.k, cache.v, table, cu, lens, cache.k_scales, cache.v_scales)
        rows = (hq * dim, dim)
        prob = g.pack(tokens, hq, tokens, q.dtype, 0.0, rows, rows)
        need = ctypes.c_size_t(0)
        _lib.check(_lib.lib().moba_paged_workspace_size(prob, ctypes.byref(need)))
        scratch = torch.full((need.value + 65536,), 0x5a, dtype=torch.uint8, device="cuda")
        g.run(_lib.lib().moba_paged_attention, prob, q.data_ptr(), *g.where, out.data_ptr(), None, scratch.data_ptr(), need.value)
        assert (scratch[need.value:] == 0x5a).all()
        # (sequences that overlap are owed nothing: rows behind the last entry, 0, are behind the batch)
        assert (out == 0).all() or batch == 40
