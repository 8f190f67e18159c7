"""Keys and values of many sequences in pages: written, read back and attended to.

The reference's operator takes whole packed sequences and keeps nothing between calls (backends/_mthreads/ops/moba/parallel.py:253-374);
`IncrementalMoba` keeps one sequence in a cache of its own.  A server has many, of any length: their rows live in one pool of pages,
in 16 bits or quantised to 8, and a call concerns a packed batch of new tokens.

    k_pages, v_pages   [pages, page_size, Hkv, D]: bfloat16, float16, float8_e4m3fn or int8, any strides with a contiguous last
                       dimension (head-major pages read fastest: see `PagedKV`); page_size a power of two, at least 16
    k_scales, v_scales [pages, Hkv, page_size] uint8, for 8-bit pages: a code c with byte s stands for c * 2**(s - 127)
    page_table         int32 [batch, pages of a sequence]: position x is slot x % page_size of page page_table[b, x // page_size];
                       an entry that is no page's number is a page that is not there
    cu_seqlens         int32 [batch + 1]: sequence b has the packed rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, its last tokens
    seq_lens           int32 [batch]: its tokens, the packed ones included

All of them stay on the device; nothing is read back to the host, so that calls may be captured in a CUDA graph and replayed
with other numbers in the same tensors.  include/moba_b200.h has the rules in full.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from .parallel import HEAD_DIMS, _on_device, _workspace

__all__ = ["PagedKV", "paged_store", "paged_load", "paged_attention", "paged_append"]

_STORES = {torch.float8_e4m3fn: _lib.STORE_E4M3, torch.int8: _lib.STORE_INT8}
_ROWS = (torch.float16, torch.bfloat16)


def _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales) -> None:
    shape, dtype, dev = k_pages.shape, k_pages.dtype, k_pages.device
    if len(shape) != 4:
        raise ValueError("k_pages and v_pages must have shape [pages, page_size, heads, head_dim]")
    if shape != v_pages.shape:
        raise ValueError(f"k_pages and v_pages must have identical shapes, got {shape} and {v_pages.shape}")
    if dtype != v_pages.dtype:
        raise TypeError("k_pages and v_pages must have the same dtype")
    if dtype not in _STORES and dtype not in _ROWS:
        raise TypeError(f"pages hold float16, bfloat16, float8_e4m3fn or int8, got {dtype}")
    if 0 in shape:
        raise ValueError("k_pages and v_pages dimensions must be non-zero")
    if dev.type != "cuda" or v_pages.device != dev:
        raise ValueError("k_pages and v_pages must be accelerator tensors on the same device")
    if shape[1] < 16 or shape[1] & (shape[1] - 1):
        raise NotImplementedError(f"page_size must be a power of two and at least 16, got {shape[1]}")
    if shape[3] not in HEAD_DIMS:
        raise NotImplementedError(f"this build supports head_dim {HEAD_DIMS} only")
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if x.stride(3) != 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if dtype in _STORES:
        want = (shape[0], shape[2], shape[1])
        for name, x in (("k_scales", k_scales), ("v_scales", v_scales)):
            if x is None or x.shape != want or x.dtype != torch.uint8 or x.device != dev or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {want} on the pages' device")
    elif k_scales is not None or v_scales is not None:
        raise ValueError("pages of 16-bit rows have no scales")
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a one-dimensional tensor of length >= 2")
    batch = cu_seqlens.numel() - 1
    if page_table.ndim != 2 or page_table.shape[0] != batch or page_table.shape[1] == 0:
        raise ValueError(f"page_table must have shape [{batch}, pages of a sequence], got {tuple(page_table.shape)}")
    if seq_lens.shape != (batch,):
        raise ValueError(f"seq_lens must have shape [{batch}], got {tuple(seq_lens.shape)}")
    for name, x in (("cu_seqlens", cu_seqlens), ("seq_lens", seq_lens), ("page_table", page_table)):
        if x.device != dev or x.dtype != torch.int32:
            raise TypeError(f"{name} must be an int32 tensor on the pages' device")
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")


def _check_rows(name, x, k_pages, heads: Optional[int], tokens: Optional[int]) -> None:
    if x.ndim != 3 or x.shape[2] != k_pages.shape[3] or (heads is not None and x.shape[1] != heads) \
            or (tokens is not None and x.shape[0] != tokens):
        raise ValueError(f"{name} must have shape [tokens, heads, head_dim] in line with the pages {tuple(k_pages.shape)}, "
                         f"got {tuple(x.shape)}")
    if x.dtype not in _ROWS:
        raise TypeError(f"only float16 and bfloat16 are supported, got {x.dtype}")
    if k_pages.dtype in _ROWS and x.dtype != k_pages.dtype:
        raise TypeError(f"{name} must have the dtype of the pages, {k_pages.dtype}, got {x.dtype}")
    if x.device != k_pages.device:
        raise ValueError(f"{name} must be on the pages' device")
    if x.shape[1] == 0:
        raise ValueError(f"{name} must have heads")
    if x.stride(2) != 1:
        raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires grad: a paged cache is state of a server, its operators have no backward")


def _problem(k_pages, v_pages, page_table, cu_seqlens, tokens: int, q_heads: int, dtype, max_new: int = 1, scale: float = 0.0):
    pages, size, heads, dim = k_pages.shape
    (kp, kt, kh, _), (vp, vt, vh, _) = k_pages.stride(), v_pages.stride()
    # a dimension of one page, slot or head may have any stride: it is never stepped over
    row = heads * size * dim
    kp, vp = (kp, vp) if pages > 1 else (row, row)
    kh, vh = (kh, vh) if heads > 1 else (size * dim, size * dim)
    return _lib.Paged(
        total_tokens=tokens, batch=cu_seqlens.numel() - 1, num_q_heads=q_heads, num_kv_heads=heads, head_dim=dim,
        num_pages=pages, page_size=size, pages_per_seq=page_table.shape[1], max_new=max_new,
        dtype=_lib.DTYPE_FP16 if dtype == torch.float16 else _lib.DTYPE_BF16, store=_STORES.get(k_pages.dtype, _lib.STORE_SAME),
        softmax_scale=scale, k_page_stride=kp, k_page_token=kt, k_page_head=kh, v_page_stride=vp, v_page_token=vt,
        v_page_head=vh, table_stride=page_table.stride(0) if page_table.shape[0] > 1 else page_table.shape[1])


def _ptr(x: Optional[torch.Tensor]):
    return None if x is None else x.data_ptr()


def _rows_strides(x) -> Tuple[int, int]:
    """Token and head stride; a single token or head may have any, and it is never stepped over."""
    t, h, _ = x.stride()
    return (t if x.shape[0] > 1 else 0), (h if x.shape[1] > 1 else 0)


def _store(prob, k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales) -> None:
    (prob.k_stride_token, prob.k_stride_head), (prob.v_stride_token, prob.v_stride_head) = _rows_strides(k), _rows_strides(v)
    _lib.check(_on_device(k.device, lambda stream: _lib.lib().moba_paged_store(
        C.byref(prob), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), stream)))
    written = [x for x in (k_pages, v_pages, k_scales, v_scales) if x is not None and not x.is_inference()]
    torch.autograd.graph.increment_version(written)          # as after an in-place torch operation


def _check_written(*tensors) -> None:
    for x in tensors:
        if x is not None and x.is_inference() and not torch.is_inference_mode_enabled():
            raise RuntimeError("pages made in inference mode can only be written in inference mode")
        if x is not None and x.requires_grad:
            raise NotImplementedError("pages that require grad cannot be written")


def paged_store(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, *, k_scales: Optional[torch.Tensor] = None,
                v_scales: Optional[torch.Tensor] = None) -> None:
    """Writes the packed rows k, v [T, Hkv, D] into the pages of their sequences; 8-bit pages are quantised to, each row
    and head with a power of two of its own.  Rows behind the last sequence, and rows whose page is not there, are not written."""
    _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    _check_rows("k", k, k_pages, k_pages.shape[2], None)
    _check_rows("v", v, k_pages, k_pages.shape[2], k.shape[0])
    if k.dtype != v.dtype:
        raise TypeError("k and v must have the same dtype")
    _check_written(k_pages, v_pages, k_scales, v_scales)
    if k.shape[0] == 0:
        return
    prob = _problem(k_pages, v_pages, page_table, cu_seqlens, k.shape[0], k.shape[1], k.dtype)
    _store(prob, k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)


def paged_load(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
               seq_lens: torch.Tensor, total_tokens: int, *, dtype: Optional[torch.dtype] = None,
               k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Reads rows back: (k, v), each [total_tokens, Hkv, D] packed as cu_seqlens says, of `dtype` (8-bit pages: bfloat16 unless
    given).  With seq_lens the lengths of whole sequences this is the packed batch that `parallel_moba` takes.  Rows whose page is not
    there are zeros; rows behind the last sequence are left as they were (undefined without `out`)."""
    _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    if not isinstance(total_tokens, int) or total_tokens < 0:
        raise ValueError(f"total_tokens must be an int that is not negative, got {total_tokens}")
    if dtype is None:
        dtype = k_pages.dtype if k_pages.dtype in _ROWS else out[0].dtype if out is not None else torch.bfloat16
    heads, dim = k_pages.shape[2:]
    if out is None:
        if dtype not in _ROWS:
            raise TypeError(f"only float16 and bfloat16 are supported, got {dtype}")
        if k_pages.dtype in _ROWS and dtype != k_pages.dtype:
            raise TypeError(f"rows of {k_pages.dtype} pages are {k_pages.dtype}, got {dtype}")
        k, v = (torch.empty(total_tokens, heads, dim, dtype=dtype, device=k_pages.device) for _ in range(2))
    else:
        k, v = out
        _check_rows("out[0]", k, k_pages, heads, total_tokens)
        _check_rows("out[1]", v, k_pages, heads, total_tokens)
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError(f"out must be of {dtype}, got {k.dtype} and {v.dtype}")
        _check_written(k, v)
    if total_tokens == 0:
        return k, v
    prob = _problem(k_pages, v_pages, page_table, cu_seqlens, total_tokens, heads, dtype)
    (prob.k_stride_token, prob.k_stride_head), (prob.v_stride_token, prob.v_stride_head) = _rows_strides(k), _rows_strides(v)
    _lib.check(_on_device(k.device, lambda stream: _lib.lib().moba_paged_load(
        C.byref(prob), cu_seqlens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(), k_pages.data_ptr(),
        v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), k.data_ptr(), v.data_ptr(), stream)))
    if out is not None:
        torch.autograd.graph.increment_version([x for x in out if not x.is_inference()])
    return k, v


def _attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, prob, k_scales, v_scales, return_lse, out):
    given = out is not None
    if not given:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if return_lse else None
    if q.shape[0] > 0:
        (prob.q_stride_token, prob.q_stride_head), (prob.o_stride_token, prob.o_stride_head) = _rows_strides(q), _rows_strides(out)
        lib, need = _lib.lib(), C.c_size_t(0)
        _lib.check(lib.moba_paged_workspace_size(C.byref(prob), C.byref(need)))
        ws = _workspace(q.device, need.value)
        _lib.check(_on_device(q.device, lambda stream: lib.moba_paged_attention(
            C.byref(prob), q.data_ptr(), cu_seqlens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(),
            k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), out.data_ptr(), _ptr(lse),
            ws.data_ptr(), need.value, stream)))
        if given and not out.is_inference():
            torch.autograd.graph.increment_version(out)
    return (out, lse) if return_lse else out


def _check_attention(q, k_pages, max_new, scale, out) -> None:
    _check_rows("q", q, k_pages, None, None)
    if q.shape[1] % k_pages.shape[2] != 0:
        raise ValueError(f"q heads ({q.shape[1]}) must be divisible by kv heads ({k_pages.shape[2]})")
    if not isinstance(max_new, int) or max_new <= 0:
        raise ValueError(f"max_new must be a positive int, got {max_new}")
    if scale is not None and not 0.0 < float(scale) < 3e38:
        raise ValueError(f"scale must be a positive number, got {scale}")
    if out is not None:
        _check_rows("out", out, k_pages, q.shape[1], q.shape[0])
        if out.dtype != q.dtype:
            raise TypeError(f"out must be of {q.dtype}, got {out.dtype}")
        _check_written(out)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, max_new: int, *, scale: Optional[float] = None,
                    k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                    return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Causal softmax attention of the packed new tokens q [T, Hq, D] over the pages of their sequences: every token sees the
    positions of its sequence up to its own, which the pages hold already (`paged_append` writes them first).  One token a sequence
    is a decode step, a few are drafted tokens, many a block of a prompt; a batch may mix them.

    `max_new`: the most new tokens that a sequence has (the kernel is chosen by it; another number costs time only).  `scale`:
    factor of the scores, head_dim ** -0.5 unless given.  Returns out [T, Hq, D], with `return_lse` (out, lse [Hq, T] fp32, natural
    log).  A token that sees nothing is zeros and -inf.  `out`: a tensor to write to; rows behind the last sequence are left as
    they were (undefined without it).  8-bit pages are attended to as the rows that `paged_load` gives; they take float16 and
    bfloat16 queries whatever they were written from."""
    _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    _check_attention(q, k_pages, max_new, scale, out)
    prob = _problem(k_pages, v_pages, page_table, cu_seqlens, q.shape[0], q.shape[1], q.dtype, max_new, float(scale or 0.0))
    return _attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, prob, k_scales, v_scales, return_lse, out)


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, max_new: int, *,
                 scale: Optional[float] = None, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """`paged_store` of the new tokens' k and v, then `paged_attention` of their q: a layer's step of a server."""
    _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    _check_attention(q, k_pages, max_new, scale, out)
    _check_rows("k", k, k_pages, k_pages.shape[2], q.shape[0])
    _check_rows("v", v, k_pages, k_pages.shape[2], q.shape[0])
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k, and v must have the same dtype")
    _check_written(k_pages, v_pages, k_scales, v_scales)
    prob = _problem(k_pages, v_pages, page_table, cu_seqlens, q.shape[0], q.shape[1], q.dtype, max_new, float(scale or 0.0))
    if q.shape[0] > 0:
        _store(prob, k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    return _attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, prob, k_scales, v_scales, return_lse, out)


class PagedKV:
    """A layer's pool of pages.  `k`, `v`: [pages, page_size, Hkv, D], in memory head by head within a page, so that the rows of
    one head that attention reads together lie together; `k_scales`, `v_scales` for 8-bit pages, else None.  `dtype` is that of the
    rows written and read, `store` that of the pages: the same, torch.float8_e4m3fn or torch.int8."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 store: Optional[torch.dtype] = None, device: Optional[torch.device] = None):
        store = dtype if store is None else store
        if dtype not in _ROWS:
            raise TypeError(f"only float16 and bfloat16 are supported, got {dtype}")
        if store != dtype and store not in _STORES:
            raise TypeError(f"pages hold the rows' own dtype, float8_e4m3fn or int8, got {store}")
        if num_pages <= 0 or num_kv_heads <= 0:
            raise ValueError(f"num_pages and num_kv_heads must be positive, got {num_pages} and {num_kv_heads}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.dtype = dtype
        self.k, self.v = (torch.zeros(num_pages, num_kv_heads, page_size, head_dim, device=device, dtype=torch.int8 if store in _STORES else store)
                          .view(store).transpose(1, 2) for _ in range(2))
        self.k_scales = self.v_scales = None
        if store in _STORES:
            self.k_scales, self.v_scales = (torch.full((num_pages, num_kv_heads, page_size), 127, device=device, dtype=torch.uint8)
                                            for _ in range(2))

    def _scales(self):
        return {"k_scales": self.k_scales, "v_scales": self.v_scales}

    def store(self, k, v, page_table, cu_seqlens, seq_lens) -> None:
        paged_store(k, v, self.k, self.v, page_table, cu_seqlens, seq_lens, **self._scales())

    def load(self, page_table, cu_seqlens, seq_lens, total_tokens: int, out=None):
        return paged_load(self.k, self.v, page_table, cu_seqlens, seq_lens, total_tokens, dtype=self.dtype, out=out, **self._scales())

    def attend(self, q, page_table, cu_seqlens, seq_lens, max_new: int, **options):
        return paged_attention(q, self.k, self.v, page_table, cu_seqlens, seq_lens, max_new, **self._scales(), **options)

    def append(self, q, k, v, page_table, cu_seqlens, seq_lens, max_new: int, **options):
        return paged_append(q, k, v, self.k, self.v, page_table, cu_seqlens, seq_lens, max_new, **self._scales(), **options)
